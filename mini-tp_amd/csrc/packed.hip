// Causal attention over packed sequences: the rows of S sequences of any
// lengths follow each other in one stream of N tokens, sequence s in rows
// offsets[s] .. offsets[s + 1] - 1. Query i of a sequence that begins at row a
// attends rows a .. i:
//     o = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,
// head h on KV head h / (Hq / Hkv). A row of no sequence gets zeros.
#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

struct PackedArgs {
  const void *q, *k, *v;  // [N, Hq, D], [N, Hkv, D] in strides of elements
  int64_t q_row, q_head, kv_row, kv_head;
  void* out;              // [N, Hq, D]
  int N, S, Hq, per;
  const int64_t* offsets;  // [S + 1]
  float scale;
};

// First row of the sequence that holds row r, -1 where none does: the last
// offset not above r begins it. (Offsets in disorder give some row up to r.)
__device__ __forceinline__ int first_row(const PackedArgs& a, int r) {
  int lo = 0, hi = a.S + 1;  // offsets[0 .. lo - 1] <= r < offsets[hi ..]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.offsets[mid] <= r)
      lo = mid + 1;
    else
      hi = mid;
  }
  if (lo == 0 || lo > a.S) return -1;
  return (int)std::min<int64_t>(std::max<int64_t>(a.offsets[lo - 1], 0), r);
}

// One query of one head by one wave, in fp32: a lane a key for the scores, a
// lane one or two dims of the output.
template <typename T, int D>
__device__ __forceinline__ void packed_row(const PackedArgs& a, int r, int first, int head) {
  constexpr int VE = Vec<T>::N, DL = D > 64 ? D / 64 : 1;
  const int lane = threadIdx.x & 63, kv = head / a.per;
  const T* q = (const T*)a.q + r * a.q_row + head * a.q_head;
  const T* k = (const T*)a.k + kv * a.kv_head;
  const T* v = (const T*)a.v + kv * a.kv_head;
  const int dim = std::min(lane * DL, D - DL);
  float m = -__builtin_inff(), l = 0.f, o[DL];
#pragma unroll
  for (int d = 0; d < DL; ++d) o[d] = 0.f;
  for (int k0 = first; k0 <= r; k0 += 64) {
    const int key = k0 + lane;
    const T* krow = k + std::min(key, r) * a.kv_row;
    float s = 0.f;
    for (int d = 0; d < D; d += VE) {
      float x[VE], y[VE];
      load_vec<T, VE>(q + d, x);
      load_vec<T, VE>(krow + d, y);
#pragma unroll
      for (int e = 0; e < VE; ++e) s = fmaf(x[e], y[e], s);
    }
    s = key <= r ? s * a.scale : -__builtin_inff();
    const float mn = fmaxf(m, wave_max(s)), ref = mn == -__builtin_inff() ? 0.f : mn;
    const float alpha = m == mn ? 1.f : expf(m - mn);
    const float p = key <= r ? expf(s - ref) : 0.f;
    m = mn;
    l = fmaf(l, alpha, wave_sum(p));
#pragma unroll
    for (int d = 0; d < DL; ++d) o[d] *= alpha;
    const int n = std::min(64, r - k0 + 1);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl(p, j, 64);
#pragma unroll
      for (int d = 0; d < DL; ++d) o[d] = fmaf(pj, load_f32<T>(v + (k0 + j) * a.kv_row, dim + d), o[d]);
    }
  }
  T* out = (T*)a.out + ((int64_t)r * a.Hq + head) * D;
  if (lane * DL < D) {
#pragma unroll
    for (int d = 0; d < DL; ++d) store_f32<T>(out, dim + d, o[d] / l);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void packed_rows_kernel(PackedArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)a.N * a.Hq) return;
  const int r = (int)(i / a.Hq), first = first_row(a, r);
  if (first >= 0) {
    packed_row<T, D>(a, r, first, (int)(i % a.Hq));
    return;
  }
  T* out = (T*)a.out + i * D;
  for (int d = threadIdx.x & 63; d < D; d += 64) store_f32<T>(out, d, 0.f);
}

template <typename T, int D>
int packed_launch(hipStream_t st, const PackedArgs& a) {
  hipLaunchKernelGGL((packed_rows_kernel<T, D>), dim3((unsigned)cdiv((int64_t)a.N * a.Hq, 4)), dim3(256), 0, st, a);
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

template <typename T>
int packed_by_d(hipStream_t st, const PackedArgs& a, int64_t D) {
  switch (D) {
    case 16:
      return packed_launch<T, 16>(st, a);
    case 32:
      return packed_launch<T, 32>(st, a);
    case 64:
      return packed_launch<T, 64>(st, a);
    default:
      return packed_launch<T, 128>(st, a);
  }
}

}  // namespace

// Whether the launch takes the shape: 32-bit row and thread numbers, and tiles
// of keys within the 2 GiB that a buffer resource's offsets reach.
int packed_check(int dtype, const PackedShape& s) {
  if (s.D != 16 && s.D != 32 && s.D != 64 && s.D != 128) {
    set_error("packed_attention: head_dim %lld not supported (16, 32, 64, 128)", (long long)s.D);
    return MINITP_ERR_UNSUPPORTED;
  }
  constexpr int64_t MOST = 1LL << 31;
  if (s.N >= MOST - 256 || s.S >= MOST - 1 || s.Hq >= MOST || s.N * s.Hq >= (1LL << 26)) {
    set_error("packed_attention: %lld rows of %lld heads in %lld sequences are too many for one call", (long long)s.N,
              (long long)s.Hq, (long long)s.S);
    return MINITP_ERR_UNSUPPORTED;
  }
  if (s.kv_row > (1LL << 24) / (dtype == MINITP_F32 ? 2 : 1)) {
    set_error("packed_attention: K/V rows %lld elements apart are too far", (long long)s.kv_row);
    return MINITP_ERR_UNSUPPORTED;
  }
  return MINITP_OK;
}

int launch_packed_attention(hipStream_t st, int dtype, const PackedShape& s, const void* q, const void* k,
                            const void* v, void* out, const int64_t* offsets) {
  const int rc = packed_check(dtype, s);
  if (rc) return rc;
  PackedArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_row = s.q_row;
  a.q_head = s.q_head;
  a.kv_row = s.kv_row;
  a.kv_head = s.kv_head;
  a.out = out;
  a.N = (int)s.N;
  a.S = (int)s.S;
  a.Hq = (int)s.Hq;
  a.per = (int)(s.Hq / s.Hkv);
  a.offsets = offsets;
  a.scale = 1.0f / sqrtf((float)s.D);
  return dtype == MINITP_F32 ? packed_by_d<float>(st, a, s.D) : packed_by_d<bf16>(st, a, s.D);
}

}  // namespace minitp
