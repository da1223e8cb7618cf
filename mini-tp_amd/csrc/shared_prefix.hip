// Attention of a batch whose rows share prefixes: G groups of W = B / G rows,
// the rows of a group over one prefix of K/V rows (kept once a group) and each
// over rows of its own after it. With P_g prefix rows and c_b cached rows of
// its own, query t of row b attends
//     prefix rows 0 .. P_g - 1 of group b / W   and   own rows 0 .. c_b + t:
//     o = sum_j softmax_j(q . k_j / sqrt(D)) v_j over both together.
//
// A softmax over two sets of keys is the two partial softmaxes joined: with
// the maximum m_i, the sum l_i of exp(s - m_i) and the unnormalised output o_i
// of set i, o = sum_i exp(m_i - m) o_i / sum_i exp(m_i - m) l_i, m = max m_i.
// The prefix part takes all W T (Hq / Hkv) queries of a (group, KV head) as the
// rows of one product, so a prefix row is read once for the group instead of
// once per batch row; the own part takes the T (Hq / Hkv) queries of one (row,
// KV head). Work items are (part, unit, query tile, key split); each writes its
// (m, l, o) and a second launch joins them in slot order.
#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct SharedArgs {
  const void *q, *kp, *vp, *kc, *vc;  // q [B, T, Hq, D]; prefix [G, Hkv, Sp, D]; own [B, Hkv, S, D]
  void* out;                          // [B, T, Hq * D]
  int B, G, T, Hq, Hkv;
  int64_t Sp, S;
  int64_t P, C;                       // prefix rows, cached own rows (bounds of the lengths below)
  const int64_t *plens, *clens;       // [G], [B], or NULL: P and C everywhere
  float scale;
  int qtiles_p, qtiles_s;             // query tiles of a unit, prefix and own part
  int splits_p, splits_s;             // key splits
  int64_t items_p;                    // items of the prefix part, which come first
  float* ml;                          // [slot][B * T * Hq][2]: maximum, sum
  float* o;                           // [slot][B * T * Hq][D]
};

// What one block computes.
struct Item {
  const void *k, *v;  // the unit's first K / V row
  int64_t n0;         // first token (b * T + t) of the unit
  int rows;           // query rows of the unit: (token, head of the KV group)
  int tile, kv, slot;
  int64_t key_lo, key_hi;  // keys of this split
  int64_t seen;            // own part: query t sees keys 0 .. seen + t; prefix: every key
  bool own;
};

// Cached own rows of batch row b, -1 for an idle row (nothing attends).
__device__ __forceinline__ int64_t own_len(const SharedArgs& a, int64_t b) {
  if (a.clens == nullptr) return a.C;
  return std::min<int64_t>(std::max<int64_t>(a.clens[b], -1), a.C);
}

template <int QT, int KT>
__device__ __forceinline__ Item shared_item(const SharedArgs& a, int64_t D_bytes) {
  const int per = a.Hq / a.Hkv;
  Item it;
  int64_t i = blockIdx.x, keys;
  int split, splits;
  it.own = i >= a.items_p;
  if (!it.own) {
    splits = a.splits_p;
    split = (int)(i % splits);
    i /= splits;
    it.tile = (int)(i % a.qtiles_p);
    i /= a.qtiles_p;
    const int64_t g = i / a.Hkv;
    it.kv = (int)(i % a.Hkv);
    const int w = a.B / a.G;
    it.n0 = g * w * a.T;
    it.rows = w * a.T * per;
    it.k = (const char*)a.kp + i * a.Sp * D_bytes;
    it.v = (const char*)a.vp + i * a.Sp * D_bytes;
    keys = a.plens == nullptr ? a.P : std::min<int64_t>(std::max<int64_t>(a.plens[g], 0), a.P);
    it.seen = 0;
    it.slot = split;
  } else {
    i -= a.items_p;
    splits = a.splits_s;
    split = (int)(i % splits);
    i /= splits;
    it.tile = (int)(i % a.qtiles_s);
    i /= a.qtiles_s;
    const int64_t b = i / a.Hkv;
    it.kv = (int)(i % a.Hkv);
    it.n0 = b * a.T;
    it.rows = a.T * per;
    it.k = (const char*)a.kc + i * a.S * D_bytes;
    it.v = (const char*)a.vc + i * a.S * D_bytes;
    it.seen = own_len(a, b);
    // the tile's last query sees the most keys
    const int last = std::min(it.tile * QT + QT, it.rows) - 1;
    keys = it.seen < 0 ? 0 : it.seen + last / per + 1;
    it.slot = a.splits_p + split;
  }
  const int64_t span = cdiv(cdiv(keys, (int64_t)KT), (int64_t)splits) * KT;
  it.key_lo = std::min<int64_t>(split * span, keys);
  it.key_hi = std::min<int64_t>(it.key_lo + span, keys);
  return it;
}

// One tile of keys through a resource of its own (a head's rows may span more
// than the 4 GiB that one reaches); rows past the item's last read zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t key_rows(const void* base, int64_t key, int64_t key_hi, int tile,
                                                           int row_bytes) {
  const int64_t n = std::min<int64_t>(std::max<int64_t>(key_hi - key, 0), tile);
  return span_rsrc((const char*)base + key * row_bytes, (uint32_t)(n * row_bytes));
}
__device__ __forceinline__ uint4 rows_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  return make_uint4(v.x, v.y, v.z, v.w);
}

// ---------------------------------------------------------------------------
// fp32 (and bf16 head dims below 32, widened on their way into LDS) on
// v_mfma_f32_16x16x4_f32. Four waves of 16 queries share each KT-key tile in
// LDS; products transposed: S^T = K Q^T leaves lane (quad, r) with keys 4 quad
// .. 4 quad + 3 of query r, which is the B operand of O^T = V^T P^T as it is.
// Score MFMA i of a chunk takes dims 16 c + 4 quad + i from both operands (one
// 16-byte LDS read a lane), output MFMA j dims E r + j; rows are padded by 16
// bytes against bank conflicts. A score is summed in four chains.
constexpr int F_QT = 64;
template <int D>
constexpr int F_KT = D >= 128 ? 32 : 64;

template <typename T, int D>
__global__ __launch_bounds__(256) void shared_attn_f32_kernel(SharedArgs a) {
  constexpr int KT = F_KT<D>, KB = KT / 16, KC = D / 16;
  constexpr int E = D / 16 < 4 ? D / 16 : 4, HALVES = D / 16 / E;
  constexpr int ROW = D + 4;
  constexpr int VE = Vec<T>::N, PIECES = KT * D / VE, PER = (PIECES + 255) / 256;
  __shared__ __attribute__((aligned(16))) float Ks[KT * ROW];
  __shared__ __attribute__((aligned(16))) float Vs[KT * ROW];
  __shared__ int odd;  // a hidden value row of this tile is not finite
  const Item it = shared_item<F_QT, KT>(a, D * (int64_t)sizeof(T));
  const int per = a.Hq / a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane % 16, lq = lane / 16;
  const int r0 = it.tile * F_QT + wave * 16, r = r0 + lr;
  const bool live = r < it.rows;
  const int64_t n = it.n0 + (live ? r : 0) / per;
  const int h = it.kv * per + (live ? r : 0) % per;
  const int64_t seen = it.own ? it.seen + (n - it.n0) : INT64_MAX;  // the last key this query sees
  const int64_t seen_first = it.own ? it.seen + (it.tile * F_QT) / per : INT64_MAX;

  f32x4 qa[KC];
  {
    const T* qrow = (const T*)a.q + (n * a.Hq + h) * D;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) qa[c][i] = load_f32<T>(qrow, 16 * c + 4 * lq + i);
  }
  f32x4 o[HALVES][E];
#pragma unroll
  for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
    for (int j = 0; j < E; ++j) o[hf][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), lsum = 0.f;

  uint4 kr[PER], vr[PER];
  auto load_tile = [&](int64_t key) {
    const __amdgpu_buffer_rsrc_t krs = key_rows(it.k, key, it.key_hi, KT, D * (int)sizeof(T));
    const __amdgpu_buffer_rsrc_t vrs = key_rows(it.v, key, it.key_hi, KT, D * (int)sizeof(T));
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const uint32_t off = (uint32_t)(tid + 256 * u) * 16;  // (past the tile: not stored)
      kr[u] = rows_load16(krs, off);
      vr[u] = rows_load16(vrs, off);
    }
  };
  if (it.key_lo < it.key_hi) load_tile(it.key_lo);
  for (int64_t k0 = it.key_lo; k0 < it.key_hi; k0 += KT) {
    __syncthreads();  // the previous tile is consumed
    if (tid == 0) odd = 0;
    __syncthreads();
    bool found = false;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = tid + 256 * u;
      if (i < PIECES) {
        const int row = i / (D / VE), at = row * ROW + i % (D / VE) * VE;
        float f[VE];
        unpack16(kr[u], f, (T*)nullptr);
#pragma unroll
        for (int e = 0; e < VE; ++e) Ks[at + e] = f[e];
        unpack16(vr[u], f, (T*)nullptr);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          Vs[at + e] = f[e];
          found |= k0 + row > seen_first && !__builtin_isfinite(f[e]);
        }
      }
    }
    if (found) odd = 1;
    __syncthreads();
    if (k0 + KT < it.key_hi) load_tile(k0 + KT);
    const bool slow = odd != 0;
    const int64_t limit = std::min<int64_t>(seen, it.key_hi - 1) - k0;  // last key of the tile this query sees
    float p[KB][4];
    float mx = -__builtin_inff();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x4 part[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) part[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const f32x4 k4 = *(const f32x4*)(Ks + (kb * 16 + lr) * ROW + 16 * c + 4 * lq);
#pragma unroll
        for (int i = 0; i < 4; ++i) part[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[i], qa[c][i], part[i], 0, 0, 0);
      }
      const f32x4 acc = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[kb][e] = kb * 16 + 4 * lq + e <= limit ? acc[e] * a.scale : -__builtin_inff();
        mx = fmaxf(mx, p[kb][e]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx);
    const float alpha = mn == -__builtin_inff() ? 1.f : expf(m - mn);
    m = mn;
    lsum *= alpha;
#pragma unroll
    for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
      for (int j = 0; j < E; ++j) o[hf][j] *= alpha;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[kb][e] = p[kb][e] == -__builtin_inff() ? 0.f : expf(p[kb][e] - mn);
        lsum += p[kb][e];
      }
    if (slow) {
      // a hidden key's value is not finite: 0 times it is no zero, so the keys
      // that this lane's query does not see are left out one by one
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll 1
          for (int src = 0; src < 4; ++src) {
            const float pk = __shfl(p[kb][e], lr + 16 * src, 64);
            const int key = kb * 16 + 4 * src + e;
            if (key > limit) continue;
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
              for (int j = 0; j < E; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  o[hf][j][x] = fmaf(pk, Vs[key * ROW + 64 * hf + E * (4 * lq + x) + j], o[hf][j][x]);
          }
      continue;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* vrow = Vs + (kb * 16 + 4 * lq + e) * ROW + E * lr;
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf) {
          float v[E];
          if constexpr (E == 4) {
            const f32x4 v4 = *(const f32x4*)(vrow + 64 * hf);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = v4[j];
          } else {
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = vrow[j];
          }
#pragma unroll
          for (int j = 0; j < E; ++j) o[hf][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], p[kb][e], o[hf][j], 0, 0, 0);
        }
      }
  }
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  if (!live) return;
  const int64_t at = (int64_t)it.slot * a.B * a.T * a.Hq + n * a.Hq + h;
  if (lq == 0) *(float2*)(a.ml + at * 2) = make_float2(m * 1.4426950408889634f, lsum);
  float* orow = a.o + at * D;
#pragma unroll
  for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < E; ++j) orow[64 * hf + E * (4 * lq + e) + j] = o[hf][j][e];
}

// The slots of each query row joined, in slot order (maxima in base 2). A
// query that saw no key, in an idle row or one without any, gets zeros.
template <typename T, int D>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
  constexpr int LPR = D / 4;  // lanes of a query row, four dims each
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  const int64_t i = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (i >= rows) return;
  const int d = threadIdx.x % LPR * 4;
  const int slots = a.splits_p + a.splits_s;
  const bool idle = own_len(a, i / a.Hq / a.T) < 0;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < slots; ++s) {
    const float2 ml = *(const float2*)(a.ml + (s * rows + i) * 2);
    const f32x4 os = *(const f32x4*)(a.o + (s * rows + i) * D + d);
    if (ml.x == -__builtin_inff()) continue;  // the split saw no key
    const float mn = fmaxf(m, ml.x);
    const float a0 = __builtin_amdgcn_exp2f(m - mn), a1 = __builtin_amdgcn_exp2f(ml.x - mn);
    l = l * a0 + ml.y * a1;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a0 + os[e] * a1;
    m = mn;
  }
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = idle || m == -__builtin_inff() ? 0.f : o[e] / l;
  store_vec<T, 4>((T*)a.out + i * D + d, r);
}

// Query tiles and key splits of a call: enough blocks to fill the CUs twice,
// no split shorter than two key tiles.
struct Plan {
  int qtiles_p, qtiles_s, splits_p, splits_s;
  int64_t items_p, items_s;
};

int64_t splits_for(int64_t blocks, int64_t keys, int kt) {
  const int64_t want = cdiv((int64_t)2 * 256, std::max<int64_t>(blocks, 1));
  return std::max<int64_t>(1, std::min<int64_t>(want, keys / (2 * kt)));
}

Plan shared_plan(int64_t B, int64_t G, int64_t T, int64_t Hq, int64_t Hkv, int64_t P, int64_t C, int qt, int kt) {
  const int64_t per = Hq / Hkv;
  Plan p;
  p.qtiles_p = (int)cdiv(B / G * T * per, qt);
  p.qtiles_s = (int)cdiv(T * per, qt);
  const int64_t bp = P > 0 ? G * Hkv * p.qtiles_p : 0, bs = B * Hkv * p.qtiles_s;
  p.splits_p = P > 0 ? (int)splits_for(bp + bs, P, kt) : 0;
  p.splits_s = (int)splits_for(bp * p.splits_p + bs, C + T, kt);
  p.items_p = bp * p.splits_p;
  p.items_s = bs * p.splits_s;
  return p;
}

Plan plan_of(int dtype, int64_t D, int64_t B, int64_t G, int64_t T, int64_t Hq, int64_t Hkv, int64_t P, int64_t C) {
  return shared_plan(B, G, T, Hq, Hkv, P, C, F_QT, D >= 128 ? 32 : 64);
}

template <typename T, int D>
int shared_launch(hipStream_t st, const SharedArgs& a, const Plan& p) {
  hipLaunchKernelGGL((shared_attn_f32_kernel<T, D>), dim3((unsigned)(p.items_p + p.items_s)), dim3(256), 0, st, a);
  MINITP_LAUNCH_CHECK();
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  hipLaunchKernelGGL((shared_join_kernel<T, D>), dim3((unsigned)cdiv(rows, 256 / (D / 4))), dim3(256), 0, st, a);
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

template <typename T>
int shared_by_d(hipStream_t st, const SharedArgs& a, const Plan& p, int64_t D) {
  switch (D) {
    case 16:
      return shared_launch<T, 16>(st, a, p);
    case 32:
      return shared_launch<T, 32>(st, a, p);
    case 64:
      return shared_launch<T, 64>(st, a, p);
    case 128:
      return shared_launch<T, 128>(st, a, p);
  }
  set_error("shared_prefix_attention: head_dim %lld not supported (16, 32, 64, 128)", (long long)D);
  return MINITP_ERR_UNSUPPORTED;
}

}  // namespace

int64_t shared_prefix_workspace_bytes(int dtype, int64_t B, int64_t G, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                      int64_t P, int64_t C) {
  if (B * T == 0) return 0;
  const Plan p = plan_of(dtype, D, B, G, T, Hq, Hkv, P, C);
  return (p.splits_p + p.splits_s) * B * T * Hq * (D + 2) * 4;
}

int launch_shared_prefix_attention(hipStream_t st, int dtype, const SharedPrefixShape& s, const void* q,
                                   const void* k_prefix, const void* v_prefix, const void* k_cache,
                                   const void* v_cache, void* out, const int64_t* prefix_lens,
                                   const int64_t* cache_lens, void* workspace, int64_t workspace_bytes) {
  const Plan p = plan_of(dtype, s.D, s.B, s.G, s.T, s.Hq, s.Hkv, s.P, s.C);
  const int64_t need = shared_prefix_workspace_bytes(dtype, s.B, s.G, s.T, s.Hq, s.Hkv, s.D, s.P, s.C);
  if (workspace_bytes < need || workspace == nullptr || !aligned16(workspace)) {
    set_error("shared_prefix_attention: workspace %p of %lld B, %lld B needed (16-byte aligned)", workspace,
              (long long)workspace_bytes, (long long)need);
    return MINITP_ERR_ARG;
  }
  const int64_t rows = s.B * s.T * s.Hq;
  if (p.items_p + p.items_s >= (1LL << 31) || rows >= (1LL << 31) || s.B / s.G * s.T * (s.Hq / s.Hkv) >= (1LL << 31)) {
    set_error("shared_prefix_attention: %lld query rows are too many for one call", (long long)rows);
    return MINITP_ERR_UNSUPPORTED;
  }
  SharedArgs a{};
  a.q = q;
  a.kp = k_prefix;
  a.vp = v_prefix;
  a.kc = k_cache;
  a.vc = v_cache;
  a.out = out;
  a.B = (int)s.B;
  a.G = (int)s.G;
  a.T = (int)s.T;
  a.Hq = (int)s.Hq;
  a.Hkv = (int)s.Hkv;
  a.Sp = s.Sp;
  a.S = s.S;
  a.P = s.P;
  a.C = s.C;
  a.plens = prefix_lens;
  a.clens = cache_lens;
  a.scale = 1.0f / sqrtf((float)s.D);
  a.qtiles_p = p.qtiles_p;
  a.qtiles_s = p.qtiles_s;
  a.splits_p = p.splits_p;
  a.splits_s = p.splits_s;
  a.items_p = p.items_p;
  a.o = (float*)workspace;
  a.ml = a.o + (p.splits_p + p.splits_s) * rows * s.D;
  return dtype == MINITP_F32 ? shared_by_d<float>(st, a, p, s.D) : shared_by_d<bf16>(st, a, p, s.D);
}

}  // namespace minitp
