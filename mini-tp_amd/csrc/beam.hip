// Beam search on the device: the selection of the next beams over beams and
// vocabulary, and the K/V caches' rows following their beams.
//
// Selection, for G groups (prompts) of W beams with cumulative log-probability
// s_w and n_w tokens each: token v continues beam w with
//     score = s_w + x_wv - log sum_u exp(x_wu),   key = score / (n_w + 1)^alpha,
// a finished beam only with the end token and its own score and length. The W
// best keys of a group win, equal ones by the lower (beam, token). A beam that
// goes on keeps its place: the first continuation of each parent stays in the
// parent's slot, the others fill the free slots in rank order, so that the
// caches move as few rows as the selection allows (and no moved row's source
// is overwritten).
//
// Two launches, as the argmax has: slices of the logits rows to (maximum, sum
// of exponentials, W best tokens), then one block a group. The order of a row's
// tokens is that of its logits, so a slice needs no sum of the whole row.
#include <cmath>

#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

constexpr int SEL_T = 256, SEL_E = 16, SEL_SLICE = SEL_T * SEL_E;  // a slice: 16 consecutive logits a thread
constexpr int MERGE_T = 1024;
constexpr int MERGE_CAP = 1024;  // contenders that a group's final ranking takes

struct SelectArgs {
  const void* logits;
  int64_t ld_group, ld_beam;  // elements between groups and between beams (0: one row for all)
  int64_t V;
  int G, W, slices;
  const float* scores;      // [G, W]
  const uint8_t* finished;  // [G, W] or NULL
  const int64_t* lengths;   // [G, W] or NULL (zeros)
  int64_t eos;              // -1: none
  double alpha;
  int64_t *tokens, *parents;
  float* scores_out;
  uint8_t* finished_out;
  int64_t* lengths_out;
  // per (row, slice)
  double* sum;
  float* top;
  float* cand_v;    // [W] a slice, best first
  int32_t* cand_i;  // token, -1: none
};

template <typename T>
__device__ __forceinline__ const T* logits_row(const SelectArgs& a, int64_t row) {
  return (const T*)a.logits + row / a.W * a.ld_group + row % a.W * a.ld_beam;
}

// A row that is read: alive (a finite cumulative score) and not finished.
__device__ __forceinline__ bool beam_open(const SelectArgs& a, int64_t row) {
  return a.scores[row] != -__builtin_inff() && !(a.finished != nullptr && a.finished[row]);
}

// Contenders of a slice without sorting it: the W-th largest of the 64 maxima
// of four threads each (64 logits) bounds the slice's W-th largest logit from
// below. Fewer than W of those sets hold a logit above the bound, at most 64
// each; of the logits equal to it the first W in order are enough.
constexpr int SEL_CAP = 31 * 64 + 32;

template <typename T>
__global__ __launch_bounds__(SEL_T) void beam_slice_kernel(SelectArgs a) {
  __shared__ __attribute__((aligned(16))) float quad_top[64];
  __shared__ float lv[SEL_CAP];
  __shared__ int32_t li[SEL_CAP];
  __shared__ int wave_cnt[4];
  __shared__ float wave_m[4];
  __shared__ double wave_s[4];
  const int64_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  if (!beam_open(a, row)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = a.W;
  const T* lr = logits_row<T>(a, row) + slice * SEL_SLICE;
  const int n = (int)std::min<int64_t>(a.V - slice * SEL_SLICE, SEL_SLICE);  // logits of this slice
  const int j0 = tid * SEL_E;

  float x[SEL_E];
  if ((((uint64_t)lr) & 15) == 0 && j0 + SEL_E <= n) {
    constexpr int VE = Vec<T>::N;
    uint4 raw[SEL_E / VE];
#pragma unroll
    for (int u = 0; u < SEL_E / VE; ++u) raw[u] = *(const uint4*)(lr + j0 + u * VE);
#pragma unroll
    for (int u = 0; u < SEL_E / VE; ++u) unpack16(raw[u], x + u * VE, (T*)nullptr);
  } else {
#pragma unroll
    for (int e = 0; e < SEL_E; ++e) x[e] = j0 + e < n ? load_f32<T>(lr, j0 + e) : -__builtin_inff();
  }

  // ---- maximum and sum of exponentials (a NaN shows in the sum) -----------
  float t = x[0];
#pragma unroll
  for (int e = 1; e < SEL_E; ++e) t = fmaxf(t, x[e]);
  t = t == t ? t : -__builtin_inff();
  const float wm = wave_max(t), ref = wm == -__builtin_inff() ? 0.f : wm;
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < SEL_E; ++e) s += expf(x[e] - ref);
  double ws = s;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) ws += __shfl_xor(ws, o, 64);
  if (lane == 0) {
    wave_m[wave] = wm;
    wave_s[wave] = ws;
  }

  // ---- the bound ------------------------------------------------------------
  float qt = fmaxf(t, dpp_f32<0xB1>(t, t));
  qt = fmaxf(qt, dpp_f32<0x4E>(qt, qt));
  if ((lane & 3) == 0) quad_top[wave * 16 + lane / 4] = qt;
  __syncthreads();
  float bound;
  {
    const float v = quad_top[lane];
    int better = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
      const float u = quad_top[j];
      better += u > v || (u == v && j < lane);
    }
    const uint64_t at = __builtin_amdgcn_ballot_w64(better == W - 1);
    bound = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), __builtin_ctzll(at)));
  }

  // ---- contenders: above the bound in the low half, equal to it in the high
  const bool low = bound == -__builtin_inff();  // (equal: not a candidate)
  int cnt = 0;
#pragma unroll
  for (int e = 0; e < SEL_E; ++e) cnt += (x[e] > bound ? 1 : 0) + (x[e] == bound && !low ? 1 << 16 : 0);
  int before = cnt;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(before, o, 64);
    if (lane >= o) before += u;
  }
  if (lane == 63) wave_cnt[wave] = before;
  before -= cnt;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w == wave) before += total;
    total += wave_cnt[w];
  }
  const int above = total & 0xffff, equal = std::min(total >> 16, W);
  if (cnt != 0) {
    int pa = before & 0xffff, pe = before >> 16;
#pragma unroll
    for (int e = 0; e < SEL_E; ++e) {
      if (x[e] > bound) {
        lv[pa] = x[e];
        li[pa++] = j0 + e;
      } else if (x[e] == bound && !low) {
        if (pe < equal) {
          lv[above + pe] = x[e];
          li[above + pe] = j0 + e;
        }
        ++pe;
      }
    }
  }
  __syncthreads();

  // ---- rank them; the W best, best first -----------------------------------
  const int c = above + equal;
  const int64_t at = row * a.slices + slice;
  float* cv = a.cand_v + at * W;
  int32_t* ci = a.cand_i + at * W;
  for (int i = tid; i < c; i += SEL_T) {
    const float v = lv[i];
    const int vi = li[i];
    int rank = 0;
    for (int j = 0; j < c; ++j) rank += lv[j] > v || (lv[j] == v && li[j] < vi);
    if (rank < W) {
      cv[rank] = v;
      ci[rank] = (int32_t)(slice * SEL_SLICE + vi);
    }
  }
  for (int i = c + tid; i < W; i += SEL_T) ci[i] = -1;
  if (tid == 0) {
    float m = wave_m[0];
    for (int w = 1; w < 4; ++w) m = fmaxf(m, wave_m[w]);
    double sum = 0.0;
    for (int w = 0; w < 4; ++w)
      sum += wave_m[w] == -__builtin_inff() ? wave_s[w] : wave_s[w] * exp((double)wave_m[w] - (double)m);
    a.top[at] = m;
    a.sum[at] = sum;
  }
}

// Keys as whole numbers in their order: 0 is no candidate (minus infinity), a
// NaN stands above every number.
__device__ __forceinline__ uint64_t order_key(double k) {
  if (k != k) return ~0ull;
  if (k == -__builtin_inf()) return 0;
  const uint64_t u = __builtin_bit_cast(uint64_t, k + 0.0);  // (-0 is 0)
  return u >> 63 ? ~u : u | (1ull << 63);
}

enum { ROW_NONE = 0, ROW_OPEN = 1, ROW_DONE = 2, ROW_NAN = 3 };

template <typename T>
__global__ __launch_bounds__(MERGE_T) void beam_merge_kernel(SelectArgs a) {
  __shared__ int kind[32];
  __shared__ float score[32];
  __shared__ double lse[32], inv[32];
  __shared__ uint64_t group_top[64];
  __shared__ uint64_t lk[MERGE_CAP], lf[MERGE_CAP];  // key; beam << 32 | token
  __shared__ uint64_t best_k[MERGE_T / 64], best_f[MERGE_T / 64];
  __shared__ int count;
  __shared__ uint64_t sel[32];
  const int W = a.W, g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row0 = (int64_t)g * W;
  const int eos32 = (int)a.eos;

  // ---- each beam's log sum, kind and length factor -------------------------
  for (int w = wave; w < W; w += MERGE_T / 64) {
    const int64_t row = row0 + w;
    const float sc = a.scores[row];
    const bool done = a.finished != nullptr && a.finished[row];
    int k = sc == -__builtin_inff() ? ROW_NONE : done ? ROW_DONE : sc != sc ? ROW_NAN : ROW_OPEN;
    double m = -__builtin_inf(), s = 0.0;
    if (k == ROW_OPEN) {
      float mf = -__builtin_inff();
      for (int i = lane; i < a.slices; i += 64) mf = fmaxf(mf, a.top[row * a.slices + i]);
      mf = wave_max(mf);
      m = mf;
      for (int i = lane; i < a.slices; i += 64) {
        const float t = a.top[row * a.slices + i];
        const double si = a.sum[row * a.slices + i];
        s += t == -__builtin_inff() ? si : si * exp((double)t - m);
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
      // no logit above minus infinity: nothing continues this beam
      if (s != s)
        k = ROW_NAN;
      else if (mf == -__builtin_inff())
        k = ROW_NONE;
    }
    if (lane == 0) {
      const int64_t len = (a.lengths != nullptr ? a.lengths[row] : 0) + (done ? 0 : 1);
      kind[w] = k;
      score[w] = sc;
      lse[w] = k == ROW_OPEN ? m + log(s) : 0.0;
      inv[w] = a.alpha == 0.0 ? 1.0 : pow((double)std::max<int64_t>(len, 1), -a.alpha);
    }
  }
  if (tid == 0) count = 0;
  __syncthreads();

  // candidate e = (beam, slice, rank): its key (0: none) and token
  const int per_row = a.slices * W, entries = per_row * W;
  auto candidate = [&](int e, uint64_t& flat) -> uint64_t {
    const int w = e / per_row, i = e - w * per_row;
    const int k = kind[w];
    int token;
    uint64_t key = 0;
    if (k == ROW_OPEN) {
      token = a.cand_i[row0 * per_row + e];
      if (token >= 0) {
        const double lp = (double)a.cand_v[row0 * per_row + e] - lse[w];
        key = order_key(((double)score[w] + lp) * inv[w]);
      }
    } else if (k == ROW_DONE) {
      token = eos32;
      if (i == 0) key = order_key((double)score[w] * inv[w]);
    } else {
      token = i;
      if (k == ROW_NAN && i < W && i < a.V) key = ~0ull;
    }
    flat = (uint64_t)w << 32 | (uint32_t)token;
    return key;
  };
  auto better = [](uint64_t ka, uint64_t fa, uint64_t kb, uint64_t fb) { return ka > kb || (ka == kb && fa < fb); };

  // ---- contenders, as in the slices: the W-th largest of 64 maxima ----------
  uint64_t top = 0, flat;
  for (int e = tid; e < entries; e += MERGE_T) top = std::max(top, candidate(e, flat));
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {
    const uint64_t u = __shfl_xor(top, o, 64);
    top = u > top ? u : top;
  }
  if (lane % 16 == 0) group_top[tid / 16] = top;
  __syncthreads();
  uint64_t bound;
  {
    const uint64_t v = group_top[lane];
    int ahead = 0;
    for (int j = 0; j < 64; ++j) {
      const uint64_t u = group_top[j];
      ahead += u > v || (u == v && j < lane);
    }
    bound = __shfl(v, __builtin_ctzll(__builtin_amdgcn_ballot_w64(ahead == W - 1)), 64);
  }
  bound = std::max<uint64_t>(bound, 1);
  for (int e = tid; e < entries; e += MERGE_T) {
    const uint64_t k = candidate(e, flat);
    if (k < bound) continue;
    const int at = atomicAdd(&count, 1);
    if (at < MERGE_CAP) {
      lk[at] = k;
      lf[at] = flat;
    }
  }
  __syncthreads();
  int n = count;
  if (n <= MERGE_CAP) {
    for (int i = tid; i < n; i += MERGE_T) {
      const uint64_t k = lk[i], f = lf[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += better(lk[j], lf[j], k, f);
      if (rank < W) sel[rank] = f;
    }
    n = std::min(n, W);
  } else {
    // more equals than the list holds: one winner at a time
    uint64_t pk = ~0ull, pf = 0;
    bool first = true;
    for (n = 0; n < W; ++n) {
      uint64_t bk = 0, bf = ~0ull;
      for (int e = tid; e < entries; e += MERGE_T) {
        const uint64_t k = candidate(e, flat);
        if (k != 0 && (first || better(pk, pf, k, flat)) && better(k, flat, bk, bf)) {
          bk = k;
          bf = flat;
        }
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t ok = __shfl_xor(bk, o, 64), of = __shfl_xor(bf, o, 64);
        if (better(ok, of, bk, bf)) {
          bk = ok;
          bf = of;
        }
      }
      __syncthreads();
      if (lane == 0) {
        best_k[wave] = bk;
        best_f[wave] = bf;
      }
      __syncthreads();
      for (int j = 0; j < MERGE_T / 64; ++j)
        if (better(best_k[j], best_f[j], bk, bf)) {
          bk = best_k[j];
          bf = best_f[j];
        }
      if (bk == 0) break;
      if (tid == 0) sel[n] = bf;
      pk = bk;
      pf = bf;
      first = false;
    }
  }
  __syncthreads();

  // ---- places, outputs (lane = rank) ----------------------------------------
  if (wave != 0) return;
  const bool chosen = lane < n;
  const int p = chosen ? (int)(sel[lane] >> 32) : 0;
  const int token = chosen ? (int)(uint32_t)sel[lane] : 0;
  bool stays = chosen;
  for (int j = 0; j < n; ++j) {
    const int pj = (int)(sel[j] >> 32);
    if (j < lane && pj == p) stays = false;
  }
  uint32_t taken = 0;
  const uint64_t stay_mask = __builtin_amdgcn_ballot_w64(stays);
  for (int j = 0; j < n; ++j)
    if (stay_mask >> j & 1) taken |= 1u << (int)(sel[j] >> 32);
  int slot = p;
  if (!stays) {
    // the k-th free slot, k = the ranks below this one that do not stay
    int k = __builtin_popcountll(~stay_mask & ((1ull << lane) - 1));
    uint32_t free = ~taken;
    for (; k > 0; --k) free &= free - 1;
    slot = free ? __builtin_ctz(free) : W;
  }
  if (lane >= W) return;
  float sc = -__builtin_inff();
  bool done = true;
  int64_t len = a.lengths != nullptr ? a.lengths[row0 + slot] : 0;
  if (chosen) {
    const bool was = a.finished != nullptr && a.finished[row0 + p];
    sc = kind[p] == ROW_DONE  ? score[p]
         : kind[p] == ROW_NAN ? __builtin_nanf("")
                              : (float)((double)score[p] + ((double)load_f32<T>(logits_row<T>(a, row0 + p), token) - lse[p]));
    done = was || token == eos32;
    len = (a.lengths != nullptr ? a.lengths[row0 + p] : 0) + (was ? 0 : 1);
  }
  // every input of the group has been read: the outputs may be the inputs
  __builtin_amdgcn_wave_barrier();
  a.tokens[row0 + slot] = chosen ? token : std::max(eos32, 0);
  a.parents[row0 + slot] = row0 + (chosen ? p : slot);
  a.scores_out[row0 + slot] = sc;
  a.finished_out[row0 + slot] = done;
  a.lengths_out[row0 + slot] = len;
}

// ---------------------------------------------------------------------------
// Rows 0 .. rows - 1 of every (layer, KV head) of beam b take those of beam
// parents[b], in place, K and V in one launch. A thread owns the same 16 bytes
// of all W beams of a group: it loads those of every moved beam's parent and
// only then stores, so it needs no copy and no order between blocks whatever
// the parents are. A beam that keeps its rows is neither read nor written (its
// resource is empty: loads return zeros, stores are dropped), and nor is one
// whose parent is not a row of its group.
struct ReorderArgs {
  void *k, *v;             // [L, B, Hkv, S, D]
  int64_t head_bytes;      // S * D elements
  int64_t row_bytes;       // Hkv * S * D elements
  uint32_t bytes;          // rows * D elements
  int Hkv, G, W;
  const int64_t* parents;  // [G, W], rows of the batch
};

template <int NB>
__global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderArgs a) {
  const int lh = blockIdx.y, l = lh / a.Hkv, h = lh % a.Hkv;
  const int g = blockIdx.z >> 1;
  char* base = (char*)(blockIdx.z & 1 ? a.v : a.k) +
               ((int64_t)l * a.G + g) * a.W * a.row_bytes + h * a.head_bytes;
  const uint32_t off = (blockIdx.x * 256 + threadIdx.x) * 16;
  u32x4 val[NB];
#pragma unroll
  for (int w = 0; w < NB; ++w) {
    const int64_t p = w < a.W ? a.parents[g * a.W + w] - (int64_t)g * a.W : w;
    const bool moved = p != w && p >= 0 && p < a.W;
    val[w] = __builtin_bit_cast(
        u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                   span_rsrc(base + (moved ? p : 0) * a.row_bytes, moved ? a.bytes : 0), off, 0, 0));
  }
#pragma unroll
  for (int w = 0; w < NB; ++w) {
    const int64_t p = w < a.W ? a.parents[g * a.W + w] - (int64_t)g * a.W : w;
    const bool moved = p != w && p >= 0 && p < a.W;
    __builtin_amdgcn_raw_buffer_store_b128(
        val[w], span_rsrc(base + (moved ? w : 0) * a.row_bytes, moved ? a.bytes : 0), off, 0, 0);
  }
}

int64_t select_slices(int64_t V) { return cdiv(V, SEL_SLICE); }

}  // namespace

int64_t beam_select_workspace_bytes(int64_t G, int64_t W, int64_t V) {
  return G * W * select_slices(V) * (8 + 4 + W * 8);
}

int launch_beam_select(hipStream_t st, int dtype, const BeamSelect& b, void* workspace, int64_t workspace_bytes) {
  const int64_t need = beam_select_workspace_bytes(b.G, b.W, b.V);
  if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)) {
    set_error("beam_select: workspace %p of %lld B, %lld B needed (16-byte aligned)", workspace,
              (long long)workspace_bytes, (long long)need);
    return MINITP_ERR_ARG;
  }
  const int64_t rows = b.G * b.W, parts = rows * select_slices(b.V);
  if (parts >= (1LL << 31) || b.W * b.W * select_slices(b.V) >= (1LL << 30)) {
    set_error("beam_select: %lld rows of %lld logits are too many for one call", (long long)rows, (long long)b.V);
    return MINITP_ERR_UNSUPPORTED;
  }
  SelectArgs a{};
  a.logits = b.logits;
  a.ld_group = b.ld_group;
  a.ld_beam = b.ld_beam;
  a.V = b.V;
  a.G = (int)b.G;
  a.W = (int)b.W;
  a.slices = (int)select_slices(b.V);
  a.scores = b.scores;
  a.finished = b.finished;
  a.lengths = b.lengths;
  a.eos = b.eos;
  a.alpha = b.alpha;
  a.tokens = b.tokens;
  a.parents = b.parents;
  a.scores_out = b.scores_out;
  a.finished_out = b.finished_out;
  a.lengths_out = b.lengths_out;
  a.sum = (double*)workspace;
  a.top = (float*)(a.sum + parts);
  a.cand_v = a.top + parts;
  a.cand_i = (int32_t*)(a.cand_v + parts * b.W);
  if (dtype == MINITP_F32) {
    beam_slice_kernel<float><<<(unsigned)parts, SEL_T, 0, st>>>(a);
    MINITP_LAUNCH_CHECK();
    beam_merge_kernel<float><<<(unsigned)b.G, MERGE_T, 0, st>>>(a);
  } else {
    beam_slice_kernel<bf16><<<(unsigned)parts, SEL_T, 0, st>>>(a);
    MINITP_LAUNCH_CHECK();
    beam_merge_kernel<bf16><<<(unsigned)b.G, MERGE_T, 0, st>>>(a);
  }
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

int launch_kv_reorder(hipStream_t st, int dtype, void* k, void* v, int64_t L, int64_t G, int64_t W, int64_t Hkv,
                      int64_t S, int64_t D, int64_t rows, const int64_t* parents) {
  const int64_t es = dtype == MINITP_F32 ? 4 : 2;
  if (rows * D * es >= (1LL << 31) || L * Hkv > 65535 || G > 32767) {
    set_error("kv_reorder: %lld rows of %lld, %lld layers of %lld heads, %lld groups are too many for one call",
              (long long)rows, (long long)D, (long long)L, (long long)Hkv, (long long)G);
    return MINITP_ERR_UNSUPPORTED;
  }
  ReorderArgs a{};
  a.k = k;
  a.v = v;
  a.head_bytes = S * D * es;
  a.row_bytes = Hkv * S * D * es;
  a.bytes = (uint32_t)(rows * D * es);
  a.Hkv = (int)Hkv;
  a.G = (int)G;
  a.W = (int)W;
  a.parents = parents;
  const dim3 grid((unsigned)cdiv(a.bytes, 4096), (unsigned)(L * Hkv), (unsigned)(2 * G));
  if (W <= 4)
    kv_reorder_kernel<4><<<grid, 256, 0, st>>>(a);
  else if (W <= 8)
    kv_reorder_kernel<8><<<grid, 256, 0, st>>>(a);
  else if (W <= 16)
    kv_reorder_kernel<16><<<grid, 256, 0, st>>>(a);
  else
    kv_reorder_kernel<32><<<grid, 256, 0, st>>>(a);
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

}  // namespace minitp
