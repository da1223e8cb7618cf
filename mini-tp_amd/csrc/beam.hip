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
// Two launches, as the argmax has. The first streams the logits: per wave a
// maximum and a sum of exponentials, per set of 64 consecutive logits their
// maximum. The second, one block a group, ranks the sets by the key of their
// maximum: whatever is among the W best tokens lies in the W best sets (W
// tokens, the sets' maxima, stand before every token of any other set), so
// only those sets' logits are read again. The order of a row's tokens is that
// of its logits, so the first launch needs no sum of the whole row.
#include <cmath>

#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

constexpr int SEL_T = 256, SEL_NV = 4;  // threads of a slice, 16-byte loads a thread
constexpr int SET = 64;                 // logits of a set
constexpr int MERGE_T = 1024;
constexpr int MERGE_CAP = 1024;  // sets that a group's ranking takes at once

template <typename T>
constexpr int SLICE = SEL_T * SEL_NV * Vec<T>::N;

struct SelectArgs {
  const void* logits;
  int64_t ld_group, ld_beam;  // elements between groups and between beams (0: one row for all)
  int64_t V;
  int G, W, slices;
  int sets;                 // of a row, padded to whole float4
  const float* scores;      // [G, W]
  const uint8_t* finished;  // [G, W] or NULL
  const int64_t* lengths;   // [G, W] or NULL (zeros)
  int64_t eos;              // -1: none
  double alpha;
  int64_t *tokens, *parents;
  float* scores_out;
  uint8_t* finished_out;
  int64_t* lengths_out;
  double* sum;     // [row][slice][wave]: sum of exponentials above ...
  float* top;      // ... this maximum
  float* set_top;  // [row][sets]
};

template <typename T>
__device__ __forceinline__ const T* logits_row(const SelectArgs& a, int64_t row) {
  return (const T*)a.logits + row / a.W * a.ld_group + row % a.W * a.ld_beam;
}

// A row that is read: alive (a cumulative score above minus infinity) and not finished.
__device__ __forceinline__ bool beam_open(const SelectArgs& a, int64_t row) {
  return a.scores[row] != -__builtin_inff() && !(a.finished != nullptr && a.finished[row]);
}

// exp(x) for x <= 0 by the hardware's 2^x, the product x log2(e) carried in two
// parts: its rounding alone, up to 2^-24 of an exponent of some tens, would be
// the sum's largest error. Below -104 the result is zero (a product of the type's
// lowest values would overflow); a NaN stays one.
__device__ __forceinline__ float exp_below(float x) {
  constexpr float L = 1.44269502f, L_LO = 1.92596299e-8f, LN2 = 0.693147182f;
  const float hi = x * L, lo = fmaf(x, L_LO, fmaf(x, L, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  return x < -104.f ? 0.f : fmaf(e, lo * LN2, e);
}

// One slice of a row a block: lanes take 16 bytes each of consecutive logits, so
// that a set is 8 (bf16) or 16 (fp32) lanes of one load. Nothing is exchanged
// between the waves. Bound by memory: 13 x 16 rows of 151,936 fp32 logits, 126 MB
// in 25 us, 5.0 TB/s; 4 rows of bf16 5 us, latency.
template <typename T>
__global__ __launch_bounds__(SEL_T) void beam_slice_kernel(SelectArgs a) {
  constexpr int VE = Vec<T>::N, LPS = SET / VE;
  const int64_t row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  if (!beam_open(a, row)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* lr = logits_row<T>(a, row) + slice * SLICE<T>;
  const int n = (int)std::min<int64_t>(a.V - slice * SLICE<T>, SLICE<T>);  // logits of this slice
  float x[SEL_NV][VE];
  if ((((uint64_t)lr) & 15) == 0) {
    const __amdgpu_buffer_rsrc_t r = span_rsrc(lr, (uint32_t)(n * (int)sizeof(T)));
    u32x4 raw[SEL_NV];
#pragma unroll
    for (int v = 0; v < SEL_NV; ++v) {
      // (whole vectors only; the others read zeros here)
      const int j = (v * SEL_T + tid) * VE;
      raw[v] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             r, j + VE <= n ? (uint32_t)(j * (int)sizeof(T)) : 0xffffffffu, 0, 0));
    }
#pragma unroll
    for (int v = 0; v < SEL_NV; ++v) {
      unpack16(make_uint4(raw[v].x, raw[v].y, raw[v].z, raw[v].w), x[v], (T*)nullptr);
      const int j = (v * SEL_T + tid) * VE;
      if (j + VE > n) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[v][e] = j + e < n ? load_f32<T>(lr, j + e) : -__builtin_inff();
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < SEL_NV; ++v)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int j = (v * SEL_T + tid) * VE + e;
        x[v][e] = j < n ? load_f32<T>(lr, j) : -__builtin_inff();
      }
  }

  const float ninf = -__builtin_inff();
  float t = ninf;
#pragma unroll
  for (int v = 0; v < SEL_NV; ++v) {
    float m = ninf;  // (a NaN is no maximum; it shows in the sum)
#pragma unroll
    for (int e = 0; e < VE; ++e) m = fmaxf(m, x[v][e]);
    t = fmaxf(t, m);
    m = fmaxf(m, dpp_f32<0xB1>(ninf, m));   // lanes of the set: quad_perm [1,0,3,2]
    m = fmaxf(m, dpp_f32<0x4E>(ninf, m));   // quad_perm [2,3,0,1]
    m = fmaxf(m, dpp_f32<0x141>(ninf, m));  // row_half_mirror
    if constexpr (LPS == 16) m = fmaxf(m, dpp_f32<0x140>(ninf, m));  // row_mirror
    const int64_t set = (slice * SLICE<T> + (v * SEL_T + tid) * VE) / SET;
    if (lane % LPS == 0 && set < a.sets) a.set_top[row * a.sets + set] = m;
  }
  const float wm = wave_max(t), ref = wm == ninf ? 0.f : wm;
  float s[SEL_NV];  // (a chain a load)
#pragma unroll
  for (int v = 0; v < SEL_NV; ++v) {
    s[v] = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) s[v] += exp_below(x[v][e] - ref);
  }
  double ws = (double)((s[0] + s[1]) + (s[2] + s[3]));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) ws += __shfl_xor(ws, o, 64);
  if (lane == 0) {
    const int64_t at = (row * a.slices + slice) * (SEL_T / 64) + wave;
    a.top[at] = wm;
    a.sum[at] = ws;
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

// The rows of a group, MERGE_T / wp threads each (wp >= W, a power of two). A
// thread keeps its sets' maxima, at most 4 NR (0: any number, read again).
// One block a group, a chain of short steps and barriers, all latency: 4 rows
// of 151,936 logits 8.5 us, 8 groups of 8 10.5, 13 groups of 16 in fp32 14.
template <typename T, int NR>
__global__ __launch_bounds__(MERGE_T) void beam_merge_kernel(SelectArgs a, int wp) {
  __shared__ int kind[32];
  __shared__ float score[32];
  __shared__ double top[32], lse[32], inv[32];             // (log sum above the row's maximum: that may be -3e38)
  __shared__ uint64_t group_top[64];
  __shared__ uint64_t lk[MERGE_CAP], lf[MERGE_CAP];        // sets: key of the maximum; beam << 32 | set
  __shared__ float lx[MERGE_CAP];                          // maximum
  __shared__ uint64_t ek[32 * SET], ef[32 * SET];          // tokens of the best sets: key; beam << 32 | token
  __shared__ uint64_t best_k[MERGE_T / 64], best_f[MERGE_T / 64];
  __shared__ int count, ecount;
  __shared__ uint64_t limit;
  __shared__ uint64_t set_k[32], set_f[32], sel[32];
  __shared__ float ex[32 * SET], sel_x[32];                // their logits
  __shared__ uint8_t ended[32];
  __shared__ int64_t length[32];
  __shared__ int first[32];                                // best rank of a parent
  const int W = a.W, g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row0 = (int64_t)g * W;
  const int eos32 = (int)a.eos;

  // This thread's sets, four at a time: f(set, maximum). (A row that is not open
  // has no maxima: what its words hold is left out below.)
  int tpr = MERGE_T / wp, mw = tid / tpr, mj = tid % tpr, quads = mw < W ? a.sets / 4 : 0;
  const float4* set_top = (const float4*)(a.set_top + (row0 + std::min(mw, W - 1)) * a.sets);
  auto four = [&](int i, const float4& x, auto f) {
    f(4 * i, x.x);
    f(4 * i + 1, x.y);
    f(4 * i + 2, x.z);
    f(4 * i + 3, x.w);
  };
  auto read_sets = [&](auto f) {
#pragma unroll 4
    for (int i = mj; i < quads; i += tpr) four(i, set_top[i], f);
  };
  float4 kept[NR > 0 ? NR : 1];
  bool keeps = NR > 0;
  auto each_set = [&](auto f) {
    if (!keeps) return read_sets(f);
#pragma unroll
    for (int u = 0; u < NR; ++u)
      if (mj + u * tpr < quads) four(mj + u * tpr, kept[u], f);
  };

  // ---- each beam's log sum, kind and length factor, a wave a beam; the first
  // ones' loads are in flight with those of the sets' maxima -----------------
  const int parts = a.slices * (SEL_T / 64);
  constexpr int PRE = 3;
  float sc = 0.f, pt[PRE];
  double ps[PRE];
  bool done = false;
  int64_t len = 0;
  auto load_beam = [&](int w) {
    const int64_t row = row0 + w;
    sc = a.scores[row];
    done = a.finished != nullptr && a.finished[row];
    len = a.lengths != nullptr ? a.lengths[row] : 0;
#pragma unroll
    for (int u = 0; u < PRE; ++u) {
      const int i = std::min(lane + 64 * u, parts - 1);
      pt[u] = a.top[row * parts + i];
      ps[u] = a.sum[row * parts + i];
    }
  };
  auto beam = [&](int w) {
    const int64_t row = row0 + w;
    int k = sc == -__builtin_inff() ? ROW_NONE : done ? ROW_DONE : sc != sc ? ROW_NAN : ROW_OPEN;
    double m = 0.0, s = 1.0;
    if (k == ROW_OPEN) {
      s = 0.0;
      float mf = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < PRE; ++u)
        if (lane + 64 * u < parts) mf = fmaxf(mf, pt[u]);
      for (int i = lane + 64 * PRE; i < parts; i += 64) mf = fmaxf(mf, a.top[row * parts + i]);
      mf = wave_max(mf);
      auto add = [&](float t, double si) { s += t == -__builtin_inff() ? si : si * (double)exp_below(t - mf); };
#pragma unroll
      for (int u = 0; u < PRE; ++u)
        if (lane + 64 * u < parts) add(pt[u], ps[u]);
      for (int i = lane + 64 * PRE; i < parts; i += 64) add(a.top[row * parts + i], a.sum[row * parts + i]);
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
      // no logit above minus infinity: nothing continues this beam
      if (s != s)
        k = ROW_NAN;
      else if (mf == -__builtin_inff())
        k = ROW_NONE;
      m = mf;
    }
    // one logarithm for both: of the sum (lane 0) and of the length (lane 1)
    const double lg = log(lane == 1 ? (double)std::max<int64_t>(len + (done ? 0 : 1), 1) : s);
    if (lane == 0) {
      kind[w] = k;
      score[w] = sc;
      ended[w] = done;
      length[w] = len;
      first[w] = 64;
      top[w] = m;
      lse[w] = lg;
    }
    if (lane == 1) inv[w] = a.alpha == 0.0 ? 1.0 : exp(-a.alpha * lg);
  };
  if (tid == 0) count = ecount = 0;
  if (wave < W) load_beam(wave);
  if constexpr (NR > 0) {
#pragma unroll
    for (int u = 0; u < NR; ++u) kept[u] = set_top[std::min(mj + u * tpr, a.sets / 4 - 1)];
  }
  float most = -__builtin_inff();
  each_set([&](int, float x) { most = fmaxf(most, x); });
  if (wave < W) beam(wave);
  if (wave + MERGE_T / 64 < W) {
    load_beam(wave + MERGE_T / 64);
    beam(wave + MERGE_T / 64);
  }
  __syncthreads();

  auto key_of = [&](int w, float x) { return order_key(((double)score[w] + (((double)x - top[w]) - lse[w])) * inv[w]); };
  auto better = [](uint64_t ka, uint64_t fa, uint64_t kb, uint64_t fb) { return ka > kb || (ka == kb && fa < fb); };
  // ranks of n entries, 32 lanes an entry: f(rank, index)
  auto rank_all = [&](const uint64_t* k, const uint64_t* f, int n, auto put) {
    for (int i = tid / 32; i < n; i += MERGE_T / 32) {
      int ahead = 0;
      for (int j = tid % 32; j < n; j += 32) ahead += better(k[j], f[j], k[i], f[i]);
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) ahead += __shfl_xor(ahead, o, 64);
      if (tid % 32 == 0 && ahead < W) put(ahead, i);
    }
  };
  // A finished beam and one that is no number have one set, the first, with a
  // key of its own: thread w's.
  const int tkind = tid < W ? kind[tid] : ROW_NONE;
  const uint64_t only = tkind == ROW_DONE ? order_key((double)score[tid] * inv[tid]) : tkind == ROW_NAN ? ~0ull : 0;

  // Few open rows (the first step has one a group): all threads on them, so that
  // the bound below comes from at least 32 of the 64 sets of threads.
  uint32_t open = (uint32_t)__builtin_amdgcn_ballot_w64(lane < W && kind[lane & 31] == ROW_OPEN);
  const int nopen = __builtin_popcount(open);
  if (2 * nopen <= wp) {
    int wq = 1;
    while (wq < nopen) wq *= 2;
    tpr = MERGE_T / wq;
    mj = tid % tpr;
    for (int j = tid / tpr; j > 0; --j) open &= open - 1;
    mw = open ? __builtin_ctz(open) : W;
    quads = mw < W ? a.sets / 4 : 0;
    set_top = (const float4*)(a.set_top + (row0 + std::min(mw, W - 1)) * a.sets);
    keeps = false;
    most = -__builtin_inff();
    read_sets([&](int, float x) { most = fmaxf(most, x); });
  }
  const bool mopen = mw < W && kind[mw] == ROW_OPEN;

  // ---- a bound: the W-th largest of the 64 maxima of 16 threads each ---------
  // (16 threads of one row: one DPP row)
  float rmost = most;
  rmost = fmaxf(rmost, dpp_f32<0xB1>(rmost, rmost));
  rmost = fmaxf(rmost, dpp_f32<0x4E>(rmost, rmost));
  rmost = fmaxf(rmost, dpp_f32<0x141>(rmost, rmost));
  rmost = fmaxf(rmost, dpp_f32<0x140>(rmost, rmost));
  if (lane % 16 == 0) group_top[tid / 16] = mopen ? key_of(mw, rmost) : 0;
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 4; ++c) {  // a wave ranks four of them
    const int i = wave * 4 + c;
    const uint64_t u = group_top[lane], v = group_top[i];
    const uint64_t ahead = __builtin_amdgcn_ballot_w64(u > v || (u == v && lane < i));
    if (lane == 0 && __builtin_popcountll(ahead) == W - 1) limit = std::max<uint64_t>(v, 1);
  }
  __syncthreads();
  const uint64_t bound = limit;

  // ---- the W best sets: first those whose maxima reach the bound, taken as a
  // logit of their row and lowered past what its rounding can be -------------
  auto take = [&](int w, int set, float x) {
    const int at = atomicAdd(&count, 1);
    if (at < MERGE_CAP) {
      lx[at] = x;
      lf[at] = (uint64_t)w << 32 | (uint32_t)set;
    }
  };
  if (mopen) {
    const double bk = __builtin_bit_cast(double, bound >> 63 ? bound ^ (1ull << 63) : ~bound);
    const double need = bk / inv[mw];
    const float bx = (float)(((need - (double)score[mw]) + lse[mw]) + top[mw]);
    const float off = (fabsf(bx) + 1.f) * 1e-5f + (float)(fabs(need) + fabs((double)score[mw])) * 1e-14f;
    // (above minus infinity at least: those are no candidates)
    const float low = bound == 1 ? -3.402823466e38f : fmaxf(bx - off, -3.402823466e38f);
    if (most >= low)
      each_set([&](int set, float x) {
        if (x >= low) take(mw, set, x);
      });
  }
  if (only >= bound) take(tid, 0, 0.f);
  __syncthreads();
  int n = count;
  uint64_t least = bound;
  for (int i = tid; i < std::min(n, MERGE_CAP); i += MERGE_T) {
    const int w = (int)(lf[i] >> 32);
    lk[i] = kind[w] == ROW_OPEN ? key_of(w, lx[i]) : kind[w] == ROW_DONE ? order_key((double)score[w] * inv[w]) : ~0ull;
  }
  __syncthreads();
  if (n <= 32) {  // few enough to take all
    if (tid < n) {
      set_k[tid] = lk[tid];
      set_f[tid] = lf[tid];
    }
  } else if (n <= MERGE_CAP) {
    rank_all(lk, lf, n, [&](int rank, int i) {
      set_k[rank] = lk[i];
      set_f[rank] = lf[i];
    });
    n = W;
  } else {
    // more equal sets than the list holds: one winner at a time
    uint64_t pk = 0, pf = 0;
    for (n = 0; n < W; ++n) {
      uint64_t bk = 0, bf = ~0ull;
      auto see = [&](uint64_t k, int w, int set) {
        const uint64_t f = (uint64_t)w << 32 | (uint32_t)set;
        if (k != 0 && (n == 0 || better(pk, pf, k, f)) && better(k, f, bk, bf)) {
          bk = k;
          bf = f;
        }
      };
      if (mopen) read_sets([&](int set, float x) { see(key_of(mw, x), mw, set); });
      see(only, tid, 0);
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
      if (tid == 0) {
        set_k[n] = bk;
        set_f[n] = bf;
      }
      pk = bk;
      pf = bf;
    }
  }
  __syncthreads();

  // ---- their tokens: those not below the last set's maximum, ranked ----------
  if (count > 32 && n == W) least = set_k[W - 1];
  for (int i = tid; i < n * SET; i += MERGE_T) {
    const int w = (int)(set_f[i / SET] >> 32), set = (int)(uint32_t)set_f[i / SET], e = i % SET;
    int token = set * SET + e;
    uint64_t k = 0;
    float x = 0.f;
    if (kind[w] == ROW_OPEN) {
      if (token < a.V) {
        x = load_f32<T>(logits_row<T>(a, row0 + w), token);
        k = key_of(w, x);
      }
    } else if (kind[w] == ROW_DONE) {
      if (e == 0) k = set_k[i / SET];
      token = eos32;
    } else if (e < W && e < a.V) {
      k = ~0ull;  // (no number: its lowest tokens)
    }
    if (k < least) continue;
    const int at = atomicAdd(&ecount, 1);
    ek[at] = k;
    ef[at] = (uint64_t)w << 32 | (uint32_t)token;
    ex[at] = x;
  }
  __syncthreads();
  n = ecount;
  rank_all(ek, ef, n, [&](int rank, int i) {
    sel[rank] = ef[i];
    sel_x[rank] = ex[i];
    atomicMin(&first[ef[i] >> 32], rank);
  });
  n = std::min(n, W);
  __syncthreads();

  // ---- places, outputs (lane = rank) ----------------------------------------
  if (wave != 0) return;
  const bool chosen = lane < n;
  const int p = chosen ? (int)(sel[lane] >> 32) : 0, token = chosen ? (int)(uint32_t)sel[lane] : 0;
  const bool stays = chosen && first[p] == lane;  // a parent's best continuation
  const uint64_t stay_mask = __builtin_amdgcn_ballot_w64(stays);
  uint32_t free = ~(uint32_t)__builtin_amdgcn_ballot_w64(lane < W && first[lane & 31] < 64);
  int slot = p;
  if (!stays) {
    // the k-th free slot, k = the ranks below this one that do not stay
    int k = __builtin_popcountll(~stay_mask & ((1ull << lane) - 1));
    for (; k > 0; --k) free &= free - 1;
    slot = free ? __builtin_ctz(free) : W;
  }
  if (lane >= W) return;
  const int from = chosen ? p : slot;  // (a slot left over is its own parent)
  const bool was = ended[from];
  float out = -__builtin_inff();
  if (chosen)
    out = kind[p] == ROW_DONE  ? score[p]
          : kind[p] == ROW_NAN ? __builtin_nanf("")
                               : (float)((double)score[p] + (((double)sel_x[lane] - top[p]) - lse[p]));
  a.tokens[row0 + slot] = chosen ? token : std::max(eos32, 0);
  a.parents[row0 + slot] = row0 + from;
  a.scores_out[row0 + slot] = out;
  a.finished_out[row0 + slot] = !chosen || was || token == eos32;
  a.lengths_out[row0 + slot] = length[from] + (chosen && !was ? 1 : 0);
}

// ---------------------------------------------------------------------------
// Rows 0 .. rows - 1 of every (layer, KV head) of beam b take those of beam
// parents[b], in place, K and V in one launch. A thread owns the same 16 bytes
// of all W beams of a group: it loads those of every moved beam's parent and
// only then stores, so it needs no copy and no order between blocks whatever
// the parents are. A beam that keeps its rows is neither read nor written (its
// resource is empty: loads return zeros, stores are dropped), and nor is one
// whose parent is not a row of its group. Bound by memory: 8 x 8 beams of which
// half move, 300 rows of 28 layers of the 7B heads, 1.1 GB in 198 us, 5.6 TB/s (a
// large copy reaches 4.9); 4 beams of 15 rows 3.4 us, a launch.
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

template <typename T>
void beam_merge(hipStream_t st, const SelectArgs& a) {
  int wp = 1;
  while (wp < a.W) wp *= 2;
  const int quads = (int)cdiv(a.sets / 4, MERGE_T / wp);  // of a thread
  auto go = [&](auto kern) { kern<<<(unsigned)a.G, MERGE_T, 0, st>>>(a, wp); };
  if (quads <= 5)
    go(beam_merge_kernel<T, 5>);
  else if (quads <= 10)
    go(beam_merge_kernel<T, 10>);
  else if (quads <= 20)
    go(beam_merge_kernel<T, 20>);
  else
    go(beam_merge_kernel<T, 0>);
}

int64_t select_slices(int64_t V) { return cdiv(V, SLICE<float>); }  // at most: fp32 has the smaller slices
int64_t select_sets(int64_t V) { return cdiv(V, 4 * SET) * 4; }

}  // namespace

int64_t beam_select_workspace_bytes(int64_t G, int64_t W, int64_t V) {
  return G * W * (select_slices(V) * (SEL_T / 64) * (8 + 4) + select_sets(V) * 4);
}

int launch_beam_select(hipStream_t st, int dtype, const BeamSelect& b, void* workspace, int64_t workspace_bytes) {
  const int64_t need = beam_select_workspace_bytes(b.G, b.W, b.V);
  if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)) {
    set_error("beam_select: workspace %p of %lld B, %lld B needed (16-byte aligned)", workspace,
              (long long)workspace_bytes, (long long)need);
    return MINITP_ERR_ARG;
  }
  const int64_t rows = b.G * b.W, slices = cdiv(b.V, dtype == MINITP_F32 ? SLICE<float> : SLICE<bf16>);
  const int64_t parts = rows * slices * (SEL_T / 64);
  // (a launch's threads are counted in 32 bits, the second's too: a block a group)
  if (rows * slices >= (1LL << 32) / SEL_T || b.G >= (1LL << 32) / MERGE_T) {
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
  a.slices = (int)slices;
  a.sets = (int)select_sets(b.V);
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
  a.set_top = (float*)workspace;  // (rows of whole float4)
  a.sum = (double*)(a.set_top + rows * a.sets);
  a.top = (float*)(a.sum + parts);
  if (dtype == MINITP_F32) {
    beam_slice_kernel<float><<<(unsigned)(rows * slices), SEL_T, 0, st>>>(a);
    MINITP_LAUNCH_CHECK();
    beam_merge<float>(st, a);
  } else {
    beam_slice_kernel<bf16><<<(unsigned)(rows * slices), SEL_T, 0, st>>>(a);
    MINITP_LAUNCH_CHECK();
    beam_merge<bf16>(st, a);
  }
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

int launch_kv_reorder(hipStream_t st, int dtype, void* k, void* v, int64_t L, int64_t G, int64_t W, int64_t Hkv,
                      int64_t S, int64_t D, int64_t rows, const int64_t* parents) {
  const int64_t es = dtype == MINITP_F32 ? 4 : 2;
  if (D >= (1LL << 31) || rows >= (1LL << 31) / (D * es) || L > 65535 || Hkv > 65535 || L * Hkv > 65535 || G > 32767) {
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
