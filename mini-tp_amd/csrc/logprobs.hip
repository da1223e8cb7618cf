// Log-probabilities of given tokens. For a row x of V logits and its token t,
// with Z = sum_v exp(x_v - r) over any reference r:
//     log p_t = (x_t - r) - log Z
//     entropy = log Z - sum_v exp(x_v - r) (x_v - r) / Z
// the number of tokens in front of t, and the first k tokens of the order:
// larger logits first, equal ones by the lower token, NaN before every number.
//
// One pass over the logits. Each wave keeps a reference, the two sums above it and
// a count of the tokens in front of t, and, of each set of 64 consecutive logits,
// the maximum. Whatever is among the k first tokens lies in the k first sets, by
// maximum and then by place (k tokens, the sets' maxima, stand before every token
// of any other set), so only those sets' logits are read again. Many rows run a
// block each, the sets' maxima in LDS; few rows are split into slices, and a
// second launch joins them.
#include <cmath>

#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

constexpr int T_ROW = 256, NC = 4;  // threads of a row or slice; 16-byte chunks a thread and turn
constexpr int SET = 64;             // logits of a set
constexpr int LIST = 1024;          // sets, then tokens, that are ranked at once
constexpr int ROW_SETS = 2560;      // sets of a row that one block takes

template <typename T>
constexpr int TURN = T_ROW * NC * Vec<T>::N;  // logits of a turn

// The sums of a wave over its logits x, in powers of 2: d = x log2(e) - ref.
struct Part {
  double z, s;  // sum of 2^d, of 2^d d
  float ref;    // (minus infinity: no logit above it)
  float top;    // maximum, a NaN above all
  int ahead;    // logits in front of the token's
  int pad;
};

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  int V, top;
  int slices, turns;  // of a row; turns of a slice
  int sets;           // words of a row's sets (a row has as many sets, or one fewer)
  const int64_t* tokens;
  float *logprobs, *entropy;
  int64_t *ranks, *top_tokens;
  float* top_logprobs;
  Part* parts;     // [row][slice][wave]
  float* set_top;  // [row][sets]
};

constexpr float LOG2E = 1.44269504f;
// Maxima from here on are left to scan_again: x log2(e) is rounded by as much as 1
// there, which its reference shares while that is far below an exponent's range.
constexpr float FAR = 0x1p23f;
constexpr double LN2 = 0.69314718055994530942;
// LOG2E is log2(e) (1 + OFF)
constexpr double OFF = (double)LOG2E * LN2 - 1.0;

// Logits as whole numbers in their order (-0 is 0, NaN above all), and with
// their place, the lower one ahead.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t place) { return (uint64_t)order_of(x) << 32 | (uint32_t)~place; }

__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A row as 16-byte chunks from the boundary at or below its first logit, `skip`
// logits before it. Sets of 64 and chunks count from there.
template <typename T>
struct Row {
  static constexpr int VE = Vec<T>::N;
  const T* x;
  int V, skip;
  int64_t chunks;
  __device__ __forceinline__ Row(const LogprobArgs& a, int64_t b) : x((const T*)a.logits + b * a.ld), V(a.V) {
    skip = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    chunks = ((int64_t)V + skip + VE - 1) / VE;
  }
};

// The logits of a turn, from chunk c0 on: x[u] is chunk c0 + 256 u + thread.
// Whole chunks come by 16-byte loads; the row's first and last, if they are not
// whole, logit by logit; minus infinity stands for what is outside the row.
template <typename T>
__device__ __forceinline__ void load_turn(const Row<T>& r, int64_t c0, float (*x)[Vec<T>::N]) {
  constexpr int VE = Vec<T>::N;
  const int tid = threadIdx.x;
  const int64_t first = r.skip ? 1 : 0, end = ((int64_t)r.V + r.skip) / VE;  // whole chunks
  const bool edge = c0 < first || c0 + T_ROW * NC > end;                     // (uniform)
  const int n = (int)std::min<int64_t>(end - c0, T_ROW * NC);
  const __amdgpu_buffer_rsrc_t rs = span_rsrc(r.x - r.skip + c0 * VE, n > 0 ? (uint32_t)n * 16 : 0);
  u32x4 raw[NC];
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int c = u * T_ROW + tid;
    raw[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                           rs, edge && c0 + c < first ? 0xffffffffu : (uint32_t)c * 16, 0, 0));
  }
#pragma unroll
  for (int u = 0; u < NC; ++u) unpack16(make_uint4(raw[u].x, raw[u].y, raw[u].z, raw[u].w), x[u], (T*)nullptr);
  if (!edge) return;
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int64_t c = c0 + u * T_ROW + tid;
    if (c >= first && c < end) continue;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int64_t i = c * VE - r.skip + e;
      x[u][e] = i >= 0 && i < r.V ? load_f32<T>(r.x, i) : -__builtin_inff();
    }
  }
}

// `turns` turns of a row from chunk c0 on: the wave's Part, by lane 0 to *part,
// and the sets' maxima to set_top.
template <typename T, bool SETS>
__device__ __forceinline__ void scan(const LogprobArgs& a, const Row<T>& r, int64_t b, int64_t c0, int turns, Part* part,
                                     float* set_top) {
  constexpr int VE = Vec<T>::N, LPS = SET / VE;  // lanes of a set
  const int tid = threadIdx.x, lane = tid & 63;
  const float ninf = -__builtin_inff();
  // the token's logit and, for logits before it, which it stands in front of only
  // if they are smaller, the number just below (a token outside: NaN, none ahead)
  const int64_t t = a.tokens[b];
  const bool given = t >= 0 && t < r.V;
  const float xt = given ? load_f32<T>(r.x, t) : __builtin_nanf("");
  const uint32_t bits = __float_as_uint(xt);
  const float below = xt == 0.f ? __uint_as_float(0x80000001u) : __uint_as_float(xt > 0.f ? bits - 1 : bits + 1);
  const int64_t tc = given ? (t + r.skip) / VE : -1;  // its chunk

  float m = ninf, ref = ninf, z = 0.f, s = 0.f;
  int ahead = 0;
  for (int turn = 0; turn < turns; ++turn, c0 += T_ROW * NC) {
    float x[NC][VE];
    load_turn<T>(r, c0, x);
    float cm[NC];
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      cm[u] = x[u][0];
#pragma unroll
      for (int e = 1; e < VE; ++e) cm[u] = max_nan(cm[u], x[u][e]);
      m = max_nan(m, cm[u]);
    }
    if constexpr (SETS) {
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        float v = cm[u];
        v = max_nan(v, dpp_f32<0xB1>(ninf, v));   // lanes of the set: quad_perm [1,0,3,2]
        v = max_nan(v, dpp_f32<0x4E>(ninf, v));   // quad_perm [2,3,0,1]
        v = max_nan(v, dpp_f32<0x141>(ninf, v));  // row_half_mirror
        if constexpr (LPS == 16) v = max_nan(v, dpp_f32<0x140>(ninf, v));  // row_mirror
        const int64_t set = (c0 + u * T_ROW + tid) / LPS;
        if (lane % LPS == 0 && set < a.sets) set_top[set] = v;
      }
    }
    // The reference moves only when the maximum passes it by 8: until then a term
    // stays below 2^8. (A NaN moves nothing, nor does a logit below -FAR: a row
    // without a greater one is scanned again.)
    const float ml = m * LOG2E;
    if (__builtin_amdgcn_ballot_w64(ml > fmaxf(ref + 8.f, -FAR * 2.f))) {
      const float to = ml > -FAR * 2.f ? fmaxf(ref, ml) : ref;
      const float off = ref - to, f = ref == ninf ? 0.f : __builtin_amdgcn_exp2f(off);
      s = f > 0.f ? f * fmaf(off, z, s) : 0.f;
      z *= f;
      ref = to;
    }
    const float rr = ref == ninf ? 0.f : ref;
    float zc[NC], sc[NC];
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      zc[u] = sc[u] = 0.f;
      const int64_t c = c0 + u * T_ROW + tid;
      const float than = c < tc ? below : xt;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        // (2^-200 is 0, and so is its product with the distance, also of minus infinity)
        const float d = fmaxf(fmaf(x[u][e], LOG2E, -rr), -200.f), p = __builtin_amdgcn_exp2f(d);
        zc[u] += p;
        sc[u] = fmaf(p, d, sc[u]);
        ahead += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[u][e] > than));
      }
    }
    z += (zc[0] + zc[1]) + (zc[2] + zc[3]);
    s += (sc[0] + sc[1]) + (sc[2] + sc[3]);
    // equal logits before the token in its own chunk
    if (tc >= c0 && tc < c0 + T_ROW * NC) {
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        const int64_t c = c0 + u * T_ROW + tid;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          ahead += __builtin_popcountll(
              __builtin_amdgcn_ballot_w64(c == tc && c * VE + e < t + r.skip && x[u][e] == xt));
      }
    }
  }
  // the lanes' sums at one reference
  const float to = wave_max(ref);
  const float off = ref - to, f = ref == ninf ? 0.f : __builtin_amdgcn_exp2f(off);
  double zd = (double)(z * f), sd = f > 0.f ? (double)f * ((double)off * (double)z + (double)s) : 0.0;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    zd += __shfl_xor(zd, o, 64);
    sd += __shfl_xor(sd, o, 64);
    m = max_nan(m, __shfl_xor(m, o, 64));
  }
  if (lane == 0) *part = Part{zd, sd, to, m, ahead, 0};
}

// What a block needs to finish a row.
struct Finish {
  uint64_t group[64], limit, wave_key[4];
  uint64_t key[LIST];
  uint32_t sel[32];
  double lz, wave_sum[4][2], ms;  // log2 Z, its reference taken in; sum of 2^d d over Z
  double ref;
  float top;
  int ahead, count;
};

// The k-th largest of the 64 groups' best keys, 4 threads a group: at least k of
// the keys that the threads look through are not below it. 0: fewer groups have any.
__device__ __forceinline__ uint64_t kth_of_groups(Finish& f, uint64_t mine, int k) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  mine = std::max<uint64_t>(mine, __shfl_xor(mine, 1, 64));
  mine = std::max<uint64_t>(mine, __shfl_xor(mine, 2, 64));
  __syncthreads();
  if (lane % 4 == 0) f.group[tid / 4] = mine;
  if (tid == 0) {
    f.limit = 0;
    f.count = 0;
  }
  __syncthreads();
  const uint64_t u = f.group[lane];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t v = f.group[wave * 16 + i];
    // (keys above 0 are all different)
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(u > v)) == k - 1 && v > 0 && lane == 0) f.limit = v;
  }
  __syncthreads();
  return f.limit;
}

// Ranks of the f.count keys listed, a thread a key: put(rank, key) for those below k.
template <typename F>
__device__ __forceinline__ void rank_list(Finish& f, int k, F put) {
  const int n = f.count;
  for (int i = threadIdx.x; i < n; i += T_ROW) {
    const uint64_t mine = f.key[i];
    int ahead = 0;
    for (int j = 0; j < n; ++j) ahead += f.key[j] > mine;
    if (ahead < k) put(ahead, mine);
  }
}

// A row whose sums say nothing: with a logit that is no number or infinite, or a
// maximum of FAR and more either way, or a token whose place the scan does not
// count (NaN or minus infinity).
template <typename T>
__device__ __forceinline__ void scan_again(const Row<T>& r, Finish& f, int64_t t) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float m = f.top, mine = t >= 0 && t < r.V ? load_f32<T>(r.x, t) : 0.f;
  const uint64_t key = order_key(mine, (uint32_t)t);
  double z = 0.0, s = 0.0;
  int ahead = 0;
  for (int64_t i = tid; i < r.V; i += T_ROW) {
    const float x = load_f32<T>(r.x, i), d = fmaxf((x - m) * LOG2E, -200.f), p = __builtin_amdgcn_exp2f(d);
    z += (double)p;
    s += (double)p * (double)d;
    ahead += order_key(x, (uint32_t)i) > key;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    z += __shfl_xor(z, o, 64);
    s += __shfl_xor(s, o, 64);
    ahead += __shfl_xor(ahead, o, 64);
  }
  __syncthreads();
  if (lane == 0) {
    f.wave_sum[wave][0] = z;
    f.wave_sum[wave][1] = s;
    f.wave_key[wave] = (uint64_t)ahead;
  }
  __syncthreads();
  if (tid == 0) {
    z = (f.wave_sum[0][0] + f.wave_sum[1][0]) + (f.wave_sum[2][0] + f.wave_sum[3][0]);
    s = (f.wave_sum[0][1] + f.wave_sum[1][1]) + (f.wave_sum[2][1] + f.wave_sum[3][1]);
    f.ahead = (int)(f.wave_key[0] + f.wave_key[1] + f.wave_key[2] + f.wave_key[3]);
    // (no number unless the maximum is one: minus infinity less itself is none)
    const bool none = !(fabsf(m) < __builtin_inff());
    f.ref = (double)m * (double)LOG2E;
    f.lz = none ? __builtin_nan("") : log2(z);
    f.ms = s / z;
  }
  __syncthreads();
}

// The row's outputs from its n parts and its sets' maxima.
template <typename T>
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int64_t b, const Part* parts, int n,
                                           const float* set_top, Finish& f) {
  const Row<T> r(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top;
  const int64_t t = a.tokens[b];
  const bool given = t >= 0 && t < r.V;
  const float xt = given ? load_f32<T>(r.x, t) : 0.f;
  if (wave == 0) {
    float ref = -__builtin_inff(), top = ref;
    int ahead = 0;
    for (int i = lane; i < n; i += 64) {
      ref = fmaxf(ref, parts[i].ref);
      top = max_nan(top, parts[i].top);
      ahead += parts[i].ahead;
    }
    ref = wave_max(ref);
    double z = 0.0, s = 0.0;
    for (int i = lane; i < n; i += 64) {
      const Part p = parts[i];
      const float off = p.ref - ref, w = p.ref == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(off);
      if (!(w > 0.f)) continue;
      z += (double)w * p.z;
      s += (double)w * ((double)off * p.z + p.s);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      z += __shfl_xor(z, o, 64);
      s += __shfl_xor(s, o, 64);
      top = max_nan(top, __shfl_xor(top, o, 64));
      ahead += __shfl_xor(ahead, o, 64);
    }
    if (lane == 0) {
      f.top = top;
      f.ahead = ahead;
      f.ref = ref;
      f.lz = log2(z);
      f.ms = s / z;
    }
  }
  // ---- the k first sets ---------------------------------------------------------
  const int sets = (int)(((int64_t)r.V + r.skip + SET - 1) / SET);
  int nsel = 0;
  if (k > 0) {
    uint64_t mine = 0;
    for (int i = tid; i < sets; i += T_ROW) mine = std::max<uint64_t>(mine, order_key(set_top[i], i));
    const uint64_t limit = kth_of_groups(f, mine, k);
    for (int i = tid; i < sets; i += T_ROW) {
      const uint64_t key = order_key(set_top[i], i);
      if (key < limit) continue;
      const int at = atomicAdd(&f.count, 1);
      if (at < LIST) f.key[at] = key;
    }
    __syncthreads();
    nsel = std::min(f.count, k);
    if (f.count <= LIST) {
      rank_list(f, k, [&](int rank, uint64_t key) { f.sel[rank] = ~(uint32_t)key; });
    } else {
      // more than the list holds (a long row whose best sets fell to few threads):
      // one set at a time
      uint64_t last = ~0ull;
      for (int i = 0; i < k; ++i) {
        uint64_t next = 0;
        for (int j = tid; j < sets; j += T_ROW) {
          const uint64_t key = order_key(set_top[j], j);
          if (key < last) next = std::max(next, key);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) next = std::max<uint64_t>(next, __shfl_xor(next, o, 64));
        __syncthreads();
        if (lane == 0) f.wave_key[wave] = next;
        __syncthreads();
        last = std::max(std::max(f.wave_key[0], f.wave_key[1]), std::max(f.wave_key[2], f.wave_key[3]));
        if (tid == 0) f.sel[i] = ~(uint32_t)last;
      }
    }
  }
  __syncthreads();
  const bool odd = !(fabsf(f.top) < FAR) || (given && !(xt > -__builtin_inff()));
  if (odd) scan_again<T>(r, f, t);
  // log-probability of a logit: LOG2E's own error, that much of x less the mean
  // logit, is taken out again
  auto logprob = [&](float x) {
    const double d = (double)x * (double)LOG2E - f.ref, lp = d - f.lz;
    return (float)(LN2 * (x == -__builtin_inff() && f.lz == f.lz ? -__builtin_inf() : lp - OFF * (d - f.ms)));
  };
  if (tid == 0) {
    a.logprobs[b] = given ? logprob(xt) : __builtin_nanf("");
    a.entropy[b] = (float)(LN2 * (f.lz - f.ms));
    a.ranks[b] = given ? f.ahead : -1;
  }
  if (k == 0) return;
  // ---- their tokens: a thread's places in the sets, in the sets' order -------------
  constexpr int PER = 32 * SET / T_ROW;
  uint64_t keys[PER], mine = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int j = u * T_ROW + tid;
    keys[u] = 0;
    if (j < nsel * SET) {
      const int64_t i = (int64_t)f.sel[j / SET] * SET + j % SET - r.skip;
      if (i >= 0 && i < r.V) keys[u] = order_key(load_f32<T>(r.x, i), (uint32_t)i);
    }
    mine = std::max(mine, keys[u]);
  }
  const uint64_t limit = std::max<uint64_t>(kth_of_groups(f, mine, k), 1);
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (keys[u] >= limit) f.key[atomicAdd(&f.count, 1)] = keys[u];  // (at most 31 groups of 32, and one)
  __syncthreads();
  rank_list(f, k, [&](int rank, uint64_t key) {
    const uint32_t token = ~(uint32_t)key;
    a.top_tokens[b * k + rank] = token;
    a.top_logprobs[b * k + rank] = logprob(load_f32<T>(r.x, token));
  });
}

template <typename T, bool SETS>
__global__ __launch_bounds__(T_ROW) void logprob_row_kernel(LogprobArgs a) {
  __shared__ Finish f;
  __shared__ Part parts[T_ROW / 64];
  __shared__ float set_top[SETS ? ROW_SETS : 1];
  const int64_t b = blockIdx.x;
  scan<T, SETS>(a, Row<T>(a, b), b, 0, a.turns, parts + (threadIdx.x >> 6), set_top);
  __syncthreads();
  finish_row<T>(a, b, parts, T_ROW / 64, set_top, f);
}

template <typename T, bool SETS>
__global__ __launch_bounds__(T_ROW) void logprob_slice_kernel(LogprobArgs a) {
  const int64_t b = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  scan<T, SETS>(a, Row<T>(a, b), b, (int64_t)slice * a.turns * T_ROW * NC, a.turns,
                a.parts + blockIdx.x * (int64_t)(T_ROW / 64) + (threadIdx.x >> 6), a.set_top + b * a.sets);
}

template <typename T>
__global__ __launch_bounds__(T_ROW) void logprob_finish_kernel(LogprobArgs a) {
  __shared__ Finish f;
  const int64_t b = blockIdx.x;
  const int n = a.slices * (T_ROW / 64);
  finish_row<T>(a, b, a.parts + b * n, n, a.set_top + b * a.sets, f);
}

struct LogprobPlan {
  int64_t turns, slices, sets;  // turns of a slice; sets padded to whole 16 bytes
  bool whole;                   // a block a row, no workspace
};
LogprobPlan logprob_plan(int dtype, int64_t B, int64_t V) {
  const int64_t turn = dtype == MINITP_F32 ? TURN<float> : TURN<bf16>, skip = dtype == MINITP_F32 ? 3 : 7;
  const int64_t all = cdiv(V + skip, turn), sets = cdiv(V + skip, SET);
  LogprobPlan p;
  // slices for about 2,048 blocks, of at most 64 turns
  p.turns = cdiv(all, std::max(std::min(all, cdiv(2048, std::max<int64_t>(B, 1))), cdiv(all, 64)));
  p.slices = cdiv(all, p.turns);
  p.sets = cdiv(sets, 4) * 4;
  p.whole = p.slices == 1 && sets <= ROW_SETS;
  return p;
}
bool logprob_fits(const LogprobPlan& p, int64_t B) {
  return B < (1LL << 24) && B * p.slices < (1LL << 24);  // (threads are counted in 32 bits)
}
int64_t logprob_bytes(const LogprobPlan& p, int64_t B, int64_t top) {
  return p.whole ? 0 : B * (p.slices * (T_ROW / 64) * (int64_t)sizeof(Part) + (top > 0 ? p.sets * 4 : 0));
}

template <typename T>
int logprob_launch(hipStream_t st, const LogprobArgs& a, bool whole, int64_t B) {
  const unsigned rows = (unsigned)B, slices = (unsigned)(B * a.slices);
  if (whole) {
    if (a.top > 0)
      logprob_row_kernel<T, true><<<rows, T_ROW, 0, st>>>(a);
    else
      logprob_row_kernel<T, false><<<rows, T_ROW, 0, st>>>(a);
    MINITP_LAUNCH_CHECK();
    return MINITP_OK;
  }
  if (a.top > 0)
    logprob_slice_kernel<T, true><<<slices, T_ROW, 0, st>>>(a);
  else
    logprob_slice_kernel<T, false><<<slices, T_ROW, 0, st>>>(a);
  MINITP_LAUNCH_CHECK();
  logprob_finish_kernel<T><<<rows, T_ROW, 0, st>>>(a);
  MINITP_LAUNCH_CHECK();
  return MINITP_OK;
}

}  // namespace

int64_t token_logprobs_workspace_bytes(int dtype, int64_t B, int64_t V, int64_t top) {
  if (B >= (1LL << 24)) return -1;
  const LogprobPlan p = logprob_plan(dtype, B, V);
  return logprob_fits(p, B) ? logprob_bytes(p, B, top) : -1;
}

int launch_token_logprobs(hipStream_t st, int dtype, const TokenLogprobs& t, void* workspace, int64_t workspace_bytes) {
  const LogprobPlan p = logprob_plan(dtype, t.B, t.V);
  if (!logprob_fits(p, t.B)) {
    set_error("token_logprobs: %lld rows of %lld logits are too many for one call", (long long)t.B, (long long)t.V);
    return MINITP_ERR_UNSUPPORTED;
  }
  const int64_t need = logprob_bytes(p, t.B, t.top);
  if (workspace_bytes < need || (workspace == nullptr && need > 0) || !aligned16(workspace)) {
    set_error("token_logprobs: workspace %p of %lld B, %lld B needed (16-byte aligned)", workspace,
              (long long)workspace_bytes, (long long)need);
    return MINITP_ERR_ARG;
  }
  LogprobArgs a{};
  a.logits = t.logits;
  a.ld = t.ld;
  a.V = (int)t.V;
  a.top = (int)t.top;
  a.slices = (int)p.slices;
  a.turns = (int)p.turns;
  a.sets = (int)p.sets;
  a.tokens = t.tokens;
  a.logprobs = t.logprobs;
  a.entropy = t.entropy;
  a.ranks = t.ranks;
  a.top_tokens = t.top_tokens;
  a.top_logprobs = t.top_logprobs;
  a.parts = (Part*)workspace;
  a.set_top = (float*)(a.parts + t.B * p.slices * (T_ROW / 64));
  return dtype == MINITP_F32 ? logprob_launch<float>(st, a, p.whole, t.B) : logprob_launch<bf16>(st, a, p.whole, t.B);
}

}  // namespace minitp
