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
//
// Many rows are bound by reading them: 8,191 rows of 151,936 bf16 logits take 432 us
// (5.8 TB/s, where a large copy reads and writes 4.9), 1,999 rows of 152,064 with the
// best five 128 us (4.7 TB/s), 331 of fp32 46 us (4.4). The arithmetic of a logit, five
// instructions beside its share of the sets and the rank, runs under the loads. One
// row is latency: 4.9 us for its slices and 6.1 to join them and rank.
#include <cmath>

#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

constexpr int T_ROW = 256;          // threads of a row or slice
constexpr int NCS = 4;              // 16-byte chunks a thread and turn (NC; 1 for a small vocabulary)
constexpr int SET = 64;             // logits of a set
constexpr int LIST = 1024;          // sets, then tokens, that are ranked at once
constexpr int NSETS = 10;           // sets that a thread keeps (NS; 1 for a small vocabulary)
constexpr int ROW_SETS = NSETS * T_ROW;  // ... a row that one block takes

template <typename T>
constexpr int TURN = T_ROW * NCS * Vec<T>::N;  // logits of a turn

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

// The logit of a key (a NaN for any).
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o);
}

// log2 of z > 0 (NaN of one): with z = 2^e m, m around 1 and s = (m - 1) / (m + 1),
// log m = 2 (s + s^3 / 3 + s^5 / 5 + ...), |s| < 0.172: terms up to s^15 leave 1e-14.
__device__ __forceinline__ double log2_of(double z) {
  double m = __builtin_amdgcn_frexp_mant(z);  // [0.5, 1)
  int e = __builtin_amdgcn_frexp_exp(z);
  const bool low = m < 0.70710678118654752;
  m = low ? m + m : m;
  e -= low;
  const double s = (m - 1.0) / (m + 1.0), q = s * s;
  double y = 1.0 / 15;
#pragma unroll
  for (int i = 13; i >= 1; i -= 2) y = fma(y, q, 1.0 / i);
  return (double)e + 2.0 / LN2 * s * y;
}

__device__ __forceinline__ float sum_of(const float (&v)[4]) { return (v[0] + v[1]) + (v[2] + v[3]); }
__device__ __forceinline__ float sum_of(const float (&v)[1]) { return v[0]; }
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
// Whole chunks come by 16-byte loads (ask), the row's first and last, if they are
// not whole, logit by logit (take); minus infinity stands for what is outside the
// row.
template <typename T, int NC>
__device__ __forceinline__ void ask_turn(const Row<T>& r, int64_t c0, u32x4 (&raw)[NC]) {
  const int64_t end = ((int64_t)r.V + r.skip) / Row<T>::VE;  // past the whole chunks
  const int n = (int)std::max<int64_t>(std::min<int64_t>(end - c0, T_ROW * NC), 0);
  const __amdgpu_buffer_rsrc_t rs = span_rsrc(r.x - r.skip + c0 * Row<T>::VE, (uint32_t)n * 16);
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const uint32_t c = u * T_ROW + threadIdx.x;
    raw[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                           rs, r.skip != 0 && c0 + c == 0 ? 0xffffffffu : c * 16, 0, 0));
  }
}
template <typename T, int NC>
__device__ __forceinline__ void take_turn(const Row<T>& r, int64_t c0, const u32x4 (&raw)[NC], float (*x)[Vec<T>::N]) {
  constexpr int VE = Vec<T>::N;
  const int64_t first = r.skip ? 1 : 0, end = ((int64_t)r.V + r.skip) / VE;  // whole chunks
#pragma unroll
  for (int u = 0; u < NC; ++u) unpack16(make_uint4(raw[u].x, raw[u].y, raw[u].z, raw[u].w), x[u], (T*)nullptr);
  if (c0 >= first && c0 + T_ROW * NC <= end) return;  // (uniform)
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int64_t c = c0 + u * T_ROW + threadIdx.x;
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
template <typename T, bool SETS, int NC>
__device__ __forceinline__ void scan(const LogprobArgs& a, const Row<T>& r, int64_t b, int64_t c0, int turns, Part* part,
                                     float* set_top) {
  constexpr int VE = Vec<T>::N, LPS = SET / VE;  // lanes of a set
  const int tid = threadIdx.x, lane = tid & 63;
  const float ninf = -__builtin_inff();
  u32x4 raw[NC];
  ask_turn<T, NC>(r, c0, raw);
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
    take_turn<T, NC>(r, c0, raw, x);
    if (turn + 1 < turns) ask_turn<T, NC>(r, c0 + T_ROW * NC, raw);
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
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = fmaf(x[u][e], LOG2E, -rr), p = __builtin_amdgcn_exp2f(d);
        zc[u] += p;
        sc[u] = fmaf(p, d, sc[u]);
      }
    }
    float st = sum_of(sc);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(st != st) != 0, 0)) {
      // 0 times an infinite distance (a masked logit) is no number, but nothing
      float r2 = rr;
      asm("" : "+v"(r2));  // (so that nothing above is kept for this)
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        sc[u] = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float d = fmaxf(fmaf(x[u][e], LOG2E, -r2), -200.f);
          sc[u] = fmaf(__builtin_amdgcn_exp2f(d), d, sc[u]);
        }
      }
      st = sum_of(sc);
    }
    z += sum_of(zc);
    s += st;
#pragma unroll
    for (int u = 0; u < NC; ++u) {
      const int64_t c = c0 + u * T_ROW + tid;
      const float than = c < tc ? below : xt;
      if (__builtin_amdgcn_ballot_w64(cm[u] > than) == 0) continue;  // (mostly: likely tokens have few in front)
#pragma unroll
      for (int e = 0; e < VE; ++e) ahead += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[u][e] > than));
    }
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
  double z, s, ref, wave_sum[4][2];  // sums of 2^d and 2^d d, d = x log2(e) - ref
  float top;
  int ahead, sets, tokens;  // sets, tokens: listed
};

template <int CTRL>
__device__ __forceinline__ uint64_t quad_of(uint64_t v) {
  const int lo = (int)(uint32_t)v, hi = (int)(uint32_t)(v >> 32);
  return (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, hi, CTRL, 0xf, 0xf, true) << 32 |
         (uint32_t)__builtin_amdgcn_update_dpp(0, lo, CTRL, 0xf, 0xf, true);
}

// The k-th largest of the 64 groups' best keys, 4 threads a group: at least k of
// the keys that the threads look through are not below it. ABSENT: fewer groups
// have any. (f.limit is ABSENT before the call; keys from there on are all different.)
constexpr uint64_t ABSENT = 1ull << 32;
__device__ __forceinline__ uint64_t kth_of_groups(Finish& f, uint64_t mine, int k) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  mine = std::max(mine, quad_of<0xB1>(mine));  // quad_perm [1,0,3,2]
  mine = std::max(mine, quad_of<0x4E>(mine));  // quad_perm [2,3,0,1]
  if (lane % 4 == 0) f.group[tid / 4] = mine;
  __syncthreads();
  const uint64_t u = f.group[lane];
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const uint64_t v = f.group[wave * 16 + i];
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(u > v)) == k - 1 && v > ABSENT && lane == 0) f.limit = v;
  }
  __syncthreads();
  return f.limit;
}

// Ranks of the n keys listed, a thread a key: put(rank, key) for those below k.
template <typename F>
__device__ __forceinline__ void rank_list(const Finish& f, int n, int k, F put) {
  for (int i = threadIdx.x; i < n; i += T_ROW) {
    const uint64_t mine = f.key[i];
    int ahead = 0;
#pragma unroll 4
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
#pragma unroll 1
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
    f.z = none ? __builtin_nan("") : z;
    f.s = s;
  }
  __syncthreads();
}

// The row's outputs from its n parts and its sets' maxima. All latency: every load
// of a step is asked for before the first is used, and what few rows take is kept
// out of the straight line.
template <typename T, int NS>
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int64_t b, const Part* parts, int n,
                                           const float* set_top, Finish& f) {
  const Row<T> r(a, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.top;
  const int sets = (int)(((int64_t)r.V + r.skip + SET - 1) / SET);
  float first[NS];  // the row's first NS * T_ROW sets
  if (k > 0) {
#pragma unroll
    for (int u = 0; u < NS; ++u) first[u] = set_top[std::min(u * T_ROW + tid, sets - 1)];
  }
  const int64_t t = a.tokens[b];
  Part p = parts[std::min(lane, n - 1)];
  const bool given = t >= 0 && t < r.V;
  const float xt = load_f32<T>(r.x, given ? t : 0);
  auto join_parts = [&]() {  // by one wave
    float ref = -__builtin_inff(), top = ref;
    double z = 0.0, s = 0.0;
    int ahead = 0;
#pragma unroll 1
    for (int i = lane; i < n; i += 64) {
      if (i >= 64) p = parts[i];
      top = max_nan(top, p.top);
      ahead += p.ahead;
      if (p.ref == -__builtin_inff()) continue;
      const float to = fmaxf(ref, p.ref), off = p.ref - to, w = __builtin_amdgcn_exp2f(off);
      const float off0 = ref - to, w0 = ref == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(off0);
      s = (w0 > 0.f ? (double)w0 * ((double)off0 * z + s) : 0.0) + (double)w * ((double)off * p.z + p.s);
      z = (double)w0 * z + (double)w * p.z;
      ref = to;
    }
    const float to = wave_max(ref), off = ref - to, w = ref == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(off);
    s = w > 0.f ? (double)w * ((double)off * z + s) : 0.0;
    z *= (double)w;
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
      f.ref = to;
      f.z = z;
      f.s = s;
    }
  };

  constexpr int PER = 32 * SET / T_ROW;
  uint32_t order[PER], at[PER], least = 0;  // of this thread's places in the selected sets
  float x[PER];
  int nsel = 0;
  if (k > 0) {
    // ---- the first sets: k of them, or all that the groups' bound leaves ---------
    if (tid == 0) {
      f.limit = ABSENT;
      f.sets = f.tokens = 0;
    }
    uint64_t mine = 0;
#pragma unroll
    for (int u = 0; u < NS; ++u)
      if (u * T_ROW + tid < sets) mine = std::max(mine, order_key(first[u], u * T_ROW + tid));
#pragma unroll 4
    for (int i = NS * T_ROW + tid; i < sets; i += T_ROW) mine = std::max(mine, order_key(set_top[i], i));
    const uint64_t limit = kth_of_groups(f, mine, k);
    auto list_set = [&](uint64_t key) {
      const int i = atomicAdd(&f.sets, 1);
      if (i < LIST) f.key[i] = key;
    };
    uint32_t hits = 0;  // (gathered first: one copy of the code that lists)
#pragma unroll
    for (int u = 0; u < NS; ++u)
      hits |= (u * T_ROW + tid < sets && order_key(first[u], u * T_ROW + tid) >= limit) << u;
    while (hits) {
      const int h = __builtin_ctz(hits);
      hits &= hits - 1;
      float x = first[0];
#pragma unroll
      for (int u = 1; u < NS; ++u) x = h == u ? first[u] : x;
      list_set(order_key(x, h * T_ROW + tid));
    }
#pragma unroll 1
    for (int i = NS * T_ROW + tid; i < sets; i += T_ROW)
      if (order_key(set_top[i], i) >= limit) list_set(order_key(set_top[i], i));
    __syncthreads();
    nsel = f.sets;
    if (nsel <= 32) {
      if (tid < nsel) f.sel[tid] = ~(uint32_t)f.key[tid];
    } else if (__builtin_expect(nsel <= LIST, 1)) {
      rank_list(f, nsel, k, [&](int rank, uint64_t key) {
        f.sel[rank] = ~(uint32_t)key;
        if (rank == k - 1) f.limit = key;
      });
      nsel = k;
    } else {
      // more than the list holds (a long row whose best sets fell to few threads):
      // one set at a time
      uint64_t last = ~0ull;
      for (int i = 0; i < k; ++i) {
        uint64_t next = 0;
#pragma unroll 1
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
        if (tid == 0) {
          f.sel[i] = ~(uint32_t)last;
          f.limit = last;
        }
      }
      nsel = k;
    }
    __syncthreads();
    // ---- their tokens not below the bound's logit, while the sums are joined ------
    least = (uint32_t)(f.limit >> 32);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (u * T_ROW >= nsel * SET) break;  // (uniform)
      const int j = u * T_ROW + tid;
      const uint32_t i = f.sel[std::min(j / SET, nsel - 1)] * SET + j % SET - r.skip;
      at[u] = j < nsel * SET && i < (uint32_t)r.V ? i : ~0u;
      x[u] = load_f32<T>(r.x, at[u] == ~0u ? 0 : i);
    }
  }
  if (wave == 3) join_parts();
  if (k > 0) {
    uint32_t hits = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      order[u] = 0;
      if (u * T_ROW >= nsel * SET) continue;
      order[u] = at[u] == ~0u ? 0 : order_of(x[u]);
      hits |= (order[u] >= least) << u;
    }
    if (least == (uint32_t)(ABSENT >> 32)) {  // (a small vocabulary: the sets give no bound)
      if (tid == 0) f.tokens = LIST;
      hits = 0;
    }
    while (hits) {
      const int h = __builtin_ctz(hits);
      hits &= hits - 1;
      uint32_t o = order[0], place = at[0];
#pragma unroll
      for (int u = 1; u < PER; ++u) {
        o = h == u ? order[u] : o;
        place = h == u ? at[u] : place;
      }
      const int i = atomicAdd(&f.tokens, 1);
      if (i < LIST) f.key[i] = (uint64_t)o << 32 | (uint32_t)~place;
    }
  }
  __syncthreads();
  if (__builtin_expect(!(fabsf(f.top) < FAR) || (given && !(xt > -__builtin_inff())), 0)) scan_again<T>(r, f, t);
  // log-probability of a logit: LOG2E's own error, that much of x less the mean
  // logit, is taken out again
  const double lz = log2_of(f.z), mean = f.s / f.z;
  auto logprob = [&](float x) {
    const double d = (double)x * (double)LOG2E - f.ref;
    const double lp = x == -__builtin_inff() && lz == lz ? d : (d - lz) - OFF * (d - mean);
    return (float)(LN2 * lp);
  };
  int listed = k > 0 ? f.tokens : 0;
  if (__builtin_expect(listed > T_ROW, 0)) {
    // many equal logits: bounded once more, by place too
    __syncthreads();
    if (tid == 0) {
      f.limit = ABSENT;
      f.tokens = 0;
    }
    uint64_t mine = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (order[u] > 0) mine = std::max(mine, (uint64_t)order[u] << 32 | (uint32_t)~at[u]);
    const uint64_t limit = kth_of_groups(f, mine, k);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const uint64_t key = (uint64_t)order[u] << 32 | (uint32_t)~at[u];
      if (order[u] > 0 && key >= limit) f.key[atomicAdd(&f.tokens, 1)] = key;  // (at most 31 groups of 32, and one)
    }
    __syncthreads();
    listed = f.tokens;
  }
  // a list entry a thread, and the row's own values by another wave's first
  if (tid == T_ROW - 64) {
    a.logprobs[b] = given ? logprob(xt) : __builtin_nanf("");
    a.entropy[b] = (float)(LN2 * (lz - mean));
    a.ranks[b] = given ? f.ahead : -1;
  }
  if (k > 0)
    rank_list(f, listed, k, [&](int rank, uint64_t key) {
      a.top_tokens[b * k + rank] = (uint32_t)~(uint32_t)key;
      a.top_logprobs[b * k + rank] = logprob(logit_of(key));
    });
}

// (A vocabulary of about 2,000 bf16 or 1,000 fp32 logits takes a chunk a thread: four are
// mostly registers and instructions for logits that there are not. 2,142 rows of 1,000
// bf16 logits 21.7 and 11.5 us, with the best five 43.7 and 22.3.)
template <typename T, bool SETS, int NC>
__global__ __launch_bounds__(T_ROW) void logprob_row_kernel(LogprobArgs a) {
  constexpr int NS = NC == 1 ? 1 : NSETS;
  __shared__ Finish f;
  __shared__ Part parts[T_ROW / 64];
  __shared__ float set_top[SETS ? NS * T_ROW : 1];
  const int64_t b = blockIdx.x;
  scan<T, SETS, NC>(a, Row<T>(a, b), b, 0, a.turns, parts + (threadIdx.x >> 6), set_top);
  __syncthreads();
  finish_row<T, NS>(a, b, parts, T_ROW / 64, set_top, f);
}

template <typename T, bool SETS>
__global__ __launch_bounds__(T_ROW) void logprob_slice_kernel(LogprobArgs a) {
  const int64_t b = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  scan<T, SETS, NCS>(a, Row<T>(a, b), b, (int64_t)slice * a.turns * T_ROW * NCS, a.turns,
                a.parts + blockIdx.x * (int64_t)(T_ROW / 64) + (threadIdx.x >> 6), a.set_top + b * a.sets);
}

template <typename T>
__global__ __launch_bounds__(T_ROW) void logprob_finish_kernel(LogprobArgs a) {
  __shared__ Finish f;
  const int64_t b = blockIdx.x;
  const int n = a.slices * (T_ROW / 64);
  finish_row<T, NSETS>(a, b, a.parts + b * n, n, a.set_top + b * a.sets, f);
}

struct LogprobPlan {
  int64_t turns, slices, sets;  // turns of a slice; sets padded to whole 16 bytes
  bool whole;                   // a block a row, no workspace
};
LogprobPlan logprob_plan(int dtype, int64_t B, int64_t V) {
  const int64_t turn = dtype == MINITP_F32 ? TURN<float> : TURN<bf16>, skip = dtype == MINITP_F32 ? 3 : 7;
  const int64_t all = cdiv(V + skip, turn), sets = cdiv(V + skip, SET);
  LogprobPlan p;
  // from 512 rows on a block a row (700 rows of 151,936 bf16 logits with the best five:
  // 54.7 us, 60.9 in three slices a row and a second launch; 331: 39.5 against 37.4),
  // below slices for about 2,048 blocks; of at most 64 turns
  p.turns = cdiv(all, std::max(B >= 512 ? 1 : std::min(all, cdiv(2048, std::max<int64_t>(B, 1))), cdiv(all, 64)));
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
    const bool small = (int64_t)a.V + Vec<T>::N - 1 <= T_ROW * Vec<T>::N;  // (in one turn of a chunk a thread)
    if (a.top > 0)
      (small ? logprob_row_kernel<T, true, 1> : logprob_row_kernel<T, true, NCS>)<<<rows, T_ROW, 0, st>>>(a);
    else
      (small ? logprob_row_kernel<T, false, 1> : logprob_row_kernel<T, false, NCS>)<<<rows, T_ROW, 0, st>>>(a);
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
