// Causal attention over packed sequences: the rows of S sequences of any
// lengths follow each other in one stream of N tokens, sequence s in rows
// offsets[s] .. offsets[s + 1] - 1. Query i of a sequence that begins at row a
// attends rows a .. i:
//     o = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,
// head h on KV head h / (Hq / Hkv). A row of no sequence gets zeros.
//
// The stream is one long causal sequence with a border in front of each
// sequence, and blocks take it as that: the queries of a KV head, (token, head
// of the group) by (token, head), in tiles of as many rows wherever the
// sequences end, each over the keys from its first token's sequence on to its
// last token. So the launch does not depend on the lengths, which stay on the
// device, and short sequences share a tile. A query's own window, first .. i, is
// its mask; tiles of keys that every query of a wave sees are not masked, tiles
// that none sees are left out.
#include "attn_tiles.h"
#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

struct PackedArgs {
  const void *q, *k, *v;  // [N, Hq, D], [N, Hkv, D] in strides of elements
  int64_t q_row, q_head, kv_row, kv_head;
  void* out;              // [N, Hq, D]
  int S, Hq, Hkv, per;    // per: query heads of a KV head
  int rows;               // N * per: query rows of a KV head
  int tiles;              // ... in tiles
  bool ranked;           // blocks take the tiles by ranked_tile
  const int64_t* offsets;  // [S + 1]
  float scale;
  Div by_per, by_hkv;
};

constexpr int NONE = INT32_MAX;  // the first row of a token of no sequence

// Where the sequences of the tokens t0 .. t1 of a tile begin. A wave finds by
// itself the offsets around t0: 64 of them, one a lane, narrowed down where there
// are more, from 64 at equal distances each time. begin() is the first row of
// t0's sequence, of(tok) of any token of the tile: the last offset not above it,
// NONE if there is none or it is the sequences' end. (Offsets in disorder give some
// row not past the token.) Those of up to 63 sequences are all loaded before the tile
// is known, which ranked_tile may choose by them. No LDS and no barrier: the first keys
// are on their way one load after the offsets.
struct Firsts {
  uint32_t lo;   // the offset that lane 0 holds
  int o, first;  // this lane's; that of t0
  int t0, t1;
  __device__ __forceinline__ int offset(const PackedArgs& a, uint32_t i) const {
    return i <= (uint32_t)a.S ? (int)std::min<int64_t>(std::max<int64_t>(a.offsets[i], 0), NONE) : NONE;
  }
  __device__ __forceinline__ explicit Firsts(const PackedArgs& a) : lo(0) {
    if (a.S < 64) o = offset(a, threadIdx.x & 63);
  }
  __device__ __forceinline__ void seek(const PackedArgs& a, int t0_, int t1_) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t span = (uint32_t)a.S + 1;
    t0 = t0_;
    t1 = t1_;
    while (span > 64) {
      const uint32_t step = (span + 63) / 64;
      const uint64_t below = __builtin_amdgcn_ballot_w64(lane * step < span && offset(a, lo + lane * step) <= t0);
      const uint32_t skip = below ? (63 - __builtin_clzll(below)) * step : 0;
      lo += skip;
      span = std::min(step, span - skip);
    }
    if (a.S >= 64) o = offset(a, lo + lane);
    const uint64_t below = __builtin_amdgcn_ballot_w64(o <= t0);
    const int at = below ? 63 - __builtin_clzll(below) : 0;
    first = below && lo + at < (uint32_t)a.S ? __builtin_amdgcn_readlane(o, at) : NONE;
  }
  // keys of the tile are those from here on
  __device__ __forceinline__ int begin() const { return first == NONE ? t0 : first; }
  template <int R>
  __device__ __forceinline__ void of(const PackedArgs& a, const int (&tok)[R], int (&f)[R]) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < R; ++i) f[i] = first;
    for (;;) {
      uint64_t inside = __builtin_amdgcn_ballot_w64(o > t0 && o <= t1);
      while (inside) {
        const int at = __builtin_ctzll(inside), b = __builtin_amdgcn_readlane(o, at);
        inside &= inside - 1;
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (b <= tok[i]) f[i] = lo + at == (uint32_t)a.S ? NONE : b;
      }
      // (a run of more offsets, of short or empty sequences)
      if (lo + 63 >= (uint32_t)a.S || __builtin_amdgcn_readlane(o, 63) > t1) return;
      lo += 64;
      o = offset(a, lo + lane);
    }
  }
};

__device__ __forceinline__ int wave_sum_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return __builtin_amdgcn_readlane(v, 63);
}

// The tile of QT rows that is taken as number `rank` where those with the most keys
// come first, for up to 63 sequences (o: the offset of each lane). A sequence's n
// tiles, those whose first row it holds, have levels 0 .. n - 1, one a QT rows; with
// C(l) the number of tiles of level l and above, the level of a rank is the greatest
// l with C(l) > rank. Tiles that begin with no sequence's row are the last. Each tile
// has one rank; offsets in disorder, which all blocks see alike, leave the order of
// the stream.
template <int QT>
__device__ __forceinline__ int ranked_tile(const PackedArgs& a, int o, int rank) {
  const int lane = threadIdx.x & 63;
  const int e = __builtin_amdgcn_update_dpp(0, o, 0x130, 0xf, 0xf, false);  // wave_shl:1
  if (__builtin_amdgcn_ballot_w64(lane < a.S && (e < o || e > a.by_per(a.rows)))) return a.tiles - 1 - rank;
  const int from = (o * a.per + QT - 1) / QT, n = lane < a.S ? (e * a.per + QT - 1) / QT - from : 0;
  const int front = __builtin_amdgcn_readfirstlane(from), end = __builtin_amdgcn_readlane(from + n, a.S - 1);
  if (rank >= end - front) {
    const int k = rank - (end - front);
    return k < front ? k : end + k - front;
  }
  int lo = 0, hi = (int)wave_max((float)n), above = 0;  // C(lo) > rank >= C(hi) = above
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, c = wave_sum_int(std::max(n - mid, 0));
    if (c > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  uint64_t there = __builtin_amdgcn_ballot_w64(n > lo);
  for (int i = rank - above; i > 0; --i) there &= there - 1;
  return __builtin_amdgcn_readlane(from, __builtin_ctzll(there)) + lo;
}

// One query of one head by one wave, in fp32, key by key and only those it sees:
// a lane a key for the scores, a lane one or two dims of the output. The tile
// kernels turn to it (rows_again) where a hidden value that is infinite or NaN
// shows in a product over a whole tile, as 0 times it is no zero, and for far scores.
template <typename T, int D>
__device__ __forceinline__ void packed_row(const PackedArgs& a, int r, int first, int head) {
  constexpr int VE = Vec<T>::N, DL = D > 64 ? D / 64 : 1;
  const int kv = head / a.per;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (or addresses are made, and kept, before they are needed)
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
#pragma unroll 2
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
    int j = 0;
    auto values = [&](auto keys) {  // as many loads at once
      constexpr int U = decltype(keys)::value;
      for (; j + U <= n; j += U) {
        float x[U][DL];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int d = 0; d < DL; ++d) x[u][d] = load_f32<T>(v + (k0 + j + u) * a.kv_row, dim + d);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float pj = __shfl(p, j + u, 64);
#pragma unroll
          for (int d = 0; d < DL; ++d) o[d] = fmaf(pj, x[u][d], o[d]);
        }
      }
    };
    values(std::integral_constant<int, 8>{});
    values(std::integral_constant<int, 1>{});
  }
  T* out = (T*)a.out + ((int64_t)r * a.Hq + head) * D;
  if (lane * DL < D) {
#pragma unroll
    for (int d = 0; d < DL; ++d) store_f32<T>(out, dim + d, o[d] / l);
  }
}

// The first of the rows from .. to of V with a value that is not finite, NONE if
// there is none.
template <typename T, int D>
__device__ __forceinline__ int odd_value(const PackedArgs& a, int kv, int from, int to) {
  constexpr int VE = Vec<T>::N, CH = D / VE, ROWS = 64 / CH, U = 4;  // rows and loads at a time
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (as in packed_row)
  const T* v = (const T*)a.v + kv * a.kv_head + lane % CH * VE;
  for (int k0 = from; k0 <= to; k0 += U * ROWS) {
    bool odd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VE];
      load_vec<T, VE>(v + std::min(k0 + u * ROWS + lane / CH, to) * a.kv_row, x);
      odd[u] = false;
#pragma unroll
      for (int e = 0; e < VE; ++e) odd[u] |= !(fabsf(x[e]) < __builtin_inff());
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t there = __builtin_amdgcn_ballot_w64(odd[u]);
      if (there) return std::min(k0 + u * ROWS + __builtin_ctzll(there) / CH, to);
    }
  }
  return NONE;
}

// Whether the dims that are not finite in the result stored for a query are so in row
// `value` of V too. (Others passed float32 on the way to a finite result: a tile's
// probabilities may be up to 2^8.)
template <typename T, int D>
__device__ __forceinline__ bool odd_like(const PackedArgs& a, int kv, int value, int r, int head) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (as in packed_row)
  const T* out = (const T*)a.out + ((int64_t)r * a.Hq + head) * D;
  const T* v = (const T*)a.v + kv * a.kv_head + value * a.kv_row;
  bool other = false;
#pragma unroll
  for (int d = 0; d < D; d += 64) {
    const int i = std::min(d + lane, D - 1);
    other |= !(fabsf(load_f32<T>(out, i)) < __builtin_inff()) && fabsf(load_f32<T>(v, i)) < __builtin_inff();
  }
  return __builtin_amdgcn_ballot_w64(other) == 0;
}

// The tiles' reference is their maximum in powers of two, rounded, so off by 2^-24 of
// itself, which probabilities share. For scores far from zero that is more than an
// exponent's range: above 2^22 the reference keeps that much and more above the
// maximum, and rows of which it leaves nothing (no sum, though they saw a key above
// minus infinity) are computed again. (Minus infinity gives NaN, which no maximum takes.)
__device__ __forceinline__ float reference_of(float x) {
  return x + fmaxf(fmaf(fabsf(x), 0x1p-22f, -1.f), 0.f);
}
__device__ __forceinline__ bool far_sum(float m, float l) { return m > -__builtin_inff() && l < 0x1p-30f; }

// Rows of a wave, by bits of their lanes in the rows' order, after their results are
// stored: the `odd` ones are not finite while the sums of their probabilities are
// numbers (a sum that is none comes from keys that the query sees, and so is the
// result), the `far` ones are far_sum's. What a query sees of infinite and NaN values
// belongs in its result. Computed again one by one are the far rows and the odd ones
// that see no such value, have one among the hidden keys of their tile too, key0 ..
// to, or are not finite in more dims than the first that they see. (One text of 8,000
// tokens, 7B heads, 490 us: 620 with an infinite value near its start, which nearly
// all rows see; 10,400 with one in the middle, for the rows of its tile in front of
// it; 44,100 with one in every row.)
template <typename T, int D>
__device__ __forceinline__ void rows_again(const PackedArgs& a, uint64_t odd, uint64_t far, int kv, int tok, int head,
                                           int first, int key0, int to) {
  int of = -1, seen = NONE, next = -1;  // the first such value of the sequence that begins at `of`; behind a row
  bool front = false;                   // one in front of it
  for (uint64_t left = odd | far; left; left &= left - 1) {
    const int lane = __builtin_ctzll(left);
    const int r = __builtin_amdgcn_readlane(tok, lane), f = __builtin_amdgcn_readlane(first, lane);
    const int hd = __builtin_amdgcn_readlane(head, lane);
    if (f != of) {
      of = f;
      seen = odd_value<T, D>(a, kv, f, to);
      front = odd_value<T, D>(a, kv, key0, f - 1) != NONE;
    }
    if (seen <= r && !(far >> lane & 1)) {
      if (next <= r) next = odd_value<T, D>(a, kv, r + 1, to);
      if (!front && next == NONE && odd_like<T, D>(a, kv, seen, r, hd)) continue;
    }
    packed_row<T, D>(a, r, f, hd);
  }
}

// What a wave's tile of keys needs: `from` .. `to` are keys that some of its
// queries see (or more), `all_from` .. `all_to` those that every one sees (or
// fewer). Its queries' tokens and first rows ascend with its 32 rows.
struct Window {
  int from, to, all_from, all_to;
};
__device__ __forceinline__ Window window_of(int tok, int first, int key0) {
  const int f = __builtin_amdgcn_readfirstlane(first);
  return Window{f == NONE ? key0 : f, __builtin_amdgcn_readlane(tok, 31), __builtin_amdgcn_readlane(first, 31),
                __builtin_amdgcn_readfirstlane(tok)};
}

// The results of a tile of QT rows that KG sets of waves hold over keys of their
// own, in LDS: po [KG][QT] rows of D, padded by 16 bytes (lanes of a wave write
// 32 rows at a time), pml [KG][QT] (maximum, as a power of two, and sum), pf [QT]
// first rows. Joined and stored by whole rows, LPR lanes a row; the ones
// that are not finite by rows_again (key0 .. to: the tile's keys).
template <typename T, int D, int KG, int QT, int THREADS>
__device__ __forceinline__ void join_rows(const PackedArgs& a, int tile, int kv, int key0, int to, const float* po,
                                          const float2* pml, const int* pf) {
  constexpr int LPR = D / 4;
  const int n = std::min(QT, a.rows - tile * QT);
  for (int i0 = 0; i0 < n * LPR; i0 += THREADS) {
    const int i = i0 + threadIdx.x, row = std::min(i / LPR, n - 1), d = i % LPR * 4;
    float m = -__builtin_inff(), l = 0.f, odd = 0.f;
    float2 ml[KG];
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      ml[g] = pml[g * QT + row];
      m = fmaxf(m, ml[g].x);
    }
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const f32x4 og = *(const f32x4*)(po + (g * QT + row) * (D + 4) + d);
      // (a set that saw nothing weighs nothing; a sum that is no number shows)
      const float sc = ml[g].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[g].x - m);
      l = fmaf(sc, ml[g].y, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        odd = fmaf(og[e], 0.f, odd);
        v[e] = fmaf(sc, og[e], v[e]);
      }
    }
    const int r = tile * QT + row, tok = a.by_per(r), head = kv * a.per + r - tok * a.per, first = pf[row];
    const bool there = i < n * LPR;
    auto rows = [](uint64_t lanes) {  // (a row: its first lane)
      uint64_t firsts = 0;
#pragma unroll
      for (int x = 0; x < 64; x += LPR)
        if (lanes >> x & ((1ull << LPR) - 1)) firsts |= 1ull << x;
      return firsts;
    };
    const uint64_t again = rows(__builtin_amdgcn_ballot_w64(there && first != NONE && odd != 0.f && l == l));
    const uint64_t far = rows(__builtin_amdgcn_ballot_w64(there && far_sum(m, l)));
    if (there) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = first == NONE ? 0.f : v[e] / l;
      store_vec<T, 4>((T*)a.out + ((int64_t)tok * a.Hq + head) * D + d, y);
    }
    if ((again | far) == 0) continue;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the rows above are stored first)
    rows_again<T, D>(a, again, far, kv, tok, head, first, key0, to);
  }
}

// ---------------------------------------------------------------------------
// bf16, on v_mfma_f32_32x32x16_bf16: a wave computes 32 query rows over all keys of
// a tile, or, where that leaves blocks too few (KG 2, 4), two or four waves the same
// rows over a half or a quarter of them each, joined at the end. A block has four or
// eight waves, a tile 64 or 128 keys (packed_form).
//
// A tile of K and V rows goes to LDS as it lies in memory, by loads that bypass
// the registers, while the tile before it is computed (two stages, one barrier a
// tile; VST 1 has one stage of V, which is loaded during its own tile's scores, and a
// second barrier, for a third block a CU). Products are transposed, S^T = K Q^T and O^T = V^T P^T, so a lane's
// scores belong to one query and its probabilities are the second product's
// operand as they are, the k-index of both operands permuted alike; V^T comes
// out of LDS transposed by ds_read_b64_tr_b16. A row's 16-byte chunks are
// permuted by its number, which the loads do on the global side, so that every
// LDS read reaches all banks.
//
// Bound by the matrix and the vector units, which hardly work at once here: 4 x 4,096
// tokens of 7B heads take 460 us (1,047 TFLOP/s; 48 + 42 % of the cycles), 8,191 of 0.5B
// heads 138 (872; 40 + 60 %, as D 64 has the exponentials of D 128 for half the
// products). What remains is instructions a score: 64 of the 73 (D 64) or 81 of a lane's
// 16 scores are their scaling, exponentials, maxima, sums and roundings.
//
// A probability is rounded to bf16 for the second product, by at most 2^-8 of
// itself, as much as the output's own rounding: the matrix cores take bf16
// there, and fp32 products run at an eighth of the rate (154 against 1,261 TFLOP/s
// of a large library product). The sums that they are divided by add the
// unrounded ones.
template <int D, int KG, int KT_, int WAVES_, int VST_ = 2>
struct Tile {
  using H = Half<D>;
  static constexpr int KT = KT_, WAVES = WAVES_, STRIPS = WAVES / KG;
  static constexpr int QT = 32 * STRIPS, NB = KT / 32 / KG;  // NB: 32-key blocks of a wave
  static constexpr int VST = VST_;  // stages of V
  static constexpr int OPER = KT * H::ROWB, STAGES = (2 + VST) * OPER;
  static constexpr int PIECES = KT / H::PIECE_ROWS, PPW = PIECES / WAVES;  // 1 KiB loads, of a wave
  static constexpr int JOIN = KG == 1 ? 0 : KG * QT * (D + 4 + 2) * 4 + QT * 4;
  static constexpr int LDS = STAGES > JOIN ? STAGES : JOIN;
  static_assert(PPW * WAVES == PIECES || 2 * PIECES == WAVES, "each wave loads alike, or half of them K and half V");
};

// The tiles of keys `key0` .. key0 + keys - 1 of a KV head through the two stages.
template <int D, typename TL>
struct KeyTiles {
  using H = Half<D>;
  const char *k, *v;
  int64_t row;  // bytes between rows
  uint32_t to, koff, voff, piece;
  int keys, n;
  __device__ __forceinline__ KeyTiles(const PackedArgs& a, int kv, int key0, int keys_, char* lds)
      : row(a.kv_row * 2), keys(keys_), n((keys_ + TL::KT - 1) / TL::KT) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = key0 * row + kv * a.kv_head * 2;
    k = (const char*)a.k + at;
    v = (const char*)a.v + at;
    to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + w * 1024;
    // piece w + WAVES j of a tile: rows WAVES PIECE_ROWS j + r; the swizzles do not depend on j
    const int r = H::PIECE_ROWS * (TL::PPW > 0 ? w : w % TL::PIECES) + lane / H::CH;
    koff = r * (uint32_t)row + ((lane % H::CH) ^ H::k_swz(r)) * 16;
    voff = r * (uint32_t)row + ((lane % H::CH) ^ H::v_swz(r)) * 16;
    piece = TL::WAVES * H::PIECE_ROWS * (uint32_t)row;
  }
  // K of tile t to stage t % 2, V to stage t % VST behind them
  __device__ __forceinline__ u32x4 rows_of(const char* base, int t) const {
    // rows past the last read zeros (or, where rows overlap, the last again)
    const int left = std::min(keys - t * TL::KT, TL::KT);
    return rows_rsrc(base + (int64_t)t * TL::KT * row, left > 0 ? (left - 1) * (uint32_t)row + H::ROWB : 0);
  }
  __device__ __forceinline__ void load_rows(u32x4 r, uint32_t off, uint32_t at) const {
    uint32_t lds = __builtin_amdgcn_readfirstlane(to + at);
    // (the sums are made anew each time: kept over the loop they take the registers of
    // a third block a CU)
    asm volatile("s_nop 4" : "+s"(lds), "+v"(off));
    // The steps go into the lanes' offsets: a scalar one may lie past the resource's
    // end by itself, where the bounds check need not hold. (At 2^24 elements a row
    // those of 128 rows are below 2^32 bytes.)
#pragma unroll
    for (int j = 0; j < std::max(TL::PPW, 1); ++j) row_dma16(r, off + j * piece, lds + j * TL::WAVES * 1024);
  }
  __device__ __forceinline__ bool mine(bool v) const {  // (few pieces: half of the waves K, half V)
    return TL::PPW > 0 || (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= TL::PIECES) == v;
  }
  __device__ __forceinline__ void load_k(int t) const {
    if ((t < n || TL::VST == 1) && mine(false)) load_rows(rows_of(k, t), koff, (t & 1) * TL::OPER);
  }
  __device__ __forceinline__ void load_v(int t) const {
    if (t < n && mine(true))
      load_rows(rows_of(v, t), voff, (2 + t % TL::VST) * TL::OPER - (TL::PPW > 0 ? 0 : TL::PIECES * 1024));
  }
};

// V of a tile has landed for the whole block: this wave's loads but the N of the
// next K (past the last tile they read nothing), and then the barrier.
template <int N>
__device__ __forceinline__ void rows_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int D, int KG, int KT, int WAVES, int VST>
__global__ __launch_bounds__(64 * WAVES, 2) void packed_bf16_kernel(PackedArgs a) {
  using H = Half<D>;
  using TL = Tile<D, KG, KT, WAVES, VST>;
  // (D = 16: the output's 32-row operand holds the 16 dims twice)
  constexpr int KS = D / 16, DB = D >= 32 ? D / 32 : 1, OC = D >= 32 ? 4 : 2;  // OC: 8-dim chunks of a block
  constexpr int NB = TL::NB, QT = TL::QT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int strip = w % TL::STRIPS, sub = w / TL::STRIPS * 32 * NB;  // of the rows; first of the wave's keys in a tile
  // The last rows, which see the most keys, first. (KV heads side by side: where
  // there are 1, 2, 4 or 8, an XCD's blocks, every eighth, share one's rows.)
  const int jb = a.by_hkv(blockIdx.x), kv = blockIdx.x - jb * a.Hkv;
  Firsts firsts(a);
  const int tile = a.ranked ? ranked_tile<QT>(a, firsts.o, jb) : a.tiles - 1 - jb;
  const int t0 = a.by_per(tile * QT), t1 = a.by_per(std::min(tile * QT + QT, a.rows) - 1);
  firsts.seek(a, t0, t1);
  const int r0 = tile * QT + strip * 32, r = std::min(r0 + n32, a.rows - 1);
  const int tok = a.by_per(r), head = kv * a.per + r - tok * a.per;
  bf16x8 qb[KS];
  {
    const bf16* q = (const bf16*)a.q + (uint32_t)tok * (uint64_t)a.q_row + (uint32_t)head * (uint64_t)a.q_head + 8 * h;
#pragma unroll
    for (int k = 0; k < KS; ++k) qb[k] = __builtin_bit_cast(bf16x8, *(const u32x4*)(q + 16 * k));
  }
  const int key0 = firsts.begin();
  const KeyTiles<D, TL> tiles(a, kv, key0, t1 - key0 + 1, lds);
  tiles.load_k(0);
  if (VST == 2) tiles.load_v(0);
  const int toks[1] = {tok};
  int first_of[1];
  firsts.of(a, toks, first_of);
  const int first = first_of[0];
  const Window win = window_of(tok, first, key0);

  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), lsum = 0.f;
  const float sl2 = a.scale * 1.4426950408889634f;

  // LDS bytes of this lane's operands: K row sub + n32, chunk 2 k + h; V rows
  // sub + 4 h + (lane % 16) / 4 (+ 8), dims 32 d + 16 ((lane / 16) % 2) + 4 (lane % 4)
  // (the swizzles do not depend on sub)
  const int kat = (sub + n32) * H::ROWB, kx = (h ^ H::k_swz(n32)) << 4;
  const int vrow = 4 * h + (lane & 15) / 4;
  const int vat = 2 * TL::OPER + (sub + vrow) * H::ROWB + 8 * (lane & 1);
  const int vx = (((D >= 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane >> 1) & 1)) ^ H::v_swz(vrow)) << 4;
  arrived(qb);

  for (int t = 0; t < tiles.n; ++t) {
    stage_wait();
    // (the readers of what is overwritten passed the barrier)
    if (VST == 1) tiles.load_v(t);
    tiles.load_k(t + 1);
    if (VST == 2) tiles.load_v(t + 1);
    const int key = key0 + t * TL::KT + sub, last = key + 32 * NB - 1;
    if (VST == 2 && (key > win.to || last < win.from)) continue;
    const char* st = lds + (t & 1) * TL::OPER;
    int sv_at = VST == 2 ? (t & 1) * TL::OPER : 0;
    asm volatile("" : "+s"(sv_at));  // (or the addresses of all reads are kept over the loop)
    const char* sv = lds + sv_at;
    f32x16 s[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {  // (two chains in turn)
        const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(st + kat + kb * 32 * H::ROWB + ((32 * k) ^ kx)));
        s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb[k], s[kb], 0, 0, 0);
      }
    }
    // lane (query, h) holds keys 32 kb + 8 (i / 4) + 4 h + i % 4 and sees first .. tok
    if (last > win.all_to) {
      const int hi = tok - key - 4 * h;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * kb + 8 * (i / 4) + i % 4 > hi) s[kb][i] = -__builtin_inff();
    }
    if (key < win.all_from) {  // (a row of no sequence sees nothing)
      const int lo = first - key - 4 * h;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * kb + 8 * (i / 4) + i % 4 < lo) s[kb][i] = -__builtin_inff();
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = reference_of(halves_max(mx) * sl2);
    if (__builtin_amdgcn_ballot_w64(mx > m + SLACK)) {
      const float mn = fmaxf(m, mx), alpha = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= alpha;
    }
    const float mref = m == -__builtin_inff() ? 0.f : m;  // (nothing seen yet)
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], sl2, -mref));
        lsum += s[kb][i];
      }
    if (VST == 1) rows_wait<TL::PPW>();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) {  // keys 16 j .. 16 j + 15
      const f32x16& p = s[j / 2];
      const int b = 8 * (j % 2);
      uint4 pk;
      pk.x = pack_bf16x2(p[b], p[b + 1]);
      pk.y = pack_bf16x2(p[b + 2], p[b + 3]);
      pk.z = pack_bf16x2(p[b + 4], p[b + 5]);
      pk.w = pack_bf16x2(p[b + 6], p[b + 7]);
      const bf16x8 pb = __builtin_bit_cast(bf16x8, pk);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const char* vp = sv + vat + 16 * j * H::ROWB + ((64 * d) ^ vx);
        const bf16x8 vf = join8(read_tr(vp), read_tr(vp + 8 * H::ROWB));
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb, o[d], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  if (VST == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no load to LDS outlives the block)

  const float l = halves_sum(lsum);
  if constexpr (KG > 1) {
    float* po = (float*)lds;                          // [KG][QT][D + 4]
    float2* pml = (float2*)(po + KG * QT * (D + 4));  // [KG][QT]
    int* pf = (int*)(pml + KG * QT);                  // [QT]
    const int row = strip * 32 + n32, at = w / TL::STRIPS * QT + row;
    __syncthreads();  // (every stage is free)
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int c = 0; c < OC; ++c)
        *(f32x4*)(po + at * (D + 4) + 32 * d + 8 * c + 4 * h) =
            f32x4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
    if (h == 0) pml[at] = make_float2(m, l);
    if (h == 0 && sub == 0) pf[row] = first;
    __syncthreads();
    join_rows<bf16, D, KG, QT, 64 * WAVES>(a, tile, kv, key0, t1, po, pml, pf);
    return;
  }
  // Through LDS, so that a wave stores whole rows (eight bytes a lane of 32 rows at
  // a time keep the address unit busy for 1 us of a block of 7 us).
  constexpr int ROW = H::ROWB + 16;
  static_assert(TL::WAVES * 32 * ROW <= TL::STAGES, "the waves' rows fit the stages");
  const bool none = first == NONE;
  float most = 0.f;  // NaN or infinite if something is
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) most = __builtin_elementwise_maximum(most, fabsf(o[d][i]));
  const bool odd = !(most < __builtin_inff());
  const uint64_t bad = __builtin_amdgcn_ballot_w64(odd && l == l && !none && r0 + n32 < a.rows);
  const uint64_t far = __builtin_amdgcn_ballot_w64(far_sum(m, l) && r0 + n32 < a.rows);
  if (__builtin_amdgcn_ballot_w64(odd && none)) {  // (0 times hidden values that are infinite or NaN)
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = none ? 0.f : o[d][i];
  }
  // (a step of the reciprocal, 2^-23, is lost in the bf16 rounding; a query that saw
  // nothing above minus infinity: NaN)
  const float f = none ? 0.f : __builtin_amdgcn_rcpf(l);
  char* mine = lds + w * 32 * ROW;
  __syncthreads();  // (every stage is free)
  if (r0 >= a.rows) return;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int c = 0; c < OC; ++c) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][4 * c + e] * f;
      store_vec<bf16, 4>((bf16*)(mine + n32 * ROW) + 32 * d + 8 * c + 4 * h, v);
    }
  __builtin_amdgcn_wave_barrier();
  // (lanes of a wave past the last row hold and store that row too)
  constexpr int RPI = 64 / H::CH;  // rows of a store
  const int out_row = tok * a.Hq + head;
  char* out = (char*)a.out + lane % H::CH * 16;
#pragma unroll
  for (int i = 0; i < 32; i += RPI) {
    const int row = i + lane / H::CH;
    const uint4 x = *(const uint4*)(mine + row * ROW + lane % H::CH * 16);
    const uint32_t at = __builtin_amdgcn_ds_bpermute(4 * row, out_row);
    *(uint4*)(out + (uint64_t)at * H::ROWB) = x;
  }
  if ((bad | far) == 0) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the rows above are stored first)
  rows_again<bf16, D>(a, (uint32_t)(bad | bad >> 32), (uint32_t)far, kv, tok, head, first, key0, t1);
}

// ---------------------------------------------------------------------------
// fp32, on v_mfma_f32_16x16x4_f32: a wave computes R strips of 16 query rows, 16
// keys at a time, straight from registers; KW of a block's four waves share rows,
// each over every KW-th 16 keys, joined at the end. Products are transposed:
// S^T = K Q^T leaves lane (quad, r) with keys 4 quad .. 4 quad + 3 of query r,
// which is the B operand of O^T = V^T P^T as it is. Score MFMA i of a chunk takes
// dims 16 c + 4 quad + i from both operands, output MFMA j dims E r + j, so that a
// lane reads K and V by 16 bytes just as it needs them, and no LDS or barrier
// stands between: the next keys are on their way during the second product, the
// values during the first. (By way of LDS, shared by the block's waves, one sequence
// of 3,000 tokens of 7B heads took 625 us, so 521: 124 TFLOP/s, where a large library
// product reaches 154. Keys and values fetched two steps ahead gained nothing.) A
// score is summed in four chains.
template <int D, int KW, int R>
constexpr int F_LDS = 64 * R * (D + 4 + 2) * 4 + 64 / KW * R * 4;

template <int D, int KW, int R>
__global__ __launch_bounds__(256, 2) void packed_f32_kernel(PackedArgs a) {
  constexpr int SW = 4 / KW, QT = 16 * R * SW, KC = D / 16;
  constexpr int E = D / 16 < 4 ? D / 16 : 4, HALVES = D / 16 / E;
  extern __shared__ __attribute__((aligned(16))) float lds_f[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane % 16, lq = lane / 16, strips = wave % SW * R * 16, part = wave / SW;
  const int jb = a.by_hkv(blockIdx.x), kv = blockIdx.x - jb * a.Hkv;
  Firsts firsts(a);
  const int tile = a.ranked ? ranked_tile<QT>(a, firsts.o, jb) : a.tiles - 1 - jb;
  const int t0 = a.by_per(tile * QT), t1 = a.by_per(std::min(tile * QT + QT, a.rows) - 1);
  firsts.seek(a, t0, t1);
  int tok[R], first[R];
  f32x4 qa[R][KC];
#pragma unroll
  for (int s = 0; s < R; ++s) {
    const int r = std::min(tile * QT + strips + 16 * s + lr, a.rows - 1);
    tok[s] = a.by_per(r);
    const float* q = (const float*)a.q + tok[s] * a.q_row + (kv * a.per + r - tok[s] * a.per) * a.q_head + 4 * lq;
#pragma unroll
    for (int c = 0; c < KC; ++c) qa[s][c] = *(const f32x4*)(q + 16 * c);
  }
  const int key0 = firsts.begin();
  firsts.of(a, tok, first);
  // this wave's steps of 16 keys, those that some of its rows see
  const int from = __builtin_amdgcn_readfirstlane(first[0]), to = __builtin_amdgcn_readlane(tok[R - 1], 15);
  const int all_from = __builtin_amdgcn_readlane(first[R - 1], 15), all_to = __builtin_amdgcn_readfirstlane(tok[0]);
  int step = from == NONE ? 0 : (from - key0) / 16;
  step += (part - step) & (KW - 1);
  const int end = (to - key0) / 16;

  const uint32_t row = (uint32_t)a.kv_row * 4;
  const char *k = (const char*)a.k + (key0 * a.kv_row + kv * a.kv_head) * 4;
  const char *v = (const char*)a.v + (key0 * a.kv_row + kv * a.kv_head) * 4;
  const uint32_t koff = lr * row + 16 * lq;
  uint32_t voff[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) voff[e] = (4 * lq + e) * row + 4 * E * lr;
  // (rows past the last, and all those of a step past the end, read zeros)
  auto rows_of = [&](const char* base, int i) {
    const uint32_t bytes = i <= end ? (std::min(t1 - key0 - 16 * i, 15)) * row + D * 4 : 0;
    return span_rsrc(base + (int64_t)(16 * i) * row, bytes);
  };
  f32x4 kr[KC];
  float vr[4][HALVES][E];
  auto load_k = [&](int i) {
    const __amdgpu_buffer_rsrc_t rs = rows_of(k, i);
#pragma unroll
    for (int c = 0; c < KC; ++c)
      kr[c] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, koff + 64 * c, 0, 0));
  };
  auto load_v = [&](int i) {
    const __amdgpu_buffer_rsrc_t rs = rows_of(v, i);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int hf = 0; hf < HALVES; ++hf) {
        if constexpr (E == 4) {
          const f32x4 x = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, voff[e] + 256 * hf, 0, 0));
#pragma unroll
          for (int j = 0; j < 4; ++j) vr[e][hf][j] = x[j];
        } else if constexpr (E == 2) {
          const float2 x = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, voff[e], 0, 0));
          vr[e][hf][0] = x.x;
          vr[e][hf][1] = x.y;
        } else {
          vr[e][hf][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, voff[e], 0, 0));
        }
      }
  };
  f32x4 o[R][HALVES][E];
  float m[R], l[R];  // (in powers of two)
#pragma unroll
  for (int s = 0; s < R; ++s) {
    m[s] = -__builtin_inff();
    l[s] = 0.f;
#pragma unroll
    for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
      for (int j = 0; j < E; ++j) o[s][hf][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale = a.scale * 1.44269504f;
  if (step <= end) load_k(step);
  for (; step <= end; step += KW) {
    const int key = key0 + 16 * step;
    load_v(step);
    f32x4 p[R];
#pragma unroll
    for (int s = 0; s < R; ++s) {
      f32x4 chain[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) chain[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          chain[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[c][i], qa[s][c][i], chain[i], 0, 0, 0);
      p[s] = (chain[0] + chain[1]) + (chain[2] + chain[3]);
    }
    load_k(step + KW);
    if (key < all_from || key + 15 > all_to) {  // (a lane sees first .. tok)
#pragma unroll
      for (int s = 0; s < R; ++s) {
        const int lo = first[s] - key - 4 * lq, hi = tok[s] - key - 4 * lq;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < lo || e > hi) p[s][e] = -__builtin_inff();
      }
    }
#pragma unroll
    for (int s = 0; s < R; ++s) {
      const float mx = quads_max(fmaxf(fmaxf(p[s][0], p[s][1]), fmaxf(p[s][2], p[s][3])));
      const float mn = fmaxf(m[s], reference_of(mx * scale)), ref = mn == -__builtin_inff() ? 0.f : mn;
      if (__builtin_amdgcn_ballot_w64(mn != m[s])) {
        const float alpha = mn == m[s] ? 1.f : __builtin_amdgcn_exp2f(m[s] - mn);
        m[s] = mn;
        l[s] *= alpha;
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
          for (int j = 0; j < E; ++j) o[s][hf][j] *= alpha;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[s][e] = __builtin_amdgcn_exp2f(fmaf(p[s][e], scale, -ref));
        l[s] += p[s][e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
        for (int s = 0; s < R; ++s)
#pragma unroll
          for (int j = 0; j < E; ++j)
            o[s][hf][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[e][hf][j], p[s][e], o[s][hf][j], 0, 0, 0);
  }
  // o[s][hf][j][x]: dim 64 hf + E (4 lq + x) + j of the lane's query; the KW waves
  // of a strip joined through LDS, and stored from there by whole rows
  float* po = lds_f;                               // [KW][QT][D + 4]
  float2* pml = (float2*)(po + 64 * R * (D + 4));  // [KW][QT]
  int* pf = (int*)(pml + 64 * R);                  // [QT]
#pragma unroll
  for (int s = 0; s < R; ++s) {
    const int at = part * QT + strips + 16 * s + lr;
#pragma unroll
    for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int j = 0; j < E; ++j) po[at * (D + 4) + 64 * hf + E * (4 * lq + x) + j] = o[s][hf][j][x];
    l[s] = quads_sum(l[s]);
    if (lq == 0) pml[at] = make_float2(m[s], l[s]);
    if (lq == 0 && part == 0) pf[strips + 16 * s + lr] = first[s];
  }
  __syncthreads();
  join_rows<float, D, KW, QT, 256>(a, tile, kv, key0, t1, po, pml, pf);
}

// The form of a call from what the host knows, blocks of 128 rows and the mean
// length (the rest is on the device; room behind the last text and empty sequences
// count in the mean: 256 places for sequences of which one text of 4,000 tokens takes
// one, 0.5B heads, 63 us instead of 50, four of 2,000 55 instead of 53): sets of waves a row, keys of a tile or step,
// waves, strips of a wave (fp32).
// Measured (us, graph replays; n x L: n sequences of L tokens, blocks in brackets):
// Four or two sets where blocks are few and the sequences longer than a tile (one
//   set, two, four):
//   0.5B heads (D 64): 2x64 (14) 5.7 5.9 5.3, 10x100 (110) 6.4 7.0 6.9, 1x500 (56) 10.4 9.7
//   7.2, 5x300 (166) 9.6 10.5 11.5, 2x1300 (286) 26.2 24.7 22.5, 8x500 (438) 16.4 17.9
//   22.8, up to L at random 4x700 (148) 16.6 13.4 (two sets), 6x700 (206) 15.5 13.0, 4x1500
//   (272) 20.9 17.3, 4x3000 (540) 47.5 35.9, 12x700 (546) 20.5 25.9; 7B heads (128):
//   1x200 (44) 10.7 10.2 8.4, 3x200 (132) 12.0 11.8 18.7 (a block a CU), 1x1300 (288) 38.0
//   28.2 51.6, 3x500 (332) 21.1 23.6 42.0.
//   Two sets over tiles of 128 keys instead of 64: 0.5B heads, 1x4096 (448) 60.4 53.3;
//   7B heads (the tiles take a CU's LDS), 1x1024 (224) 25.6 30.1.
// Tiles of 128 keys for long sequences: fewer barriers and lane exchanges a key.
//   7B heads, 256 rows and eight waves a block: 3x(20011 .. 8882) (9,768) 5,575 5,240,
//   1x4096 (896) 143 138, 3x2500 (1,644) 180 178, 4x2000 (1,752) 147 149.
//   D 64, where a CU holds four blocks of 64-key tiles, so that about 1,024 are resident
//   at once and the longest is what counts, and two of 128-key tiles, whose light
//   blocks fill in behind (64 keys, 128, 128 with two sets of eight waves):
//   0.5B heads: 1x5000 (548) 82 75 71, 1x6000 (658) 98 90 89, 1x6900 (756) 119 107 112,
//   1x7500 (822) 135 121 129, 1x9500 (1,040) 191 179 189, 1x10500 (1,150) 226 221 228,
//   1x12000 (1,314) 284 291 293; 2x3400 (744) 72 67 63, 2x4500 (986) 105 93 97, 2x5000
//   (1,094) 121 110 116, 3x2600 (854) 61 56 58; 16 heads on 8: 1x5000 (632) 81 76 74,
//   1x6000 (752) 104 94 98, 1x9000 (1,128) 192 188 196; 8 on 8: 1x11000 (688) 177 162 157,
//   1x12500 (784) 214 193 196, 1x16600 (1,040) 328 304 320.
// fp32: four sets as long as the blocks are few for the lengths, of two strips for long
//   sequences, one set for many short ones (n x up to L: random lengths; one, two, four
//   sets of one strip, four of two):
//   0.5B heads: 1x200 (22) 14.2 9.7 7.4 10.7, 5x668 (216) 47.2 37.3 33.8 37.8, 40x192 (404)
//   29.8 23.6 25.0 26.2, 3x2846 (734) 305 284 284 266; 7B heads: 8x665 (548) 135 117 103
//   108, 20x397 (844) 104 102 113 117, 100x200 (2,136) 158 167 209 216, 300x60 (2,016)
//   91.7 107 151 160, 3x2846 (1,468) 1,055 999 1,011 936.
struct PackedForm {
  int sets, keys, waves, strips = 1;
};
PackedForm packed_form(bool half, int D, int64_t rows, int64_t heads, int64_t tokens, int64_t sequences) {
  const int64_t blocks = cdiv(rows, 128) * heads, mean = tokens / std::max<int64_t>(sequences, 1);
  if (half) {
    if (mean >= 64 && blocks <= std::min<int64_t>(64 + (D < 128 ? mean * 64 / (5 * D) : 0), 20480 / D)) return {4, 128, 4};
    if (D < 128 && mean >= 300 && blocks <= std::min<int64_t>(mean / 2 + 64, 34816 / D)) return {2, 128, 4};
    if (D == 128 && mean >= 300 && blocks <= std::min<int64_t>(mean * 2 / 5, 512)) return {2, 64, 4};
    if (D == 128 && mean >= 2500) return {1, 128, 8};
    if (D == 64 && mean >= 2500 && blocks <= 704) return {2, 128, 8};
    if (D == 64 && mean >= 2500 && blocks <= 1152) return {1, 128, 4};
    return {1, 64, 4};
  }
  if (mean >= 700 && blocks >= 300) return {4, 16, 4, 2};
  return {blocks <= 2 * mean ? 4 : blocks * D < 1024 * mean ? 2 : 1, 16, 4};
}

template <typename T, int D>
int packed_launch(hipStream_t st, PackedArgs a, const PackedForm& f) {
  auto go = [&](auto kern, int rows, int lds) -> int {
    a.tiles = (int)cdiv(a.rows, rows);
    // Ranked where the blocks outnumber what runs at once and the texts are few; of
    // many, some are short enough for an even end, and keys of all at once do not stay
    // in the L2s. In stream order and by rank (us): 7B heads, 16 texts of up to 1,500
    // tokens 141 131, 8x1500 161 152, 6x2000 199 187, 40x400 81 89; 0.5B heads, 24 texts of
    // up to 1,500 54 47, 6x2000 73 62, 50x100 in fp32 25.6 27.2.
    a.ranked = a.S >= 2 && a.S < 32 && (int64_t)a.tiles * a.Hkv > 512;
    const int rc = ensure_lds_limit((const void*)kern, lds);
    if (rc) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.tiles * a.Hkv)), dim3(64 * f.waves), lds, st, a);
    MINITP_LAUNCH_CHECK();
    return MINITP_OK;
  };
  if constexpr (sizeof(T) == 2) {
    constexpr int KEYS2 = D < 128 ? 128 : 64;  // (of the form with two sets)
    if (f.sets == 4) return go(packed_bf16_kernel<D, 4, 128, 4, 2>, 32, Tile<D, 4, 128, 4>::LDS);
    if (f.sets == 2 && f.waves == 4) return go(packed_bf16_kernel<D, 2, KEYS2, 4, 2>, 64, Tile<D, 2, KEYS2, 4>::LDS);
    if constexpr (D == 128) {
      if (f.keys == 128) return go(packed_bf16_kernel<D, 1, 128, 8, 2>, 256, Tile<D, 1, 128, 8>::LDS);
    }
    if constexpr (D == 64) {
      if (f.sets == 2) return go(packed_bf16_kernel<D, 2, 128, 8, 2>, 128, Tile<D, 2, 128, 8>::LDS);
      if (f.keys == 128) return go(packed_bf16_kernel<D, 1, 128, 4, 2>, 128, Tile<D, 1, 128, 4>::LDS);
    }
    constexpr int VST = D == 128 ? 1 : 2;
    return go(packed_bf16_kernel<D, 1, 64, 4, VST>, 128, Tile<D, 1, 64, 4, VST>::LDS);
  } else {
    if (f.strips == 2) return go(packed_f32_kernel<D, 4, 2>, 32, F_LDS<D, 4, 2>);
    if (f.sets == 4) return go(packed_f32_kernel<D, 4, 1>, 16, F_LDS<D, 4, 1>);
    if (f.sets == 2) return go(packed_f32_kernel<D, 2, 1>, 32, F_LDS<D, 2, 1>);
    return go(packed_f32_kernel<D, 1, 1>, 64, F_LDS<D, 1, 1>);
  }
}

template <typename T>
int packed_by_d(hipStream_t st, const PackedArgs& a, int64_t D, const PackedForm& f) {
  switch (D) {
    case 16:
      return packed_launch<T, 16>(st, a, f);
    case 32:
      return packed_launch<T, 32>(st, a, f);
    case 64:
      return packed_launch<T, 64>(st, a, f);
    default:
      return packed_launch<T, 128>(st, a, f);
  }
}

}  // namespace

// Whether the launch takes the shape: 32-bit row and thread numbers, and tiles of up
// to 128 keys within the 4 GiB that a buffer resource's offsets reach.
int packed_check(int dtype, const PackedShape& s) {
  if (s.D != 16 && s.D != 32 && s.D != 64 && s.D != 128) {
    set_error("packed_attention: head_dim %lld not supported (16, 32, 64, 128)", (long long)s.D);
    return MINITP_ERR_UNSUPPORTED;
  }
  // (query rows are counted in 31 bits; a block of 256 threads takes 16 at least)
  constexpr int64_t MOST = 1LL << 28;
  if (s.N >= MOST || s.Hq >= MOST || s.N * s.Hq >= MOST - 16 * s.Hkv || s.S >= (1LL << 31) - 64) {
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
  a.S = (int)s.S;
  a.Hq = (int)s.Hq;
  a.Hkv = (int)s.Hkv;
  a.per = (int)(s.Hq / s.Hkv);
  a.rows = (int)s.N * a.per;
  a.by_per = make_div(a.per);
  a.by_hkv = make_div(s.Hkv);
  a.offsets = offsets;
  a.scale = 1.0f / sqrtf((float)s.D);
  const PackedForm f = packed_form(dtype == MINITP_BF16, (int)s.D, a.rows, s.Hkv, s.N, s.S);
  return dtype == MINITP_F32 ? packed_by_d<float>(st, a, s.D, f) : packed_by_d<bf16>(st, a, s.D, f);
}

}  // namespace minitp
