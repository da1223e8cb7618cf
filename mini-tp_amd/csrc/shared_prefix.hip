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
// (m, l, o) and a second launch joins them in slot order, or, where that costs
// more than it saves, one item takes both parts (shared_plan).
//
// Bounds: few keys are all latency (4 rows on 128 + 16 keys, 0.5B heads: 5.5 us);
// a long prefix under few rows is two launches and the partial results (32 rows
// on 8,191 + up to 400 keys, 7B heads: 37 MB, 16 us and 6 us for the join); many
// rows are bound by the matrix cores (256 rows on 32,256 + 512 keys: 120 GFLOP
// in 150 us, 0.80 PFLOP/s where a large library product reaches 1.22, and 9 us
// for the join).
#include <type_traits>

#include "attn_tiles.h"
#include "common.h"
#include "kernels.h"

namespace minitp {

namespace {

struct SharedArgs {
  const void *q, *kp, *vp, *kc, *vc;  // q [B, T, Hq, D]; prefix [G, Hkv, Sp, D]; own [B, Hkv, S, D]
  void* out;                          // [B, T, Hq * D]
  int B, T, Hq, Hkv;
  int w, per;                         // batch rows of a group, query heads of a KV head
  int64_t Sp, S;
  int64_t query_rows;                 // B * T * Hq
  int P, C;                           // prefix rows, cached own rows (bounds of the lengths below)
  const int64_t *plens, *clens;       // [G], [B], or NULL: P and C everywhere
  float scale;
  int qtiles_p, qtiles_s;             // query tiles of a unit, prefix and own part
  int splits_p, splits_s;             // key splits
  int items_p, items_s;               // items of the two parts
  int run_p, run_s;                   // ... of one XCD
  Div by_qtiles_p, by_qtiles_s, by_splits_p, by_splits_s, by_hkv, by_w, by_per;
  bool joined;                        // an item takes both parts and writes the output: no slots
  float* ml;                          // [slot][B * T * Hq][2]: maximum, sum
  float* o;                           // [slot][B * T * Hq][D]
};

// Consecutive K/V rows, n of them; the queries of a unit's token t see those up
// to seen + t.
struct Keys {
  const void *k, *v;
  int n, seen;
  bool own;
};

// The last of the keys that token t sees (-1: none).
__device__ __forceinline__ int last_seen(const Keys& k, int t) {
  return k.own ? std::max(std::min(k.seen + t, k.n - 1), -1) : k.n - 1;
}

// What one block computes: a tile of a unit's query rows over the keys of the
// prefix (part 0), of the own rows (part 1) or of one after the other.
struct Item {
  Keys pre, own;
  int first, last;  // parts: 0 the prefix, 1 the own rows
  int n0;           // first token (b * T + t) of the unit
  int rows;         // query rows of the unit: (token, head of the KV group)
  int tile, kv, slot;
};

// Cached own rows of batch row b, -1 for an idle row (nothing attends).
__device__ __forceinline__ int own_len(const SharedArgs& a, int b) {
  if (a.clens == nullptr) return a.C;
  return (int)std::min<int64_t>(std::max<int64_t>(a.clens[b], -1), a.C);
}

// Rows of a prefix or of a batch row's cache, those of one split.
template <int KT>
__device__ __forceinline__ void set_keys(Keys& k, const void* kb, const void* vb, int64_t row0, int64_t row_bytes,
                                         int keys, int split, int splits, const Div& by_splits) {
  const uint32_t tiles = ((uint32_t)keys + KT - 1) / KT;
  const uint32_t span = (uint32_t)by_splits((int)tiles + splits - 1) * KT;
  const int lo = (int)std::min<uint32_t>(split * span, (uint32_t)keys);
  k.k = (const char*)kb + (row0 + lo) * row_bytes;
  k.v = (const char*)vb + (row0 + lo) * row_bytes;
  k.n = (int)std::min<uint32_t>(span, (uint32_t)(keys - lo));
  k.seen = -lo;
}

// Block -> item. Blocks go to the eight XCDs round robin, each with an L2 of
// its own, so every XCD takes a run of each part's items, in which the query
// tiles of one (unit, split) follow each other and share its K/V rows. The
// prefix part, bound by the matrix cores where the groups are large, goes
// first; blocks of the own part, bound by memory, take the places it leaves.
// False: no item.
template <int QT, int KT>
__device__ __forceinline__ bool shared_item(const SharedArgs& a, int64_t row_bytes, Item& it) {
  const int xcd = blockIdx.x % 8, seq = blockIdx.x / 8;
  const bool own = seq >= a.run_p;
  int i = own ? xcd * a.run_s + seq - a.run_p : xcd * a.run_p + seq;
  if (i >= (own ? a.items_s : a.items_p)) return false;
  const int splits = own ? a.splits_s : a.splits_p;
  const Div by_qtiles = own ? a.by_qtiles_s : a.by_qtiles_p, by_splits = own ? a.by_splits_s : a.by_splits_p;
  const int j = by_qtiles(i), unit = by_splits(j), head0 = a.by_hkv(unit);  // (unit: group or batch row, KV head)
  it.tile = i - j * (own ? a.qtiles_s : a.qtiles_p);
  const int split = j - unit * splits;
  it.kv = unit - head0 * a.Hkv;
  const int b = own ? head0 : head0 * a.w, g = own ? a.by_w(head0) : head0;
  it.n0 = b * a.T;
  it.rows = (own ? 1 : a.w) * a.T * a.per;
  it.slot = own ? a.splits_p + split : split;
  it.first = own && (!a.joined || a.P == 0) ? 1 : 0;
  it.last = own ? 1 : 0;
  it.pre.own = false;
  it.own.own = true;
  if (it.first == 0) {
    const int keys = a.plens == nullptr ? a.P : (int)std::min<int64_t>(std::max<int64_t>(a.plens[g], 0), a.P);
    set_keys<KT>(it.pre, a.kp, a.vp, ((int64_t)g * a.Hkv + it.kv) * a.Sp, row_bytes, keys, own ? 0 : split,
                 own ? 1 : splits, own ? Div{1u << 31, 31} : by_splits);
  }
  if (own) {
    const int seen = own_len(a, b);
    const int last = std::min(it.tile * QT + QT, it.rows) - 1;  // (the tile's last query sees the most keys)
    set_keys<KT>(it.own, a.kc, a.vc, (int64_t)unit * a.S, row_bytes, seen < 0 ? 0 : seen + a.by_per(last) + 1, split,
                 splits, by_splits);
    it.own.seen += seen;
    if (seen < 0) it.own.n = it.pre.n = 0;  // an idle row
  }
  return true;
}

// Query row r of an item: its token of the unit, and its row of q and out.
struct Query {
  int t;
  int64_t row;
};
__device__ __forceinline__ Query query_of(const SharedArgs& a, const Item& it, int r) {
  const int t = a.by_per(r);
  return Query{t, (int64_t)(it.n0 + t) * a.Hq + it.kv * a.per + (r - t * a.per)};
}

// One tile of keys through a resource of its own (a head's rows may span more
// than the 4 GiB that one reaches); rows past the item's last read zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t key_rows(const void* base, int key, int keys, int tile,
                                                           int row_bytes) {
  const int n = std::min(keys - key, tile);
  return span_rsrc((const char*)base + (int64_t)key * row_bytes, (uint32_t)(n * row_bytes));
}
__device__ __forceinline__ uint4 rows_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  return make_uint4(v.x, v.y, v.z, v.w);
}

// A maximum to join by. Scores that are no numbers are no maximum but show in
// the sum; what has none above minus infinity and such a sum is no empty set.
__device__ __forceinline__ float join_max(float m, float l) { return l != l ? 0.f : m; }

// Results of query rows [0, rows) from base row r0 of the item that KW waves
// hold over keys of their own, in LDS: po [KW][cap][D], pml [KW][cap] (maximum,
// sum; exp2 or expf by BASE2). Joined, they go to the output or to the slot.
template <typename T, int D, int KW, bool BASE2>
__device__ __forceinline__ void finish_rows(const SharedArgs& a, const Item& it, const float* po, const float2* pml,
                                            int cap, int r0, int rows) {
  constexpr int LPR = D / 4;
  for (int i = threadIdx.x; i < rows * LPR; i += 256) {
    const int row = i / LPR, d = i % LPR * 4;
    float2 ml[KW];
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      ml[j] = pml[j * cap + row];
      m = fmaxf(m, ml[j].x);
    }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      if (ml[j].x == -__builtin_inff()) continue;
      const float sc = BASE2 ? __builtin_amdgcn_exp2f(ml[j].x - m) : expf(ml[j].x - m);
      l = fmaf(sc, ml[j].y, l);
      const f32x4 oj = *(const f32x4*)(po + (j * cap + row) * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(sc, oj[e], o[e]);
    }
    const int64_t n = query_of(a, it, r0 + row).row;
    if (a.joined) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = m == -__builtin_inff() ? 0.f : o[e] / l;
      store_vec<T, 4>((T*)a.out + n * D + d, v);
    } else {
      const int64_t at = it.slot * a.query_rows + n;
      *(f32x4*)(a.o + at * D + d) = o;
      if (d == 0) *(float2*)(a.ml + at * 2) = make_float2(m, l);
    }
  }
}

// ---------------------------------------------------------------------------
// fp32, on v_mfma_f32_16x16x4_f32. Four waves share each 64-key tile in LDS: 4 / KW
// strips of 16 queries, KW waves a strip over 64 / KW keys each (a unit of few
// rows is bound by the latency of one wave's keys); products transposed: S^T =
// K Q^T leaves lane (quad, r) with keys 4 quad .. 4 quad + 3 of query r, which
// is the B operand of O^T = V^T P^T as it is. Score MFMA i of a chunk takes
// dims 16 c + 4 quad + i from both operands (one 16-byte LDS read a lane),
// output MFMA j dims E r + j; rows are padded by 16 bytes against bank
// conflicts. A score is summed in four chains. Measured: 3 x 5 rows on 777 + 100
// keys, 0.5B heads, 8 us and 4 us for the join (latency); 11 x 116 rows on 421 +
// up to 206 keys, 7B heads, 10.4 GFLOP in 171 us (572 blocks on 512 places; 220
// us before the bound of two blocks a CU, which kept D = 128 to one).
constexpr int F_QT = 64, F_KT = 64;
template <int D>
constexpr int F_LDS = 2 * F_KT * (D + 4) * 4;

template <int D, int KW>
__device__ __forceinline__ void shared_rows_f32(const SharedArgs& a, const Item& it, float* lds, int* odd) {
  constexpr int KT = F_KT, KB = KT / 16 / KW, KC = D / 16, SW = 4 / KW;
  constexpr int E = D / 16 < 4 ? D / 16 : 4, HALVES = D / 16 / E;
  constexpr int ROW = D + 4;
  constexpr int PIECES = KT * D / 4, PER = (PIECES + 255) / 256;
  float *Ks = lds, *Vs = lds + KT * ROW;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane % 16, lq = lane / 16, strip = wave % SW, key0 = wave / SW * KB * 16;
  const int t0 = it.tile * F_QT, r = t0 + strip * 16 + lr;
  const Query me = query_of(a, it, r < it.rows ? r : 0);

  f32x4 qa[KC];
  {
    const float* qrow = (const float*)a.q + me.row * D;
#pragma unroll
    for (int c = 0; c < KC; ++c) qa[c] = *(const f32x4*)(qrow + 16 * c + 4 * lq);
  }
  f32x4 o[HALVES][E];
#pragma unroll
  for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
    for (int j = 0; j < E; ++j) o[hf][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), lsum = 0.f;

  for (int part = it.first; part <= it.last; ++part) {
    const Keys ks = part == 0 ? it.pre : it.own;
    const int seen = last_seen(ks, me.t), all_see = last_seen(ks, a.by_per(t0));
    uint4 kr[PER], vr[PER];
    auto load_tile = [&](int key) {
      const __amdgpu_buffer_rsrc_t krs = key_rows(ks.k, key, ks.n, KT, D * 4);
      const __amdgpu_buffer_rsrc_t vrs = key_rows(ks.v, key, ks.n, KT, D * 4);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const uint32_t off = (uint32_t)(tid + 256 * u) * 16;  // (past the tile: not stored)
        kr[u] = rows_load16(krs, off);
        vr[u] = rows_load16(vrs, off);
      }
    };
    if (ks.n > 0) load_tile(0);
    for (int k0 = 0; k0 < ks.n; k0 += KT) {
      __syncthreads();  // the previous tile is consumed
      if (tid == 0) *odd = 0;
      __syncthreads();
      bool found = false;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int i = tid + 256 * u;
        if (i < PIECES) {
          const int row = i / (D / 4), at = row * ROW + i % (D / 4) * 4;
          *(uint4*)(Ks + at) = kr[u];
          *(uint4*)(Vs + at) = vr[u];
          if (k0 + row > all_see) {
            // a key that some query does not see: is its value finite?
            const f32x4 f = __builtin_bit_cast(f32x4, vr[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= !__builtin_isfinite(f[e]);
          }
        }
      }
      if (found) *odd = 1;
      __syncthreads();
      if (k0 + KT < ks.n) load_tile(k0 + KT);
      const bool slow = *odd != 0;
      if (k0 + key0 >= ks.n) continue;  // (none of this wave's keys)
      const int limit = seen - k0 - key0;  // last of the wave's keys that this query sees
      float p[KB][4];
      float mx = -__builtin_inff();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        f32x4 chain[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) chain[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const f32x4 k4 = *(const f32x4*)(Ks + (key0 + kb * 16 + lr) * ROW + 16 * c + 4 * lq);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            chain[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4[i], qa[c][i], chain[i], 0, 0, 0);
        }
        const f32x4 acc = (chain[0] + chain[1]) + (chain[2] + chain[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[kb][e] = kb * 16 + 4 * lq + e <= limit ? acc[e] * a.scale : -__builtin_inff();
          mx = fmaxf(mx, p[kb][e]);
        }
      }
      mx = quads_max(mx);
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
              const float* vrow = Vs + (key0 + key) * ROW;
#pragma unroll
              for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
                for (int j = 0; j < E; ++j)
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const float v = vrow[64 * hf + E * (4 * lq + x) + j];
                    o[hf][j][x] = key <= limit ? fmaf(pk, v, o[hf][j][x]) : o[hf][j][x];
                  }
            }
        continue;
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* vrow = Vs + (key0 + kb * 16 + 4 * lq + e) * ROW + E * lr;
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
            for (int j = 0; j < E; ++j)
              o[hf][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], p[kb][e], o[hf][j], 0, 0, 0);
          }
        }
    }
  }
  // o[hf][j][x]: dim 64 hf + E (4 lq + x) + j of the lane's query
  lsum = quads_sum(lsum);
  constexpr int CAP = SW * 16;
  float* po = lds;                        // [KW][CAP][D]
  float2* pml = (float2*)(po + 64 * D);   // [KW][CAP]
  const int at = wave / SW * CAP + strip * 16 + lr;
  __syncthreads();  // (the last tile is consumed)
#pragma unroll
  for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int j = 0; j < E; ++j) po[at * D + 64 * hf + E * (4 * lq + x) + j] = o[hf][j][x];
  if (lq == 0) pml[at] = make_float2(join_max(m, lsum), lsum);
  __syncthreads();
  finish_rows<float, D, KW, false>(a, it, po, pml, CAP, t0, std::min(CAP, it.rows - t0));
}

template <int D>
__global__ __launch_bounds__(256, 2) void shared_attn_f32_kernel(SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds_f[];
  static_assert(F_LDS<D> >= 64 * (D + 2) * 4, "the waves' results fit the tiles");
  __shared__ int odd;
  Item it;
  if (!shared_item<F_QT, F_KT>(a, D * 4, it)) return;
  const int rows = it.rows - it.tile * F_QT;
  if (rows <= 16)
    shared_rows_f32<D, 4>(a, it, lds_f, &odd);
  else if (rows <= 32)
    shared_rows_f32<D, 2>(a, it, lds_f, &odd);
  else
    shared_rows_f32<D, 1>(a, it, lds_f, &odd);
}

// ---------------------------------------------------------------------------
// bf16. A block takes 128 query rows of a unit over the keys of its split, four
// waves of 32 rows (v_mfma_f32_32x32x16_bf16), or, where the unit has at most 16
// rows (one token of a row's own part), those rows over 64 keys at a time, 16
// keys a wave (16x16 MFMAs).
//
// A tile of 64 K and V rows goes to LDS as it lies in memory, by loads that
// bypass the registers, while the tile before it is computed (two stages, one
// barrier a tile). Products are transposed, S^T = K Q^T and O^T = V^T P^T, so
// a lane's scores belong to one query: its maximum takes one lane exchange, its
// sum none until the end, and its probabilities are the second product's
// operand as they are, the k-index of both operands permuted alike. V^T comes
// out of LDS transposed by ds_read_b64_tr_b16: in each group of 16 lanes, lane
// i gives the address of four columns of row i / 4 and receives column i of
// the four rows.
//
// The 16-byte chunks of a row are permuted by its row number, which the loads
// do on the global side, so that every LDS read reaches all banks: a K read
// takes one chunk column of 16 rows, a V read 64 bytes of four rows.
//
// A probability is rounded to bf16 for the second product, by at most 2^-8 of
// itself, as much as the output's own rounding: the matrix cores take bf16
// there, and fp32 products would run at an eighth of the rate (153 against 1,223
// TFLOP/s of a large library product). The sums that they are divided by add
// the unrounded ones.
//
// Two blocks a CU (64 KiB of LDS each at D = 128) cover each other's softmax:
// 512 even blocks (16 rows of 128 tokens, 32 heads, 8,192 keys) run at 1.04 to
// 1.07 PFLOP/s. Not faster, each against the kernel as it stood then: a tile's
// scores computed before the tile in front of it is used (946 against 961
// TFLOP/s), the next loads issued behind the scores (-7 %) or spread over the
// product.
constexpr int H_QT = 128, H_SMALL = 16;

// one of eight bf16 values is infinite or NaN
__device__ __forceinline__ bool not_finite(const uint4& x) {
  const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) odd |= (wd[e] & 0x7f80u) == 0x7f80u || (wd[e] & 0x7f800000u) == 0x7f800000u;
  return odd;
}
// The tiles of consecutive rows through the two stages (tile t in stage t % 2).
template <int D>
struct Tiles {
  using H = Half<D>;
  const char *k, *v;
  uint32_t to, koff, voff;
  int keys, n;
  __device__ __forceinline__ Tiles(const Keys& ks, char* lds)
      : k((const char*)ks.k), v((const char*)ks.v), keys(ks.n), n((ks.n + H_KT - 1) / H_KT) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + w * 1024;
    // piece w + 4 j of a tile: rows 4 PIECE_ROWS j + row; the swizzles do not depend on j
    const int row = H::PIECE_ROWS * (H::PPW > 0 ? w : w & 1) + lane / H::CH;
    koff = row * H::ROWB + ((lane % H::CH) ^ H::k_swz(row)) * 16;
    voff = row * H::ROWB + ((lane % H::CH) ^ H::v_swz(row)) * 16;
  }
  __device__ __forceinline__ void load(int t) const {
    if (t >= n) return;
    const int left = std::min(keys - t * H_KT, H_KT) * H::ROWB;
    const u32x4 kr = rows_rsrc(k + (int64_t)t * H::OPER, left), vr = rows_rsrc(v + (int64_t)t * H::OPER, left);
    uint32_t at = __builtin_amdgcn_readfirstlane(to + (t & 1) * H::STAGE);
    asm volatile("s_nop 4" : "+s"(at));
    if constexpr (H::PPW == 0) {
      if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 7) == 0)
        row_dma16(kr, koff, at);
      else
        row_dma16(vr, voff, at);
    }
#pragma unroll
    for (int j = 0; j < H::PPW; ++j) row_dma16(kr, koff + j * 4096, at + j * 4096);
#pragma unroll
    for (int j = 0; j < H::PPW; ++j) row_dma16(vr, voff + j * 4096, at + H::OPER + j * 4096);
  }
  // compute(t, stage, masked) for each tile, tile 0 being on its way; the tiles
  // from `masked_from` on have keys that some query does not see
  template <typename F>
  __device__ __forceinline__ void each(const char* lds, int masked_from, F&& compute) const {
    int t = 0;
    for (; t < masked_from; ++t) {
      stage_wait();
      load(t + 1);  // (the stage's readers passed the barrier)
      compute(t, lds + (t & 1) * H::STAGE, std::false_type{});
    }
    for (; t < n; ++t) {
      stage_wait();
      load(t + 1);
      compute(t, lds + (t & 1) * H::STAGE, std::true_type{});
    }
  }
};

// AHEAD: a wave's second products go before other waves' work (below).
template <int D, bool AHEAD>
__device__ __forceinline__ void shared_rows128(const SharedArgs& a, const Item& it, char* lds) {
  using H = Half<D>;
  // (D = 16: the output's 32-row operand holds the 16 dims twice)
  constexpr int KS = D / 16, DB = D >= 32 ? D / 32 : 1, OC = D >= 32 ? 4 : 2;  // OC: 8-dim chunks of a block
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  Keys ks = it.first == 0 ? it.pre : it.own;
  Tiles<D> tiles(ks, lds);
  tiles.load(0);
  const int r0 = it.tile * H_QT + w * 32, r = r0 + n32;
  const Query me = query_of(a, it, r < it.rows ? r : 0);

  bf16x8 qb[KS];
  {
    const bf16* q = (const bf16*)a.q + me.row * D + 8 * h;
#pragma unroll
    for (int k = 0; k < KS; ++k) qb[k] = __builtin_bit_cast(bf16x8, *(const u32x4*)(q + 16 * k));
  }
  const int t_first = a.by_per(it.tile * H_QT), t_last = a.by_per(r0 + 31);  // of the block, of the wave
  f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), lsum = 0.f;
  const float sl2 = a.scale * 1.4426950408889634f;

  // LDS bytes of this lane's operands: K row n32, chunk 2 k + h; V rows
  // 4 h + (lane % 16) / 4 (+ 8), dims 32 d + 16 ((lane / 16) % 2) + 4 (lane % 4)
  const int kat = n32 * H::ROWB, kx = (h ^ H::k_swz(n32)) << 4;
  const int vrow = 4 * h + (lane & 15) / 4;
  const int vat = H::OPER + vrow * H::ROWB + 8 * (lane & 1);
  const int vx = (((D >= 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane >> 1) & 1)) ^ H::v_swz(vrow)) << 4;
  arrived(qb);

  for (int part = it.first; part <= it.last; ++part) {
    if (part != it.first) {
      ks = it.own;
      tiles = Tiles<D>(ks, lds);
      __syncthreads();  // (every stage is free)
      tiles.load(0);
    }
    const int seen = last_seen(ks, me.t), seen_last = last_seen(ks, t_last);
    const int all_see = last_seen(ks, t_first);  // the last key that every query of the block sees
    tiles.each(lds, (all_see + 1) / H_KT, [&](int t, const char* st, auto masked) {
      if (r0 >= it.rows || (masked && t * H_KT > seen_last)) return;
      f32x16 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {  // (two chains in turn)
          const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(st + kat + kb * 32 * H::ROWB + ((32 * k) ^ kx)));
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb[k], s[kb], 0, 0, 0);
        }
      }
      bool odd = false;
      const int limit = seen - t * H_KT;
      if constexpr (masked) {
        // lane (query, h) holds keys 32 kb + 8 (i / 4) + 4 h + i % 4
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * kb + 8 * (i / 4) + i % 4 > limit - 4 * h) s[kb][i] = -__builtin_inff();
        if (all_see < ks.n - 1) {
          // hidden keys that other queries see: are their values finite?
          for (int c = lane; c < H_KT * H::CH; c += 64) odd |= not_finite(*(const uint4*)(st + H::OPER + c * 16));
          odd = __builtin_amdgcn_ballot_w64(odd) != 0;
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
      mx = halves_max(mx) * sl2;
      if (__builtin_amdgcn_ballot_w64(mx > m + SLACK)) {
        const float mn = fmaxf(m, mx), alpha = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        lsum *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= alpha;
      }
      const float mref = m == -__builtin_inff() ? 0.f : m;  // (nothing seen yet)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], sl2, -mref));
          lsum += s[kb][i];
        }
      if (masked && odd) {
        // a value that some query may not touch is not finite (0 times it is no
        // zero): key by key, for the queries that see it
#pragma unroll 1
        for (int key = 0; key < H_KT; ++key) {
          const int idx = (key >> 5) * 16 + ((key >> 3) & 3) * 4 + (key & 3);
          float p = 0.f;
#pragma unroll
          for (int c = 0; c < 32; ++c) p = c == idx ? s[c / 16][c % 16] : p;
          p = __shfl(p, n32 + 32 * ((key >> 2) & 1), 64);
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int c = 0; c < OC; ++c) {
              const char* vp = st + H::OPER + key * H::ROWB + (((4 * d + c) ^ H::v_swz(key)) << 4) + 8 * h;
              const uint2 x = *(const uint2*)vp;
              const float v[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u),
                                  __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u)};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float old = o[d][4 * c + e];
                o[d][4 * c + e] = key <= limit ? fmaf(p, v[e], old) : old;
              }
            }
        }
        return;
      }
      if (AHEAD) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // keys 16 j .. 16 j + 15
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
          const char* vp = st + vat + 16 * j * H::ROWB + ((64 * d) ^ vx);
          const bf16x8 vf = join8(read_tr(vp), read_tr(vp + 8 * H::ROWB));
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb, o[d], 0, 0, 0);
        }
      }
      if (AHEAD) __builtin_amdgcn_s_setprio(0);
    });
  }
  if (r >= it.rows) return;
  const float l = halves_sum(lsum);
  m = join_max(m, l);
  if (a.joined) {
    const float f = m == -__builtin_inff() ? 0.f : 1.f / l;
    bf16* orow = (bf16*)a.out + me.row * D + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int c = 0; c < OC; ++c) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[d][4 * c + e] * f;
        store_vec<bf16, 4>(orow + 32 * d + 8 * c, v);
      }
    return;
  }
  const int64_t at = it.slot * a.query_rows + me.row;
  if (h == 0) *(float2*)(a.ml + at * 2) = make_float2(m, l);
  float* orow = a.o + at * D + 4 * h;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int c = 0; c < OC; ++c)
      *(f32x4*)(orow + 32 * d + 8 * c) = f32x4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
}

template <int D>
__device__ __forceinline__ void shared_rows16(const SharedArgs& a, const Item& it, char* lds) {
  using H = Half<D>;
  constexpr int KS = D >= 32 ? D / 32 : 1, DB = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, q4 = lane >> 4;
  Keys ks = it.first == 0 ? it.pre : it.own;
  Tiles<D> tiles(ks, lds);
  tiles.load(0);
  const int r = n16;  // (one tile)
  const Query me = query_of(a, it, r < it.rows ? r : 0);

  bf16x8 qb[KS];  // (D = 16: four dims a lane, in the low half)
  {
    const bf16* q = (const bf16*)a.q + me.row * D + (D >= 32 ? 8 : 4) * q4;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if constexpr (D >= 32) {
        qb[k] = __builtin_bit_cast(bf16x8, *(const u32x4*)(q + 32 * k));
      } else {
        const uint2 x = *(const uint2*)q;
        qb[k] = __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, 0, 0));
      }
    }
  }
  f32x4 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), lsum = 0.f;
  const float sl2 = a.scale * 1.4426950408889634f;

  // K row 16 w + n16, chunk 4 k + q4; V rows 16 w + 4 q4 + n16 / 4, dims 16 d + 4 (lane % 4)
  // (D = 16: 8 bytes, half q4 % 2 of chunk q4 / 2)
  const int krow = 16 * w + n16, kat = krow * H::ROWB + (D >= 32 ? 0 : 8 * (q4 & 1));
  const int kx = ((D >= 32 ? q4 : q4 >> 1) ^ H::k_swz(krow)) << 4;
  const int vrow = 16 * w + 4 * q4 + n16 / 4;
  const int vat = H::OPER + vrow * H::ROWB + 8 * (lane & 1), vx = (((lane >> 1) & 1) ^ H::v_swz(vrow)) << 4;
  arrived(qb);

  for (int part = it.first; part <= it.last; ++part) {
    if (part != it.first) {
      ks = it.own;
      tiles = Tiles<D>(ks, lds);
      __syncthreads();  // (every stage is free)
      tiles.load(0);
    }
    const int seen = last_seen(ks, me.t), all_see = last_seen(ks, 0);
    tiles.each(lds, (all_see + 1) / H_KT, [&](int t, const char* st, auto masked) {
      const int kw = t * H_KT + 16 * w;
      if (masked && kw >= ks.n) return;
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if constexpr (D >= 32) {
          const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(st + kat + ((64 * k) ^ kx)));
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qb[k], s, 0, 0, 0);
        } else {
          const s16x4 kf = *(const s16x4*)(st + kat + kx);
          const auto q = __builtin_bit_cast(s16x8, qb[0]);
          s = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(kf, s16x4{q[0], q[1], q[2], q[3]}, s, 0, 0, 0);
        }
      }
      const int limit = seen - kw;
      if constexpr (masked) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * q4 + i > limit) s[i] = -__builtin_inff();
      }
      const float mx = quads_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))) * sl2;
      if (__builtin_amdgcn_ballot_w64(mx > m)) {
        const float mn = fmaxf(m, mx), alpha = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        lsum *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= alpha;
      }
      const float mref = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sl2, -mref));
        lsum += s[i];
      }
      // (several tokens: a hidden key's value may not be finite)
      if (masked && all_see < ks.n - 1) {
        bool odd = false;
        for (int c = lane; c < 16 * H::CH; c += 64)
          odd |= not_finite(*(const uint4*)(st + H::OPER + 16 * w * H::ROWB + c * 16));
        if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
          for (int key = 0; key < 16; ++key) {
            const float pi = (key & 3) == 0 ? s[0] : (key & 3) == 1 ? s[1] : (key & 3) == 2 ? s[2] : s[3];
            const float p = __shfl(pi, n16 + 16 * (key >> 2), 64);
            const int row = 16 * w + key;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
              const int chunk = (2 * d + (q4 >> 1)) ^ H::v_swz(row);
              const char* vp = st + H::OPER + row * H::ROWB + (chunk << 4) + 8 * (q4 & 1);
              const uint2 x = *(const uint2*)vp;
              const float v[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u),
                                  __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u)};
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][e] = key <= limit ? fmaf(p, v[e], o[d][e]) : o[d][e];
            }
          }
          return;
        }
      }
      const s16x4 pb = __builtin_bit_cast(s16x4, make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])));
#pragma unroll
      for (int d = 0; d < DB; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(read_tr(st + vat + ((32 * d) ^ vx)), pb, o[d], 0, 0, 0);
    });
  }

  // ---- the four waves' keys joined through LDS ------------------------------
  const float l = quads_sum(lsum);
  float* po = (float*)lds;                     // [wave][16][D]
  float2* pml = (float2*)(po + 4 * H_SMALL * D);  // [wave][16]
  __syncthreads();                             // (every stage is free)
#pragma unroll
  for (int d = 0; d < DB; ++d) *(f32x4*)(po + (w * H_SMALL + r) * D + 16 * d + 4 * q4) = o[d];
  if (q4 == 0) pml[w * H_SMALL + r] = make_float2(join_max(m, l), l);
  __syncthreads();
  finish_rows<bf16, D, 4, true>(a, it, po, pml, H_SMALL, 0, it.rows);
}

// FEW: the own part's units have at most 16 rows. Where they have more, all blocks
// are alike and the two on a CU fall into step best, one in its softmax while
// the other multiplies, when a wave's second products go first: 16 rows of 100
// tokens on 4,096 keys, 7B heads, 123 -> 115 us. Beside blocks of few rows it
// costs them their turns (256 rows of one token on 32,256 keys 158 -> 164 us).
template <int D, bool FEW>
__global__ __launch_bounds__(256, 2) void shared_attn_bf16_kernel(SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  static_assert(Half<D>::LDS >= 4 * H_SMALL * (D + 2) * 4, "the waves' join fits the stages");
  Item it;
  if (!shared_item<H_QT, H_KT>(a, D * 2, it)) return;
  if (FEW && it.rows <= H_SMALL)
    shared_rows16<D>(a, it, lds);
  else
    shared_rows128<D, !FEW>(a, it, lds);
}

// The slots of each query row joined, by powers of the base that their maxima are
// in (fp32 e, bf16 2: changing it would round a maximum once more, and so weigh
// the parts by as much as 2^-24 of it); every LPR = D / 4 lanes take four dims
// each. SG sets of lanes share a row, set j the slots j, j + SG, ...: one set a row
// where there are many rows or few slots. A query that saw no key, in an idle
// row or one without any, gets zeros.
template <typename T, int D, int SG>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
  constexpr int LPR = D / 4, RB = 256 / (LPR * SG);
  static_assert(RB == 1 || SG == 1, "a block's sets share one row, or each has its own");
  __shared__ f32x4 po[4][LPR];
  __shared__ float2 pml[4];
  const int64_t rows = a.query_rows;
  const int lane = threadIdx.x % LPR, sg = threadIdx.x / LPR % SG, rb = threadIdx.x / (LPR * SG);
  const int64_t i = (int64_t)blockIdx.x * RB + rb;
  const int64_t row = std::min<int64_t>(i, rows - 1);
  const int slots = a.splits_p + a.splits_s;
  const bool idle = a.clens != nullptr && own_len(a, (int)((uint32_t)row / (uint32_t)(a.Hq * a.T))) < 0;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto power = [](float x) { return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(x) : expf(x); };
  auto add = [&](float ms, float ls, const f32x4& os, float mn) {
    if (ms == -__builtin_inff()) return;  // the split saw no key
    const float a1 = power(ms - mn);
    l = fmaf(ls, a1, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(os[e], a1, o[e]);
  };
  constexpr int NB = 4;  // slots whose loads are in flight together
  for (int s0 = sg; s0 < slots; s0 += NB * SG) {
    float2 ml[NB];
    f32x4 os[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int64_t at = std::min(s0 + u * SG, slots - 1) * rows + row;  // (past the last: read again, left out)
      ml[u] = *(const float2*)(a.ml + at * 2);
      os[u] = *(const f32x4*)(a.o + at * D + 4 * lane);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (s0 + u * SG >= slots) ml[u].x = -__builtin_inff();
      mn = fmaxf(mn, ml[u].x);
    }
    if (mn == -__builtin_inff()) continue;
    const float a0 = power(m - mn);
    l *= a0;
    o *= a0;
#pragma unroll
    for (int u = 0; u < NB; ++u) add(ml[u].x, ml[u].y, os[u], mn);
    m = mn;
  }
  if constexpr (SG > 1) {
    // the sets of a wave by lane exchange, then the four waves through LDS
    auto fold = [&](float mo, float lo, const f32x4& oo) {
      const float mn = fmaxf(m, mo);
      const float a0 = m == -__builtin_inff() ? 0.f : power(m - mn);
      const float a1 = mo == -__builtin_inff() ? 0.f : power(mo - mn);
      l = l * a0 + lo * a1;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * a0 + oo[e] * a1;
      m = mn;
    };
#pragma unroll
    for (int x = LPR; x < 64; x *= 2) {
      f32x4 oo;
#pragma unroll
      for (int e = 0; e < 4; ++e) oo[e] = __shfl_xor(o[e], x, 64);
      const float mo = __shfl_xor(m, x, 64), lo = __shfl_xor(l, x, 64);
      fold(mo, lo, oo);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < LPR) {
      po[wave][lane] = o;
      if (lane == 0) pml[wave] = make_float2(m, l);
    }
    __syncthreads();
    if (threadIdx.x >= LPR) return;
#pragma unroll
    for (int j = 1; j < 4; ++j) fold(pml[j].x, pml[j].y, po[j][lane]);
  }
  if (i >= rows) return;
  const bool empty = idle || m == -__builtin_inff();
  float r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = empty ? 0.f : o[e] / l;
  store_vec<T, 4>((T*)a.out + i * D + 4 * lane, r);
}

// Query tiles and key splits of a call.
struct Plan {
  int qtiles_p, qtiles_s, splits_p, splits_s;
  int64_t items_p, items_s;
  bool joined;
};

// Splits: the prefix part takes 256 blocks, each of at least two key tiles (one
// on the fp32 path, whose tiles take three times as long), or, where that
// leaves a block 16 tiles and more, 448 of the 512 places that there are; the
// own part 256 blocks of at least two tiles. Measured (us a call): 32 rows of
// the 7B heads on 8,191 and up to 400 keys, 8 units: 16 splits 24.0, 32 (taken)
// 22.1, 48 25.3, 64 30.2; 256 rows on 32,256 and 511, 56 units: 7 splits 159.7, 8
// (taken) 161.8, 9 176.1, 12 170.7; 8 rows x 4 of the 0.5B heads on 2,048: 8 splits
// 12.2, 16 11.6, 32 12.4; fp32, 5 rows x 3 on 777: 6 19.3, 13 12.6.
//
// Joined, one item a query tile over both parts and straight to the output, where
// a second launch and the partial results cost more than the prefix computed
// for half-empty tiles. Measured (us, joined against apart; own: tiles of all rows):
//   own < 256: bf16, up to 10 key tiles in all, fp32, rows of at most 16 queries
//     and up to 7 tiles, two of them the prefix's: own 128, 7B heads, 512 + 65 keys
//     10.4 against 12.0, 1,024 + 1 14.2 against 12.9; fp32 128 + 257 25.3 against
//     27.9, 256 + 1 17.6 against 16.2;
//   rows of at most 16 queries, whose tiles are not shared: own x prefix tiles
//     up to 8,192 (fp32 131,072 / D): own 512, 7B heads, 1,024 + 1 keys 18.4
//     against 24.7, own 2,048 256 + 65 39.5 against 36.4; fp32 own 256 256 + 65
//     20.9 against 23.4, own 512 256 + 65 42.7 against 37.8;
//   longer rows: the empty part of their tiles, in queries x prefix keys a
//     query, up to 1,200 (fp32 100): 7B heads, 63 queries of 128, own 512, 1,024
//     keys 34.8 against 40.3, 4,096 101 against 102; 98: 4,096 132 against 136;
//     700 of 768, 4,096 keys 114 against 120; fp32 98 of 128, own 512, 256 keys
//     156 against 163, 1,024 486 against 465.
Plan shared_plan(int dtype, int64_t D, int64_t B, int64_t G, int64_t T, int64_t Hq, int64_t Hkv, int64_t P, int64_t C) {
  const bool tiles16 = dtype == MINITP_BF16;
  const int64_t qt = tiles16 ? H_QT : F_QT, kt = tiles16 ? H_KT : F_KT, per = Hq / Hkv;
  Plan p;
  p.qtiles_p = (int)cdiv(B / G * T * per, qt);
  p.qtiles_s = (int)cdiv(T * per, qt);
  const int64_t bp = G * Hkv * p.qtiles_p, bs = B * Hkv * p.qtiles_s;
  const int64_t tiles_p = cdiv(P, kt), tiles_s = cdiv(C + T, kt);
  auto within = [](int64_t v, int64_t most) { return (int)std::max<int64_t>(1, std::min(v, most)); };
  const int64_t most_p = tiles16 ? tiles_p / 2 : tiles_p;
  p.splits_p = P > 0 ? within(std::min(448 / bp, std::max(256 / bp, tiles_p / 16)), most_p) : 0;
  p.splits_s = within(256 / bs, tiles_s / 2);
  const bool few = T * per <= H_SMALL;
  if (P == 0 && p.splits_s == 1)
    p.joined = true;
  else if (bs < 256)
    p.joined = tiles16 ? tiles_p + tiles_s <= 10 : few && tiles_p <= 2 && tiles_p + tiles_s <= 7;
  else if (few)
    p.joined = tiles_p <= 16 && bs * tiles_p <= (tiles16 ? 8192 : 131072 / D) && (tiles_p <= 4 || tiles_p + tiles_s <= 20);
  else
    p.joined = (qt * p.qtiles_s - T * per) * P <= (tiles16 ? 1200 : 100) * T * per;
  if (p.joined) {
    p.splits_p = 0;
    p.splits_s = 1;
  }
  p.items_p = bp * p.splits_p;
  p.items_s = bs * p.splits_s;
  return p;
}

template <typename T, int D>
int shared_launch(hipStream_t st, const SharedArgs& a, const Plan& p) {
  const dim3 grid((unsigned)(8 * (a.run_p + a.run_s)));
  if constexpr (sizeof(T) == 2) {
    const auto kern = a.T * a.per <= H_SMALL ? shared_attn_bf16_kernel<D, true> : shared_attn_bf16_kernel<D, false>;
    const int rc = ensure_lds_limit((const void*)kern, Half<D>::LDS);
    if (rc) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(256), Half<D>::LDS, st, a);
  } else {
    const int rc = ensure_lds_limit((const void*)shared_attn_f32_kernel<D>, F_LDS<D>);
    if (rc) return rc;
    hipLaunchKernelGGL((shared_attn_f32_kernel<D>), grid, dim3(256), F_LDS<D>, st, a);
  }
  MINITP_LAUNCH_CHECK();
  if (p.joined) return MINITP_OK;
  const int64_t rows = a.query_rows;
  constexpr int SG = 256 / (D / 4);
  // (several sets of lanes a row while there are few rows: 7,168 rows of 9
  // slots 8.3 us with one set, 18.3 with eight; 896 rows of 33 slots 5.7 us with
  // eight)
  if (p.splits_p + p.splits_s >= 4 && rows * (D / 4) < 131072)
    hipLaunchKernelGGL((shared_join_kernel<T, D, SG>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((shared_join_kernel<T, D, 1>), dim3((unsigned)cdiv(rows, SG)), dim3(256), 0, st, a);
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
    default:
      return shared_launch<T, 128>(st, a, p);
  }
}

}  // namespace

// Whether the launches take the shape: 32-bit row, key and thread numbers, of
// the join too (a thread for four elements of the output, where parts are joined).
int shared_prefix_check(int dtype, const SharedPrefixShape& s) {
  if (s.D != 16 && s.D != 32 && s.D != 64 && s.D != 128) {
    set_error("shared_prefix_attention: head_dim %lld not supported (16, 32, 64, 128)", (long long)s.D);
    return MINITP_ERR_UNSUPPORTED;
  }
  constexpr int64_t MOST = 1LL << 31;
  if (s.P >= MOST - 64 || s.C >= MOST || s.T >= MOST || s.C + s.T >= MOST - 64) {
    set_error("shared_prefix_attention: %lld prefix and %lld + %lld own rows are too many", (long long)s.P,
              (long long)s.C, (long long)s.T);
    return MINITP_ERR_UNSUPPORTED;
  }
  bool fits = s.B < MOST && s.Hq < MOST && s.B * s.T < MOST && s.B * s.T * s.Hq < MOST - 256;
  if (fits && s.B * s.T > 0) {
    const Plan p = shared_plan(dtype, s.D, s.B, s.G, s.T, s.Hq, s.Hkv, s.P, s.C);
    fits = p.items_p + p.items_s < (1LL << 24) - 16 && (p.joined || cdiv(s.B * s.T * s.Hq, 1024 / s.D) < (1LL << 24));
  }
  if (!fits) {
    set_error("shared_prefix_attention: %lld x %lld x %lld query rows are too many for one call", (long long)s.B,
              (long long)s.T, (long long)s.Hq);
    return MINITP_ERR_UNSUPPORTED;
  }
  return MINITP_OK;
}

int64_t shared_prefix_workspace_bytes(int dtype, const SharedPrefixShape& s) {
  if (s.B == 0 || s.T == 0) return 0;
  if (shared_prefix_check(dtype, s)) return -1;
  const Plan p = shared_plan(dtype, s.D, s.B, s.G, s.T, s.Hq, s.Hkv, s.P, s.C);
  return p.joined ? 0 : (p.splits_p + p.splits_s) * s.B * s.T * s.Hq * (s.D + 2) * 4;
}

int launch_shared_prefix_attention(hipStream_t st, int dtype, const SharedPrefixShape& s, const void* q,
                                   const void* k_prefix, const void* v_prefix, const void* k_cache,
                                   const void* v_cache, void* out, const int64_t* prefix_lens,
                                   const int64_t* cache_lens, void* workspace, int64_t workspace_bytes) {
  const int rc = shared_prefix_check(dtype, s);
  if (rc) return rc;
  const Plan p = shared_plan(dtype, s.D, s.B, s.G, s.T, s.Hq, s.Hkv, s.P, s.C);
  const int64_t rows = s.B * s.T * s.Hq;
  const int64_t need = p.joined ? 0 : (p.splits_p + p.splits_s) * rows * (s.D + 2) * 4;
  if (workspace_bytes < need || (workspace == nullptr && need > 0) || !aligned16(workspace)) {
    set_error("shared_prefix_attention: workspace %p of %lld B, %lld B needed (16-byte aligned)", workspace,
              (long long)workspace_bytes, (long long)need);
    return MINITP_ERR_ARG;
  }
  SharedArgs a{};
  a.q = q;
  a.kp = k_prefix;
  a.vp = v_prefix;
  a.kc = k_cache;
  a.vc = v_cache;
  a.out = out;
  a.B = (int)s.B;
  a.w = (int)(s.B / s.G);
  a.per = (int)(s.Hq / s.Hkv);
  a.query_rows = rows;
  a.T = (int)s.T;
  a.Hq = (int)s.Hq;
  a.Hkv = (int)s.Hkv;
  a.Sp = s.Sp;
  a.S = s.S;
  a.P = (int)s.P;
  a.C = (int)s.C;
  a.plens = prefix_lens;
  a.clens = cache_lens;
  a.scale = 1.0f / sqrtf((float)s.D);
  a.qtiles_p = p.qtiles_p;
  a.qtiles_s = p.qtiles_s;
  a.splits_p = p.splits_p;
  a.splits_s = p.splits_s;
  a.items_p = (int)p.items_p;
  a.items_s = (int)p.items_s;
  a.run_p = (int)cdiv(p.items_p, 8);
  a.run_s = (int)cdiv(p.items_s, 8);
  a.by_qtiles_p = make_div(p.qtiles_p);
  a.by_qtiles_s = make_div(p.qtiles_s);
  a.by_splits_p = make_div(std::max(p.splits_p, 1));
  a.by_splits_s = make_div(p.splits_s);
  a.by_hkv = make_div(s.Hkv);
  a.by_w = make_div(a.w);
  a.by_per = make_div(a.per);
  a.joined = p.joined;
  a.o = (float*)workspace;
  a.ml = a.o + (p.splits_p + p.splits_s) * rows * s.D;
  return dtype == MINITP_F32 ? shared_by_d<float>(st, a, p, s.D) : shared_by_d<bf16>(st, a, p, s.D);
}

}  // namespace minitp
