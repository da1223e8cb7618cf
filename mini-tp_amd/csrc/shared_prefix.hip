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

// ---------------------------------------------------------------------------
// bf16, head dims 32, 64 and 128. A block takes 128 query rows of a unit over
// the keys of its split, four waves of 32 rows (v_mfma_f32_32x32x16_bf16), or,
// where the unit has at most 16 rows (one token of a row's own part), those
// rows over 64 keys at a time, 16 keys a wave (16x16 MFMAs).
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
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int H_QT = 128, H_KT = 64, H_SMALL = 16;

template <int D>
struct Half {
  static constexpr int ROWB = D * 2, CH = D / 8;
  static constexpr int OPER = H_KT * ROWB, STAGE = 2 * OPER, LDS = 2 * STAGE;
  static constexpr int PIECE_ROWS = 64 / CH, PIECES = H_KT / PIECE_ROWS, PPW = PIECES / 4;  // 1 KiB loads
  // chunk c of row r lies at chunk c ^ swz(r)
  __device__ static int k_swz(int r) { return r * ROWB / 256 % CH; }
  __device__ static int v_swz(int r) { return r * ROWB / 256 % 4 * 4 % CH; }
};

// 16 bytes a lane from the resource at voff to LDS at lds_addr + 16 lane
// (m0, wave-uniform; zeros past the resource's end). asm, so that the compiler
// does not wait for these loads at every LDS read: stage_wait does. The s_nop
// is the wait state between the write of m0 and a load to LDS.
__device__ __forceinline__ void row_dma16(u32x4 r, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(lds_addr) : "memory");
}
__device__ __forceinline__ u32x4 rows_rsrc(const void* base, int64_t key, int64_t key_hi, int row_bytes) {
  const uint64_t p = (uint64_t)base + key * row_bytes;
  u32x4 r;
  r.x = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p);
  r.y = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  r.z = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)std::min<int64_t>(key_hi - key, H_KT) * row_bytes);
  r.w = 0x00020000u;
  return r;
}
// this wave's loads have landed and its LDS reads are done; then the block's
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
__device__ __forceinline__ bf16x8 join8(s16x4 lo, s16x4 hi) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// maximum / sum over lanes l and l ^ 32 (and, for the 16-lane form, l ^ 16)
__device__ __forceinline__ float halves_max(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float quads_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float quads_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halves_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// Tiles of an item through the two stages; compute(k0, stage) for each.
template <int D, typename F>
__device__ __forceinline__ void over_tiles(const Item& it, char* lds, F&& compute) {
  using H = Half<D>;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // piece w + 4 j of a tile: rows 4 PIECE_ROWS j + row; the swizzles do not depend on j
  const int row = H::PIECE_ROWS * w + lane / H::CH;
  const uint32_t koff = row * H::ROWB + ((lane % H::CH) ^ H::k_swz(row)) * 16;
  const uint32_t voff = row * H::ROWB + ((lane % H::CH) ^ H::v_swz(row)) * 16;
  auto issue = [&](int64_t k0, int st) {
    const u32x4 kr = rows_rsrc(it.k, k0, it.key_hi, H::ROWB), vr = rows_rsrc(it.v, k0, it.key_hi, H::ROWB);
    const uint32_t to = lds0 + st * H::STAGE + w * 1024;
#pragma unroll
    for (int j = 0; j < H::PPW; ++j) row_dma16(kr, koff + j * 4096, to + j * 4096);
#pragma unroll
    for (int j = 0; j < H::PPW; ++j) row_dma16(vr, voff + j * 4096, to + H::OPER + j * 4096);
  };
  if (it.key_lo < it.key_hi) issue(it.key_lo, 0);
  int st = 0;
  for (int64_t k0 = it.key_lo; k0 < it.key_hi; k0 += H_KT, st ^= 1) {
    stage_wait();
    if (k0 + H_KT < it.key_hi) issue(k0 + H_KT, st ^ 1);  // (its readers passed the barrier)
    compute(k0, lds + st * H::STAGE);
  }
}

// The running maximum moves only when some lane's passes it by this much (base
// 2): until then probabilities stay below 2^8 and nothing is rescaled.
constexpr float SLACK = 8.f;

template <int D>
__device__ __forceinline__ void shared_rows128(const SharedArgs& a, const Item& it, char* lds) {
  using H = Half<D>;
  constexpr int KS = D / 16, DB = D / 32;
  const int per = a.Hq / a.Hkv;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int r0 = it.tile * H_QT + w * 32, r = r0 + n32;
  const bool live = r < it.rows;
  const int64_t n = it.n0 + (live ? r : 0) / per;
  const int head = it.kv * per + (live ? r : 0) % per;
  const int64_t seen = it.own ? it.seen + (n - it.n0) : INT64_MAX;  // the last key this query sees
  const int64_t seen_first = it.own ? it.seen + r0 / per : INT64_MAX, seen_last = it.own ? it.seen + (r0 + 31) / per : INT64_MAX;

  bf16x8 qb[KS];
  {
    const bf16* q = (const bf16*)a.q + (n * a.Hq + head) * D + 8 * h;
#pragma unroll
    for (int k = 0; k < KS; ++k) qb[k] = __builtin_bit_cast(bf16x8, *(const uint4*)(q + 16 * k));
  }
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
  const int vx = ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ H::v_swz(vrow)) << 4;

  over_tiles<D>(it, lds, [&](int64_t k0, const char* st) {
    if (r0 >= it.rows || k0 > seen_last) return;
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(st + kat + kb * 32 * H::ROWB + ((32 * k) ^ kx)));
        s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb[k], s[kb], 0, 0, 0);
      }
    }
    bool odd = false;
    const int limit = (int)std::min<int64_t>(std::min<int64_t>(seen, it.key_hi - 1) - k0, H_KT);
    if (k0 + H_KT - 1 > std::min<int64_t>(seen_first, it.key_hi - 1)) {
      // some query does not see some key: lane (query, h) holds keys
      // 32 kb + 8 (i / 4) + 4 h + i % 4
      __asm__ volatile("");  // (a branch, not selects on every tile)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * kb + 8 * (i / 4) + i % 4 > limit - 4 * h) s[kb][i] = -__builtin_inff();
      if (seen_first < it.key_hi - 1) {
        // hidden keys that other queries see: are their values finite?
        for (int c = lane; c < H_KT * H::CH; c += 64) {
          const uint4 x = *(const uint4*)(st + H::OPER + c * 16);
          const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            odd |= (wd[e] & 0x7f80u) == 0x7f80u || (wd[e] & 0x7f800000u) == 0x7f800000u;
        }
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
    if (odd) {
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
          for (int c = 0; c < 4; ++c) {
            const uint2 x = *(const uint2*)(st + H::OPER + key * H::ROWB + (((4 * d + c) ^ H::v_swz(key)) << 4) + 8 * h);
            const float v[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u),
                                __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u)};
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][4 * c + e] = key <= limit ? fmaf(p, v[e], o[d][4 * c + e]) : o[d][4 * c + e];
          }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // keys 16 j .. 16 j + 15
      const f32x16& p = s[j / 2];
      const int b = 8 * (j % 2);
      const bf16x8 pb = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(p[b], p[b + 1]), pack_bf16x2(p[b + 2], p[b + 3]),
                                                              pack_bf16x2(p[b + 4], p[b + 5]), pack_bf16x2(p[b + 6], p[b + 7])));
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const char* vp = st + vat + 16 * j * H::ROWB + ((64 * d) ^ vx);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join8(read_tr(vp), read_tr(vp + 8 * H::ROWB)), pb, o[d], 0, 0, 0);
      }
    }
  });
  if (!live) return;
  const float l = halves_sum(lsum);
  const int64_t at = (int64_t)it.slot * a.B * a.T * a.Hq + n * a.Hq + head;
  if (h == 0) *(float2*)(a.ml + at * 2) = make_float2(m, l);
  float* orow = a.o + at * D + 4 * h;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *(float4*)(orow + 32 * d + 8 * c) = make_float4(o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]);
}

template <int D>
__device__ __forceinline__ void shared_rows16(const SharedArgs& a, const Item& it, char* lds) {
  using H = Half<D>;
  constexpr int KS = D / 32, DB = D / 16;
  const int per = a.Hq / a.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, q4 = lane >> 4;
  const int r = n16;  // (one tile)
  const bool live = r < it.rows;
  const int64_t n = it.n0 + (live ? r : 0) / per;
  const int head = it.kv * per + (live ? r : 0) % per;
  const int64_t seen = it.own ? it.seen + (n - it.n0) : INT64_MAX;

  bf16x8 qb[KS];
  {
    const bf16* q = (const bf16*)a.q + (n * a.Hq + head) * D + 8 * q4;
#pragma unroll
    for (int k = 0; k < KS; ++k) qb[k] = __builtin_bit_cast(bf16x8, *(const uint4*)(q + 32 * k));
  }
  f32x4 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), lsum = 0.f;
  const float sl2 = a.scale * 1.4426950408889634f;

  // K row 16 w + n16, chunk 4 k + q4; V rows 16 w + 4 q4 + n16 / 4, dims 16 d + 4 (lane % 4)
  const int krow = 16 * w + n16, kat = krow * H::ROWB, kx = (q4 ^ H::k_swz(krow)) << 4;
  const int vrow = 16 * w + 4 * q4 + n16 / 4;
  const int vat = H::OPER + vrow * H::ROWB + 8 * (lane & 1), vx = (((lane >> 1) & 1) ^ H::v_swz(vrow)) << 4;

  over_tiles<D>(it, lds, [&](int64_t k0, const char* st) {
    const int64_t kw = k0 + 16 * w;
    if (kw >= it.key_hi) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(st + kat + ((64 * k) ^ kx)));
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qb[k], s, 0, 0, 0);
    }
    const int limit = (int)std::min<int64_t>(std::min<int64_t>(seen, it.key_hi - 1) - kw, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * q4 + i > limit) s[i] = -__builtin_inff();
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
    if (__builtin_amdgcn_ballot_w64(limit < std::min<int64_t>(it.key_hi - 1 - kw, 15))) {
      bool odd = false;
      for (int c = lane; c < 16 * H::CH; c += 64) {
        const uint4 x = *(const uint4*)(st + H::OPER + 16 * w * H::ROWB + c * 16);
        const uint32_t wd[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (wd[e] & 0x7f80u) == 0x7f80u || (wd[e] & 0x7f800000u) == 0x7f800000u;
      }
      if (__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
          const float pi = (key & 3) == 0 ? s[0] : (key & 3) == 1 ? s[1] : (key & 3) == 2 ? s[2] : s[3];
          const float p = __shfl(pi, n16 + 16 * (key >> 2), 64);
          const int row = 16 * w + key;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const uint2 x = *(const uint2*)(st + H::OPER + row * H::ROWB + (((2 * d + (q4 >> 1)) ^ H::v_swz(row)) << 4) +
                                            8 * (q4 & 1));
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

  // ---- the four waves' keys joined through LDS ------------------------------
  const float l = quads_sum(lsum);
  float* po = (float*)lds;             // [wave][16][D]
  float* pml = po + 4 * H_SMALL * D;   // [wave][16][2]
  __syncthreads();                     // (every stage is free)
  if (live) {
#pragma unroll
    for (int d = 0; d < DB; ++d) *(f32x4*)(po + (w * H_SMALL + r) * D + 16 * d + 4 * q4) = o[d];
    if (q4 == 0) *(float2*)(pml + (w * H_SMALL + r) * 2) = make_float2(m, l);
  }
  __syncthreads();
  constexpr int LPR = D / 4;
  for (int i = tid; i < it.rows * LPR; i += 256) {
    const int row = i / LPR, d = i % LPR * 4;
    float2 ml[4];
    float mx = -__builtin_inff(), ls = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ml[j] = *(const float2*)(pml + (j * H_SMALL + row) * 2);
      mx = fmaxf(mx, ml[j].x);
    }
    f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float sc = ml[j].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[j].x - mx);
      ls = fmaf(sc, ml[j].y, ls);
      const f32x4 oj = *(const f32x4*)(po + (j * H_SMALL + row) * D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) os[e] = fmaf(sc, oj[e], os[e]);
    }
    const int64_t nn = it.n0 + row / per;
    const int64_t at = (int64_t)it.slot * a.B * a.T * a.Hq + nn * a.Hq + it.kv * per + row % per;
    *(f32x4*)(a.o + at * D + d) = os;
    if (d == 0) *(float2*)(a.ml + at * 2) = make_float2(mx, ls);
  }
}

template <int D>
__global__ __launch_bounds__(256, 2) void shared_attn_bf16_kernel(SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  static_assert(Half<D>::LDS >= 4 * H_SMALL * (D + 2) * 4, "the waves' join fits the stages");
  const Item it = shared_item<H_QT, H_KT>(a, D * 2);
  if (it.rows <= H_SMALL)
    shared_rows16<D>(a, it, lds);
  else
    shared_rows128<D>(a, it, lds);
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
  constexpr int NB = 8;  // slots whose loads are in flight together
  for (int s0 = 0; s0 < slots; s0 += NB) {
    float2 ml[NB];
    f32x4 os[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int64_t at = std::min(s0 + u, slots - 1) * rows + i;  // (past the last: read again, left out)
      ml[u] = *(const float2*)(a.ml + at * 2);
      os[u] = *(const f32x4*)(a.o + at * D + d);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (s0 + u >= slots) ml[u].x = -__builtin_inff();
      mn = fmaxf(mn, ml[u].x);
    }
    if (mn == -__builtin_inff()) continue;  // no split so far saw a key
    const float a0 = __builtin_amdgcn_exp2f(m - mn);
    l *= a0;
    o *= a0;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (ml[u].x == -__builtin_inff()) continue;
      const float a1 = __builtin_amdgcn_exp2f(ml[u].x - mn);
      l = fmaf(ml[u].y, a1, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(os[u][e], a1, o[e]);
    }
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

bool bf16_tiles(int dtype, int64_t D) { return dtype == MINITP_BF16 && D >= 32; }

Plan plan_of(int dtype, int64_t D, int64_t B, int64_t G, int64_t T, int64_t Hq, int64_t Hkv, int64_t P, int64_t C) {
  if (bf16_tiles(dtype, D)) return shared_plan(B, G, T, Hq, Hkv, P, C, H_QT, H_KT);
  return shared_plan(B, G, T, Hq, Hkv, P, C, F_QT, D >= 128 ? 32 : 64);
}

template <typename T, int D>
int shared_launch(hipStream_t st, const SharedArgs& a, const Plan& p) {
  const dim3 grid((unsigned)(p.items_p + p.items_s));
  if constexpr (sizeof(T) == 2 && D >= 32) {
    const int rc = ensure_lds_limit((const void*)shared_attn_bf16_kernel<D>, Half<D>::LDS);
    if (rc) return rc;
    hipLaunchKernelGGL(shared_attn_bf16_kernel<D>, grid, dim3(256), Half<D>::LDS, st, a);
  } else {
    hipLaunchKernelGGL((shared_attn_f32_kernel<T, D>), grid, dim3(256), 0, st, a);
  }
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
