// What the attention kernels of tiles in LDS share: index arithmetic, lane
// exchanges, loads that go straight to LDS and transposed reads of them.
#pragma once

#include "common.h"

namespace minitp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Division by a number the host knows: n / d for 0 <= n < 2^31 as one product
// (m = ceil(2^(31 + l) / d) with 2^l >= d: n (m d - 2^(31 + l)) < 2^(31 + l)). The
// index arithmetic in front of a block's first load is all latency: with the
// compiler's divisions, most of them in 64 bits, a 5.6 us call took 6.2.
struct Div {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

inline Div make_div(int64_t d) {
  int l = 0;
  while ((1LL << l) < d) ++l;
  return Div{(uint32_t)(((1ull << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d), 31 + l};
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

// ---- bf16 tiles of 64 K or V rows, as they lie in memory ---------------------
constexpr int H_KT = 64;

template <int D>
struct Half {
  static constexpr int ROWB = D * 2, CH = D / 8;
  static constexpr int OPER = H_KT * ROWB, STAGE = 2 * OPER, LDS = 2 * STAGE;
  // 1 KiB loads of a tile: PPW of K and of V a wave (D = 16: one of either)
  static constexpr int PIECE_ROWS = 64 / CH, PIECES = H_KT / PIECE_ROWS, PPW = PIECES / 4;
  static_assert(PPW >= 1 || PIECES == 2, "each wave loads alike, or waves 0, 1 K and waves 2, 3 V");
  // chunk c of row r lies at chunk c ^ swz(r)
  __device__ static int k_swz(int r) { return r * ROWB / 256 % CH; }
  __device__ static int v_swz(int r) { return r * ROWB / 256 % 4 * 4 % CH; }
};

// 16 bytes a lane from the resource at voff to LDS at lds_addr + 16 lane
// (m0, wave-uniform; zeros past the resource's end). asm, so that the compiler
// does not wait for these loads at every LDS read: stage_wait does. It also
// keeps the compiler from adding the wait states that the hardware asks for:
// one between the write of m0 and a load to LDS (the s_nop 0), and five between
// a vector instruction's write of a scalar register (v_readfirstlane) and a
// load that reads it, which rows_rsrc leaves.
__device__ __forceinline__ void row_dma16(u32x4 r, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(lds_addr) : "memory");
}
__device__ __forceinline__ u32x4 rows_rsrc(const void* base, int bytes) {
  const uint64_t p = (uint64_t)base;
  u32x4 r;
  r.x = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p);
  r.y = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  r.z = (uint32_t)__builtin_amdgcn_readfirstlane(bytes);
  r.w = 0x00020000u;
  asm volatile("s_nop 4" : "+s"(r));
  return r;
}
// this wave's loads have landed and its LDS reads are done; then the block's
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The queries are waited for here. Without it the compiler would wait for them
// at their first use in the tile loop, every time round, and so for the next
// tile's loads, which are counted with them.
template <int N>
__device__ __forceinline__ void arrived(bf16x8 (&q)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int k = 0; k < N; k += 4) asm volatile("" : "+v"(q[k]), "+v"(q[k + 1]), "+v"(q[k + 2]), "+v"(q[k + 3]));
  } else if constexpr (N == 2) {
    asm volatile("" : "+v"(q[0]), "+v"(q[1]));
  } else {
    asm volatile("" : "+v"(q[0]));
  }
}

__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
__device__ __forceinline__ bf16x8 join8(s16x4 lo, s16x4 hi) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The running maximum moves only when some lane's passes it by this much (base
// 2): until then probabilities stay below 2^8 and nothing is rescaled. (It is a
// score times log2(e), rounded: off by 2^-24 of its size, which scales all of a
// part's probabilities alike and goes out in the division. Scores of up to 2^29
// leave that within 2^32.)
constexpr float SLACK = 8.f;

}  // namespace minitp
