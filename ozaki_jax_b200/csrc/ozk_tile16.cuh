// Building blocks shared by the 16-bit (BF16 / FP16) tile kernels of the
// low-rank adapter products and the checkpointed weight gradient: instruction
// and shared-memory descriptors for operands in either major order, MMAs that
// leave masked TMEM lanes alone, the per-tile adapter lists, tensor maps.
#pragma once

#include "ozk_device.cuh"
#include "ozk_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ozk {

// Element types of the 16-bit kernels (OZK_DT_*).
__host__ __device__ constexpr bool dt_is_16bit(int dt) { return dt == OZK_DT_BF16 || dt == OZK_DT_F16; }

// Instruction descriptor, kind::f16, FP32 accumulator: bf16 selects BF16 or
// FP16 operands, amn / bmn a row-contiguous (MN-major) A / B tile.
__host__ __device__ constexpr uint32_t umma_idesc_16(bool bf16, int M, int N, bool amn, bool bmn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((amn ? 1u : 0u) << 15) |
         ((bmn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Descriptor of an MN-major tile with 128-byte swizzle: blocks of 64 elements
// (128 B) along M or N, `lbo` bytes apart; inside a block each contraction
// index is a 128-byte row, 8 of them an atom of 1024 B.
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t saddr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// D (+)= A B^T where the lanes whose bit is set in m0..m3 (lanes 0-31, ...)
// keep their accumulators.
__device__ __forceinline__ void umma_16_masked(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                               uint32_t acc, uint32_t m0, uint32_t m1, uint32_t m2,
                                               uint32_t m3) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(m0), "r"(m1), "r"(m2), "r"(m3)
      : "memory");
}
// The same over a CTA pair: m[0..3] are the even CTA's lanes, m[4..7] the odd one's.
__device__ __forceinline__ void umma_16_masked_pair(uint32_t d, uint64_t a, uint64_t b,
                                                    uint32_t idesc, uint32_t acc,
                                                    const uint32_t (&m)[8]) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, "
      "{%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3]), "r"(m[4]),
      "r"(m[5]), "r"(m[6]), "r"(m[7])
      : "memory");
}

// A grid launched with programmatic serialisation waits here for the grid
// before it; that grid lets it start early with grid_release().
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Two FP32 values as a packed pair of 16-bit ones, rounded to nearest even
// (the low half holds `a`).
__device__ __forceinline__ uint32_t pack16(bool bf16, float a, float b) {
  uint32_t r;
  if (bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint16_t round16(bool bf16, float a) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(a)) : __half_as_ushort(__float2half_rn(a));
}
__device__ __forceinline__ float widen16(bool bf16, uint16_t u) {
  return bf16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

// ------------------------------------------------- adapters of a row tile

// Adapter of row `row`: -1 for none (an id outside [0, E)).  Without ids every
// row belongs to adapter 0.
__device__ __forceinline__ int row_adapter(const int32_t* ids, int64_t row, int64_t M, int E) {
  if (row >= M) return -1;
  const int v = ids ? ids[row] : 0;
  return v >= 0 && v < E ? v : -1;
}

// The distinct adapters of a tile of 32 NW rows, in order of their first row,
// each with the mask of the lanes that do NOT belong to it.
template <int NW>
struct SlotList {
  int n;
  int id[32 * NW];
  uint32_t off[32 * NW][NW];
};

// Built by one warp.
template <int NW>
__device__ __forceinline__ void build_slots(const int32_t* ids, int64_t row0, int64_t M, int E,
                                            SlotList<NW>* out, int lane) {
  int v[NW];
  uint32_t todo[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) v[w] = row_adapter(ids, row0 + 32 * w + lane, M, E);
#pragma unroll
  for (int w = 0; w < NW; ++w) todo[w] = __ballot_sync(~0u, v[w] >= 0);
  int n = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    while (todo[w]) {
      const int id = __shfl_sync(~0u, v[w], __ffs(todo[w]) - 1);
#pragma unroll
      for (int u = 0; u < NW; ++u) {
        const uint32_t m = __ballot_sync(~0u, v[u] == id);
        todo[u] &= ~m;
        if (lane == 0) out->off[n][u] = ~m;
      }
      if (lane == 0) out->id[n] = id;
      ++n;
    }
  }
  if (lane == 0) out->n = n;
}

// ------------------------------------------------- host side

// Tensor map of a [d2][d1][d0] array of elements of `esz` bytes (2, or 1 for
// codes), row stride s1 and plane stride s2 in bytes, box b0 x b1, 128-byte
// swizzle when swz.  Elements outside the array read as 0.
int make_map(CUtensorMap* map, const void* base, int esz, int64_t d0, int64_t d1, int64_t d2,
             int64_t s1, int64_t s2, int b0, int b1, bool swz);

// Whether a row-major operand can be read by TMA as it is: 16-byte base and row stride.
inline bool tma_ready(const void* p, int64_t ld) {
  return ((uintptr_t)p & 15) == 0 && (ld * 2) % 16 == 0;
}

// Shared memory that a CTA of these kernels asks for at least when it holds
// `cols` TMEM columns: its share of the SM's 227 KB.  CTAs that fit an SM
// together then never want more than its 512 columns, so an allocation cannot
// block one CTA of a cluster while its peers wait for it.
inline size_t tmem_share(int cols) {
  int c = 32;
  while (c < cols) c *= 2;
  return (size_t)c * 456;
}

// Carves aligned areas out of a caller's workspace (or, with base NULL, only counts them).
struct Arena {
  char* base;
  size_t used = 0;
  explicit Arena(void* b) : base((char*)b) {}
  template <typename T = void>
  T* take(size_t bytes) {
    char* p = base ? base + used : nullptr;
    used += (bytes + 1023) & ~(size_t)1023;
    return (T*)p;
  }
};

// Copies `rows` rows of `cols` 16-bit elements to rows of `ldd` elements, the rest of a row 0.
int launch_pad_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows,
                    int64_t cols, cudaStream_t stream);

}  // namespace ozk
