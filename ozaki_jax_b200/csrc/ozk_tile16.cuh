// Building blocks shared by the 16-bit (BF16 / FP16) tile kernels of the
// low-rank adapter products and the checkpointed weight gradient: instruction
// and shared-memory descriptors for operands in either major order, MMAs that
// leave masked TMEM lanes alone, the per-tile adapter lists, tensor maps.
#pragma once

#include "ozk_device.cuh"
#include "ozk_internal.h"

#include <atomic>

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

// mbar_wait that acquires at cluster scope: what a peer CTA's threads wrote
// before their arrivals (mbar_arrive_cluster).
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity,
                                                  volatile int* abort, int32_t* status,
                                                  uint64_t budget_ns) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (i == 1) t0 = global_ns();
    if ((i & 63) == 0) {
      if (abort && *abort) return false;
      if (global_ns() - t0 > budget_ns) {
        if (abort) *abort = 1;
        raise_flag(status, OZK_FLAG_TIMEOUT);
        return false;
      }
    }
  }
}

// Ring of shared-memory stages: the index and phase parity of the current step.
struct Ring {
  int n;
  int s = 0;
  uint32_t ph = 0;
  __device__ explicit Ring(int stages) : n(stages) {}
  __device__ Ring(int stages, int step) : n(stages), s(step % stages), ph((step / stages) & 1) {}
  __device__ void next() {
    if (++s == n) {
      s = 0;
      ph ^= 1;
    }
  }
};

// Waits for the last copies of a ring that has run `steps` steps, so that its
// shared memory may be reused or released.
__device__ __forceinline__ void ring_drain(uint64_t* full, int stages, int steps, int32_t* status,
                                           uint64_t budget_ns) {
  const int first = steps > stages ? steps - stages : 0;
  Ring b(stages, first);
  for (int i = first; i < steps; ++i, b.next())
    mbar_wait(&full[b.s], b.ph, nullptr, status, budget_ns);
}

// Columns of the split T of rank r, high or low half: 32 up to rank 32, else
// ceil(r / 64) blocks of 64.
__host__ __device__ inline int split_half(int r) { return r <= 32 ? 32 : (r + 63) / 64 * 64; }

// Low parts that a product of their own multiplies are held 2^11 times as large
// in FP16, whose smallest number is 2^-24: the value is then held to 2^-36
// instead of 2^-25.  (What rounding to FP16 leaves of a value below 65520 is at most 16, so
// nothing overflows.)  BF16 has FP32's range.
__host__ __device__ constexpr float low_up(bool bf16) { return bf16 ? 1.0f : 2048.0f; }
__host__ __device__ constexpr float low_down(bool bf16) { return bf16 ? 1.0f : 1.0f / 2048.0f; }

// Two FP32 values as high and low 16-bit parts, packed; `up`: what the low
// parts are multiplied by, a power of two.
__device__ __forceinline__ void split16(bool bf16, float a, float b, float up, uint32_t& hi,
                                        uint32_t& lo) {
  hi = pack16(bf16, a, b);
  float ra = a - widen16(bf16, (uint16_t)hi), rb = b - widen16(bf16, (uint16_t)(hi >> 16));
  if (!(fabsf(ra) <= 3.0e38f)) ra = 0.0f;  // not finite: the high part says so by itself
  if (!(fabsf(rb) <= 3.0e38f)) rb = 0.0f;
  lo = pack16(bf16, ra * up, rb * up);
}

// Rounds t to its high and low 16-bit parts and stores them in the split T.
__device__ __forceinline__ void store_split(uint16_t* split, int64_t row, int half, int c, float t,
                                            bool bf16, float up) {
  uint32_t hi, lo;
  split16(bf16, t, 0.0f, up, hi, lo);
  split[row * 2 * half + c] = (uint16_t)hi;
  split[row * 2 * half + half + c] = (uint16_t)lo;
}

// ------------------------------------------------- int8 checkpoint codes

constexpr int kGroup = 128;      // columns of a row that share an exponent
constexpr int kExpNaN = -128;    // exponent of a group that held a NaN or infinity

// 2^e as a packed pair of 16-bit values (NaN for kExpNaN): exact for the
// exponents that checkpoint_rows writes for the type.
__device__ __forceinline__ uint32_t exp_pair(bool bf16, int e) {
  if (e == kExpNaN) return bf16 ? 0x7FC07FC0u : 0x7E007E00u;
  const float f = pow2f(e);
  return pack16(bf16, f, f);
}

// Four int8 codes times 2^e as two packed pairs, exactly.
// BF16 holds 128 + m exactly for m in [0, 127] (0x4300 | m), so with the code
// q = (q & 127) - 128 [q < 0]: q = (0x4300 | (q & 127)) - (0x4300 | (q & 128)),
// the second being 128 or 256.  FP16 holds 1024 + u for a byte u (0x6400 | u):
// q = (0x6400 | (q ^ 128)) - 1152.
__device__ __forceinline__ void codes_to_16(bool bf16, uint32_t q4, uint32_t scale, uint32_t& lo,
                                            uint32_t& hi) {
  if (bf16) {
    const uint32_t a = __byte_perm(q4, 0x43434343u, 0x4140);
    const uint32_t b = __byte_perm(q4, 0x43434343u, 0x4342);
    const uint32_t a0 = a & 0xFF7FFF7Fu, a1 = a & 0xFF80FF80u;
    const uint32_t b0 = b & 0xFF7FFF7Fu, b1 = b & 0xFF80FF80u;
    const __nv_bfloat162 s = *(const __nv_bfloat162*)&scale;
    const __nv_bfloat162 x =
        __hmul2(__hsub2(*(const __nv_bfloat162*)&a0, *(const __nv_bfloat162*)&a1), s);
    const __nv_bfloat162 y =
        __hmul2(__hsub2(*(const __nv_bfloat162*)&b0, *(const __nv_bfloat162*)&b1), s);
    lo = *(const uint32_t*)&x;
    hi = *(const uint32_t*)&y;
  } else {
    const uint32_t u = q4 ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t c = 0x64806480u;  // 1152
    const __half2 s = *(const __half2*)&scale;
    const __half2 x = __hmul2(__hsub2(*(const __half2*)&a, *(const __half2*)&c), s);
    const __half2 y = __hmul2(__hsub2(*(const __half2*)&b, *(const __half2*)&c), s);
    lo = *(const uint32_t*)&x;
    hi = *(const uint32_t*)&y;
  }
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

// 256 x 256 tiles on CTA pairs (ozk_wide16.cu).
enum WideMode {
  kWideForward = 0,  // A [M][C], B [N][C]: both operands' rows run along the contraction C
  kWideBack = 1,     // A [M][C], B [C][N]
  kWideWeight = 2    // A [C][M], B [C][N] as int8 codes and exponents
};
struct WideProduct {
  WideMode mode;
  bool bf16;
  int64_t M, N, C;
  const void* A;
  int64_t lda;
  const void* B;           // 16-bit elements, or int8 codes
  int64_t ldb;
  const int8_t* exps;      // kWideWeight: [ceil(N / 128)][C]
  // Further contraction: adapters' T B_i^T (kWideForward, kWideBack), r = 0: none.
  const int32_t* ids;
  int r, E;
  const uint16_t* split;   // [M][2 split_half(r)]
  const void* Bi;          // [E][N][r] (forward) or [E][r][N] (back)
  int64_t ldbi;
  bool early;              // launch while the kernel before it (which writes split) still runs
  void* out;               // [M][N], 16-bit of the operands' type or FP32
  int64_t ldo;
  bool out_f32, accumulate;
  float* partial;          // kWideWeight: room for wide_partial_bytes, or NULL
  int32_t* status;
};
int launch_wide(const WideProduct& p, int dev, cudaStream_t stream);
// Scratch of a kWideWeight product: FP32 partials when its contraction is split.
size_t wide_partial_bytes(int64_t M, int64_t N, int64_t C, int dev);

// Shared memory that a CTA of these kernels asks for at least when it holds
// `cols` TMEM columns: a little more than its share of the SM's 228 KB, less what
// a CTA has besides (544 columns' shares exceed the SM, 2 x 256's fit).  CTAs that
// fit an SM together then never want more than its 512 columns, so an allocation cannot
// block one CTA of a cluster while its peers wait for it.
inline size_t tmem_share(int cols) {
  int c = 32;
  while (c < cols) c *= 2;
  return (size_t)c * 432;
}

// Lets kernel K use `bytes` of dynamic shared memory on device dev.  The limit
// is an attribute of the kernel that a call sets, not raises: so it is set once,
// to all that the device gives a CTA besides K's static shared memory, and
// threads whose calls need different sizes cannot lower it under each other.
// (A launch's own size, not the limit, decides how many CTAs fit an SM.)
template <auto K>
int allow_smem(size_t bytes, int dev) {
  static std::atomic<int> allowed[64];
  if (dev < 0 || dev >= 64) return set_error(OZK_ERR_ARG, "device %d", dev);
  int most = allowed[dev].load(std::memory_order_acquire);
  if (!most) {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, K);
    if (e == cudaSuccess)
      e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e == cudaSuccess) {
      most -= (int)a.sharedSizeBytes;
      e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    }
    if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute", e);
    allowed[dev].store(most, std::memory_order_release);
  }
  if (bytes > (size_t)most)
    return set_error(OZK_ERR_UNSUPPORTED, "%zu bytes of shared memory needed, %d there", bytes, most);
  return OZK_OK;
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
