// Rows kept in 8 bits between the forward and the backward pass.
//
// Each row is cut into groups of 128 columns.  A group with largest magnitude
// m has the step 2^e, the smallest power of two for which m / 2^e rounds to at
// most 127 (floor(log2 m) - 6, one more when m / 2^e >= 127.5), and the codes
// q = RN(x / 2^e): |x - q 2^e| <= 2^e / 2 < m / 127.  The step is a power of
// two, as in the slice extraction, so every value q 2^e is exact in the type
// it came from (7 bits of BF16's 8 or FP16's 11) and a product with the codes
// is a product with the restored matrix.  e is held within the type's range
// (the smallest steps are FP16's and FP32's subnormal and normal limits), and
// at its upper end codes saturate at 127.  A group that holds a NaN or an
// infinity gets the exponent -128 and reads back as NaN.
//
// Layout: codes [M][round_up(K, 128)] (0 beyond K), exponents [groups][M], so
// that the weight gradient, which contracts over rows, finds the exponents of
// a column block's rows side by side.
//
// Both kernels are bound by HBM: one read and one write of each element.  A
// CTA takes 32 rows x 256 columns, a warp 4 rows, each lane 16 bytes of each
// (four loads in flight).  65536 x 4096 BF16: saved in 134 us (6.0 TB/s), restored
// in 121 us (6.6 TB/s); a plain copy of the matrix runs at 6.4 TB/s.  With the
// maxima and codes computed element by element in FP32 (17 instructions an
// element instead of 11) saving was bound by instructions: 220 us.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "ozk_tile16.cuh"

namespace ozk {

namespace {

constexpr int kTileRows = 32;
constexpr int kTileCols = 256;
constexpr int kWarpRows = 4;

template <int DT>
struct Elem {
  using type = uint16_t;
  static constexpr int VEC = 8;
  static constexpr int EMIN = DT == OZK_DT_F16 ? -24 : -126;
  static constexpr int EMAX = DT == OZK_DT_F16 ? 9 : 121;
};
template <>
struct Elem<OZK_DT_F32> {
  using type = float;
  static constexpr int VEC = 4;
  static constexpr int EMIN = -126;
  static constexpr int EMAX = 121;
};

// Larger of two packed pairs of non-negative 16-bit values, NaN if one is.
template <int DT>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == OZK_DT_BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Step exponent of a group whose largest magnitude has the FP32 bits `top`.
template <int DT>
__device__ __forceinline__ int group_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return kExpNaN;
  int e = (int)(top >> 23) - 127 - 6;
  if (e < Elem<DT>::EMIN) e = Elem<DT>::EMIN;
  if (__uint_as_float(top) * __uint_as_float((uint32_t)(127 - e) << 23) >= 127.5f) ++e;
  return e < Elem<DT>::EMAX ? e : Elem<DT>::EMAX;
}

template <int DT>
__global__ void __launch_bounds__(256)
    k_checkpoint_rows(const typename Elem<DT>::type* X, int64_t ldx, int64_t M, int64_t K,
                      int8_t* codes, int64_t ldc, int8_t* exps, int vec) {
  using E = Elem<DT>;
  constexpr int VEC = E::VEC;
  constexpr int HALVES = kTileCols / (32 * VEC);  // 16-byte pieces of a lane per row
  constexpr int LANES = kGroup / VEC;             // lanes of a group
  __shared__ int8_t s_exp[2][kTileRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.y * kTileRows;
  const int64_t col0 = (int64_t)blockIdx.x * kTileCols;
  uint32_t x[kWarpRows][HALVES][4];  // 16 bytes of elements
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int64_t row = row0 + warp * kWarpRows + j;
      const int64_t col = col0 + (h * 32 + lane) * VEC;
      uint4 q = make_uint4(0, 0, 0, 0);
      if (row < M && vec && col + VEC <= K) {
        q = __ldcs((const uint4*)(X + row * ldx + col));
      } else if (row < M) {
        typename E::type u[VEC] = {};
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (col + i < K) u[i] = X[row * ldx + col + i];
        memcpy(&q, u, 16);
      }
      x[j][h][0] = q.x, x[j][h][1] = q.y, x[j][h][2] = q.z, x[j][h][3] = q.w;
    }
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j)
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int r = warp * kWarpRows + j;
      const int64_t row = row0 + r;
      const int64_t col = col0 + (h * 32 + lane) * VEC;
      const uint32_t(&w)[4] = x[j][h];
      // Largest magnitude, NaN if there is one: 16-bit elements two to a word,
      // FP32 ones as the unsigned integers that they order like.
      uint32_t top;
      if constexpr (VEC == 8) {
        const uint32_t m = 0x7fff7fffu;
        top = max_pair<DT>(max_pair<DT>(w[0] & m, w[1] & m), max_pair<DT>(w[2] & m, w[3] & m));
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) top = max_pair<DT>(top, __shfl_xor_sync(~0u, top, o));
        const uint32_t hi = __float_as_uint(widen16(DT == OZK_DT_BF16, (uint16_t)(top >> 16)));
        const uint32_t lo = __float_as_uint(widen16(DT == OZK_DT_BF16, (uint16_t)top));
        top = max(hi, lo);
      } else {
        const uint32_t m = 0x7fffffffu;
        top = max(max(w[0] & m, w[1] & m), max(w[2] & m, w[3] & m));
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
      }
      const int e = group_exponent<DT>(top);
      const float inv = e == kExpNaN ? 0.0f : __uint_as_float((uint32_t)(127 - e) << 23);
      // x / 2^e is exact; the fused sum with 1.5 2^23 rounds it to the integer
      // whose two's complement is the low byte.
      auto element = [&](int i) {
        if constexpr (VEC == 8) return widen16(DT == OZK_DT_BF16, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
        else return __uint_as_float(w[i]);
      };
      auto low_bytes = [](float a, float b, float c, float d) {
        return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                           __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
      };
      constexpr float kRound = 12582912.0f;
      uint32_t q[VEC / 4];
#pragma unroll
      for (int i = 0; i < VEC; i += 4)
        q[i / 4] = low_bytes(__fmaf_rn(element(i), inv, kRound), __fmaf_rn(element(i + 1), inv, kRound),
                             __fmaf_rn(element(i + 2), inv, kRound), __fmaf_rn(element(i + 3), inv, kRound));
      // A step at the type's upper limit may be too small for the group: those
      // codes saturate.  (A branch of the warp's, so that no other group pays.)
      if (__any_sync(~0u, e == E::EMAX) && e == E::EMAX) {
        auto clamp = [&](float v) { return fminf(fmaxf(v * inv, -127.0f), 127.0f) + kRound; };
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
          q[i / 4] = low_bytes(clamp(element(i)), clamp(element(i + 1)), clamp(element(i + 2)),
                               clamp(element(i + 3)));
      }
      if (e == kExpNaN)
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) q[i] = 0;
      if (row < M && col < ldc) {
        int8_t* c = codes + row * ldc + col;
        if constexpr (VEC == 8) *(uint2*)c = make_uint2(q[0], q[1]);
        else *(uint32_t*)c = q[0];
      }
      if (lane % LANES == 0) s_exp[VEC == 8 ? lane / LANES : h][r] = (int8_t)e;
    }
  __syncthreads();
  if (threadIdx.x < 2 * kTileRows) {
    const int gr = threadIdx.x / kTileRows, r = threadIdx.x % kTileRows;
    const int64_t group = (int64_t)blockIdx.x * 2 + gr;
    if (group * kGroup < K && row0 + r < M) exps[group * M + row0 + r] = s_exp[gr][r];
  }
}

template <int DT>
__global__ void __launch_bounds__(256)
    k_restore_rows(const int8_t* codes, int64_t ldc, const int8_t* exps, int64_t M, int64_t K,
                   typename Elem<DT>::type* out, int64_t ldo, int vec) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.y * kTileRows + warp * kWarpRows;
  const int64_t col = (int64_t)blockIdx.x * kTileCols + lane * 8;
  if (col >= K) return;
  uint2 q[kWarpRows];
  int e[kWarpRows];
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j)
    if (row0 + j < M) {
      q[j] = __ldcs((const uint2*)(codes + (row0 + j) * ldc + col));
      e[j] = __ldg(exps + (col / kGroup) * M + row0 + j);
    }
#pragma unroll
  for (int j = 0; j < kWarpRows; ++j) {
    if (row0 + j >= M) break;
    typename Elem<DT>::type* o = out + (row0 + j) * ldo + col;
    if constexpr (DT == OZK_DT_F32) {
      const float s = e[j] == kExpNaN ? __uint_as_float(0x7fc00000u) : pow2f(e[j]);
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // 2^23 + u is exact in FP32 for the byte u = q + 128
        const uint32_t u = (i < 4 ? q[j].x : q[j].y) ^ 0x80808080u;
        f[i] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + (i & 3))) - 8388736.0f) * s;
      }
      if (vec && col + 8 <= K) {
        __stcs((float4*)o, make_float4(f[0], f[1], f[2], f[3]));
        __stcs((float4*)(o + 4), make_float4(f[4], f[5], f[6], f[7]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < K) o[i] = f[i];
      }
    } else {
      constexpr bool bf16 = DT == OZK_DT_BF16;
      const uint32_t s = exp_pair(bf16, e[j]);
      uint32_t w[4];
      codes_to_16(bf16, q[j].x, s, w[0], w[1]);
      codes_to_16(bf16, q[j].y, s, w[2], w[3]);
      if (vec && col + 8 <= K) {
        __stcs((uint4*)o, make_uint4(w[0], w[1], w[2], w[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < K) o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
}

__global__ void k_zero(uint8_t* out, int64_t pitch, int64_t width, int64_t rows) {
  const int64_t n = rows * width;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    out[i / width * pitch + i % width] = 0;
}

int saved_args(const void* codes, int64_t ldc, const void* exps, int64_t M, int64_t K) {
  if (M < 0 || K < 1) return set_error(OZK_ERR_ARG, "need M >= 0 and K >= 1");
  if (M > ((int64_t)1 << 30) || K > ((int64_t)1 << 30))
    return set_error(OZK_ERR_UNSUPPORTED, "M and K are limited to 2^30");
  if (ldc != round_up(K, kGroup))
    return set_error(OZK_ERR_ARG, "ldc must be K rounded up to %d", kGroup);
  if (M && (!codes || !exps)) return set_error(OZK_ERR_ARG, "NULL pointer");
  if ((uintptr_t)codes & 15) return set_error(OZK_ERR_ARG, "codes not 16-byte aligned");
  return OZK_OK;
}

}  // namespace

}  // namespace ozk

using namespace ozk;

extern "C" {

int ozk_checkpoint_rows(const void* X, int64_t ldx, int64_t M, int64_t K, int dt, void* codes,
                        int64_t ldc, void* exps, void* stream) {
  if (dt != OZK_DT_F32 && !dt_is_16bit(dt)) return set_error(OZK_ERR_ARG, "unknown dtype %d", dt);
  int rc = saved_args(codes, ldc, exps, M, K);
  if (rc || M == 0) return rc;
  if (!X || ldx < K) return set_error(OZK_ERR_ARG, "NULL X or ldx < K");
  const int64_t tiles = (M + kTileRows - 1) / kTileRows, cols = (K + kTileCols - 1) / kTileCols;
  const int size = dt == OZK_DT_F32 ? 4 : 2;
  const int vec = ((uintptr_t)X & 15) == 0 && ldx * size % 16 == 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (tiles > 65535) return set_error(OZK_ERR_UNSUPPORTED, "more than %d rows", 65535 * kTileRows);
  const dim3 grid((unsigned)cols, (unsigned)tiles);
  int8_t *c = (int8_t*)codes, *x = (int8_t*)exps;
  if (dt == OZK_DT_BF16)
    k_checkpoint_rows<OZK_DT_BF16><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, M, K, c, ldc, x, vec);
  else if (dt == OZK_DT_F16)
    k_checkpoint_rows<OZK_DT_F16><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, M, K, c, ldc, x, vec);
  else
    k_checkpoint_rows<OZK_DT_F32><<<grid, 256, 0, s>>>((const float*)X, ldx, M, K, c, ldc, x, vec);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_checkpoint_rows launch", e);
}

int ozk_restore_rows(const void* codes, int64_t ldc, const void* exps, int64_t M, int64_t K,
                     void* out, int64_t ldo, int dt, void* stream) {
  if (dt != OZK_DT_F32 && !dt_is_16bit(dt)) return set_error(OZK_ERR_ARG, "unknown dtype %d", dt);
  int rc = saved_args(codes, ldc, exps, M, K);
  if (rc || M == 0) return rc;
  if (!out || ldo < K) return set_error(OZK_ERR_ARG, "NULL out or ldo < K");
  const int64_t tiles = (M + kTileRows - 1) / kTileRows, cols = (K + kTileCols - 1) / kTileCols;
  if (tiles > 65535) return set_error(OZK_ERR_UNSUPPORTED, "more than %d rows", 65535 * kTileRows);
  const int size = dt == OZK_DT_F32 ? 4 : 2;
  const int vec = ((uintptr_t)out & 15) == 0 && ldo * size % 16 == 0;
  const dim3 grid((unsigned)cols, (unsigned)tiles);
  cudaStream_t s = (cudaStream_t)stream;
  const int8_t *c = (const int8_t*)codes, *x = (const int8_t*)exps;
  if (dt == OZK_DT_BF16)
    k_restore_rows<OZK_DT_BF16><<<grid, 256, 0, s>>>(c, ldc, x, M, K, (uint16_t*)out, ldo, vec);
  else if (dt == OZK_DT_F16)
    k_restore_rows<OZK_DT_F16><<<grid, 256, 0, s>>>(c, ldc, x, M, K, (uint16_t*)out, ldo, vec);
  else
    k_restore_rows<OZK_DT_F32><<<grid, 256, 0, s>>>(c, ldc, x, M, K, (float*)out, ldo, vec);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_restore_rows launch", e);
}

size_t ozk_checkpoint_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int aligned) {
  if (M < 1 || N < 1 || K < 1) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  Arena ws(nullptr);
  if (!aligned) ws.take((size_t)M * round_up(N, 8) * 2);  // room for dY's copy
  ws.take(wide_partial_bytes(N, K, M, dev));
  return ws.used;
}

int ozk_checkpoint_grad(const void* dY, int64_t ldy, const void* codes, int64_t ldc,
                        const void* exps, void* out, int64_t ldo, int64_t M, int64_t N, int64_t K,
                        int dt, int out_dt, int accumulate, void* workspace, size_t ws_bytes,
                        int32_t* status_dev, void* stream) {
  if (!dt_is_16bit(dt)) return set_error(OZK_ERR_ARG, "dtype must be OZK_DT_BF16 or OZK_DT_F16");
  if (out_dt != dt && out_dt != OZK_DT_F32)
    return set_error(OZK_ERR_ARG, "the output is of the operands' type or OZK_DT_F32");
  int rc = saved_args(codes, ldc, exps, M, K);
  if (rc) return rc;
  if (N < 0 || N > ((int64_t)1 << 30)) return set_error(OZK_ERR_ARG, "N must be 0 to 2^30");
  if (N == 0) return OZK_OK;
  if (!out || ldo < K) return set_error(OZK_ERR_ARG, "NULL out or ldo < K");
  cudaStream_t s = (cudaStream_t)stream;
  const int size = out_dt == OZK_DT_F32 ? 4 : 2;
  if (M == 0) {
    if (accumulate) return OZK_OK;
    k_zero<<<148, 256, 0, s>>>((uint8_t*)out, ldo * size, K * size, N);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? OZK_OK : set_cuda_error("k_zero launch", e);
  }
  if (!dY || ldy < N) return set_error(OZK_ERR_ARG, "NULL dY or ldy < N");
  int dev = 0;
  cudaGetDevice(&dev);
  const bool ready = tma_ready(dY, ldy);
  Arena ws(workspace);
  void* copy = ready ? nullptr : ws.take<void>((size_t)M * round_up(N, 8) * 2);
  const size_t pb = wide_partial_bytes(N, K, M, dev);
  float* partial = pb ? ws.take<float>(pb) : nullptr;
  if (ws.used && (!workspace || ws.used > ws_bytes || ((uintptr_t)workspace & 127)))
    return set_error(OZK_ERR_WORKSPACE, "workspace of %zu bytes, aligned to 128, needed", ws.used);
  WideProduct p = {};
  p.mode = kWideWeight;
  p.bf16 = dt == OZK_DT_BF16;
  p.M = N;
  p.N = K;
  p.C = M;
  p.A = dY;
  p.lda = ldy;
  if (!ready) {
    if ((rc = launch_pad_rows(dY, ldy, copy, round_up(N, 8), M, N, s))) return rc;
    p.A = copy;
    p.lda = round_up(N, 8);
  }
  p.B = codes;
  p.ldb = ldc;
  p.exps = (const int8_t*)exps;
  p.out = out;
  p.ldo = ldo;
  p.out_f32 = out_dt == OZK_DT_F32;
  p.accumulate = accumulate != 0;
  p.partial = partial;
  p.status = status_dev;
  return launch_wide(p, dev, s);
}

}  // extern "C"
