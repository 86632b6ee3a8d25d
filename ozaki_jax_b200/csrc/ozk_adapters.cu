// Low-rank adapters of many requests beside a shared projection:
//   T = s_i X A_i^T,  Y = X W^T + T B_i^T,  i = ids[row]
// and the gradient's first half, which is the same product read the other way:
//   U = s_i dY B_i,   dX = dY W + U A_i.
//
// Both run as two kernels, the second started while the first still runs:
//   k_low_rank / k_low_rank_rows   T (FP32) and its split T = hi + lo into two
//                                  16-bit values;
//   k_linear                       the shared product, with T's columns as
//                                  further columns of the contraction.
//
// The adapters of a tile's rows.  A tile of 128 rows may belong to many
// adapters.  A TMEM lane of an MMA with M = 128 is a row of the tile, and
// tcgen05.mma can leave lanes alone: so for each distinct adapter of the tile
// one MMA chain T B_i^T runs over the whole tile with the lanes of the other
// rows masked.  No row is moved, no zero is multiplied by another adapter's
// NaN, and any order of ids is right; contiguous requests cost one or two
// chains per tile.
//
// T between the kernels.  Rounded once to BF16, T would be up to 2^-8 of itself
// off; as hi + lo it is 2^-16 (BF16) or 2^-22 (FP16) off, at the price of r more
// columns of the contraction.  FP16 ends at 2^-24, so there T is also up to 2^-25
// off whatever its size: with |B| below 1 / sqrt(r) that is less than what Y's
// own rounding costs.  The sums over rows in dA get a split of U that keeps more
// (see low_up).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "ozk_adapters.h"
#include "ozk_tile16.cuh"

namespace ozk {

namespace {

constexpr int kRows = 128;       // rows of a tile (TMEM lanes)
constexpr int kKB = 64;          // contraction elements per stage: 128 bytes
constexpr int kMaxRank = 128;
constexpr int kMaxStages = 16;
constexpr int kThreads = 192;    // producer warp, MMA warp, four epilogue warps

struct LinearArgs {
  const int32_t* ids;
  void* Y;
  int64_t ldy;
  int64_t M;
  int N, nkb, E, r;
  int bf16, y_vec;
  int stages, xrows, tiles_n;
  int32_t* status;
  uint64_t budget_ns;
};

// Sum over the CTAs of the cluster (at most 8), in rank order, of the four FP32
// partials at shared-memory address `a` of each.  The loads are independent, so
// their round trips overlap.
__device__ __forceinline__ float4 cluster_sum4(uint32_t a, int splits) {
  float4 v[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (q < splits) {
      uint32_t ra;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(q));
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                   : "r"(ra)
                   : "memory");
    }
  }
  float4 s = v[0];
#pragma unroll
  for (int q = 1; q < 8; ++q)
    if (q < splits) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
  return s;
}

// ---------------------------------------------------------------- k_linear
//
// Few rows: bound by reading W once (one row of 4096 x 4096: the call takes 12 to
// 17 us in a graph, of which W's 33.5 MB need 5.1; 64 rows of 8192 x 4096 with 64
// adapters: 25 to 29 us, 12.9 by their bytes).  The tokens are the MMA's M side even
// then: 128 lanes of which few are used cost N / 2 clocks per 16 indexes, less
// than the 1.4 N that W's bytes take from memory.
// One CTA per 128 x BN tile, or a cluster of CTAs per tile that split the
// contraction (and the adapters) between them and add their FP32 partials in
// rank order through distributed shared memory: deterministic, no scratch.
// MNB: the shared operand's rows are contraction indexes (W of dX = dY W),
// read as MN-major tiles.
template <int BN, bool MNB>
__global__ void __launch_bounds__(kThreads)
    k_linear(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW,
             const __grid_constant__ CUtensorMap mapT, const __grid_constant__ CUtensorMap mapB,
             const __grid_constant__ LinearArgs g) {
  constexpr int B_BYTES = BN * 128;
  constexpr int TMEM_COLS = BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int a_bytes = g.xrows * 128;
  uint8_t* sA = smem;
  uint8_t* sB = smem + g.stages * a_bytes;
  __shared__ SlotList<4> slots;
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done, slots_ready;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_word;
  volatile int* s_abort = &s_abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t splits, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
  rank = cluster_ctarank();
  const int tile = blockIdx.x / splits;
  const int tm = tile / g.tiles_n, tn = tile - tm * g.tiles_n;
  const int64_t row0 = (int64_t)tm * kRows;
  const int col0 = tn * BN;
  const int kb0 = (int)((int64_t)g.nkb * rank / splits);
  const int kb1 = (int)((int64_t)g.nkb * (rank + 1) / splits);
  const int half = split_half(g.r);
  const int blocks = half < 64 ? 1 : half / 64 * 2;  // stages per adapter

  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&slots_ready, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&s_tmem, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_release();
  const uint32_t tmem = s_tmem;

  if (warp == 0) {
    if (lane == 0) {
      Ring rg(g.stages);
      bool ok = true;
      int issued = 0;
      const uint32_t bytes = (uint32_t)(a_bytes + B_BYTES);
      auto load = [&](const CUtensorMap* ma, int ax, const CUtensorMap* mb, int bx, int bz) {
        if (!mbar_wait(&empty[rg.s], rg.ph ^ 1, s_abort, g.status, g.budget_ns)) return false;
        mbar_arrive_expect_tx(&full[rg.s], bytes);
        tma_load_3d(sA + rg.s * a_bytes, ma, &full[rg.s], ax, (int)row0, 0);
        uint8_t* b = sB + rg.s * B_BYTES;
        if constexpr (MNB) {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j)
            tma_load_3d(b + j * 8192, mb, &full[rg.s], col0 + 64 * j, bx, bz);
        } else {
          tma_load_3d(b, mb, &full[rg.s], bx, col0, bz);
        }
        rg.next();
        ++issued;
        return true;
      };
      for (int kb = kb0; ok && kb < kb1; ++kb) ok = load(&mapX, kb * kKB, &mapW, kb * kKB, 0);
      // The split T comes from the kernel before this one.
      grid_wait();
      ok = ok && mbar_wait(&slots_ready, 0, s_abort, g.status, g.budget_ns);
      const int n = ok ? slots.n : 0;
      for (int j = rank; ok && j < n; j += splits)
        for (int b = 0; ok && b < blocks; ++b) {
          // hi and lo blocks of the same ranks in turn, against the same B_i
          const int ax = blocks == 1 ? 0 : (b & 1) * half + (b >> 1) * 64;
          ok = load(&mapT, ax, &mapB, blocks == 1 ? 0 : (b >> 1) * 64, slots.id[j]);
        }
      // Every copy lands before the shared memory is reused or released.
      ring_drain(full, g.stages, issued, g.status, g.budget_ns);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_16(g.bf16, kRows, BN, false, MNB);
      Ring rg(g.stages);
      bool ok = true;
      auto desc_b = [&](uint32_t b0, int kk) {
        return MNB ? umma_desc_mn128(b0 + kk * 2048, 8192) : umma_desc_sw128(b0 + kk * 32);
      };
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a0 = smem_u32(sA + rg.s * a_bytes), b0 = smem_u32(sB + rg.s * B_BYTES);
#pragma unroll
        for (int kk = 0; kk < kKB / 16; ++kk)
          umma_bf16(tmem, umma_desc_sw128(a0 + kk * 32), desc_b(b0, kk), idesc,
                    (kb != kb0) || kk != 0);
        umma_commit(&empty[rg.s]);
        rg.next();
      }
      ok = ok && mbar_wait(&slots_ready, 0, s_abort, g.status, g.budget_ns);
      const int n = ok ? slots.n : 0;
      for (int j = rank; ok && j < n; j += splits) {
        const uint32_t m0 = slots.off[j][0], m1 = slots.off[j][1], m2 = slots.off[j][2],
                       m3 = slots.off[j][3];
        for (int b = 0; b < blocks; ++b) {
          if (!mbar_wait(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + rg.s * a_bytes), b0 = smem_u32(sB + rg.s * B_BYTES);
          const int left = g.r - (b >> 1) * 64;
          const int steps = left >= 64 ? 4 : (left + 15) / 16;
          for (int kk = 0; kk < steps; ++kk) {
            umma_16_masked(tmem, umma_desc_sw128(a0 + kk * 32), desc_b(b0, kk), idesc, 1, m0, m1,
                           m2, m3);
            if (blocks == 1)
              umma_16_masked(tmem, umma_desc_sw128(a0 + 64 + kk * 32), desc_b(b0, kk), idesc, 1, m0,
                             m1, m2, m3);
          }
          umma_commit(&empty[rg.s]);
          rg.next();
        }
      }
      umma_commit(&done);
      mbar_wait(&done, 0, nullptr, g.status, g.budget_ns);
    }
    __syncwarp();
  } else {
    if (warp == 2) {
      build_slots<4>(g.ids, row0, g.M, g.E, &slots, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&slots_ready);
    }
    mbar_wait(&done, 0, nullptr, g.status, g.budget_ns);
  }
  // The MMAs are done and the copies have landed: the stages are free.
  __syncthreads();
  tc_fence_after();
  const int mrows = g.M - row0 < kRows ? (int)(g.M - row0) : kRows;
  if (splits == 1 && g.y_vec && col0 + BN <= g.N) {
    // 16-byte stores of each row's columns.
    if (warp >= 2) {
      const int q = warp & 3;
      const int64_t row = row0 + q * 32 + lane;
#pragma unroll
      for (int c = 0; c < BN; c += 32) {
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c, v);
        tmem_wait_ld();
        if (row < g.M) {
          uint4* y = (uint4*)((uint16_t*)g.Y + row * g.ldy + col0 + c);
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              w[j] = pack16(g.bf16, __uint_as_float(v[i + 2 * j]), __uint_as_float(v[i + 2 * j + 1]));
            y[i / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  } else {
    // Parts to be added up, or rows that take no vector stores: by way of shared
    // memory, [row][BN + 4]: rows of 16-byte pieces, eight of them across all
    // banks.
    constexpr int LDP = BN + 4;
    float* part = (float*)smem;
    if (warp >= 2) {
      const int q = warp & 3;
      const int r = q * 32 + lane;
      if (q * 32 < mrows) {
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          uint32_t v[32];
          tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c, v);
          tmem_wait_ld();
          if (r < mrows)
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *(uint4*)&part[r * LDP + c + i] = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    cluster_sync();
    const int share = BN / 4 / (int)splits;  // pieces of a row for this CTA
    const int c0 = (int)rank * share;
    for (int e = threadIdx.x; e < mrows * share; e += kThreads) {
      const int r = e / share, c = 4 * (c0 + e - r * share);
      const float4 s = cluster_sum4(smem_u32(&part[r * LDP + c]), (int)splits);
      const int n = g.N - (col0 + c);
      uint16_t* y = (uint16_t*)g.Y + (row0 + r) * g.ldy + col0 + c;
      if (g.y_vec && n >= 4) {
        *(uint2*)y = make_uint2(pack16(g.bf16, s.x, s.y), pack16(g.bf16, s.z, s.w));
      } else {
        if (n > 0) y[0] = round16(g.bf16, s.x);
        if (n > 1) y[1] = round16(g.bf16, s.y);
        if (n > 2) y[2] = round16(g.bf16, s.z);
        if (n > 3) y[3] = round16(g.bf16, s.w);
      }
    }
    cluster_sync();  // no CTA leaves while a peer reads its partials
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- low rank

struct LowArgs {
  const int32_t* ids;
  const float* scale;
  float alpha;
  float* low;        // [M][r] FP32, or NULL
  uint16_t* split;   // [M][2 half], or NULL
  uint16_t* outer;   // the same with low parts times low_up, or NULL
  int64_t M;
  int nkb, E, r, rp;  // rp: r rounded up to 16
  int batch;          // adapters of a tile that are multiplied at once
  int bf16;
  int stages, xrows;
  int32_t* status;
  uint64_t budget_ns;
};

// T of a tile of 128 rows, for up to `batch` of the tile's adapters at once,
// each into TMEM columns of its own; a row then takes its own adapter's.  A
// stage holds 64 contraction elements of X and of those adapters; a tile with
// more adapters walks X again for the next ones.  The CTAs of a cluster split
// the contraction.  Bound by reading X (requests of many rows: one batch).
//
// An MMA this narrow lasts some 250 clocks when the next one waits for its
// sum, so the four steps of 16 elements in a stage go to four accumulators
// (two from rank 65 on), which are added in FP32 at the end.  That also keeps
// the chains short: the tensor cores cut off, rather than round, what a sum's
// exponent leaves no room for, and T was 1.2e-6 off after chains of 1024
// elements, 3.5e-7 after 256.
template <bool MNB>
__global__ void __launch_bounds__(kThreads)
    k_low_rank(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapA,
               const __grid_constant__ LowArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int x_bytes = g.xrows * 128;
  const int a_bytes = MNB ? (g.rp + 63) / 64 * 8192 : g.rp * 128;
  uint8_t* sX = smem;
  uint8_t* sA = smem + g.stages * x_bytes;
  float* part = (float*)(sA + g.stages * g.batch * a_bytes);  // [row][rp + 4], in 16-byte pieces
  const int ldp = g.rp + 4;
  __shared__ SlotList<4> slots;
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done, taken;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_word;
  volatile int* s_abort = &s_abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t splits, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
  rank = cluster_ctarank();
  const int64_t row0 = (int64_t)(blockIdx.x / splits) * kRows;
  const int kb0 = (int)((int64_t)g.nkb * rank / splits);
  const int kb1 = (int)((int64_t)g.nkb * (rank + 1) / splits);
  const int accs = g.rp <= 64 ? 4 : 2;
  uint32_t cols = 32;
  while (cols < (uint32_t)(accs * g.batch * g.rp)) cols *= 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&taken, 4);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&s_tmem, cols);
  if (warp == 2) build_slots<4>(g.ids, row0, g.M, g.E, &slots, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_release();  // after the allocation: the next kernel's CTAs cannot take this CTA's TMEM
  const uint32_t tmem = s_tmem;
  const int n = slots.n;

  if (warp == 0) {
    if (lane == 0) {
      Ring rg(g.stages);
      bool ok = true;
      int issued = 0;
      for (int j0 = 0; ok && j0 < n; j0 += g.batch) {
        const int cnt = n - j0 < g.batch ? n - j0 : g.batch;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&empty[rg.s], rg.ph ^ 1, s_abort, g.status, g.budget_ns);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[rg.s], (uint32_t)(x_bytes + cnt * a_bytes));
          tma_load_3d(sX + rg.s * x_bytes, &mapX, &full[rg.s], kb * kKB, (int)row0, 0);
          uint8_t* d = sA + rg.s * g.batch * a_bytes;
          for (int j = 0; j < cnt; ++j, d += a_bytes) {
            if constexpr (MNB) {
              for (int c = 0; c < g.rp; c += 64)
                tma_load_3d(d + c * 128, &mapA, &full[rg.s], c, kb * kKB, slots.id[j0 + j]);
            } else {
              tma_load_3d(d, &mapA, &full[rg.s], kb * kKB, 0, slots.id[j0 + j]);
            }
          }
          rg.next();
          ++issued;
        }
      }
      ring_drain(full, g.stages, issued, g.status, g.budget_ns);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      Ring rg(g.stages);
      bool ok = true;
      int batch = 0;
      for (int j0 = 0; ok && j0 < n; j0 += g.batch, ++batch) {
        const int cnt = n - j0 < g.batch ? n - j0 : g.batch;
        if (batch > 0) ok = mbar_wait(&taken, (batch - 1) & 1, s_abort, g.status, g.budget_ns);
        if (!ok) break;
        tc_fence_after();
        // K-major adapters lie side by side: one MMA takes them all.
        const uint32_t idesc = umma_idesc_16(g.bf16, kRows, MNB ? g.rp : cnt * g.rp, false, MNB);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns);
          if (!ok) break;
          tc_fence_after();
          const uint32_t x0 = smem_u32(sX + rg.s * x_bytes);
          const uint32_t a0 = smem_u32(sA + rg.s * g.batch * a_bytes);
          for (int j = 0; j < (MNB ? cnt : 1); ++j)
#pragma unroll
            for (int kk = 0; kk < kKB / 16; ++kk) {
              const uint32_t d = tmem + (uint32_t)(((kk & (accs - 1)) * g.batch + j) * g.rp);
              umma_bf16(d, umma_desc_sw128(x0 + kk * 32),
                        MNB ? umma_desc_mn128(a0 + j * a_bytes + kk * 2048, 8192)
                            : umma_desc_sw128(a0 + kk * 32),
                        idesc, kb != kb0 || kk >= accs);
            }
          umma_commit(&empty[rg.s]);
          rg.next();
        }
        umma_commit(&done);
      }
      // Whatever is in flight ends before TMEM is released.
      if (!ok) umma_commit(&done);
      if (n > 0) mbar_wait(&done, (ok ? batch - 1 : batch) & 1, nullptr, g.status, g.budget_ns);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int r = q * 32 + lane;
    int batch = 0;
    for (int j0 = 0; j0 < n; j0 += g.batch, ++batch) {
      const int cnt = n - j0 < g.batch ? n - j0 : g.batch;
      if (!mbar_wait(&done, batch & 1, s_abort, g.status, g.budget_ns)) break;
      tc_fence_after();
      for (int j = 0; j < cnt; ++j) {
        const uint32_t off = slots.off[j0 + j][q];
        if (off == ~0u) continue;  // no row of this warp's
        const bool mine = !((off >> lane) & 1);
        for (int c = 0; c < g.rp; c += 16) {
          uint32_t v[4][16];
#pragma unroll
          for (int a = 0; a < 4; ++a)
            if (a < accs)
              tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + (a * g.batch + j) * g.rp + c, v[a]);
          tmem_wait_ld();
          float sum[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sum[i] = __uint_as_float(v[0][i]) + __uint_as_float(v[1][i]);
            if (accs == 4) sum[i] += __uint_as_float(v[2][i]) + __uint_as_float(v[3][i]);
          }
          if (mine)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *(float4*)&part[r * ldp + c + i] =
                  make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&taken);
    }
  }
  cluster_sync();
  // The kernel before this one may still run (the backward pass's row lists):
  // whoever waits for this kernel has waited for that one too.
  if (threadIdx.x == 0) grid_wait();
  // Rows of the tile are dealt to the CTAs of the cluster.
  const int mrows = g.M - row0 < kRows ? (int)(g.M - row0) : kRows;
  const int half = split_half(g.r);
  const int r0 = mrows * (int)rank / (int)splits, r1 = mrows * ((int)rank + 1) / (int)splits;
  for (int e = threadIdx.x; e < (r1 - r0) * (half / 4); e += kThreads) {
    const int r = r0 + e / (half / 4), c = e % (half / 4) * 4;
    const int64_t row = row0 + r;
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int i = row_adapter(g.ids, row, g.M, g.E);
    if (i >= 0 && c < g.r) {
      t = cluster_sum4(smem_u32(&part[r * ldp + c]), (int)splits);
      const float f = g.scale ? g.alpha * g.scale[i] : g.alpha;
      t.x *= f, t.y *= f, t.z *= f, t.w *= f;
      // Beyond rank r the adapter read as zeros, but an infinity in the row has
      // made NaNs of them.
      if (c + 1 >= g.r) t.y = 0.0f;
      if (c + 2 >= g.r) t.z = 0.0f;
      if (c + 3 >= g.r) t.w = 0.0f;
    }
    if (g.low) {
      float* o = g.low + row * g.r + c;
      if (c < g.r) o[0] = t.x;
      if (c + 1 < g.r) o[1] = t.y;
      if (c + 2 < g.r) o[2] = t.z;
      if (c + 3 < g.r) o[3] = t.w;
    }
    auto store = [&](uint16_t* split, float up) {
      uint32_t hi[2], lo[2];
      split16(g.bf16, t.x, t.y, up, hi[0], lo[0]);
      split16(g.bf16, t.z, t.w, up, hi[1], lo[1]);
      uint16_t* o = split + row * 2 * half + c;
      *(uint2*)o = make_uint2(hi[0], hi[1]);
      *(uint2*)(o + half) = make_uint2(lo[0], lo[1]);
    };
    if (g.split) store(g.split, 1.0f);
    if (g.outer) store(g.outer, low_up(g.bf16));
  }
  cluster_sync();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// T of few rows (decoding): one CTA per row and four ranks, the contraction
// split over its threads.  Every row reads its own A_i, so nothing is shared
// that a matrix instruction could use; bound by the latency of the reads.
constexpr int kLowThreads = 256;
constexpr int kLowRanks = 4;

__global__ void __launch_bounds__(kLowThreads)
    k_low_rank_rows(const uint16_t* X, int64_t ldx, const uint16_t* A, int64_t lda, int64_t K,
                    LowArgs g) {
  grid_release();
  __shared__ float part[kLowThreads / 32][kLowRanks];
  const int half = split_half(g.r);
  const int64_t row = blockIdx.x;
  const int c0 = blockIdx.y * kLowRanks;
  const int i = row_adapter(g.ids, row, g.M, g.E);
  float acc[kLowRanks] = {};
  if (i >= 0 && c0 < g.r) {
    const uint16_t* x = X + row * ldx;
    const uint16_t* a[kLowRanks];
#pragma unroll
    for (int j = 0; j < kLowRanks; ++j) {
      const int c = c0 + j < g.r ? c0 + j : g.r - 1;
      a[j] = A + ((int64_t)i * g.r + c) * lda;
    }
    // X's and A's rows start on 16 bytes (padded before this kernel otherwise).
    const int64_t K8 = K & ~(int64_t)7;
#pragma unroll 2
    for (int64_t k = threadIdx.x * 8; k < K8; k += kLowThreads * 8) {
      const uint4 xv = *(const uint4*)(x + k);
      uint4 av[kLowRanks];
#pragma unroll
      for (int j = 0; j < kLowRanks; ++j) av[j] = __ldg((const uint4*)(a[j] + k));
      const uint32_t* xw = (const uint32_t*)&xv;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float x0 = widen16(g.bf16, (uint16_t)xw[w]), x1 = widen16(g.bf16, xw[w] >> 16);
#pragma unroll
        for (int j = 0; j < kLowRanks; ++j) {
          const uint32_t u = ((const uint32_t*)&av[j])[w];
          acc[j] = fmaf(x0, widen16(g.bf16, (uint16_t)u), acc[j]);
          acc[j] = fmaf(x1, widen16(g.bf16, u >> 16), acc[j]);
        }
      }
    }
    const int64_t k = K8 + threadIdx.x;
    if (k < K) {
      const float xv = widen16(g.bf16, x[k]);
#pragma unroll
      for (int j = 0; j < kLowRanks; ++j) acc[j] = fmaf(xv, widen16(g.bf16, a[j][k]), acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kLowRanks; ++j)
    for (int o = 16; o; o >>= 1) acc[j] += __shfl_xor_sync(~0u, acc[j], o);
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int j = 0; j < kLowRanks; ++j) part[threadIdx.x >> 5][j] = acc[j];
  __syncthreads();
  if (threadIdx.x < kLowRanks) {
    const int c = c0 + threadIdx.x;
    float t = 0.0f;
    if (i >= 0 && c < g.r) {
      for (int w = 0; w < kLowThreads / 32; ++w) t += part[w][threadIdx.x];
      t *= g.scale ? g.alpha * g.scale[i] : g.alpha;
    }
    if (g.low && c < g.r) g.low[row * g.r + c] = t;
    if (g.split && c < half) store_split(g.split, row, half, c, t, g.bf16, 1.0f);
  }
}

// A thread copies 8 elements, read one by one (a warp reads 512 bytes side by
// side) and written as 16 bytes; a CTA takes 256 columns of 32 rows.
__global__ void __launch_bounds__(256)
    k_pad_rows(const uint16_t* src, int64_t lds, uint16_t* dst, int64_t ldd, int64_t rows,
               int64_t cols) {
  const int64_t c = ((int64_t)blockIdx.x * 32 + threadIdx.x % 32) * 8;
  if (c >= ldd) return;
  for (int64_t r = (int64_t)blockIdx.y * 32 + threadIdx.x / 32; r < rows;
       r += (int64_t)gridDim.y * 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t row = r + 8 * j;
      if (row >= rows) break;
      const uint16_t* p = src + row * lds + c;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (c + 2 * i < cols ? p[2 * i] : 0u) |
               ((c + 2 * i + 1 < cols ? (uint32_t)p[2 * i + 1] : 0u) << 16);
      *(uint4*)(dst + row * ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace

int launch_pad_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows,
                    int64_t cols, cudaStream_t stream) {
  if (rows == 0 || cols == 0) return OZK_OK;
  const int64_t tiles = (rows + 31) / 32;
  const dim3 grid((unsigned)((ldd + 255) / 256), (unsigned)(tiles < 65535 ? tiles : 65535));
  k_pad_rows<<<grid, 256, 0, stream>>>((const uint16_t*)src, lds, (uint16_t*)dst, ldd, rows, cols);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_pad_rows launch", e);
}

// ---------------------------------------------------------------- launches

namespace {

template <auto K, typename... Args>
int launch_cluster(const char* what, int64_t tiles, int splits, int threads, size_t smem,
                   bool early, int dev, cudaStream_t stream, const Args&... args) {
  int rc = allow_smem<K>(smem, dev);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * splits));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, K, args...);
  return e == cudaSuccess ? OZK_OK : set_cuda_error(what, e);
}

struct Operand {
  const void* p;
  int64_t ld;
};

// One product X W^T + (s X A_i^T) B_i^T, or with `back` set the same read the
// other way: X is dY [M][N], W and the A of the low-rank step lie as [N][K] and
// [E][N][r] with the contraction along their rows.
struct Product {
  Operand X, W, A, B;        // A: the adapters of the first step, B: of the second
  int64_t M, n_out, n_in;    // rows, output columns, contraction
  int r, E;
  bool back, bf16;
};

int run_low_rank(const Product& p, const int32_t* ids, const float* scale, float alpha, float* low,
                 uint16_t* split, uint16_t* outer, int32_t* status, int dev, cudaStream_t stream) {
  LowArgs g = {};
  g.ids = ids;
  g.scale = scale;
  g.alpha = alpha;
  g.low = low;
  g.split = split;
  g.outer = outer;
  g.M = p.M;
  g.E = p.E;
  g.r = p.r;
  g.rp = (p.r + 15) / 16 * 16;
  g.bf16 = p.bf16;
  g.nkb = (int)((p.n_in + kKB - 1) / kKB);
  g.status = status;
  g.budget_ns = wait_budget_ns();
  // Few rows (decoding): each may have an adapter of its own.  Up to 128 rows
  // are taken one by one, up to 256 if that is cheaper than tiles in which
  // every adapter has a row (about 1000 clocks for each batch's stage, against
  // 2.5 KB of adapters read per clock).
  const int accs = g.rp <= 64 ? 4 : 2;
  const int64_t most = p.E < kRows ? p.E : kRows;
  const int64_t by_tile = (most * accs * g.rp + 255) / 256 * (g.nkb / 8 + 1) * 1000;
  const int64_t by_row = p.M * p.r * p.n_in * 2 / 2500;
  if (!p.back && (p.M <= kRows || (p.M <= 2 * kRows && by_row < by_tile))) {
    const int half = split_half(p.r);
    k_low_rank_rows<<<dim3((unsigned)p.M, (unsigned)(half / kLowRanks)), kLowThreads, 0, stream>>>(
        (const uint16_t*)p.X.p, p.X.ld, (const uint16_t*)p.A.p, p.A.ld, p.n_in, g);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? OZK_OK : set_cuda_error("k_low_rank_rows launch", e);
  }
  g.xrows = p.M >= kRows ? kRows : (int)round_up(p.M, 8);
  const int64_t tiles = (p.M + kRows - 1) / kRows;
  // Two CTAs per SM at most (a second wave doubles the time), clusters of four
  // where there are tiles enough (of eight, only 15 fit the GPU at 100 KB of
  // shared memory a CTA), and chains of at most 512 elements up to a contraction of
  // 16384 (8192 from rank 65 on; beyond, they grow with it).
  int splits = 1;
  while (splits < (tiles <= 8 ? 8 : 4) && tiles * splits * 2 <= 2 * device_sm_count(dev) &&
         g.nkb >= splits * 4)
    splits *= 2;
  while (splits < 8 && g.nkb > 8 * splits * accs) splits *= 2;
  const int a_bytes = p.back ? (g.rp + 63) / 64 * 8192 : g.rp * 128;
  // TMEM for two CTAs per SM: 256 columns.
  g.batch = 256 / (accs * g.rp);
  if (p.back && g.batch > 2) g.batch = 2;
  const size_t stage = (size_t)g.xrows * 128 + (size_t)g.batch * a_bytes;
  const size_t red = (size_t)kRows * (g.rp + 4) * 4;
  // (Stages for one CTA per SM where there are no more: a stage takes its copy's
  // latency divided by the stages in flight.)
  const bool alone = g.rp > 64 || tiles * splits <= device_sm_count(dev);
  const size_t room = (alone ? 180 : 108) * 1024 - red;
  g.stages = (int)(room / stage);
  if (g.stages > 8) g.stages = 8;
  size_t area = g.stages * stage + red;
  // (The MMA reads 128 rows of X's last stage even if fewer were loaded: what
  // lies behind belongs to this CTA.)
  const size_t need = (size_t)(g.stages - 1) * g.xrows * 128 + kRows * 128;
  if (area < need) area = need;
  if (area < tmem_share(accs * g.batch * g.rp)) area = tmem_share(accs * g.batch * g.rp);
  CUtensorMap mx, ma;
  int rc;
  if ((rc = make_map(&mx, p.X.p, 2, p.n_in, p.M, 1, p.X.ld * 2, p.X.ld * 2 * p.M, kKB, g.xrows,
                     true)))
    return rc;
  if (p.back)
    rc = make_map(&ma, p.A.p, 2, p.r, p.n_in, p.E, p.A.ld * 2, p.A.ld * 2 * p.n_in, 64, kKB, true);
  else
    rc = make_map(&ma, p.A.p, 2, p.n_in, p.r, p.E, p.A.ld * 2, p.A.ld * 2 * p.r, kKB, g.rp, true);
  if (rc) return rc;
  return p.back ? launch_cluster<k_low_rank<true>>("k_low_rank", tiles, splits, kThreads,
                                                   area + 1024, true, dev, stream, mx, ma, g)
                : launch_cluster<k_low_rank<false>>("k_low_rank", tiles, splits, kThreads,
                                                    area + 1024, false, dev, stream, mx, ma, g);
}

template <int BN, bool MNB>
int run_linear_bn(const Product& p, LinearArgs g, const uint16_t* split, int splits,
                  int dev, cudaStream_t stream) {
  const int half = split_half(p.r);
  g.tiles_n = (int)((p.n_out + BN - 1) / BN);
  const int64_t tiles = (p.M + kRows - 1) / kRows * g.tiles_n;
  const size_t stage = (size_t)g.xrows * 128 + BN * 128;
  g.stages = (int)(96 * 1024 / stage);
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  size_t area = g.stages * stage;
  const size_t need = (size_t)(g.stages - 1) * g.xrows * 128 + kRows * 128;
  const size_t red = (size_t)g.xrows * (BN + 4) * 4;
  if (area < need) area = need;
  if (area < red) area = red;
  if (area < tmem_share(BN)) area = tmem_share(BN);
  CUtensorMap mx, mw, mt, mb;
  int rc;
  if ((rc = make_map(&mx, p.X.p, 2, p.n_in, p.M, 1, p.X.ld * 2, p.X.ld * 2 * p.M, kKB, g.xrows,
                     true)))
    return rc;
  if ((rc = make_map(&mt, split, 2, 2 * half, p.M, 1, 4 * half, 4 * half * p.M, 64, g.xrows, true)))
    return rc;
  if (MNB) {
    rc = make_map(&mw, p.W.p, 2, p.n_out, p.n_in, 1, p.W.ld * 2, p.W.ld * 2 * p.n_in, 64, kKB, true);
    if (!rc)
      rc = make_map(&mb, p.B.p, 2, p.n_out, p.r, p.E, p.B.ld * 2, p.B.ld * 2 * p.r, 64, 64, true);
  } else {
    rc = make_map(&mw, p.W.p, 2, p.n_in, p.n_out, 1, p.W.ld * 2, p.W.ld * 2 * p.n_out, kKB, BN,
                  true);
    if (!rc)
      rc = make_map(&mb, p.B.p, 2, p.r, p.n_out, p.E, p.B.ld * 2, p.B.ld * 2 * p.n_out, 64, BN,
                    true);
  }
  if (rc) return rc;
  return launch_cluster<k_linear<BN, MNB>>("k_linear", tiles, splits, kThreads, area + 1024, true,
                                           dev, stream, mx, mw, mt, mb, g);
}

int run_linear(const Product& p, const int32_t* ids, const uint16_t* split, void* Y, int64_t ldy,
               int32_t* status, int dev, cudaStream_t stream) {
  LinearArgs g = {};
  g.ids = ids;
  g.Y = Y;
  g.ldy = ldy;
  g.M = p.M;
  g.N = (int)p.n_out;
  g.nkb = (int)((p.n_in + kKB - 1) / kKB);
  g.E = p.E;
  g.r = p.r;
  g.bf16 = p.bf16;
  g.y_vec = ((uintptr_t)Y & 15) == 0 && ldy % 8 == 0;
  g.xrows = p.M >= kRows ? kRows : (int)round_up(p.M, 8);
  g.status = status;
  g.budget_ns = wait_budget_ns();
  const int64_t tiles_m = (p.M + kRows - 1) / kRows;
  const int sms = device_sm_count(dev);
  if (((p.M + 255) / 256) * ((p.n_out + 255) / 256) >= sms / 2) {
    WideProduct w = {};
    w.mode = p.back ? kWideBack : kWideForward;
    w.bf16 = p.bf16;
    w.M = p.M;
    w.N = p.n_out;
    w.C = p.n_in;
    w.A = p.X.p;
    w.lda = p.X.ld;
    w.B = p.W.p;
    w.ldb = p.W.ld;
    w.ids = ids;
    w.r = p.r;
    w.E = p.E;
    w.split = split;
    w.Bi = p.B.p;
    w.ldbi = p.B.ld;
    w.early = true;
    w.out = Y;
    w.ldo = ldy;
    w.status = status;
    return launch_wide(w, dev, stream);
  }
  // 128 columns per CTA; the contraction split over a cluster as long as two
  // CTAs per SM hold them all (a second wave adds half: 64 x 8192 x 4096, its
  // inputs in the L2 cache, took 20 us with 256 CTAs and 30 us with 512).  Full tiles have more to add
  // up: they are split in four at most, into parts of sixteen stages or more
  // (1023 x 2048 x 1000 took 17 us whole and 22 us halved, 1777 x 1001 x 2000
  // 37 us whole and 24 us halved).
  const int64_t tiles = tiles_m * ((p.n_out + 127) / 128);
  const int most = p.M > 64 ? 4 : 8, least = p.M > 64 ? 16 : 4;
  int splits = 1;
  while (splits < most && tiles * splits * 2 <= 2 * sms && g.nkb >= splits * 2 * least) splits *= 2;
  return p.back ? run_linear_bn<128, true>(p, g, split, splits, dev, stream)
                : run_linear_bn<128, false>(p, g, split, splits, dev, stream);
}

// Copies an operand that TMA cannot read into the workspace, its rows padded
// to 16 bytes; `launch` false only counts the bytes.
int align_operand(Operand& o, int64_t rows, int64_t cols, Arena& ws, bool launch,
                  cudaStream_t stream) {
  if (tma_ready(o.p, o.ld)) return OZK_OK;
  const int64_t ld = round_up(cols, 8);
  void* d = ws.take<void>((size_t)(rows * ld * 2));
  if (launch) {
    int rc = launch_pad_rows(o.p, o.ld, d, ld, rows, cols, stream);
    if (rc) return rc;
  }
  o.p = d;
  o.ld = ld;
  return OZK_OK;
}

}  // namespace

}  // namespace ozk

using namespace ozk;

static int adapter_args(const void* X, int64_t ldx, const void* W, int64_t ldw, const void* A,
                        const void* B, int64_t M, int64_t N, int64_t K, int r, int E, int dt) {
  if (!dt_is_16bit(dt)) return set_error(OZK_ERR_ARG, "dtype must be OZK_DT_BF16 or OZK_DT_F16");
  if (M < 0 || N < 0 || K < 1) return set_error(OZK_ERR_ARG, "need M, N >= 0 and K >= 1");
  if (M > (1 << 30) || N > (1 << 30) || K > (1 << 30))
    return set_error(OZK_ERR_UNSUPPORTED, "M, N and K are limited to 2^30");
  if (r < 1 || r > kMaxRank)
    return set_error(OZK_ERR_ARG, "rank %d; expected 1 to %d", r, kMaxRank);
  if (E < 1 || E > (1 << 20)) return set_error(OZK_ERR_ARG, "need 1 <= E <= 2^20 adapters");
  if (M == 0 || N == 0) return OZK_OK;
  if (!X || !W || !A || !B) return set_error(OZK_ERR_ARG, "NULL pointer");
  if (ldw < K) return set_error(OZK_ERR_ARG, "ldw < K");
  return OZK_OK;
}

extern "C" {

size_t ozk_matmul_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int r, int E,
                                           int aligned) {
  if (M < 1 || N < 0 || K < 1 || r < 1 || r > kMaxRank || E < 1) return 0;
  Arena ws(nullptr);
  ws.take<uint16_t>((size_t)M * 4 * split_half(r));
  if (aligned) return ws.used;
  // The worst case: every operand has to be copied.
  ws.take((size_t)M * round_up(K, 8) * 2);
  ws.take((size_t)N * round_up(K, 8) * 2);
  ws.take((size_t)E * r * round_up(K, 8) * 2);
  ws.take((size_t)E * N * round_up(r, 8) * 2);
  return ws.used;
}

int ozk_matmul_adapters(const void* X, int64_t ldx, const void* W, int64_t ldw, const void* A,
                        const void* B, const int32_t* ids, const float* scale, double alpha,
                        void* Y, int64_t ldy, float* low, int64_t M, int64_t N, int64_t K, int r,
                        int E, int dt, void* workspace, size_t ws_bytes, int32_t* status_dev,
                        void* stream) {
  int rc = adapter_args(X, ldx, W, ldw, A, B, M, N, K, r, E, dt);
  if (rc) return rc;
  if (M == 0 || (N == 0 && !low)) return OZK_OK;
  if (ldx < K || !X || !A) return set_error(OZK_ERR_ARG, "NULL X or A, or ldx < K");
  if (N && (!Y || ldy < N)) return set_error(OZK_ERR_ARG, "NULL Y or ldy < N");
  cudaStream_t s = (cudaStream_t)stream;
  int dev;
  cudaGetDevice(&dev);
  Product p = {{X, ldx}, {W, ldw}, {A, K}, {B, r}, M, N, K, r, E, false, dt == OZK_DT_BF16};
  Arena ws(workspace);
  uint16_t* split = ws.take<uint16_t>((size_t)M * 4 * split_half(r));
  for (int pass = 0; pass < 2; ++pass) {  // count first, then copy
    Product q = p;
    Arena w = ws;
    if ((rc = align_operand(q.X, M, K, w, pass, s)) ||
        (rc = align_operand(q.A, (int64_t)E * r, K, w, pass, s)) ||
        (N && (rc = align_operand(q.W, N, K, w, pass, s))) ||
        (N && (rc = align_operand(q.B, (int64_t)E * N, r, w, pass, s))))
      return rc;
    if (pass) p = q;
    else if (!workspace || w.used > ws_bytes || ((uintptr_t)workspace & 127))
      return set_error(OZK_ERR_WORKSPACE, "workspace of %zu bytes, aligned to 128, needed", w.used);
  }
  if ((rc = run_low_rank(p, ids, scale, (float)alpha, low, split, nullptr, status_dev, dev,
                         s)) ||
      N == 0)
    return rc;
  return run_linear(p, ids, split, Y, ldy, status_dev, dev, s);
}

size_t ozk_adapters_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int r, int E,
                                         int aligned) {
  if (M < 1 || N < 1 || K < 1 || r < 1 || r > kMaxRank || E < 1) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  Arena ws(nullptr);
  ws.take((size_t)M * 4 * split_half(r));
  ws.take((size_t)M * 4 * split_half(r));
  ws.take(outer_scratch_bytes(M, N, K, r, E, dev));
  if (aligned) return ws.used;
  ws.take((size_t)M * round_up(N, 8) * 2);
  ws.take((size_t)N * round_up(K, 8) * 2);
  ws.take((size_t)E * r * round_up(K, 8) * 2);
  ws.take((size_t)E * N * round_up(r, 8) * 2);
  ws.take((size_t)M * round_up(K, 8) * 2);
  return ws.used;
}

int ozk_adapters_grad(const void* dY, int64_t ldy, const void* X, int64_t ldx, const void* exps,
                      const void* W, int64_t ldw, const void* A, const void* B, const int32_t* ids,
                      const float* T, const float* scale, double alpha, void* dX, int64_t lddx,
                      void* dA, void* dB, int64_t M, int64_t N, int64_t K, int r, int E, int dt,
                      void* workspace, size_t ws_bytes, int32_t* status_dev, void* stream) {
  int rc = adapter_args(X, ldx, W, ldw, A, B, M, N, K, r, E, dt);
  if (rc) return rc;
  if (E > 65535) return set_error(OZK_ERR_UNSUPPORTED, "at most 65535 adapters");
  if (!dA || (N && !dB)) return set_error(OZK_ERR_ARG, "NULL dA or dB");
  if (dX && lddx < K) return set_error(OZK_ERR_ARG, "lddx < K");
  cudaStream_t s = (cudaStream_t)stream;
  if (M == 0 || N == 0) {
    // No rows or no outputs: the gradients are zero.
    cudaError_t e = cudaMemsetAsync(dA, 0, (size_t)E * r * K * 2, s);
    if (e == cudaSuccess && N) e = cudaMemsetAsync(dB, 0, (size_t)E * N * r * 2, s);
    if (e == cudaSuccess && M && dX)
      e = cudaMemset2DAsync(dX, (size_t)lddx * 2, 0, (size_t)K * 2, (size_t)M, s);
    return e == cudaSuccess ? OZK_OK : set_cuda_error("cudaMemsetAsync", e);
  }
  if (!dY || !T || ldy < N) return set_error(OZK_ERR_ARG, "NULL dY or T, or ldy < N");
  if (exps ? (ldx != round_up(K, kGroup) || ((uintptr_t)X & 15)) : ldx < K)
    return set_error(OZK_ERR_ARG, exps ? "codes need 16 bytes of alignment and ldx = K rounded up to 128"
                                       : "ldx < K");
  int dev;
  cudaGetDevice(&dev);
  Product p = {{dY, ldy}, {W, ldw}, {B, r}, {A, K}, M, K, N, r, E, true, dt == OZK_DT_BF16};
  Arena ws(workspace);
  uint16_t* split = ws.take<uint16_t>((size_t)M * 4 * split_half(r));
  // U for dA: in BF16 the same split serves.
  uint16_t* outer = p.bf16 ? split : ws.take<uint16_t>((size_t)M * 4 * split_half(r));
  void* scratch = ws.take(outer_scratch_bytes(M, N, K, r, E, dev));
  Operand in = {X, ldx};
  for (int pass = 0; pass < 2; ++pass) {
    Product q = p;
    Operand x = in;
    Arena w = ws;
    if ((rc = align_operand(q.X, M, N, w, pass, s)) || (rc = align_operand(q.W, N, K, w, pass, s)) ||
        (rc = align_operand(q.A, (int64_t)E * N, r, w, pass, s)) ||
        (rc = align_operand(q.B, (int64_t)E * r, K, w, pass, s)) ||
        (!exps && (rc = align_operand(x, M, K, w, pass, s))))
      return rc;
    if (pass) p = q, in = x;
    else if (!workspace || w.used > ws_bytes || ((uintptr_t)workspace & 127))
      return set_error(OZK_ERR_WORKSPACE, "workspace of %zu bytes, aligned to 128, needed", w.used);
  }
  OuterProduct o = {};
  o.bf16 = p.bf16;
  o.M = M;
  o.N = N;
  o.K = K;
  o.r = r;
  o.E = E;
  o.ids = ids;
  o.X = in.p;
  o.ldx = in.ld;
  o.exps = (const int8_t*)exps;
  o.dY = p.X.p;
  o.ldy = p.X.ld;
  o.U = outer;
  o.T = T;
  o.dA = dA;
  o.dB = dB;
  o.status = status_dev;
  if ((rc = launch_outer_rows(o, scratch, dev, s))) return rc;
  if ((rc = run_low_rank(p, ids, scale, (float)alpha, nullptr,
                         p.bf16 || dX ? split : nullptr, p.bf16 ? nullptr : outer, status_dev, dev,
                         s)))
    return rc;
  if (dX && (rc = run_linear(p, ids, split, dX, lddx, status_dev, dev, s))) return rc;
  return launch_outer(o, scratch, dev, s);
}

}  // extern "C"
