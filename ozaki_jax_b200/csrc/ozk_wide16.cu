// k_wide: 16-bit products on 256 x 256 tiles of CTA pairs, FP32 accumulators.
//
//   forward  Y  = X W^T  (+ T B_i^T)     both operands K-major
//   back     dX = dY W   (+ U A_i)       W and A_i MN-major
//   weight   dW = dY^T X^                dY MN-major, X^ from int8 codes
//
// Persistent: each CTA pair (cta_group::2, M = 256) walks its tiles; each CTA
// stages its 128 rows of A and half of B's 256 columns per 64 contraction
// indexes.  Bound by shared memory, by this count: a stage of 4 MMAs lasts 512
// clocks on the tensor cores, in which the MMAs read 32 KB of each SM's shared
// memory and the copies write 32 KB; that is all of its 128 B/clk, and a stage
// took 714 clocks (859 with the converters' traffic).  So where there are tiles enough,
// a pair takes two tiles one below the other (SUB = 2, 512 x 256) that share
// B: 112 KB instead of 128 KB for the same work, and in the weight product
// each code is converted for 512 rows instead of 256.
//
// 16384 x 8192 x 8192 from codes: 1.63 ms in a burst and 1.88 ms under the power
// limit (1.35 and 1.17 PFLOP/s; restoring the rows and cuBLAS's BF16 product
// 1.33 and 1.56 ms in the same runs).  To FP32, with SUB = 1 and every chain's
// sums added in the output, 3.74 ms.  8192 x 8192 x 4096 with a rank of 64, the
// whole call: 388 us in a burst, 456 us under the power limit (cuBLAS without
// the adapters 408 us there).
//
// SUB = 1: two TMEM accumulators (all 512 columns) let the epilogue of one tile
// run under the MMAs of the next.  SUB = 2: they belong to the two halves of a
// tile; the first stages' MMAs into the upper half run while the lower half is
// still being read.
//
// Warps: 0 TMA producer, 1 MMA issuer (one thread of the even CTA), 2-9
// epilogue, 10 the tile's list of adapters (forward, back) or 10-18 (weight):
// 10-17 convert each CTA's 128 columns x 64 rows of codes (TMA'd into a ring of
// their own) into 16-bit values in the MMA's layout, 16 codes per clock and SM
// at the MMA's full rate, at about 2.5 instructions a code; two groups of four
// warps take alternate stages, so that a group has two stages' time for its
// chain of loads, conversions, stores and fence.  Warp 18 turns the exponents
// into 16-bit steps and copies the codes in, some stages ahead of the MMA.  The
// steps are powers of two, so a code times its step is exact in the operand type
// and the product is that of the restored matrix.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "ozk_tile16.cuh"

namespace ozk {

namespace {

constexpr int kTile = 256;
constexpr int kHalf = 128;       // rows of A, columns of B per CTA
constexpr int kKB = 64;          // contraction indexes per stage
constexpr int kABytes = kHalf * kKB * 2;
constexpr int kRawBytes = kHalf * kKB;
constexpr int kConvWarps = 4;    // of one of the two converter groups

constexpr int kTurnBytes = 32 * 9 * 4;  // a warp's buffer for turning 8 columns of its 32 rows
constexpr int kEpiWarps = 8;     // four lane quadrants, two column halves
constexpr int kWork = 2 + kEpiWarps;  // first warp after the epilogue's

template <WideMode MODE, int SUB>
struct WideCfg {
  static constexpr bool W = MODE == kWideWeight;
  static constexpr int STAGE_BYTES = (SUB + 1) * kABytes;
  static constexpr int STAGES = SUB == 2 ? 4 : W ? 5 : 6;
  static constexpr int RAW = W ? (SUB == 2 ? 3 : 6) : 0;
  static constexpr int THREADS = 32 * (W ? kWork + 2 * kConvWarps + 1 : kWork + 1);
  // Most of an SM's shared memory, and in any case more than half: a CTA holds all
  // TMEM columns, so no other TMEM kernel may fit beside it.
  static constexpr int SMEM = 227 * 1024 - (W ? (SUB == 2 ? 1 : 3) : SUB == 2 ? 20 : 11) * 1024;
  static_assert(1024 + STAGES * STAGE_BYTES + RAW * kRawBytes + kEpiWarps * kTurnBytes <= SMEM, "");
};

struct WideArgs {
  int64_t M, N;
  int nkb, tiles_m, tiles_n, group_m, splits;
  int chain;           // stages summed in one accumulator before FP32 takes over
  int bf16, out_f32, accumulate, o_vec;
  void* out;
  int64_t ldo;
  float* partial;      // [splits][M][ldp] when splits > 1
  int64_t ldp;
  const int8_t* exps;  // [groups][C]
  int64_t C;
  const int32_t* ids;
  int r, E;
  int32_t* status;
  uint64_t budget_ns;
};

// Tiles walk down groups of group_m tile rows before moving right, so the
// tiles in flight share few panels.
__device__ __forceinline__ void tile_at(const WideArgs& g, int t, int& tm, int& tn) {
  const int per = g.group_m * g.tiles_n;
  const int grp = t / per, first = grp * g.group_m;
  const int rows = g.tiles_m - first < g.group_m ? g.tiles_m - first : g.group_m;
  const int r = t - grp * per;
  tm = first + r % rows;
  tn = r / rows;
}

// 32 bytes at once (p on 32 bytes): a store of a warp touches 32 rows here, and
// costs the same whether it writes a half or a whole sector of each.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 32 consecutive outputs of one row, added to what is there with `add`.  wide:
// the row takes 32-byte stores, else 16-byte ones.
__device__ __forceinline__ void store_f32(float* o, bool wide, const uint32_t (&v)[32], bool add) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    uint32_t f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v[i + j];
    if (add) {
      const float4 p = *(const float4*)(o + i), q = *(const float4*)(o + i + 4);
      const float w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __float_as_uint(__uint_as_float(f[j]) + w[j]);
    }
    if (wide) {
      store32(o + i, f);
    } else {
      *(uint4*)(o + i) = make_uint4(f[0], f[1], f[2], f[3]);
      *(uint4*)(o + i + 4) = make_uint4(f[4], f[5], f[6], f[7]);
    }
  }
}
__device__ __forceinline__ void store_16(uint16_t* o, bool wide, const uint32_t (&v)[32], bool add,
                                         bool bf16) {
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    uint32_t q[8];
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(v[i + h + j]);
      if (add) {
        const uint4 p = *(const uint4*)(o + i + h);
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] += widen16(bf16, (uint16_t)w[j]);
          f[2 * j + 1] += widen16(bf16, (uint16_t)(w[j] >> 16));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) q[h / 2 + j] = pack16(bf16, f[2 * j], f[2 * j + 1]);
    }
    if (wide) {
      store32(o + i, q);
    } else {
      *(uint4*)(o + i) = make_uint4(q[0], q[1], q[2], q[3]);
      *(uint4*)(o + i + 8) = make_uint4(q[4], q[5], q[6], q[7]);
    }
  }
}

// The same for rows that take no vector stores, or the last n < 32 columns:
// through the warp's own shared memory, so that a store writes along a row (a
// lane storing its own row element by element touches 32 lines each time: a
// 5905 x 7048 output took 447 us).  `out` is the warp's first row, `rows` of its
// 32 lie inside the matrix.
template <typename F>
__device__ __forceinline__ void store_turned(uint8_t* turn, const uint32_t (&v)[32], int rows, int n,
                                             F&& put) {
  uint32_t* t = (uint32_t*)turn;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = 0; h < 32; h += 8) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) t[lane * 9 + i] = v[h + i];
    __syncwarp();
    const int c = h + (lane & 7);
#pragma unroll
    for (int r = 0; r < 32; r += 4) {
      const int row = r + (lane >> 3);
      if (row < rows && c < n) put(row, c, __uint_as_float(t[row * 9 + (lane & 7)]));
    }
  }
}

template <WideMode MODE, bool BF16, int SUB>
__global__ void __launch_bounds__(WideCfg<MODE, SUB>::THREADS, 1)
    k_wide(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
           const __grid_constant__ CUtensorMap mapT, const __grid_constant__ CUtensorMap mapBi,
           const __grid_constant__ WideArgs g) {
  using Cfg = WideCfg<MODE, SUB>;
  constexpr int STAGES = Cfg::STAGES, RAW = Cfg::RAW, kStageBytes = Cfg::STAGE_BYTES;
  constexpr int kBOff = SUB * kABytes;  // B behind the tile halves of A
  constexpr bool AMN = MODE == kWideWeight, BMN = MODE != kWideForward;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sRaw = smem + STAGES * kStageBytes;
  __shared__ uint64_t full[STAGES], empty[STAGES], rfull[RAW + 1], rempty[RAW + 1], accf[2],
      acce[2], sfull, sempty, done;
  __shared__ SlotList<MODE == kWideWeight ? 1 : 8> slots[SUB];
  __shared__ uint32_t steps[MODE == kWideWeight ? RAW : 1][kKB];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_word;
  volatile int* s_abort = &s_abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int unit = (int)(blockIdx.x >> 1), n_units = (int)(gridDim.x >> 1);
  const int tiles = g.tiles_m * g.tiles_n, items = tiles * g.splits;
  const int half = split_half(g.r);
  const int blocks = half < 64 ? 1 : half / 64 * 2;  // stages per adapter

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], MODE == kWideWeight ? 1 + 2 * kConvWarps : 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&rfull[i], 2);  // the codes' bytes, the steps
      mbar_init(&rempty[i], kConvWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accf[i], 1);
      mbar_init(&acce[i], 2 * kEpiWarps);
    }
    mbar_init(&sfull, 1);
    mbar_init(&sempty, rank == 0 ? 2 : 1);
    mbar_init(&done, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  grid_release();
  const uint32_t tmem = s_tmem;

  auto item_at = [&](int i, int& tm, int& tn, int& sp, int& kb0, int& kb1) {
    sp = i / tiles;
    tile_at(g, i - sp * tiles, tm, tn);
    kb0 = (int)((int64_t)g.nkb * sp / g.splits);
    kb1 = (int)((int64_t)g.nkb * (sp + 1) / g.splits);
  };

  if (warp == 0) {
    if (lane == 0) {
      Ring rg(STAGES);
      bool ok = true, waited = false;
      int issued = 0;
      uint32_t sph = 0;
      for (int i = unit; ok && i < items; i += n_units) {
        int tm, tn, sp, kb0, kb1;
        item_at(i, tm, tn, sp, kb0, kb1);
        const int arow = tm * SUB * kTile + (int)rank * kHalf;
        const int bcol = tn * kTile + (int)rank * kHalf;
        // The halves [s0, s1) of A at contraction index ax, and B.
        auto load = [&](const CUtensorMap* ma, int ax, int s0, int s1, const CUtensorMap* mb, int bx,
                        int bz) {
          if (!mbar_wait(&empty[rg.s], rg.ph ^ 1, s_abort, g.status, g.budget_ns)) return false;
          if (rank == 0)
            mbar_arrive_expect_tx(&full[rg.s],
                                  2 * (s1 - s0 + (MODE == kWideWeight ? 0 : 1)) * kABytes);
          const uint32_t fb = mapa_u32(&full[rg.s], 0);
          uint8_t* st = smem + rg.s * kStageBytes;
          for (int s = s0; s < s1; ++s) {
            uint8_t* a = st + s * kABytes;
            const int row = arow + s * kTile;
            if constexpr (AMN) {
              tma_load_3d_pair(a, ma, fb, row, ax, 0);
              tma_load_3d_pair(a + 8192, ma, fb, row + 64, ax, 0);
            } else {
              tma_load_3d_pair(a, ma, fb, ax, row, 0);
            }
          }
          uint8_t* b = st + kBOff;
          if constexpr (MODE == kWideForward) {
            tma_load_3d_pair(b, mb, fb, bx, bcol, bz);
          } else if constexpr (MODE == kWideBack) {
            tma_load_3d_pair(b, mb, fb, bcol, bx, bz);
            tma_load_3d_pair(b + 8192, mb, fb, bcol + 64, bx, bz);
          }
          rg.next();
          ++issued;
          return true;
        };
        for (int kb = kb0; ok && kb < kb1; ++kb) ok = load(&mapA, kb * kKB, 0, SUB, &mapB, kb * kKB, 0);
        if (MODE != kWideWeight && g.r > 0) {
          if (!waited) grid_wait();  // the split T comes from the kernel before this one
          waited = true;
          ok = ok && mbar_wait(&sfull, sph, s_abort, g.status, g.budget_ns);
          for (int s = 0; ok && s < SUB; ++s)
            for (int j = 0; ok && j < slots[s].n; ++j)
              for (int b = 0; ok && b < blocks; ++b)
                ok = load(&mapT, blocks == 1 ? 0 : (b & 1) * half + (b >> 1) * 64, s, s + 1, &mapBi,
                          blocks == 1 ? 0 : (b >> 1) * 64, slots[s].id[j]);
          if (ok) mbar_arrive(&sempty);
          sph ^= 1;
        }
      }
      if (!waited) grid_wait();
      // Drain: every copy lands before shared memory is released (the even
      // CTA's full barriers count both CTAs' bytes).
      if (rank == 0) ring_drain(full, STAGES, issued, g.status, g.budget_ns);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = umma_idesc_16(BF16, kTile, kTile, AMN, BMN);
      Ring rg(STAGES);
      bool ok = true;
      int it = 0;
      uint32_t sph = 0;
      auto desc_a = [](uint32_t a, int kk) {
        return AMN ? umma_desc_mn128(a + kk * 2048, 8192) : umma_desc_sw128(a + kk * 32);
      };
      auto desc_b = [](uint32_t b, int kk) {
        return BMN ? umma_desc_mn128(b + kk * 2048, 8192) : umma_desc_sw128(b + kk * 32);
      };
      // One stage's MMAs into accumulator `buf` from half s of A.
      auto multiply = [&](int slot, int s, int buf, bool fresh) {
        const uint32_t a0 = smem_u32(smem + slot * kStageBytes) + s * kABytes;
        const uint32_t b0 = smem_u32(smem + slot * kStageBytes) + kBOff;
#pragma unroll
        for (int kk = 0; kk < kKB / 16; ++kk)
          umma_bf16_pair(tmem + buf * kTile, desc_a(a0, kk), desc_b(b0, kk), idesc, !fresh || kk != 0);
      };
      // The converters of both CTAs arrive at the stages of a weight product.
      auto loaded = [&] {
        const bool k = MODE == kWideWeight
                           ? mbar_wait_cluster(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns)
                           : mbar_wait(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns);
        tc_fence_after();
        return k;
      };
      auto free_acc = [&](int buf, uint32_t parity) {
        const bool k = mbar_wait(&acce[buf], parity, s_abort, g.status, g.budget_ns);
        tc_fence_after();
        return k;
      };
      for (int i = unit; ok && i < items; i += n_units) {
        int tm, tn, sp, kb0, kb1;
        item_at(i, tm, tn, sp, kb0, kb1);
        int buf = 0;
        if constexpr (SUB == 1) {
          int head = kb0;  // first stage of this accumulator's chain
          for (int kb = kb0; kb < kb1; ++kb) {
            if (kb == kb0 || kb - head == g.chain) {
              if (kb != kb0) umma_commit_pair(&accf[buf], 0x3);
              buf = it & 1;
              head = kb;
              if (!(ok = free_acc(buf, ((it >> 1) & 1) ^ 1))) break;
              ++it;
            }
            if (!(ok = loaded())) break;
            multiply(rg.s, 0, buf, kb == head);
            umma_commit_pair(&empty[rg.s], 0x3);
            rg.next();
          }
        } else {
          // The upper half's MMAs of the first stages, as many as the ring
          // holds, while the epilogue still reads the lower half.
          const int first = kb1 - kb0 < STAGES ? kb1 - kb0 : STAGES;
          if (!(ok = free_acc(0, (it & 1) ^ 1))) break;
          Ring low = rg;
          for (int k = 0; k < first; ++k) {
            if (!(ok = loaded())) break;
            multiply(rg.s, 0, 0, k == 0);
            rg.next();
          }
          if (!ok || !(ok = free_acc(1, (it & 1) ^ 1))) break;
          for (int k = 0; k < first; ++k) {
            multiply(low.s, 1, 1, k == 0);
            umma_commit_pair(&empty[low.s], 0x3);
            low.next();
          }
          for (int kb = kb0 + first; kb < kb1; ++kb) {
            if (!(ok = loaded())) break;
            multiply(rg.s, 0, 0, false);
            multiply(rg.s, 1, 1, false);
            umma_commit_pair(&empty[rg.s], 0x3);
            rg.next();
          }
          ++it;
        }
        if constexpr (MODE != kWideWeight) {
          if (g.r > 0) {
            ok = ok && mbar_wait(&sfull, sph, s_abort, g.status, g.budget_ns);
            for (int s = 0; ok && s < SUB; ++s) {
              const uint32_t d = tmem + (SUB == 1 ? buf : s) * kTile;
              for (int j = 0; ok && j < slots[s].n; ++j) {
                uint32_t off[8];
#pragma unroll
                for (int w = 0; w < 8; ++w) off[w] = slots[s].off[j][w];
                for (int b = 0; b < blocks; ++b) {
                  ok = mbar_wait(&full[rg.s], rg.ph, s_abort, g.status, g.budget_ns);
                  if (!ok) break;
                  tc_fence_after();
                  const uint32_t a0 = smem_u32(smem + rg.s * kStageBytes) + s * kABytes;
                  const uint32_t b0 = smem_u32(smem + rg.s * kStageBytes) + kBOff;
                  const int left = g.r - (b >> 1) * 64;
                  const int steps = left >= 64 ? 4 : (left + 15) / 16;
                  for (int kk = 0; kk < steps; ++kk) {
                    umma_16_masked_pair(d, desc_a(a0, kk), desc_b(b0, kk), idesc, 1, off);
                    if (blocks == 1)
                      umma_16_masked_pair(d, umma_desc_sw128(a0 + 64 + kk * 32), desc_b(b0, kk),
                                          idesc, 1, off);
                  }
                  umma_commit_pair(&empty[rg.s], 0x3);
                  rg.next();
                }
              }
              if (SUB == 2 && ok) umma_commit_pair(&accf[s], 0x3);
            }
            if (ok) mbar_arrive(&sempty);
            sph ^= 1;
          }
        }
        if (!ok) break;
        if (SUB == 1) {
          umma_commit_pair(&accf[buf], 0x3);
        } else if (MODE == kWideWeight || g.r == 0) {
          umma_commit_pair(&accf[0], 0x3);
          umma_commit_pair(&accf[1], 0x3);
        }
      }
      umma_commit_pair(&done, 0x1);
      mbar_wait(&done, 0, nullptr, g.status, g.budget_ns);
    }
    __syncwarp();
  } else if (warp < kWork) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, cbeg = (warp - 2) / 4 * (kTile / 2);
    uint8_t* turn = sRaw + RAW * kRawBytes + (warp - 2) * kTurnBytes;
    int it = 0;
    bool ok = true;
    auto drain = [&](int buf, uint32_t parity, int64_t row0, int tn, int sp, bool add) {
      if (!mbar_wait(&accf[buf], parity, s_abort, g.status, g.budget_ns)) return false;
      tc_fence_after();
      const int64_t row = row0 + rank * kHalf + q * 32 + lane;
      const int64_t col0 = (int64_t)tn * kTile + cbeg;
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + buf * kTile + cbeg;
#pragma unroll 1
      for (int c = 0; c < kTile / 2; c += 32) {
        uint32_t v[32];
        tmem_ld32(acc + c, v);
        tmem_wait_ld();
        if (c == kTile / 2 - 32) {
          // This half of the accumulator is read.
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(&acce[buf], 0));
        }
        const int64_t left = g.N - (col0 + c), first = row - lane;
        if (first >= g.M || left <= 0) continue;
        const int n = left < 32 ? (int)left : 32;
        if (g.splits > 1) {
          if (row < g.M)  // (padded to whole pieces)
            store_f32(g.partial + ((int64_t)sp * g.M + row) * g.ldp + col0 + c, true, v, add);
        } else if (g.o_vec && n == 32) {
          if (row >= g.M) continue;
          if (g.out_f32)
            store_f32((float*)g.out + row * g.ldo + col0 + c, g.o_vec > 1, v, add || g.accumulate);
          else
            store_16((uint16_t*)g.out + row * g.ldo + col0 + c, g.o_vec > 1, v, g.accumulate, BF16);
        } else {
          const int rows = g.M - first < 32 ? (int)(g.M - first) : 32;
          const int64_t at = first * g.ldo + col0 + c;
          store_turned(turn, v, rows, n, [&](int r, int i, float x) {
            if (g.out_f32) {
              float* o = (float*)g.out + at + r * g.ldo + i;
              *o = x + (add || g.accumulate ? *o : 0.0f);
            } else {
              uint16_t* o = (uint16_t*)g.out + at + r * g.ldo + i;
              *o = round16(BF16, x + (g.accumulate ? widen16(BF16, *o) : 0.0f));
            }
          });
        }
      }
      return true;
    };
    for (int i = unit; ok && i < items; i += n_units) {
      int tm, tn, sp, kb0, kb1;
      item_at(i, tm, tn, sp, kb0, kb1);
      const int64_t row0 = (int64_t)tm * SUB * kTile;
      if constexpr (SUB == 1) {
        // (Each thread adds to sums that it has written itself.)
        for (int head = kb0; ok && head < kb1; head += g.chain, ++it)
          ok = drain(it & 1, (it >> 1) & 1, row0, tn, sp, head != kb0);
      } else {
        for (int s = 0; ok && s < 2; ++s) ok = drain(s, it & 1, row0 + s * kTile, tn, sp, false);
        ++it;
      }
    }
  } else if constexpr (MODE == kWideWeight) {
    if (warp == kWork + 2 * kConvWarps) {
      // ------------------------------------------- codes' copies and steps
      Ring rr(RAW);
      bool ok = true;
      int raws = 0;
      for (int i = unit; ok && i < items; i += n_units) {
        int tm, tn, sp, kb0, kb1;
        item_at(i, tm, tn, sp, kb0, kb1);
        const int64_t group = (int64_t)tn * 2 + rank;
        const bool inside = group * kGroup < g.N;
        const int8_t* ex = g.exps + (inside ? group * g.C : 0);
        constexpr int AHEAD = 4;  // stages whose exponents are in flight
        int e[AHEAD][2];
        auto fetch = [&](int kb, int (&v)[2]) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t m = (int64_t)kb * kKB + h * 32 + lane;
            v[h] = inside && kb < kb1 && m < g.C ? (int)__ldg(ex + m) : 0;
          }
        };
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) fetch(kb0 + a, e[a]);
        for (int kb = kb0; ok && kb < kb1; kb += AHEAD) {
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            if (kb + a >= kb1) break;
            ok = mbar_wait(&rempty[rr.s], rr.ph ^ 1, s_abort, g.status, g.budget_ns);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&rfull[rr.s], kRawBytes);
              tma_load_3d(sRaw + rr.s * kRawBytes, &mapB, &rfull[rr.s],
                          tn * kTile + (int)rank * kHalf, (kb + a) * kKB, 0);
            }
            ++raws;
            steps[rr.s][lane] = exp_pair(BF16, e[a][0]);
            steps[rr.s][lane + 32] = exp_pair(BF16, e[a][1]);
            fetch(kb + a + AHEAD, e[a]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&rfull[rr.s]);
            rr.next();
          }
        }
      }
      ring_drain(rfull, RAW, raws, g.status, g.budget_ns);
    } else {
      // ---------------------------------------------------------- converters
      // Thread: rows t / 16 + 8 j of the stage, 8 columns at 8 (t % 16); lanes
      // of a half warp write one row's 16-byte pieces, eight to a 128-byte line.
      const int cg = (warp - kWork) / kConvWarps;  // converter group
      const int t = (threadIdx.x - 32 * kWork) % (32 * kConvWarps);
      const int piece = t & 15, r0 = t >> 4;
      const uint32_t to = smem_u32(smem) + kBOff + (piece >> 3) * 8192;
      Ring rg(STAGES), rr(RAW);
      bool ok = true;
      int turn = 0;
      for (int i = unit; ok && i < items; i += n_units) {
        int tm, tn, sp, kb0, kb1;
        item_at(i, tm, tn, sp, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb, turn ^= 1, rg.next(), rr.next()) {
          if (turn != cg) continue;
          ok = mbar_wait(&rfull[rr.s], rr.ph, s_abort, g.status, g.budget_ns);
          if (!ok) break;
          uint2 q[8];
          uint32_t sc[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            q[j] = *(const uint2*)(sRaw + rr.s * kRawBytes + (r0 + 8 * j) * kHalf + piece * 8);
            sc[j] = steps[rr.s][r0 + 8 * j];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&rempty[rr.s]);
          ok = mbar_wait(&empty[rg.s], rg.ph ^ 1, s_abort, g.status, g.budget_ns);
          if (!ok) break;
          const uint32_t at0 = to + rg.s * kStageBytes + r0 * 128 +
                               (((uint32_t)(piece & 7) ^ (uint32_t)(r0 & 7)) << 4);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
            codes_to_16(BF16, q[j].x, sc[j], w[0], w[1]);
            codes_to_16(BF16, q[j].y, sc[j], w[2], w[3]);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at0 + j * 1024), "r"(w[0]),
                         "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(&full[rg.s], 0));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ adapter lists
    uint32_t ph = 0;
    for (int i = unit; g.r > 0 && i < items; i += n_units) {
      int tm, tn, sp, kb0, kb1;
      item_at(i, tm, tn, sp, kb0, kb1);
      if (!mbar_wait(&sempty, ph ^ 1, s_abort, g.status, g.budget_ns)) break;
      for (int s = 0; s < SUB; ++s)
        build_slots<8>(g.ids, ((int64_t)tm * SUB + s) * kTile, g.M, g.E,
                       (SlotList<8>*)(void*)&slots[s], lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sfull);
      ph ^= 1;
    }
  }
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Sum of the contraction's parts, in order, into the output.
__global__ void k_wide_join(const float* part, int splits, int64_t M, int64_t N, int64_t ldp,
                            void* out, int64_t ldo, int out_f32, int bf16, int accumulate) {
  const int64_t n = M * N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / N, c = i - r * N, at = r * ldo + c;
    float s = 0.0f;
    for (int q = 0; q < splits; ++q) s += part[(q * M + r) * ldp + c];
    if (out_f32) {
      float* o = (float*)out + at;
      *o = s + (accumulate ? *o : 0.0f);
    } else {
      uint16_t* o = (uint16_t*)out + at;
      *o = round16(bf16, s + (accumulate ? widen16(bf16, *o) : 0.0f));
    }
  }
}

// Parts of a weight product's contraction: as many as give every CTA pair a
// tile, each of at least 8 stages (512 indexes).
int wide_splits(int64_t M, int64_t N, int64_t C, int dev) {
  const int64_t tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
  const int units = device_sm_count(dev) / 2;
  const int64_t nkb = (C + kKB - 1) / kKB;
  int64_t s = units / tiles;
  if (s > nkb / 8) s = nkb / 8;
  return s < 2 ? 1 : (int)s;
}

// Rows of the output take 32-byte (2), 16-byte (1) or no (0) vector stores.
int wide_vec(const void* out, int64_t ldo, bool f32) {
  const uintptr_t bits = (uintptr_t)out | (uintptr_t)(ldo * (f32 ? 4 : 2));
  return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
}

template <WideMode MODE, int SUB>
int launch_mode(const WideProduct& p, WideArgs g, int dev, cudaStream_t stream) {
  using Cfg = WideCfg<MODE, SUB>;
  CUtensorMap ma, mb, mt, mbi;
  memset(&mt, 0, sizeof(mt));
  memset(&mbi, 0, sizeof(mbi));
  int rc;
  if (MODE == kWideWeight)
    rc = make_map(&ma, p.A, 2, p.M, p.C, 1, p.lda * 2, p.lda * 2 * p.C, 64, kKB, true);
  else
    rc = make_map(&ma, p.A, 2, p.C, p.M, 1, p.lda * 2, p.lda * 2 * p.M, kKB, kHalf, true);
  if (rc) return rc;
  if (MODE == kWideForward)
    rc = make_map(&mb, p.B, 2, p.C, p.N, 1, p.ldb * 2, p.ldb * 2 * p.N, kKB, kHalf, true);
  else if (MODE == kWideBack)
    rc = make_map(&mb, p.B, 2, p.N, p.C, 1, p.ldb * 2, p.ldb * 2 * p.C, 64, kKB, true);
  else
    rc = make_map(&mb, p.B, 1, p.ldb, p.C, 1, p.ldb, p.ldb * p.C, kHalf, kKB, false);
  if (rc) return rc;
  if (p.r > 0) {
    const int half = split_half(p.r);
    if ((rc = make_map(&mt, p.split, 2, 2 * half, p.M, 1, 4 * half, 4 * half * p.M, 64, kHalf,
                       true)))
      return rc;
    if (MODE == kWideForward)
      rc = make_map(&mbi, p.Bi, 2, p.r, p.N, p.E, p.ldbi * 2, p.ldbi * 2 * p.N, 64, kHalf, true);
    else
      rc = make_map(&mbi, p.Bi, 2, p.N, p.r, p.E, p.ldbi * 2, p.ldbi * 2 * p.r, 64, 64, true);
    if (rc) return rc;
  }
  auto kern = p.bf16 ? k_wide<MODE, true, SUB> : k_wide<MODE, false, SUB>;
  if ((rc = p.bf16 ? allow_smem<k_wide<MODE, true, SUB>>(Cfg::SMEM, dev)
                   : allow_smem<k_wide<MODE, false, SUB>>(Cfg::SMEM, dev)))
    return rc;
  const int items = g.tiles_m * g.tiles_n * g.splits;
  const int units = device_sm_count(dev) / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (items < units ? items : units)));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.early ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, ma, mb, mt, mbi, g);
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_wide launch", e);
}

}  // namespace

size_t wide_partial_bytes(int64_t M, int64_t N, int64_t C, int dev) {
  const int s = wide_splits(M, N, C, dev);
  return s > 1 ? (size_t)s * M * round_up(N, 32) * 4 : 0;
}

int launch_wide(const WideProduct& p, int dev, cudaStream_t stream) {
  WideArgs g = {};
  g.M = p.M;
  g.N = p.N;
  g.C = p.C;
  g.nkb = (int)((p.C + kKB - 1) / kKB);
  const int64_t tm = (p.M + kTile - 1) / kTile, tn = (p.N + kTile - 1) / kTile;
  if (tm * tn > (1 << 26)) return set_error(OZK_ERR_UNSUPPORTED, "too many output tiles");
  g.tiles_m = (int)tm;
  g.tiles_n = (int)tn;
  g.group_m = 8;
  g.splits = p.mode == kWideWeight && p.partial ? wide_splits(p.M, p.N, p.C, dev) : 1;
  // The tensor cores cut off what a sum's exponent leaves no room for, so an
  // error grows with the length of the chain: an FP32 result was 1.7e-5 off
  // after 16384 FP16 rows, 7e-7 after 1024.  FP32 results are summed in chains
  // of 1024.  16-bit results are not: 1.7e-5 changes 0.13% of the BF16 values of a
  // sum of 16384, each by one step.
  g.chain = p.out_f32 || g.splits > 1 ? 16 : 1 << 30;
  g.bf16 = p.bf16;
  g.out_f32 = p.out_f32;
  g.accumulate = p.accumulate;
  g.out = p.out;
  g.ldo = p.ldo;
  g.o_vec = wide_vec(p.out, p.ldo, p.out_f32);
  g.partial = p.partial;
  g.ldp = round_up(p.N, 32);
  g.exps = p.exps;
  g.ids = p.ids;
  g.r = p.r;
  g.E = p.E;
  g.status = p.status;
  g.budget_ns = wait_budget_ns();
  // Two tiles at once where that does not leave more CTA pairs idle in the last
  // round (a round of double tiles lasts 1.7 of a round of single ones).  FP32
  // results change accumulators every 1024 indexes, which only single tiles do
  // without a pause.
  const int units = device_sm_count(dev) / 2;
  const int64_t one = (tm * tn + units - 1) / units;
  const int64_t two = ((p.M + 2 * kTile - 1) / (2 * kTile) * tn + units - 1) / units;
  const bool twice = g.splits == 1 && !p.out_f32 && 17 * two <= 10 * one;
  if (twice) g.tiles_m = (int)((p.M + 2 * kTile - 1) / (2 * kTile));
  int rc;
  if (p.mode == kWideForward)
    rc = twice ? launch_mode<kWideForward, 2>(p, g, dev, stream)
               : launch_mode<kWideForward, 1>(p, g, dev, stream);
  else if (p.mode == kWideBack)
    rc = twice ? launch_mode<kWideBack, 2>(p, g, dev, stream)
               : launch_mode<kWideBack, 1>(p, g, dev, stream);
  else
    rc = twice ? launch_mode<kWideWeight, 2>(p, g, dev, stream)
               : launch_mode<kWideWeight, 1>(p, g, dev, stream);
  if (rc || g.splits == 1) return rc;
  int64_t blocks = (p.M * p.N + 255) / 256;
  if (blocks > 148 * 8) blocks = 148 * 8;
  k_wide_join<<<(unsigned)blocks, 256, 0, stream>>>(p.partial, g.splits, p.M, p.N, g.ldp, p.out,
                                                    p.ldo, p.out_f32, p.bf16, p.accumulate);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_wide_join launch", e);
}

}  // namespace ozk
