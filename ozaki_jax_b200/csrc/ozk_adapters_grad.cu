// Gradients of the low-rank adapters themselves:
//   dA_i = sum over the rows of adapter i of U_m^T X_m      [r][K]
//   dB_i = sum over the rows of adapter i of dY_m^T T_m     [N][r]
// Both are sums of outer products of a row of an FP32 matrix of r columns (U or
// T) with a long 16-bit row (X, or X^ from its int8 codes, or dY), over the
// rows that share an adapter: tall contractions with small outputs, bound by
// reading X and dY once.
//
// k_sort_rows lists the rows by adapter (stable, one CTA per adapter, no
// atomics on memory) and splits T into high and low 16-bit parts, as U already
// is.  k_outer cuts the list into chunks; a CTA takes one chunk and 256 columns,
// gathers 64 rows at a time into a ring of shared-memory stages (cp.async, three
// stages in flight: 96 KB per SM; codes are converted on the way to the tensor
// cores) and multiplies them: D[256 columns][2 r] += Z^T [hi | lo], the halves
// being added at the end (in FP16 lo is held 2^11 times as large, so that U and
// T count to 2^-36 however small they are; rows of a gradient of 1e-7 add up to
// values that FP16 holds).  One warp issues the MMAs (about 90 clocks each at
// these widths, bound by reading Z from shared memory) and one looks the next
// rows up, beside the sixteen that fetch: with the issue and the lookup in the
// fetching warps a stage took 5400 clocks.  Rows of other
// adapters are never read, so a NaN in them cannot reach this one's gradient.
// 4096 rows, N = K = 4096, r = 16: 34 us; 8192 rows, N = 4096, K = 8192 as codes,
// r = 32: 96 us, a stage of 64 rows taking about 3700 clocks, most of it the
// fetching warps' own chain of copies, conversion and barriers.
// A chunk that holds all of an adapter's rows writes its gradient at once;
// otherwise the chunks' FP32 sums are added in order by k_outer_join: the
// result does not depend on scheduling.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "ozk_adapters.h"
#include "ozk_tile16.cuh"

namespace ozk {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kOuterWarps = 16;  // that fetch and convert; two more issue MMAs and look rows up
constexpr int kOuterFetch = 32 * kOuterWarps;
constexpr int kOuterThreads = kOuterFetch + 64;
constexpr int kCols = 256;       // columns of Z per CTA: two accumulators of 128
constexpr int kStep = 64;        // rows per stage
constexpr int kZBytes = kCols * kStep * 2;

// order: the rows of adapters 0, 1, ... in turn, each adapter's in ascending
// order; start[e]: the first place of adapter e.
__global__ void __launch_bounds__(kSortThreads)
    k_sort_rows(const int32_t* ids, int64_t M, int E, int32_t* order, int32_t* start,
                const float* T, int r, uint16_t* split, int bf16) {
  grid_release();
  if ((int)blockIdx.x >= E) {  // the CTAs after the adapters': the split of T
    const int half = split_half(r);
    const int64_t n = M * half;
    for (int64_t i = (int64_t)((int)blockIdx.x - E) * kSortThreads + threadIdx.x; i < n;
         i += (int64_t)((int)gridDim.x - E) * kSortThreads) {
      const int64_t m = i / half;
      const int c = (int)(i - m * half);
      store_split(split, m, half, c, c < r ? T[m * r + c] : 0.0f, bf16, low_up(bf16));
    }
    return;
  }
  __shared__ int s_less, s_eq;
  __shared__ int s_warp[kSortThreads / 32];
  const int e = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  if (t == 0) s_less = s_eq = 0;
  __syncthreads();
  int less = 0, eq = 0;
  for (int64_t m = t; m < M; m += kSortThreads) {
    const int v = row_adapter(ids, m, M, E);
    less += v >= 0 && v < e;
    eq += v == e;
  }
  for (int o = 16; o; o >>= 1) {
    less += __shfl_xor_sync(~0u, less, o);
    eq += __shfl_xor_sync(~0u, eq, o);
  }
  if (lane == 0) {
    atomicAdd(&s_less, less);  // integers: the order of the additions does not matter
    atomicAdd(&s_eq, eq);
  }
  __syncthreads();
  int pos = s_less;
  if (t == 0) {
    start[e] = pos;
    if (e == E - 1) start[E] = pos + s_eq;
  }
  if (s_eq == 0) return;
  for (int64_t m0 = 0; m0 < M; m0 += kSortThreads) {
    const bool mine = row_adapter(ids, m0 + t, M, E) == e;
    const uint32_t b = __ballot_sync(~0u, mine);
    if (lane == 0) s_warp[warp] = __popc(b);
    __syncthreads();
    const int c = s_warp[lane];  // as many warps as lanes
    const int before = __reduce_add_sync(~0u, lane < warp ? c : 0), all = __reduce_add_sync(~0u, c);
    if (mine) order[pos + before + __popc(b & ((1u << lane) - 1))] = (int32_t)(m0 + t);
    pos += all;
    __syncthreads();
  }
}

struct OuterJob {
  const void* Z;         // 16-bit [M][C], or int8 codes when exps is set
  int64_t ldz, C;
  const int8_t* exps;    // [groups][M]
  const uint16_t* L;     // [M][2 split_half(r)]: high parts, low parts times low_up
  float* partial;        // [2 chunks][r C], see below
  void* out;             // [E][r][C], or [E][C][r] when trans
  int trans, tiles;
};

// Of the adapters in a chunk, only the first (continued from the chunk before)
// and the last (continued in the next) can have rows elsewhere: two places of
// partial sums per chunk, the second for an adapter that does not start it.

struct OuterArgs {
  OuterJob job[2];
  const int32_t *order, *start;
  int64_t M;
  int E, r, rp, bf16;
  int len;               // places of the order per chunk, a multiple of kStep
  int32_t* status;
  uint64_t budget_ns;
};

// A word of the row lists.  k_sort_rows may still be writing them when a later
// kernel of the call starts, so they are read after grid_wait() and by an
// ordinary load that stays there: __ldg's path wants data that nobody writes
// while the kernel runs, and its loads may be moved before the wait.
__device__ __forceinline__ int32_t load_listed(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// The stages of a chunk: up to 64 places [pos, end) of one adapter's rows at a time.
struct Walk {
  int e, pos, end, first;  // end: of this adapter's rows in the chunk
  __device__ void seek(const int32_t* start, int E, int limit) {
    while (e < E && load_listed(start + e + 1) <= pos) ++e;
    if (e >= E || pos >= limit) {
      e = E;
      return;
    }
    const int b = load_listed(start + e + 1);
    end = b < limit ? b : limit;
    first = pos;
  }
  __device__ bool last() const { return pos + kStep >= end; }
  __device__ void next(const int32_t* start, int E, int limit) {
    if (e >= E) return;
    if (!last()) {
      pos += kStep;
    } else {
      pos = end;
      seek(start, E, limit);
    }
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kRowSlots = 8;  // stages whose row numbers are held

struct OuterShared {
  uint64_t empty[4], done;
  uint32_t tmem;
  int abort;
  int rows[kRowSlots][kStep];
};

// One chunk and 256 columns.  A stage holds Z (32 KB, or 16 KB of codes) and
// L's rows, high parts then low parts; with CODES two buffers of 32 KB behind the ring take
// the converted Z in turn.
template <bool BF16, bool CODES, int S>
__device__ void outer_body(const OuterArgs& g, const OuterJob& job, int64_t col0, int chunk,
                           int limit, uint8_t* smem, OuterShared& sh) {
  constexpr int Z_STAGE = CODES ? kZBytes / 2 : kZBytes;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int stage_bytes = Z_STAGE + (2 * g.rp + 63) / 64 * 8192;
  uint8_t* conv = smem + S * stage_bytes;
  const uint32_t tmem = sh.tmem;
  volatile int* s_abort = &sh.abort;
  const int half = split_half(g.r);
  const bool fetcher = warp < kOuterWarps;

  // The first adapter of the chunk: the last e with start[e] <= its first place.
  Walk cur;
  cur.pos = chunk * g.len;
  {
    int lo = 0, hi = g.E - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (load_listed(g.start + mid) <= cur.pos) lo = mid;
      else hi = mid - 1;
    }
    cur.e = lo;
    cur.seek(g.start, g.E, limit);
  }
  // cur: the stage being multiplied; ahead: the one whose row numbers come next.
  Walk ahead = cur;
  auto number_rows = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kStep; i += 32) {
      const int p = ahead.pos + i + lane;
      sh.rows[stage % kRowSlots][i + lane] = ahead.e < g.E && p < ahead.end ? load_listed(g.order + p) : -1;
    }
    ahead.next(g.start, g.E, limit);
  };
  // A thread fetches 16 bytes of each of FETCH rows: 8 columns of four rows, a
  // warp a row; or 16 codes of two rows, a half warp a row.
  constexpr int FETCH = CODES ? 2 : 4;
  const int row0 = CODES ? 2 * warp + (lane >> 4) : warp;
  constexpr int ROW_STEP = CODES ? 2 * kOuterWarps : kOuterWarps;
  const int at_col = CODES ? (lane & 15) * 16 : lane * 8;
  const int64_t col = col0 + at_col;
  // This thread's 16-byte pieces of L's parts: the row, where it comes from in
  // that row, where it goes in a stage.
  const int lp = g.rp / 8, pieces = 2 * kStep * lp;
  int l_row[4], l_from[4];
  uint32_t l_to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = t + i * kOuterFetch;
    const int r = q / (2 * lp), c = q - r * 2 * lp;  // piece c of the row's 2 lp
    const int part = c >= lp;
    l_row[i] = q < pieces ? r : -1;
    l_from[i] = 2 * (part * half + (c - part * lp) * 8);
    l_to[i] = Z_STAGE + (c >> 3) * 8192 + r * 128 + (((uint32_t)(c & 7) ^ (uint32_t)(r & 7)) << 4);
  }
  // What does not change from stage to stage: this lane's bytes of a row of Z
  // (its 8 columns, or those of them inside the matrix) and where they go.
  const int64_t left = (CODES ? job.ldz : job.C) - col;
  const uint32_t z_bytes = left <= 0 ? 0 : CODES ? 16 : left < 8 ? 2 * (uint32_t)left : 16;
  const int64_t z_pitch = job.ldz * (CODES ? 1 : 2);
  const char* z_from = (const char*)job.Z + (z_bytes ? col * (CODES ? 1 : 2) : 0);
  // Where 8 columns of row r belong in the MMA's layout.
  auto place = [](int r, int c) {
    return (uint32_t)((c >> 6) * 8192 + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4));
  };
  uint32_t z_to[FETCH];
#pragma unroll
  for (int j = 0; j < FETCH; ++j) {
    const int r = row0 + ROW_STEP * j;
    z_to[j] = CODES ? r * 256 + at_col : place(r, at_col);
  }
  const char* l_base = (const char*)job.L;
  const int l_pitch = 4 * half;
  auto load = [&](uint32_t zb, const int* rows) {
#pragma unroll
    for (int j = 0; j < FETCH; ++j) {
      const int row = rows[row0 + ROW_STEP * j];
      const char* p = z_from + (row >= 0 ? row : 0) * z_pitch;
      const uint32_t n = row >= 0 ? z_bytes : 0;
      cp_async16(zb + z_to[j], p, n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (l_row[i] < 0) break;
      const int row = rows[l_row[i]];
      cp_async16(zb + l_to[i], l_base + (int64_t)(row >= 0 ? row : 0) * l_pitch + l_from[i],
                 row >= 0 ? 16 : 0);
    }
  };
  // Exponents of a stage: lane 4 j + 2 h + g holds row row0 + 32 j of half warp h
  // in column group g.  (Turned into 16-bit steps when they are used, an
  // iteration later.)
  auto exponents = [&](int stage) {
    if (!CODES || !fetcher || lane >= 8) return 0;
    const int row = sh.rows[stage % kRowSlots][2 * warp + (lane >> 1 & 1) + ROW_STEP * (lane >> 2)];
    const int64_t group = col0 / kGroup + (lane & 1);
    return row >= 0 && group * kGroup < job.ldz ? (int)__ldg(job.exps + group * g.M + row) : 0;
  };

  if (warp == kOuterWarps + 1)
    for (int k = 0; k < S; ++k) number_rows(k);
  __syncthreads();
  if (fetcher)
    for (int k = 0; k < S - 1; ++k) {
      load(smem_u32(smem) + k * stage_bytes, sh.rows[k]);
      cp_async_commit();
    }
  int ex = exponents(0);
  const uint32_t idesc = umma_idesc_16(BF16, 128, 2 * g.rp, true, true);
  uint32_t done_ph = 0;
  bool ok = true;
  int slot = 0, before = S - 1;        // ring places of this stage and of the one before it
  uint32_t ph = 0, before_ph = 1;      // phase parity of their uses
  for (int it = 0; cur.e < g.E; ++it) {
    uint8_t* st = smem + slot * stage_bytes;
    cp_async_wait<S - 2>();
    const uint32_t z0 = CODES ? smem_u32(conv + (it & 1) * kZBytes) : smem_u32(st);
    if (CODES && fetcher) {
      const uint32_t steps = exp_pair(BF16, ex);
      // Every thread converts the pieces that it fetched.  (The multiplication
      // two stages ago, which read this buffer, has been waited for.)
#pragma unroll
      for (int j = 0; j < FETCH; ++j) {
        const int r = row0 + ROW_STEP * j;
        const uint4 q = *(const uint4*)(st + z_to[j]);
        const uint32_t step = __shfl_sync(~0u, steps, 4 * j + 2 * (lane >> 4) + (at_col >> 7));
        uint32_t w[8];
        codes_to_16(BF16, q.x, step, w[0], w[1]);
        codes_to_16(BF16, q.y, step, w[2], w[3]);
        codes_to_16(BF16, q.z, step, w[4], w[5]);
        codes_to_16(BF16, q.w, step, w[6], w[7]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(z0 + place(r, at_col + 8 * h)),
                       "r"(w[4 * h]), "r"(w[4 * h + 1]), "r"(w[4 * h + 2]), "r"(w[4 * h + 3])
                       : "memory");
      }
    }
    fence_proxy_async_smem();
    if (__syncthreads_or(!ok)) break;  // all threads leave together
    const bool fresh = cur.pos == cur.first, last = cur.last();
    if (t == kOuterFetch) {
      tc_fence_after();
      const uint32_t l0 = smem_u32(st) + Z_STAGE;
#pragma unroll
      for (int kk = 0; kk < kStep / 16; ++kk)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          umma_bf16(tmem + mb * 2 * g.rp, umma_desc_mn128(z0 + mb * 16384 + kk * 2048, 8192),
                    umma_desc_mn128(l0 + kk * 2048, 8192), idesc, !fresh || kk != 0);
        }
      umma_commit(&sh.empty[slot]);
      if (last) umma_commit(&sh.done);
    }
    // Refill: the stage before this one is free once its multiplication is done.
    if (fetcher) {
      if (it > 0) ok = mbar_wait(&sh.empty[before], before_ph, s_abort, g.status, g.budget_ns);
      if (ok) load(smem_u32(smem) + before * stage_bytes, sh.rows[(it + S - 1) % kRowSlots]);
      cp_async_commit();
      ex = exponents(it + 1);
    } else if (warp == kOuterWarps + 1) {
      number_rows(it + S);
    }
    __syncwarp();
    before = slot;
    before_ph = ph;
    if (++slot == S) {
      slot = 0;
      ph ^= 1;
    }
    const Walk was = cur;
    cur.next(g.start, g.E, limit);
    if (last) {
      // One adapter's rows are through: its sums of this chunk.
      ok = mbar_wait(&sh.done, done_ph, s_abort, g.status, g.budget_ns) && ok;
      done_ph ^= 1;
      if (__syncthreads_or(!ok)) break;
      tc_fence_after();
      const bool whole = was.first == load_listed(g.start + was.e) && was.end == load_listed(g.start + was.e + 1);
      const int mb = (warp >> 2) & 1, q = warp & 3;
      const int64_t c = col0 + mb * 128 + q * 32 + lane;
      const int64_t part = (int64_t)(2 * chunk + (was.first != chunk * g.len)) * g.r * job.C;
      const int64_t base = (int64_t)was.e * g.r * job.C;
      for (int k0 = (warp >> 3) * 16; fetcher && k0 < g.rp; k0 += 32) {  // two warps share a quadrant
        uint32_t v[16], w[16];
        const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + mb * 2 * g.rp + k0;
        tmem_ld16(at, v);
        tmem_ld16(at + g.rp, w);
        tmem_wait_ld();
        if (c >= job.C) continue;
        float sum[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          // An infinity says so in the high parts' sum; times a low part that is
          // zero or of the other sign it would become a NaN.
          const float h = __uint_as_float(v[k]);
          sum[k] = fabsf(h) < INFINITY ? fmaf(__uint_as_float(w[k]), low_down(BF16), h) : h;
        }
        if (job.trans && (g.r & 7) == 0) {
          // a thread's ranks lie side by side: 8 at a time
#pragma unroll
          for (int k = 0; k < 16; k += 8) {
            if (k0 + k >= g.r) break;
            const int64_t to = c * g.r + k0 + k;
            if (whole) {
              *(uint4*)((uint16_t*)job.out + base + to) =
                  make_uint4(pack16(BF16, sum[k], sum[k + 1]), pack16(BF16, sum[k + 2], sum[k + 3]),
                             pack16(BF16, sum[k + 4], sum[k + 5]), pack16(BF16, sum[k + 6], sum[k + 7]));
            } else {
              float4* o = (float4*)(job.partial + part + to);
              o[0] = make_float4(sum[k], sum[k + 1], sum[k + 2], sum[k + 3]);
              o[1] = make_float4(sum[k + 4], sum[k + 5], sum[k + 6], sum[k + 7]);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (k0 + k >= g.r) break;
            const int64_t to = job.trans ? c * g.r + k0 + k : (int64_t)(k0 + k) * job.C + c;
            if (whole) ((uint16_t*)job.out)[base + to] = round16(BF16, sum[k]);
            else job.partial[part + to] = sum[k];
          }
        }
      }
      tc_fence_before();
      __syncthreads();
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  if (*s_abort) {
    // MMAs still in flight after a wait that gave up end before TMEM is freed.
    if (t == kOuterFetch) umma_commit(&sh.done);
    mbar_wait(&sh.done, done_ph, nullptr, g.status, g.budget_ns);
  }
}

template <bool BF16, int S>
__global__ void __launch_bounds__(kOuterThreads, 1)
    k_outer(const __grid_constant__ OuterArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ OuterShared sh;
  grid_release();
  grid_wait();  // for U, by way of the kernels between them for the row lists
  const bool second = (int)blockIdx.x >= g.job[0].tiles;
  const OuterJob& job = g.job[second];
  const int64_t col0 = (int64_t)((int)blockIdx.x - (second ? g.job[0].tiles : 0)) * kCols;
  const int chunk = blockIdx.y;
  const int total = load_listed(g.start + g.E);
  const int limit = (chunk + 1) * g.len < total ? (chunk + 1) * g.len : total;
  if (chunk * g.len >= limit) return;  // the whole CTA: nothing is allocated yet
  uint32_t cols = 32;
  while (cols < 4u * g.rp) cols *= 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&sh.empty[i], 1);
    mbar_init(&sh.done, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < 32) tmem_alloc(&sh.tmem, cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (job.exps) outer_body<BF16, true, S>(g, job, col0, chunk, limit, smem, sh);
  else outer_body<BF16, false, S>(g, job, col0, chunk, limit, smem, sh);
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x < 32) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, cols);
  }
}

// Adapters whose rows lie in several chunks (or that have none).
__global__ void k_outer_join(const __grid_constant__ OuterArgs g) {
  grid_wait();
  const int e = blockIdx.y;
  const OuterJob& job = g.job[blockIdx.z];
  const int a = load_listed(g.start + e), b = load_listed(g.start + e + 1);
  const int c0 = a / g.len, c1 = b > a ? (b - 1) / g.len : c0 - 1;
  if (c0 == c1) return;
  const int64_t n = (int64_t)g.r * job.C;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    float s = 0.0f;
    for (int c = c0; c <= c1; ++c)
      s += job.partial[(int64_t)(2 * c + (c == c0 && a != c0 * g.len)) * n + i];
    ((uint16_t*)job.out)[e * n + i] = round16(g.bf16, s);
  }
}

// Rows per chunk: the most chunks that run at once, one CTA per SM, each of at
// least one stage (a second wave of a few CTAs would double the time).
int chunk_len(int64_t M, int64_t tiles, int sms) {
  int64_t chunks = sms / tiles;
  if (chunks < 1) chunks = 1;
  int64_t len = round_up((M + chunks - 1) / chunks, kStep);
  if (len > 8192) len = 8192;
  return (int)len;
}

}  // namespace

namespace {

// The scratch of one call.
struct OuterScratch {
  int32_t *order, *start;
  uint16_t* split;  // of T
  float *pa, *pb;
  int len;
  int64_t chunks, tiles;
};

OuterScratch outer_scratch(int64_t M, int64_t N, int64_t K, int r, int E, int dev, Arena& ws) {
  OuterScratch s;
  s.tiles = (N + kCols - 1) / kCols + (K + kCols - 1) / kCols;
  s.len = chunk_len(M, s.tiles, device_sm_count(dev));
  s.chunks = (M + s.len - 1) / s.len;
  s.order = ws.take<int32_t>((size_t)M * 4);
  s.start = ws.take<int32_t>((size_t)(E + 1) * 4);
  s.split = ws.take<uint16_t>((size_t)M * 4 * split_half(r));
  s.pa = ws.take<float>((size_t)2 * s.chunks * r * K * 4);
  s.pb = ws.take<float>((size_t)2 * s.chunks * r * N * 4);
  return s;
}

// A launch that may begin while the kernel before it, which has released it,
// still runs; the kernel waits for that one itself.
template <typename K>
int launch_early(const char* what, K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                 const OuterArgs& g) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, g);
  return e == cudaSuccess ? OZK_OK : set_cuda_error(what, e);
}

}  // namespace

size_t outer_scratch_bytes(int64_t M, int64_t N, int64_t K, int r, int E, int dev) {
  Arena ws(nullptr);
  outer_scratch(M, N, K, r, E, dev, ws);
  return ws.used;
}

int launch_outer_rows(const OuterProduct& p, void* scratch, int dev, cudaStream_t stream) {
  Arena ws(scratch);
  const OuterScratch o = outer_scratch(p.M, p.N, p.K, p.r, p.E, dev, ws);
  int64_t more = (p.M * split_half(p.r) + 4 * kSortThreads - 1) / (4 * kSortThreads);
  if (more > 148) more = 148;
  k_sort_rows<<<(unsigned)(p.E + more), kSortThreads, 0, stream>>>(
      p.ids, p.M, p.E, o.order, o.start, p.T, p.r, o.split, p.bf16);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_sort_rows launch", e);
}

int launch_outer(const OuterProduct& p, void* scratch, int dev, cudaStream_t stream) {
  Arena ws(scratch);
  const OuterScratch sc = outer_scratch(p.M, p.N, p.K, p.r, p.E, dev, ws);
  if (sc.chunks > 65535) return set_error(OZK_ERR_UNSUPPORTED, "too many rows");
  OuterArgs g = {};
  g.M = p.M;
  g.E = p.E;
  g.r = p.r;
  g.rp = (p.r + 15) / 16 * 16;
  g.bf16 = p.bf16;
  g.status = p.status;
  g.budget_ns = wait_budget_ns();
  g.order = sc.order;
  g.start = sc.start;
  g.len = sc.len;
  OuterJob& a = g.job[0];
  a.Z = p.X;
  a.ldz = p.ldx;
  a.C = p.K;
  a.exps = p.exps;
  a.L = p.U;
  a.partial = sc.pa;
  a.out = p.dA;
  a.tiles = (int)((p.K + kCols - 1) / kCols);
  OuterJob& b = g.job[1];
  b.Z = p.dY;
  b.ldz = p.ldy;
  b.C = p.N;
  b.L = sc.split;
  b.partial = sc.pb;
  b.out = p.dB;
  b.trans = 1;
  b.tiles = (int)((p.N + kCols - 1) / kCols);
  // One CTA per SM: as many stages, up to four, as fit.
  const int l_bytes = (2 * g.rp + 63) / 64 * 8192;
  const int stages = l_bytes > 16384 ? 3 : 4;
  size_t smem = (size_t)stages * (kZBytes + l_bytes);
  const size_t coded = (size_t)stages * (kZBytes / 2 + l_bytes) + 2 * kZBytes;
  if (p.exps && smem < coded) smem = coded;
  smem += 1024;
  if (smem < tmem_share(4 * g.rp)) smem = tmem_share(4 * g.rp);
  auto kern = p.bf16 ? (stages == 4 ? k_outer<true, 4> : k_outer<true, 3>)
                     : (stages == 4 ? k_outer<false, 4> : k_outer<false, 3>);
  int rc = p.bf16 ? (stages == 4 ? allow_smem<k_outer<true, 4>>(smem, dev)
                                 : allow_smem<k_outer<true, 3>>(smem, dev))
                  : (stages == 4 ? allow_smem<k_outer<false, 4>>(smem, dev)
                                 : allow_smem<k_outer<false, 3>>(smem, dev));
  if (rc) return rc;
  rc = launch_early("k_outer launch", kern, dim3((unsigned)sc.tiles, (unsigned)sc.chunks),
                    kOuterThreads, smem, stream, g);
  if (rc) return rc;
  const int64_t most = (int64_t)p.r * (p.K > p.N ? p.K : p.N);
  int64_t blocks = (most + 1023) / 1024;
  if (blocks > 256) blocks = 256;
  return launch_early("k_outer_join launch", k_outer_join,
                      dim3((unsigned)blocks, (unsigned)p.E, 2), 256, 0, stream, g);
}

}  // namespace ozk
