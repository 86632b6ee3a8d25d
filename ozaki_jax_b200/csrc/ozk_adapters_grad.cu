// Gradients of the low-rank adapters themselves:
//   dA_i = sum over the rows of adapter i of U_m^T X_m      [r][K]
//   dB_i = sum over the rows of adapter i of dY_m^T T_m     [N][r]
// Both are sums of outer products of a row of an FP32 matrix of r columns (U or
// T) with a long 16-bit row (X, or X^ from its int8 codes, or dY), over the
// rows that share an adapter: tall contractions with small outputs, bound by
// reading X and dY once.
//
// k_sort_rows lists the rows by adapter (stable, one CTA per adapter, no
// atomics).  k_outer cuts that list into chunks; a CTA takes one chunk and 256
// columns, gathers 64 rows at a time into shared memory (converting codes, and
// splitting U or T into high and low 16-bit parts, on the way) and multiplies
// them on the tensor cores: D[256 columns][r] += Z^T [hi | lo].  Rows of other
// adapters are never read, so a NaN in them cannot reach this one's gradient.
// A chunk that holds all of an adapter's rows writes its gradient at once;
// otherwise the chunks' FP32 sums are added in order by k_outer_join: the
// result does not depend on scheduling.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "ozk_adapters.h"
#include "ozk_tile16.cuh"

namespace ozk {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kOuterThreads = 256;
constexpr int kCols = 256;       // columns of Z per CTA: two accumulators of 128
constexpr int kStep = 64;        // rows per stage
constexpr int kZBytes = kCols * kStep * 2;

// order: the rows of adapters 0, 1, ... in turn, each adapter's in ascending
// order; start[e]: the first place of adapter e.
__global__ void __launch_bounds__(kSortThreads)
    k_sort_rows(const int32_t* ids, int64_t M, int E, int32_t* order, int32_t* start) {
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
    int before = 0, all = 0;
    for (int w = 0; w < kSortThreads / 32; ++w) {
      const int c = s_warp[w];
      before += w < warp ? c : 0;
      all += c;
    }
    if (mine) order[pos + before + __popc(b & ((1u << lane) - 1))] = (int32_t)(m0 + t);
    pos += all;
    __syncthreads();
  }
}

struct OuterJob {
  const void* Z;         // 16-bit [M][C], or int8 codes when exps is set
  int64_t ldz, C;
  const int8_t* exps;    // [groups][M]
  const float* L;        // [M][r]
  float* partial;        // [chunks + E][r C]
  void* out;             // [E][r][C], or [E][C][r] when trans
  int trans, tiles, vec;
};

struct OuterArgs {
  OuterJob job[2];
  const int32_t *order, *start;
  int64_t M;
  int E, r, rp, bf16;
  int len;               // places of the order per chunk, a multiple of kStep
  int32_t* status;
  uint64_t budget_ns;
};

// The stages of a chunk: up to 64 places [pos, end) of one adapter's rows at a time.
struct Walk {
  int e, pos, end, first;  // end: of this adapter's rows in the chunk
  __device__ void seek(const int32_t* start, int E, int limit) {
    while (e < E && __ldg(start + e + 1) <= pos) ++e;
    if (e >= E || pos >= limit) {
      e = E;
      return;
    }
    const int b = __ldg(start + e + 1);
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

template <bool BF16>
__global__ void __launch_bounds__(kOuterThreads, 2)
    k_outer(const __grid_constant__ OuterArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t empty[2], done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_rows[2][kStep];
  __shared__ int s_abort_word;
  volatile int* s_abort = &s_abort_word;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const bool second = (int)blockIdx.x >= g.job[0].tiles;
  const OuterJob& job = g.job[second];
  const int64_t col0 = (int64_t)((int)blockIdx.x - (second ? g.job[0].tiles : 0)) * kCols;
  const int chunk = blockIdx.y;
  const int total = __ldg(g.start + g.E);
  const int c0 = chunk * g.len;
  const int limit = c0 + g.len < total ? c0 + g.len : total;
  if (c0 >= limit) return;  // the whole CTA: nothing is allocated yet
  const int lblk = (g.rp + 63) / 64;  // 8 KB blocks of a part of L
  const int stage_bytes = kZBytes + 2 * lblk * 8192;
  uint32_t cols = 32;
  while (cols < 2u * g.rp) cols *= 2;

  if (t == 0) {
    mbar_init(&empty[0], 1);
    mbar_init(&empty[1], 1);
    mbar_init(&done, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0) tmem_alloc(&s_tmem, cols);

  // The first adapter of the chunk: the last e with start[e] <= c0 and rows there.
  Walk cur, nxt;
  {
    int lo = 0, hi = g.E - 1;  // start[lo] <= c0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(g.start + mid) <= c0) lo = mid;
      else hi = mid - 1;
    }
    cur.e = lo;
    cur.pos = c0;
    cur.seek(g.start, g.E, limit);
  }
  nxt = cur;
  nxt.next(g.start, g.E, limit);
  auto rows_of = [&](const Walk& w, int slot) {
    if (t < kStep) s_rows[slot][t] = w.e < g.E && w.pos + t < w.end ? __ldg(g.order + w.pos + t) : -1;
  };
  rows_of(cur, 0);
  rows_of(nxt, 1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  // A stage in registers: Z rows warp + 8 j, 8 columns at 8 lane; L pieces of 8
  // ranks, piece t + 256 i being row (t + 256 i) / (rp / 8).
  uint4 z[8];
  uint32_t sc[8];
  float l[4][8];
  const int lp = g.rp / 8;
  const int64_t col = col0 + lane * 8;
  auto fetch = [&](int slot) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = s_rows[slot][warp + 8 * j];
      z[j] = make_uint4(0, 0, 0, 0);
      sc[j] = 0;
      if (row < 0) continue;
      if (job.exps) {
        const int64_t ldc = job.ldz;
        if (col < ldc) {
          const uint2 q = __ldg((const uint2*)((const int8_t*)job.Z + (int64_t)row * ldc + col));
          z[j].x = q.x;
          z[j].y = q.y;
          sc[j] = (uint32_t)(int)__ldg(job.exps + (col / kGroup) * g.M + row);
        }
      } else {
        const uint16_t* p = (const uint16_t*)job.Z + (int64_t)row * job.ldz + col;
        if (job.vec && col + 8 <= job.C) {
          z[j] = __ldg((const uint4*)p);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a = col + 2 * i < job.C ? p[2 * i] : 0;
            const uint32_t b = col + 2 * i + 1 < job.C ? p[2 * i + 1] : 0;
            w[i] = a | (b << 16);
          }
          z[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = t + kOuterThreads * i;
      if (q >= kStep * lp) break;
      const int row = s_rows[slot][q / lp], c = q % lp * 8;
      const float* p = job.L + (int64_t)row * g.r + c;
#pragma unroll
      for (int k = 0; k < 8; ++k) l[i][k] = row >= 0 && c + k < g.r ? __ldg(p + k) : 0.0f;
    }
  };
  auto put = [&](uint8_t* st) {
    const uint32_t zb = smem_u32(st) + (lane >> 3) * 8192;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = warp + 8 * j;
      uint32_t w[4] = {z[j].x, z[j].y, z[j].z, z[j].w};
      if (job.exps) {
        const uint32_t s = exp_pair(BF16, (int)sc[j]);
        codes_to_16(BF16, z[j].y, s, w[2], w[3]);
        codes_to_16(BF16, z[j].x, s, w[0], w[1]);
      }
      const uint32_t at = zb + row * 128 + (((uint32_t)(lane & 7) ^ (uint32_t)(row & 7)) << 4);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]),
                   "r"(w[2]), "r"(w[3])
                   : "memory");
    }
    const uint32_t lb = smem_u32(st) + kZBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = t + kOuterThreads * i;
      if (q >= kStep * lp) break;
      const int row = q / lp, c8 = q % lp;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float a = l[i][2 * k], b = l[i][2 * k + 1];
        hi[k] = pack16(BF16, a, b);
        float ra = a - widen16(BF16, (uint16_t)hi[k]), rb = b - widen16(BF16, (uint16_t)(hi[k] >> 16));
        if (!(fabsf(ra) <= 3.0e38f)) ra = 0.0f;
        if (!(fabsf(rb) <= 3.0e38f)) rb = 0.0f;
        lo[k] = pack16(BF16, ra, rb);
      }
      const uint32_t at = lb + (c8 >> 3) * 8192 + row * 128 +
                          (((uint32_t)(c8 & 7) ^ (uint32_t)(row & 7)) << 4);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(hi[0]), "r"(hi[1]),
                   "r"(hi[2]), "r"(hi[3])
                   : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lblk * 8192), "r"(lo[0]),
                   "r"(lo[1]), "r"(lo[2]), "r"(lo[3])
                   : "memory");
    }
  };

  const uint32_t idesc = umma_idesc_16(BF16, 128, g.rp, true, true);
  fetch(0);
  uint32_t done_ph = 0;
  bool ok = true;
  for (int it = 0; cur.e < g.E; ++it) {
    const int buf = it & 1;
    uint8_t* st = smem + buf * stage_bytes;
    ok = mbar_wait(&empty[buf], ((it >> 1) & 1) ^ 1, s_abort, g.status, g.budget_ns);
    if (__syncthreads_or(!ok)) break;  // all threads leave together
    put(st);
    fence_proxy_async_smem();
    __syncthreads();
    const bool fresh = cur.pos == cur.first, last = cur.last();
    if (t == 0) {
      tc_fence_after();
      const uint32_t z0 = smem_u32(st), l0 = z0 + kZBytes;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk) {
          const uint64_t da = umma_desc_mn128(z0 + mb * 16384 + kk * 2048, 8192);
          umma_bf16(tmem + mb * g.rp, da, umma_desc_mn128(l0 + kk * 2048, 8192), idesc,
                    !fresh || kk != 0);
          umma_bf16(tmem + mb * g.rp, da, umma_desc_mn128(l0 + lblk * 8192 + kk * 2048, 8192),
                    idesc, 1);
        }
      umma_commit(&empty[buf]);
      if (last) umma_commit(&done);
    }
    const Walk was = cur;
    cur = nxt;
    nxt.next(g.start, g.E, limit);
    rows_of(nxt, buf);
    if (cur.e < g.E) fetch(buf ^ 1);
    if (last) {
      // One adapter's rows are through: its sums of this chunk.
      ok = mbar_wait(&done, done_ph, s_abort, g.status, g.budget_ns);
      done_ph ^= 1;
      if (__syncthreads_or(!ok)) break;
      tc_fence_after();
      const bool whole = was.first == __ldg(g.start + was.e) && was.end == __ldg(g.start + was.e + 1);
      const int mb = warp >> 2, q = warp & 3;
      const int64_t c = col0 + mb * 128 + q * 32 + lane;
      const int64_t slot = (int64_t)(chunk + was.e) * g.r * job.C;
      const int64_t base = (int64_t)was.e * g.r * job.C;
      for (int k0 = 0; k0 < g.rp; k0 += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + mb * g.rp + k0, v);
        tmem_wait_ld();
        if (c < job.C)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            if (k0 + k >= g.r) break;
            const int64_t at = job.trans ? c * g.r + k0 + k : (int64_t)(k0 + k) * job.C + c;
            if (whole) ((uint16_t*)job.out)[base + at] = round16(BF16, __uint_as_float(v[k]));
            else job.partial[slot + at] = __uint_as_float(v[k]);
          }
      }
      tc_fence_before();
      __syncthreads();
    }
  }
  // MMAs still in flight after a wait that gave up end before TMEM is freed.
  __syncthreads();
  if (!ok || *s_abort) {
    if (t == 0) umma_commit(&done);
    mbar_wait(&done, done_ph, nullptr, g.status, g.budget_ns);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// Adapters whose rows lie in several chunks (or that have none).
__global__ void k_outer_join(const __grid_constant__ OuterArgs g) {
  const int e = blockIdx.y;
  const OuterJob& job = g.job[blockIdx.z];
  const int a = __ldg(g.start + e), b = __ldg(g.start + e + 1);
  const int c0 = a / g.len, c1 = b > a ? (b - 1) / g.len : c0 - 1;
  if (c0 == c1) return;
  const int64_t n = (int64_t)g.r * job.C;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    float s = 0.0f;
    for (int c = c0; c <= c1; ++c) s += job.partial[(int64_t)(c + e) * n + i];
    ((uint16_t*)job.out)[e * n + i] = round16(g.bf16, s);
  }
}

// Rows per chunk: the most chunks that run at once, two CTAs per SM, each of at
// least 256 rows (a second wave of a few CTAs would double the time).
int chunk_len(int64_t M, int64_t tiles, int sms) {
  int64_t chunks = 2 * sms / tiles;
  if (chunks < 1) chunks = 1;
  int64_t len = round_up((M + chunks - 1) / chunks, kStep);
  if (len < 256) len = 256;
  if (len > 8192) len = 8192;
  return (int)len;
}

}  // namespace

size_t outer_scratch_bytes(int64_t M, int64_t N, int64_t K, int r, int E, int dev) {
  const int64_t tiles = (N + kCols - 1) / kCols + (K + kCols - 1) / kCols;
  const int64_t chunks = (M + chunk_len(M, tiles, device_sm_count(dev)) - 1) /
                         chunk_len(M, tiles, device_sm_count(dev));
  Arena ws(nullptr);
  ws.take((size_t)M * 4);
  ws.take((size_t)(E + 1) * 4);
  ws.take((size_t)(chunks + E) * r * K * 4);
  ws.take((size_t)(chunks + E) * r * N * 4);
  return ws.used;
}

int launch_outer(const OuterProduct& p, void* scratch, int dev, cudaStream_t stream) {
  OuterArgs g = {};
  g.M = p.M;
  g.E = p.E;
  g.r = p.r;
  g.rp = (p.r + 15) / 16 * 16;
  g.bf16 = p.bf16;
  g.status = p.status;
  g.budget_ns = wait_budget_ns();
  OuterJob& a = g.job[0];
  a.Z = p.X;
  a.ldz = p.ldx;
  a.C = p.K;
  a.exps = p.exps;
  a.L = p.U;
  a.out = p.dA;
  a.tiles = (int)((p.K + kCols - 1) / kCols);
  a.vec = ((uintptr_t)p.X & 15) == 0 && p.ldx % 8 == 0;
  OuterJob& b = g.job[1];
  b.Z = p.dY;
  b.ldz = p.ldy;
  b.C = p.N;
  b.L = p.T;
  b.out = p.dB;
  b.trans = 1;
  b.tiles = (int)((p.N + kCols - 1) / kCols);
  b.vec = ((uintptr_t)p.dY & 15) == 0 && p.ldy % 8 == 0;
  const int64_t tiles = a.tiles + b.tiles;
  g.len = chunk_len(p.M, tiles, device_sm_count(dev));
  const int64_t chunks = (p.M + g.len - 1) / g.len;
  if (chunks > 65535) return set_error(OZK_ERR_UNSUPPORTED, "too many rows");
  Arena ws(scratch);
  int32_t* order = ws.take<int32_t>((size_t)p.M * 4);
  int32_t* start = ws.take<int32_t>((size_t)(p.E + 1) * 4);
  a.partial = ws.take<float>((size_t)(chunks + p.E) * p.r * p.K * 4);
  b.partial = ws.take<float>((size_t)(chunks + p.E) * p.r * p.N * 4);
  g.order = order;
  g.start = start;
  k_sort_rows<<<p.E, kSortThreads, 0, stream>>>(p.ids, p.M, p.E, order, start);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("k_sort_rows launch", e);
  size_t smem = 1024 + 2 * (size_t)(kZBytes + 2 * ((g.rp + 63) / 64) * 8192);
  if (smem < tmem_share(2 * g.rp)) smem = tmem_share(2 * g.rp);
  auto kern = p.bf16 ? k_outer<true> : k_outer<false>;
  int rc = p.bf16 ? allow_smem<k_outer<true>>(smem, dev) : allow_smem<k_outer<false>>(smem, dev);
  if (rc) return rc;
  kern<<<dim3((unsigned)tiles, (unsigned)chunks), kOuterThreads, smem, stream>>>(g);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("k_outer launch", e);
  const int64_t most = (int64_t)p.r * (p.K > p.N ? p.K : p.N);
  int64_t blocks = (most + 1023) / 1024;
  if (blocks > 256) blocks = 256;
  k_outer_join<<<dim3((unsigned)blocks, (unsigned)p.E, 2), 256, 0, stream>>>(g);
  e = cudaGetLastError();
  return e == cudaSuccess ? OZK_OK : set_cuda_error("k_outer_join launch", e);
}

}  // namespace ozk
