// What weight every cached row received from a chunk of new tokens: sums[b, g, j] += sum
// over the rows of key head g's group of exp(s - lse), with the scores s computed again and
// the rows' lse from the attention (paged_chunk.cu).
//
// Why again: a weight is known only when its row's total is, which is after the last key,
// and a chunk's scores are too many to keep (rows x keys x 4 bytes; the rows of a single
// token are few, and paged_rows.cu keeps theirs).  The second product is half of the
// attention's operations and needs no values.
//
// Transposed tiles: S^T[128 keys][128 rows] = K Q^T, so that a thread owns one key, adds
// up its columns in registers, and no reduction across threads, no atomics and no order
// that could change are needed; a unit (128 keys of a sequence and key head) stays in
// shared memory while the rows' tiles pass by.  Rows are packed as in paged_chunk.cu
// (token * G + head).  Four warpgroups take 32 columns each.  Bound by the exponentials
// (128 x 128 of them against 128 x 128 x D products): the S buffers, four, keep the
// tensor pipe ahead.  (A share of the exponentials on the FMA pipe, or the next tile's scores fetched into registers
// ahead, made it 1 and 10 % slower.)
//
// 880 tokens over 13200 rows, 24 heads of 128: 109 us of the call's 250 to 290, the exponentials' unit 71 % busy.
#include "paged_chunk.h"
#include "paged_tiles.cuh"

namespace rw {
namespace weigh {

using paged::Pool;
using paged::Seq;
using namespace tiles;

constexpr int NS = 4;                        // S buffers (and row parameters)
constexpr int NQ = 4;                        // row tiles in shared memory
constexpr int NK = 2;                        // key tiles
constexpr int NWG = 4;                       // warpgroups that take 128 / NWG columns each
constexpr int CW = BM / NWG;
constexpr int SUM_THREADS = 128 * NWG;
constexpr int NUM_THREADS = SUM_THREADS + 128;
constexpr int WARP_LOAD = 4 * NWG, WARP_MMA = WARP_LOAD + 1, WARP_ROWS = WARP_LOAD + 2;

struct Params {
  Pool pool;
  int T, Hq, G, causal, tpc;
  int kbox, k_head, k_page;
  float scale_log2;
  const float* row_b;                        // [T, Hq]: -(m + log2 l)
  float* sums;
  long long sums_sb, sums_sh;
  int* status;
};

struct __align__(8) Barriers {
  uint64_t k_full[NK], k_free[NK], q_full[NQ], q_free[NQ], s_full[NS], s_free[NS], r_full[NS];
  uint64_t part_full[2], part_free[2];
  uint32_t tmem_base;
  int abort_flag;
};

struct Unit {
  int b, hk, key0, first, n;                 // row tiles [first, first + n) see any of the keys
  Seq s;
};

template <bool HALF, int D>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    weigh_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ Params p) {
  constexpr int TILE_BYTES = BM * D * 2;
  constexpr int Q_BOX = BM * 128;
  constexpr int K_GROUP = 1024 * (D / 64);
  extern __shared__ uint8_t dsmem_raw[];
  __shared__ Barriers sb;
  __shared__ int before[chunk::MAX_BATCH + 1];   // units before each sequence
  __shared__ int3 seq[chunk::MAX_BATCH];         // s0, lq, kv
  __shared__ __align__(16) float par[NS][BM];    // -(m + log2 l) of the columns' rows
  __shared__ float part_sum[2][NWG - 1][BM];
  __shared__ int unit_nan[2 * NS];               // whether a row of the unit has a total of NaN
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ks = smem;
  uint8_t* qs = smem + NK * TILE_BYTES;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const int used = p.tpc * p.G;

  if (threadIdx.x == WARP_LOAD * 32) {
    for (int i = 0; i < NK; ++i) { mbar_init(&sb.k_full[i], 1); mbar_init(&sb.k_free[i], 1); }
    for (int i = 0; i < NQ; ++i) { mbar_init(&sb.q_full[i], 1); mbar_init(&sb.q_free[i], 1); }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sb.s_full[i], 1);
      mbar_init(&sb.s_free[i], SUM_THREADS);
      mbar_init(&sb.r_full[i], 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sb.part_full[i], SUM_THREADS - 128);
      mbar_init(&sb.part_free[i], 128);
    }
    sb.abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
  }
  if (warp == WARP_MMA) {
    tmem_alloc(&sb.tmem_base, 512);
    tmem_relinquish();
  }
  // rows of the row tiles that hold no token stay zero: no load reaches them
  for (int i = threadIdx.x; i < NQ * (BM - used) * (D / 8); i += NUM_THREADS) {
    const int c = i % (D / 8), r = used + (i / (D / 8)) % (BM - used), st = i / (D / 8) / (BM - used);
    *reinterpret_cast<uint4*>(qs + st * TILE_BYTES + (c >> 3) * Q_BOX + r * 128 + ((c & 7) << 4)) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  griddep_wait();
  for (int b = threadIdx.x; b < p.pool.B; b += NUM_THREADS) {
    const Seq s = paged::load_seq(p.pool, b, p.T, nullptr);
    seq[b] = make_int3(s.s0, s.lq, s.kv);
    before[b + 1] = s.lq > 0 ? (int)min(0x7fffffffll, (long long)((s.kv + BM - 1) / BM) * p.pool.Hkv) : 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {
    long long c = 0;
    for (int b0 = 0; b0 < p.pool.B; b0 += 32) {
      long long u = b0 + lane < p.pool.B ? before[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long z = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) u += z;
      }
      if (b0 + lane < p.pool.B) before[b0 + lane + 1] = (int)(c + u);
      c += __shfl_sync(0xffffffffu, u, 31);
    }
    if (lane == 0) {
      before[0] = 0;
      if (c >= 0x7fffffffll) {   // (as many as that would take hours)
        report_status(p.status, RW_STATUS_BAD_SLOT);
        before[p.pool.B] = 0;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = sb.tmem_base;
  const int U = before[p.pool.B];
  volatile int* abort_flag = &sb.abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t parity, int err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, err));
  };
  // neighbouring units cost about the same, and CTAs at work at the same time share a head's rows
  auto unit = [&](int u) {
    Unit x;
    int lo = 0, hi = p.pool.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= u) lo = mid; else hi = mid - 1;
    }
    x.b = lo;
    const int3 s = seq[lo];
    x.s = Seq{s.x, s.y, s.z};
    const int nk = (x.s.kv + BM - 1) / BM, r = u - before[lo];
    x.hk = r / nk;
    x.key0 = (r - x.hk * nk) * BM;
    // the first token that sees key0
    const int tok = p.causal ? max(0, x.key0 - (x.s.kv - x.s.lq)) : 0;
    x.first = tok / p.tpc;
    x.n = (x.s.lq + p.tpc - 1) / p.tpc - x.first;
    return x;
  };

  if (warp == WARP_LOAD) {
    int i = 0, k = 0;                          // row tiles and units so far
    bool ok = true;
    const int nkp = BM / p.kbox, mask = (1 << p.pool.page_shift) - 1;
    for (int u = blockIdx.x; u < U && ok; u += gridDim.x, ++k) {
      const Unit x = unit(u);
      const int row = x.key0 + lane * p.kbox;
      int pg = lane < nkp && row < x.s.kv ? paged::raw_page_of(p.pool, x.b, row) : 0;
      const int sk = k % NK;
      if (k >= NK && !(ok = wait(&sb.k_free[sk], (uint32_t)(k / NK - 1) & 1u, RW_STATUS_TIMEOUT_LOAD))) break;
      if (lane == 0) mbar_expect_tx(&sb.k_full[sk], TILE_BYTES);
      pg = paged::checked_page(p.pool, pg, p.status);
      __syncwarp();
      const int row0 = nkp == 1 ? x.key0 & mask : 0;
      for_pages(x.hk * p.k_head + pg * p.k_page, nkp, [&](int j, int line) {
        load_5d<1>(smem_u32(ks) + sk * TILE_BYTES + j * p.kbox * 2 * D, &tm_k, smem_u32(&sb.k_full[sk]), 0, 0, 0,
                   row0 >> 3, line);
      });
      for (int j = 0; j < x.n; ++j, ++i) {
        const int sq = i % NQ;
        if (i >= NQ && !(ok = wait(&sb.q_free[sq], (uint32_t)(i / NQ - 1) & 1u, RW_STATUS_TIMEOUT_LOAD))) break;
        if (elect_one()) {
          mbar_expect_tx(&sb.q_full[sq], (D / 64) * used * 128);
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            load_3d<1>(smem_u32(qs) + sq * TILE_BYTES + c * Q_BOX, &tm_q, smem_u32(&sb.q_full[sq]), 64 * c, x.hk * p.G,
                       x.s.s0 + (x.first + j) * p.tpc);
        }
        __syncwarp();
      }
    }
  } else if (warp == WARP_MMA) {
    constexpr uint32_t ID = idesc<HALF>(BM, BM, 0);
    const uint64_t dk = umma_desc(smem_u32(ks), 16, K_GROUP), dq = umma_desc(smem_u32(qs), 16, 1024);
    int i = 0, k = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < U && ok; u += gridDim.x, ++k) {
      const int n = unit(u).n, sk = k % NK;
      if (!(ok = wait(&sb.k_full[sk], (uint32_t)(k / NK) & 1u, RW_STATUS_TIMEOUT_MMA))) break;
      for (int j = 0; j < n; ++j, ++i) {
        const int sq = i % NQ, s = i % NS;
        if (!(ok = wait(&sb.q_full[sq], (uint32_t)(i / NQ) & 1u, RW_STATUS_TIMEOUT_MMA))) break;
        if (i >= NS && !(ok = wait(&sb.s_free[s], (uint32_t)(i / NS - 1) & 1u, RW_STATUS_TIMEOUT_MMA))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = dk + (uint64_t)((sk * TILE_BYTES) >> 4), b = dq + (uint64_t)((sq * TILE_BYTES) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss(tmem + 128u * s, a + (uint64_t)(((kk >> 2) * 1024 + (kk & 3) * 32) >> 4),
                   b + (uint64_t)(((kk >> 2) * Q_BOX + (kk & 3) * 32) >> 4), ID, kk > 0 ? 1u : 0u);
          tc_commit(&sb.s_full[s]);
          tc_commit(&sb.q_free[sq]);
          if (j == n - 1) tc_commit(&sb.k_free[sk]);
        }
        __syncwarp();
      }
    }
    // the last row tiles' MMAs are seen to end by the warpgroups; their releases land before the CTA leaves
    if (ok)
      for (int t = max(0, i - NQ); t < i; ++t) mbar_wait_drain(&sb.q_free[t % NQ], (uint32_t)(t / NQ) & 1u);
    if (ok)
      for (int t = max(0, k - NK); t < k; ++t) mbar_wait_drain(&sb.k_free[t % NK], (uint32_t)(t / NK) & 1u);
  } else if (warp == WARP_ROWS) {
    // -(m + log2 l) of a row tile's rows, fetched one tile ahead; -inf (no weight) for a row that is none.  Also for one
    // whose total is NaN: that would reach keys that the row does not see (-inf + NaN), so such units are marked (this warp
    // is at most NS units ahead of the sums) and the keys that do see it get their NaN behind the unit.
    int i = 0, k = 0;
    bool ok = true;
    float next[4];
    for (int u = blockIdx.x; u < U && ok; u += gridDim.x, ++k) {
      const Unit x = unit(u);
      bool nan = false;
      auto fetch = [&](int j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * lane + e, t = r / p.G, tok = (x.first + j) * p.tpc + t;
          next[e] = r < used && tok < x.s.lq && j < x.n
                        ? __ldg(p.row_b + (long long)(x.s.s0 + tok) * p.Hq + x.hk * p.G + (r - t * p.G))
                        : -INFINITY;
        }
      };
      fetch(0);
      for (int j = 0; j < x.n; ++j, ++i) {
        const int s = i % NS;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bad = bad || next[e] != next[e];
          next[e] = next[e] == next[e] ? next[e] : -INFINITY;
        }
        nan = __any_sync(0xffffffffu, bad) || nan;
        const float4 now = make_float4(next[0], next[1], next[2], next[3]);
        fetch(j + 1);
        if (i >= NS && !(ok = wait(&sb.s_free[s], (uint32_t)(i / NS - 1) & 1u, RW_STATUS_TIMEOUT_LOAD))) break;
        *reinterpret_cast<float4*>(par[s] + 4 * lane) = now;
        if (lane == 0) unit_nan[k % (2 * NS)] = nan;
        mbar_arrive(&sb.r_full[s]);
      }
    }
  } else if (warp < 4 * NWG) {
    const int w = warp >> 2;                   // columns [CW w, CW w + CW)
    const int r = threadIdx.x & 127;           // the thread's key
    const uint32_t t0 = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(CW * w);
    const uint64_t s2 = f2_pack(p.scale_log2, p.scale_log2);
    int i = 0, k = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < U; u += gridDim.x, ++k) {
      const Unit x = unit(u);
      uint64_t acc[2] = {0ull, 0ull};
      // rows (token * G + head) of the sequence that see the thread's key begin here
      const long long from = p.causal ? (long long)max(0, x.key0 + r - (x.s.kv - x.s.lq)) * p.G : 0;
      const int all = p.causal ? max(0, x.key0 + BM - 1 - (x.s.kv - x.s.lq)) : 0;  // first token that sees all keys
      for (int j = 0; j < x.n; ++j, ++i) {
        const int s = i % NS;
        ok = ok && wait(&sb.s_full[s], (uint32_t)(i / NS) & 1u, RW_STATUS_TIMEOUT_SOFTMAX) &&
             wait(&sb.r_full[s], (uint32_t)(i / NS) & 1u, RW_STATUS_TIMEOUT_SOFTMAX);
        if (!ok) break;
        tc_fence_after();
        const int tok0 = (x.first + j) * p.tpc;
        const bool masked = tok0 < all || tok0 + p.tpc > x.s.lq;  // (columns without a row hold 0 and have no weight)
        // columns [lo, hi) count; the scores of the others are whatever lies there
        const int lo = (int)max(0ll, min((long long)BM, from - (long long)tok0 * p.G)) - CW * w;
        const int hi = min(used, (x.s.lq - tok0) * p.G) - CW * w;
        const float4* pr = reinterpret_cast<const float4*>(par[s] + CW * w);
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(t0 + 128u * s + 32 * c, v);
          tmem_wait_ld();
          reg_fence32(v);
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * c + e < lo || 32 * c + e >= hi) v[e] = __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 q = pr[8 * c + e];
            float a0, a1, a2, a3;
            f2_unpack(ffma2(f2_pack(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1])), s2, f2_pack(q.x, q.y)),
                      a0, a1);
            f2_unpack(ffma2(f2_pack(__uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3])), s2,
                            f2_pack(q.z, q.w)), a2, a3);
            acc[0] = fadd2(acc[0], f2_pack(fast_exp2(a0), fast_exp2(a1)));
            acc[1] = fadd2(acc[1], f2_pack(fast_exp2(a2), fast_exp2(a3)));
          }
        }
        tc_fence_before();
        mbar_arrive(&sb.s_free[s]);
      }
      float a, b;
      f2_unpack(fadd2(acc[0], acc[1]), a, b);
      // the first warpgroup joins the others' sums while they go on
      const int h = k & 1;
      const uint32_t ph = (uint32_t)(k >> 1) & 1u;
      if (w > 0) {
        ok = ok && (k < 2 || wait(&sb.part_free[h], ph ^ 1u, RW_STATUS_TIMEOUT_SOFTMAX));
        if (!ok) break;
        part_sum[h][w - 1][r] = a + b;
        mbar_arrive(&sb.part_full[h]);
      } else {
        ok = ok && wait(&sb.part_full[h], ph, RW_STATUS_TIMEOUT_SOFTMAX);
        if (!ok) break;
        float sum = a + b;
#pragma unroll
        for (int i = 0; i < NWG - 1; ++i) sum += part_sum[h][i][r];
        mbar_arrive(&sb.part_free[h]);
        if (unit_nan[k % (2 * NS)]) {
#pragma unroll 1
          for (long long e = from; e < (long long)x.s.lq * p.G; ++e) {
            const float y = __ldg(p.row_b + (x.s.s0 + e / p.G) * p.Hq + x.hk * p.G + e % p.G);
            if (y != y) sum = y;
          }
        }
        // one thread of one CTA adds to a row's sum: an addition without a return value, whose order is no matter
        if (x.key0 + r < x.s.kv) atomicAdd(p.sums + x.b * p.sums_sb + x.hk * p.sums_sh + x.key0 + r, sum);
      }
    }
  }

  if (warp == WARP_LOAD && lane == 0 && *abort_flag) {
    const uint64_t t0 = globaltimer_ns();      // after a timeout: copies in flight get time to land
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  if (threadIdx.x == 0) griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool HALF, int D>
int launch_one(const CUtensorMap& mq, const CUtensorMap& mk, const Params& p, int sms, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int SMEM = (NK + NQ) * BM * D * 2 + 1024;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(weigh_kernel<HALF, D>), SMEM, &done)) return RW_ERR_CUDA;
  return launch_dependent(weigh_kernel<HALF, D>, dim3(sms), dim3(NUM_THREADS), SMEM, st, mq, mk, p) == cudaSuccess
             ? RW_OK : RW_ERR_CUDA;
}

int launch(const rw_paged_t* cache, const Pool& pool, const chunk::Call& c, float* sums, long long sums_sb,
           long long sums_sh, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return RW_ERR_CUDA;
  const long long units = (long long)pool.B * pool.Hkv * (((long long)cache->table_width * cache->page_size + BM - 1) / BM);
  if (units == 0) return RW_OK;
  if (units < sms) sms = (int)units;
  Params p{};
  p.pool = pool;
  p.T = c.T; p.Hq = c.Hq; p.G = c.Hq / pool.Hkv; p.causal = c.causal;
  p.tpc = BM / p.G;
  p.kbox = cache->page_size < BM ? cache->page_size : BM;
  const KeyLines kl = key_lines(cache);
  p.k_head = cache->Hkv == 1 ? 0 : (int)(cache->k_sh / kl.step);
  p.k_page = cache->num_pages == 1 ? 0 : (int)(cache->k_sp / kl.step);
  p.scale_log2 = c.scale_log2;
  p.row_b = c.row_b;
  p.sums = sums;
  p.sums_sb = sums_sb;
  p.sums_sh = sums_sh;
  p.status = c.status;
  CUtensorMap mq, mk;
  if (q_map(&mq, c.q, cache->dtype, c.T, c.Hq, cache->D, c.q_sl, c.q_sh, p.G, p.tpc) || key_map(&mk, cache, p.kbox))
    return RW_ERR_DRIVER;
  if (cache->dtype == RW_DTYPE_FP16)
    return cache->D == 128 ? launch_one<true, 128>(mq, mk, p, sms, st) : launch_one<true, 64>(mq, mk, p, sms, st);
  return cache->D == 128 ? launch_one<false, 128>(mq, mk, p, sms, st) : launch_one<false, 64>(mq, mk, p, sms, st);
}

}  // namespace weigh
}  // namespace rw
