// Eviction from a paged cache by accumulated attention weight: of the kv rows of a
// sequence and key head, the first n_sink and the last n_recent stay, and of the others
// the ones with the largest sums (equal sums: the lower row), until `keep` rows are
// left.  Kept rows keep their order and go to the pages of a second table, so that
// pages shared with other sequences stay whole and every row can move at once.
//
// select_kernel, a cluster of one to eight CTAs for a sequence and key head: finds the smallest kept sum by
// radix selection (three passes over the sums, which stay in L2, with histograms of 11, 11
// and 10 bits: 11 bits hold the exponent and three more, so that sums of a similar size
// do not all meet in one counter), then numbers the kept rows with one scan for every
// 16384 rows and writes their indices and sums.  Each CTA of the cluster has its part of
// the rows; they add up one another's histograms and counts through distributed shared
// memory (64 units of 32768 rows leave more than half of the SMs idle otherwise).  move_kernel copies the kept rows of k and
// v, 16 bytes a thread; it is bound by memory (a kept row is read and written once).
#include "paged.cuh"

namespace rw {
namespace evict {

using paged::Pool;

constexpr int BINS = 2048;
constexpr int PER = 16;              // sums of a thread under way at once

struct Params {
  Pool pool;
  const float* sums;
  long long sums_sb, sums_sh;
  float* new_sums;                   // [B, Hkv, new_cap], entries behind the kept rows zeroed
  long long new_cap;
  int* kept;                         // [B, Hkv, keep], -1 behind the kept rows
  int* new_lens;                     // [B]
  int keep, n_sink, n_recent;
  int cs;                            // CTAs of a cluster
  const int* dst_table;
  long long dst_stride;
  int dst_width;
  int* status;
};

// Unsigned order of the floats; NaN counts as less than everything, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0u;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ int rows_of(const Params& p, int b, int* status) {
  const int n = __ldg(p.pool.kv_lens + b);
  const int kv = (int)min((long long)max(n, 0), (long long)p.pool.width << p.pool.page_shift);
  if (kv != n) report_status(status, RW_STATUS_BAD_SLOT);
  return kv;
}

// Inclusive sums over the block of a value of every thread, in thread order; `all` is their total.
template <int THREADS>
__device__ __forceinline__ unsigned block_scan(unsigned x, unsigned* scan, unsigned* all) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scan[warp] = x;
  __syncthreads();
  // every warp sums up the warps' totals for itself
  unsigned w = lane < WARPS ? scan[lane] : 0u;
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *all = __shfl_sync(0xffffffffu, w, WARPS - 1);
  return x + (warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0u);
}

// Word at the same shared address in CTA `rank` of the cluster.
__device__ __forceinline__ unsigned ld_cluster(const unsigned* p, int rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), (uint32_t)rank)) : "memory");
  return v;
}

template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 1) select_kernel(const __grid_constant__ Params p) {
  constexpr int WARPS = THREADS / 32, STEP = THREADS * PER, DIGITS = BINS / THREADS;
  __shared__ unsigned hist[BINS];
  __shared__ unsigned scan[WARPS];
  __shared__ unsigned count[PER * WARPS];    // kept (low half) and tied (high half) rows of every 32
  __shared__ unsigned s_digit, s_left, s_keep, s_ties;
  griddep_launch_dependents();
  griddep_wait();
  const int cs = CLUSTER ? p.cs : 1, rank = CLUSTER ? blockIdx.x % cs : 0;
  const int hk = CLUSTER ? blockIdx.x / cs : blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kv = rows_of(p, b, p.status);
  const float* x = p.sums + b * p.sums_sb + hk * p.sums_sh;
  int* kept = p.kept + ((long long)b * p.pool.Hkv + hk) * p.keep;
  float* ns = p.new_sums + ((long long)b * p.pool.Hkv + hk) * p.new_cap;
  const int n_new = min(kv, p.keep);
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = n_new;
  const int first = rank * THREADS + tid, step = cs * THREADS;
  for (long long i = n_new + first; i < p.new_cap; i += step) ns[i] = 0.f;
  for (int i = n_new + first; i < p.keep; i += step) kept[i] = -1;
  if (kv <= p.keep) {
    for (int i = first; i < kv; i += step) {
      kept[i] = i;
      ns[i] = x[i];
    }
    return;
  }
  const int lo = min(p.n_sink, kv), hi = kv - p.n_recent;   // rows [lo, hi) compete; lo <= hi since sink + recent <= keep < kv
  const unsigned need = (unsigned)(p.keep - p.n_sink - p.n_recent);
  // this CTA's rows [begin, end); a short part's sums are read once
  const int per = (kv + cs - 1) / cs, begin = min(kv, rank * per), end = min(kv, begin + per);
  const bool once = end - begin <= STEP;
  auto sync_all = [&]() {
    if constexpr (CLUSTER) cluster_sync(); else __syncthreads();
  };
  float v[PER];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = i0 + j * THREADS + tid;
      v[j] = i < end ? x[i] : 0.f;
    }
  };
  if (once) fetch(begin);
  if (tid == 0) s_keep = s_ties = 0;
  // ---- the need-th largest sum of [lo, hi): its bits from the top
  uint32_t prefix = 0;
  unsigned left = need;                      // of the rows with this prefix
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      for (int i = tid; i < BINS; i += THREADS) hist[i] = 0;
      __syncthreads();
      for (int i0 = begin; i0 < end; i0 += STEP) {
        if (!once) fetch(i0);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int i = i0 + j * THREADS + tid;
          if (i0 + j * THREADS >= end) break;
          const uint32_t o = order_of(v[j]);
          if (i < end && i >= lo && i < hi && (pass == 0 || (o >> (shift + bits)) == prefix))
            atomicAdd(&hist[(o >> shift) & ((1u << bits) - 1u)], 1u);
        }
      }
      sync_all();
      // a thread has DIGITS digits, thread 0 the largest: how many rows have a larger one
      unsigned n[DIGITS], mine = 0, all;
#pragma unroll
      for (int i = 0; i < DIGITS; ++i) n[i] = hist[BINS - 1 - DIGITS * tid - i];
      for (int c = 1; c < cs; ++c) {
#pragma unroll
        for (int i = 0; i < DIGITS; ++i) n[i] += ld_cluster(&hist[BINS - 1 - DIGITS * tid - i], (rank + c) % cs);
      }
#pragma unroll
      for (int i = 0; i < DIGITS; ++i) mine += n[i];
      unsigned above = block_scan<THREADS>(mine, scan, &all) - mine;
#pragma unroll
      for (int i = 0; i < DIGITS; ++i) {
        if (above < left && left <= above + n[i]) {
          s_digit = BINS - 1 - DIGITS * tid - i;
          s_left = left - above;
        }
        above += n[i];
      }
      __syncthreads();
      prefix = (prefix << bits) | s_digit;
      left = s_left;
      sync_all();                            // the histograms are read
    }
  }
  // what a row is: 1 kept whatever the ties, 2 tied, 0 neither
  auto kind = [&](int i, float s) {
    if (i >= end) return 0;
    if (i < lo || i >= hi) return 1;
    if (need == 0) return 0;
    const uint32_t o = order_of(s);
    return o > prefix ? 1 : (o == prefix ? 2 : 0);
  };
  // ---- number the kept rows: sink, recent, sums above the threshold, and the first `left` equal to it
  unsigned done_keep = 0, done_ties = 0;     // kept without the ties, ties seen, before this step
  if constexpr (CLUSTER) {
    // those of the CTAs before this one
    unsigned k = 0, e = 0;
    for (int i0 = begin; i0 < end; i0 += STEP) {
      if (!once) fetch(i0);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int is = kind(i0 + j * THREADS + tid, v[j]);
        k += is == 1;
        e += is == 2;
      }
    }
    k = __reduce_add_sync(0xffffffffu, k);
    e = __reduce_add_sync(0xffffffffu, e);
    __syncthreads();                         // (the totals are zeroed)
    if (lane == 0) {
      atomicAdd(&s_keep, k);
      atomicAdd(&s_ties, e);
    }
    cluster_sync();
    for (int c = 0; c < rank; ++c) {
      done_keep += ld_cluster(&s_keep, c);
      done_ties += ld_cluster(&s_ties, c);
    }
  }
  for (int i0 = begin; i0 < end; i0 += STEP) {
    unsigned keep_m[PER], tie_m[PER];        // of the warp's 32 rows
    if (!once) fetch(i0);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (i0 + j * THREADS >= end) {
        if (lane == 0) count[j * WARPS + warp] = 0;
        continue;
      }
      const int is = kind(i0 + j * THREADS + tid, v[j]);
      keep_m[j] = __ballot_sync(0xffffffffu, is == 1);
      tie_m[j] = __ballot_sync(0xffffffffu, is == 2);
      if (lane == 0) count[j * WARPS + warp] = (unsigned)__popc(keep_m[j]) | ((unsigned)__popc(tie_m[j]) << 16);
    }
    __syncthreads();
    // the groups of 32 in their order (at most 16384 rows a step: the halves do not run over); exclusive sums
    unsigned all;
    const unsigned mine = tid < PER * WARPS ? count[tid] : 0u;
    const unsigned upto = block_scan<THREADS>(mine, scan, &all);
    if (tid < PER * WARPS) count[tid] = upto - mine;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (i0 + j * THREADS >= end) break;
      const unsigned before = count[j * WARPS + warp], under = (1u << lane) - 1u;
      const unsigned nk = done_keep + (before & 0xffffu) + __popc(keep_m[j] & under);
      const unsigned nt = done_ties + (before >> 16) + __popc(tie_m[j] & under);
      const bool tie = (tie_m[j] >> lane) & 1u;
      if (((keep_m[j] >> lane) & 1u) || (tie && nt < left)) {
        const unsigned at = nk + min(nt, left);
        kept[at] = i0 + j * THREADS + tid;
        ns[at] = v[j];
      }
    }
    done_keep += all & 0xffffu;
    done_ties += all >> 16;
    __syncthreads();
  }
  if constexpr (CLUSTER) cluster_sync();     // no CTA leaves while another may read its counts
}

constexpr int MOVE_THREADS = 128;

template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(const __grid_constant__ Params p) {
  constexpr int CH = D / 8;
  constexpr int ROWS = 2;                    // rows of a thread, all loaded before the first is stored
  constexpr int RSTEP = MOVE_THREADS / CH;
  griddep_launch_dependents();
  griddep_wait();
  const int hk = blockIdx.x % p.pool.Hkv, b = blockIdx.y;
  const int c = threadIdx.x % CH;
  const int n_new = min(rows_of(p, b, nullptr), p.keep);
  const int j0 = blockIdx.x / p.pool.Hkv * (ROWS * RSTEP) + threadIdx.x / CH;
  const int* kept = p.kept + ((long long)b * p.pool.Hkv + hk) * p.keep;
  const int mask = (1 << p.pool.page_shift) - 1;
  uint4 kr[ROWS], vr[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int j = j0 + i * RSTEP;
    if (j < n_new) {
      const int row = kept[j];
      const long long pg = paged::page_of(p.pool, b, row, p.status);
      kr[i] = __ldcs(reinterpret_cast<const uint4*>(p.pool.k + pg * p.pool.k_sp + (row & mask) * p.pool.k_sl +
                                                    hk * p.pool.k_sh + 16 * c));
      vr[i] = __ldcs(reinterpret_cast<const uint4*>(p.pool.v + pg * p.pool.v_sp + (row & mask) * p.pool.v_sl +
                                                    hk * p.pool.v_sh + 16 * c));
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int j = j0 + i * RSTEP;
    if (j < n_new) {
      const int pg = __ldg(p.dst_table + b * p.dst_stride + (j >> p.pool.page_shift));
      if ((unsigned)pg >= (unsigned)p.pool.num_pages) {
        report_status(p.status, RW_STATUS_BAD_SLOT);
        continue;
      }
      uint8_t* kd = const_cast<uint8_t*>(p.pool.k) + pg * p.pool.k_sp + (j & mask) * p.pool.k_sl + hk * p.pool.k_sh;
      uint8_t* vd = const_cast<uint8_t*>(p.pool.v) + pg * p.pool.v_sp + (j & mask) * p.pool.v_sl + hk * p.pool.v_sh;
      __stcs(reinterpret_cast<uint4*>(kd + 16 * c), kr[i]);
      __stcs(reinterpret_cast<uint4*>(vd + 16 * c), vr[i]);
    }
  }
}

}  // namespace evict
}  // namespace rw

extern "C" int rw_paged_evict(const rw_paged_t* cache, const float* sums, long long sums_sb, long long sums_sh,
                              float* new_sums, long long new_cap, int* kept, int* new_lens, int keep, int n_sink,
                              int n_recent, const int* dst_table, long long dst_stride, int dst_width, int* status,
                              void* stream) {
  using namespace rw;
  evict::Params p{};
  if (int e = paged::make_pool(cache, &p.pool)) return e;
  if (keep < 1 || n_sink < 0 || n_recent < 0 || (long long)n_sink + n_recent > keep || new_cap < 0 || sums_sb < 0 ||
      sums_sh < 0 || dst_width < 0 || dst_stride < dst_width)
    return RW_ERR_INVALID_ARG;
  if (cache->B == 0) return RW_OK;
  if (!sums || !new_sums || !kept || !new_lens || !dst_table) return RW_ERR_INVALID_ARG;
  if ((long long)dst_width * cache->page_size < keep || new_cap < keep) return RW_ERR_CAPACITY;
  const int rows = 2 * evict::MOVE_THREADS / (cache->D / 8);   // of a block of move_kernel
  const long long blocks = ((long long)keep + rows - 1) / rows;
  if (blocks * p.pool.Hkv > 0x7fffffffll) return RW_ERR_CAPACITY;
  p.sums = sums;
  p.sums_sb = sums_sb; p.sums_sh = sums_sh;
  p.new_sums = new_sums; p.new_cap = new_cap;
  p.kept = kept; p.new_lens = new_lens;
  p.keep = keep; p.n_sink = n_sink; p.n_recent = n_recent;
  p.dst_table = dst_table; p.dst_stride = dst_stride; p.dst_width = dst_width;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // A short row needs few threads, and barriers cost less with few (evicting from 1000 rows 10.3 us, with 1024 threads
  // 12.9; from 4000 rows 14.7 and 16.0).  A long one gets more CTAs while SMs are idle: 8 units of
  // 32768 rows 56.0 -> 50.0 us, of 200000 rows 223 -> 81, 64 units of 32768 rows 212.8 -> 205.3; not one that a CTA
  // holds in its registers (16 units of 10000 rows 25.7 -> 32.2 with four).
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return RW_ERR_CUDA;
  const long long cap = (long long)cache->table_width * cache->page_size, units = (long long)p.pool.Hkv * cache->B;
  const bool few = cap <= 4096;
  p.cs = 1;
  while (cap > 16384 && p.cs < 8 && units * p.cs * 2 <= sms && cap >= 4096ll * p.cs) p.cs *= 2;
  {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.pool.Hkv * p.cs, cache->B);
    cfg.blockDim = dim3(few ? 256 : 1024);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.cs;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.cs > 1 ? 2 : 1;
    auto kernel = p.cs > 1 ? evict::select_kernel<1024, true>
                           : (few ? evict::select_kernel<256, false> : evict::select_kernel<1024, false>);
    if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess)
      return RW_ERR_CUDA;
  }
  const dim3 grid((unsigned)(blocks * p.pool.Hkv), cache->B);
  auto kernel = cache->D == 128 ? evict::move_kernel<128> : evict::move_kernel<64>;
  return launch_dependent(kernel, grid, dim3(evict::MOVE_THREADS), 0, st, p) == cudaSuccess ? RW_OK : RW_ERR_CUDA;
}
