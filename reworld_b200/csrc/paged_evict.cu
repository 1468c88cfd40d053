// Eviction from a paged cache by accumulated attention weight: of the kv rows of a
// sequence and key head, the first n_sink and the last n_recent stay, and of the others
// the ones with the largest sums (equal sums: the lower row), until `keep` rows are
// left.  Kept rows keep their order and go to the pages of a second table, so that
// pages shared with other sequences stay whole and every row can move at once.
//
// select_kernel, a cluster of one to eight CTAs for a sequence and key head: finds the smallest kept sum by
// radix selection (three passes over the sums, which stay in registers or L2, with histograms of 11, 11
// and 10 bits: 11 bits hold the exponent and three more, so that sums of a similar size
// do not all meet in one counter), then numbers the kept rows with one scan for every
// 16384 rows and writes their indices and sums.  Each CTA of the cluster has its part of
// the rows; through distributed shared memory each adds up its slice of the histograms, and
// the one whose slice has the threshold tells the others (all of them adding up all of the histograms
// took 5 us a pass with eight CTAs).  move_kernel copies the kept rows of k and
// v, 16 bytes a thread; it is bound by memory (a kept row is read and written once).
//
// 64 units of 32768 rows of 128 channels, half kept: 199 us, 1.09 GB, 5.5 TB/s; 8 units of 1000 rows: 7.2 us,
// the chain of the selection's barriers and the second launch.
#include "paged.cuh"

namespace rw {
namespace evict {

using paged::Pool;

constexpr int BINS = 2048;
constexpr int PER = 16;              // sums of a thread under way at once
constexpr int MAX_CLUSTER = 8;

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
__device__ __forceinline__ void st_cluster(unsigned* p, int rank, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), (uint32_t)rank)), "r"(v) : "memory");
}

template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 1) select_kernel(const __grid_constant__ Params p) {
  constexpr int WARPS = THREADS / 32, STEP = THREADS * PER, DIGITS = BINS / THREADS;
  __shared__ unsigned hist[BINS];
  __shared__ unsigned scan[WARPS];
  __shared__ unsigned s_digit, s_left, s_keep, s_ties;
  __shared__ unsigned s_slice[MAX_CLUSTER];  // counts of the CTAs' parts of the histogram
  griddep_launch_dependents();
  griddep_wait();
  const int cs = CLUSTER ? p.cs : 1, rank = CLUSTER ? blockIdx.x % cs : 0;
  const int hk = CLUSTER ? blockIdx.x / cs : blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kv = rows_of(p, b, p.status);
  const float* x = p.sums + b * p.sums_sb + hk * p.sums_sh;
  int* kept = p.kept + ((long long)b * p.pool.Hkv + hk) * p.keep;
  float* ns = p.new_sums + ((long long)b * p.pool.Hkv + hk) * p.new_cap;
  const int n_new = min(kv, p.keep);
  // this CTA's rows [begin, end); a short part's sums are read once.  A warp has 32 * pe rows of a step, 32 at a time
  const int part = (kv + cs - 1) / cs, begin = min(kv, rank * part), end = min(kv, begin + part);
  const bool once = end - begin <= STEP;
  const int pe = once ? (end - begin + THREADS - 1) / THREADS : PER;
  const int own = warp * (32 * pe) + lane;
  float v[PER];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = i0 + own + 32 * j;
      v[j] = j < pe && i < end ? x[i] : 0.f;
    }
  };
  if (once) fetch(begin);
  if (tid == 0) s_keep = s_ties = 0;
  const int first = rank * THREADS + tid, step = cs * THREADS;
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = n_new;
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
  // ---- the need-th largest sum of [lo, hi): its bits from the top
  uint32_t prefix = 0;
  unsigned left = need;                      // of the rows with this prefix
  if (need > 0) {
    const unsigned span = (unsigned)max(0, min(hi, end) - lo);
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      for (int i = tid; i < BINS; i += THREADS) hist[i] = 0;
      __syncthreads();
      for (int i0 = begin; i0 < end; i0 += STEP) {
        if (!once) fetch(i0);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (j >= pe) break;
          const uint32_t o = order_of(v[j]);
          if ((unsigned)(i0 + own + 32 * j - lo) < span && (pass == 0 || (o >> (shift + bits)) == prefix))
            atomicAdd(&hist[(o >> shift) & ((1u << bits) - 1u)], 1u);
        }
      }
      if constexpr (CLUSTER) {
        // a CTA adds up its slice of the cluster's histograms, a thread a digit, thread 0 the largest
        const int slice = BINS / cs;
        cluster_sync();
        unsigned n = 0, all;
        const int digit = slice * (rank + 1) - 1 - tid;
        if (tid < slice) {
          unsigned m[MAX_CLUSTER];
#pragma unroll
          for (int c = 0; c < MAX_CLUSTER; ++c) m[c] = c < cs ? ld_cluster(&hist[digit], c) : 0u;
#pragma unroll
          for (int c = 0; c < MAX_CLUSTER; ++c) n += m[c];
        }
        const unsigned upto = block_scan<THREADS>(n, scan, &all);
        if (tid < cs) st_cluster(&s_slice[rank], tid, all);
        cluster_sync();
        unsigned above = upto - n;
        for (int c = rank + 1; c < cs; ++c) above += s_slice[c];
        if (above < left && left <= above + n)
          for (int c = 0; c < cs; ++c) {
            st_cluster(&s_digit, c, (unsigned)digit);
            st_cluster(&s_left, c, left - above);
          }
        cluster_sync();
      } else {
        __syncthreads();
        // a thread has DIGITS digits, thread 0 the largest: how many rows have a larger one
        unsigned n[DIGITS], mine = 0, all;
#pragma unroll
        for (int i = 0; i < DIGITS; ++i) mine += n[i] = hist[BINS - 1 - DIGITS * tid - i];
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
      }
      prefix = (prefix << bits) | s_digit;
      left = s_left;
      __syncthreads();                       // (they are read)
    }
  }
  // What a thread's rows of a step are, two bits each: 1 kept whatever the ties, 2 tied, 0 neither.
  unsigned code = 0;
  auto classify = [&](int i0) {
    code = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j >= pe) break;
      const int i = i0 + own + 32 * j;
      const uint32_t o = order_of(v[j]);
      unsigned is = o > prefix ? 1u : (o == prefix ? 2u : 0u);
      if (need == 0) is = 0u;
      if (i < lo || i >= hi) is = 1u;
      if (i < end) code |= is << (2 * j);
    }
    return (unsigned)(__popc(code & 0x55555555u) | (__popc(code & 0xAAAAAAAAu) << 16));
  };
  // ---- number the kept rows: sink, recent, sums above the threshold, and the first `left` equal to it
  unsigned done_keep = 0, done_ties = 0;     // kept without the ties, ties seen, before this step
  unsigned mine = 0;                         // kept (low half) and tied (high half) rows of the thread in the step
  if constexpr (CLUSTER) {
    // those of the CTAs before this one
    unsigned k = 0, e = 0;
    for (int i0 = begin; i0 < end; i0 += STEP) {
      if (!once) fetch(i0);
      mine = classify(i0);
      k += mine & 0xffffu;
      e += mine >> 16;
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
    if (!once) fetch(i0);
    if (!CLUSTER || !once) mine = classify(i0);
    // (at most 16384 rows a step: the halves do not run over)
    const unsigned in_warp = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) scan[warp] = in_warp;
    __syncthreads();
    unsigned w = lane < WARPS ? scan[lane] : 0u;
    const unsigned all = __reduce_add_sync(0xffffffffu, w), before = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0u);
    unsigned nk = done_keep + (before & 0xffffu), nt = done_ties + (before >> 16);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j >= pe) break;
      const unsigned is = (code >> (2 * j)) & 3u, under = (1u << lane) - 1u;
      const unsigned km = __ballot_sync(0xffffffffu, is & 1u), tm = __ballot_sync(0xffffffffu, is & 2u);
      const unsigned t = nt + __popc(tm & under);
      if ((is & 1u) || ((is & 2u) && t < left)) {
        const unsigned at = nk + __popc(km & under) + min(t, left);
        kept[at] = i0 + own + 32 * j;
        ns[at] = v[j];
      }
      nk += __popc(km);
      nt += __popc(tm);
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
  // Barriers cost less with few threads, and the work on a sum less with many: 600 rows 6.7 us with 256 threads, 7.2 with
  // 1024; 1500 rows 7.7 and 8.0; 4000 rows 11.1 and 9.7.  A long row gets a cluster while SMs are idle: 1 unit of 16384
  // rows 17.9 us with one CTA, 16.4 with eight, 8 units 25.8 and 24.6, but of 10000 rows 18.4 and 20.6.
  // Clusters of more than two leave some SMs of a group of SMs unused: 16 units of 32768 rows 74.9 us with eight CTAs,
  // some of which then wait for others to leave, 62.4 with four.
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return RW_ERR_CUDA;
  const long long cap = (long long)cache->table_width * cache->page_size, units = (long long)p.pool.Hkv * cache->B;
  p.cs = 1;
  while (cap > 12288 && p.cs < 8 && units * p.cs * 2 <= (p.cs == 1 ? sms : sms * 3 / 4) && cap >= 4096ll * p.cs) p.cs *= 2;
  const bool few = p.cs == 1 && cap <= 1536;
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
