// Eviction from a paged cache by accumulated attention weight: of the kv rows of a
// sequence and key head, the first n_sink and the last n_recent stay, and of the others
// the ones with the largest sums (equal sums: the lower row), until `keep` rows are
// left.  Kept rows keep their order and go to the pages of a second table, so that
// pages shared with other sequences stay whole and every row can move at once.
//
// select_kernel, one CTA for a sequence and key head: finds the smallest kept sum by
// radix selection (four passes over the sums with an 8-bit histogram each; the sums,
// 4 bytes a row, stay in L2), then one pass that numbers the kept rows with a running
// scan and writes their indices and sums.  move_kernel copies the kept rows of k and v,
// 16 bytes a thread; it is bound by memory (a kept row is read and written once).
#include "paged.cuh"

namespace rw {
namespace evict {

using paged::Pool;

constexpr int THREADS = 1024;
constexpr int WARPS = THREADS / 32;
constexpr int PER = 4;               // rows of a thread in a step of the last pass
constexpr int STEP = THREADS * PER;

struct Params {
  Pool pool;
  const float* sums;
  long long sums_sb, sums_sh;
  float* new_sums;                   // [B, Hkv, new_cap], entries behind the kept rows zeroed
  long long new_cap;
  int* kept;                         // [B, Hkv, keep], -1 behind the kept rows
  int* new_lens;                     // [B]
  int keep, n_sink, n_recent;
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

__global__ void __launch_bounds__(THREADS) select_kernel(const __grid_constant__ Params p) {
  __shared__ unsigned hist[WARPS][256];
  __shared__ unsigned scan[WARPS];
  __shared__ unsigned s_digit, s_left;
  griddep_launch_dependents();
  griddep_wait();
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kv = rows_of(p, b, p.status);
  const float* x = p.sums + b * p.sums_sb + hk * p.sums_sh;
  int* kept = p.kept + ((long long)b * p.pool.Hkv + hk) * p.keep;
  float* ns = p.new_sums + ((long long)b * p.pool.Hkv + hk) * p.new_cap;
  const int n_new = min(kv, p.keep);
  if (hk == 0 && tid == 0) p.new_lens[b] = n_new;
  for (long long i = n_new + tid; i < p.new_cap; i += THREADS) ns[i] = 0.f;
  for (int i = n_new + tid; i < p.keep; i += THREADS) kept[i] = -1;
  if (kv <= p.keep) {
    for (int i = tid; i < kv; i += THREADS) {
      kept[i] = i;
      ns[i] = x[i];
    }
    return;
  }
  const int lo = min(p.n_sink, kv), hi = kv - p.n_recent;   // rows [lo, hi) compete; lo <= hi since sink + recent <= keep < kv
  unsigned need = (unsigned)(p.keep - p.n_sink - p.n_recent);
  // ---- the need-th largest sum of [lo, hi): its bits from the top, 8 at a time
  uint32_t prefix = 0;
  unsigned left = need;                      // of the rows with this prefix
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = lane; i < 256; i += 32) hist[warp][i] = 0;
      __syncwarp();
      for (int i = lo + tid; i < hi; i += THREADS) {
        const uint32_t o = order_of(x[i]);
        if (shift == 24 || (o >> (shift + 8)) == prefix) atomicAdd(&hist[warp][(o >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid < 256) {
        unsigned n = 0;
        for (int w = 0; w < WARPS; ++w) n += hist[w][tid];
        hist[0][tid] = n;
      }
      __syncthreads();
      if (warp == 0) {
        // rows with a larger digit than each: lane holds digits 8 lane .. 8 lane + 7
        unsigned mine = 0;
        for (int i = 0; i < 8; ++i) mine += hist[0][8 * lane + i];
        unsigned above = mine;               // suffix sum over lanes
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned y = __shfl_down_sync(0xffffffffu, above, o);
          if (lane + o < 32) above += y;
        }
        above -= mine;
        for (int i = 7; i >= 0; --i) {
          const unsigned n = hist[0][8 * lane + i];
          if (above < left && left <= above + n) {
            s_digit = 8 * lane + i;
            s_left = left - above;
          }
          above += n;
        }
      }
      __syncthreads();
      prefix = (prefix << 8) | s_digit;
      left = s_left;
      __syncthreads();
    }
  }
  // ---- number the kept rows: sink, recent, sums above the threshold, and the first `left` equal to it
  unsigned done_keep = 0, done_ties = 0;     // kept without the ties, ties seen, before this step
  for (int i0 = 0; i0 < kv; i0 += STEP) {
    unsigned flag[PER], mine = 0;            // low half: kept without the ties, high half: ties (a step has 4096 rows)
    float val[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = i0 + tid * PER + j;
      flag[j] = 0;
      val[j] = 0.f;
      if (i < kv) {
        val[j] = x[i];
        if (i < lo || i >= hi) {
          flag[j] = 1u;
        } else if (need > 0) {
          const uint32_t o = order_of(val[j]);
          flag[j] = o > prefix ? 1u : (o == prefix ? 0x10000u : 0u);
        }
      }
      mine += flag[j];
    }
    unsigned s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) scan[warp] = s;
    __syncthreads();
    if (warp == 0) {
      unsigned w = scan[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      scan[lane] = w;
    }
    __syncthreads();
    unsigned before = s - mine + (warp > 0 ? scan[warp - 1] : 0u);
    const unsigned total = scan[WARPS - 1];
    unsigned nk = done_keep + (before & 0xffffu), nt = done_ties + (before >> 16);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const bool tie = flag[j] == 0x10000u;
      if (flag[j] == 1u || (tie && nt < left)) {
        const unsigned at = nk + min(nt, left);
        kept[at] = i0 + tid * PER + j;
        ns[at] = val[j];
      }
      nk += flag[j] & 0xffffu;
      nt += flag[j] >> 16;
    }
    done_keep += total & 0xffffu;
    done_ties += total >> 16;
    __syncthreads();
  }
}

constexpr int MOVE_THREADS = 256;

template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(const __grid_constant__ Params p) {
  constexpr int CH = D / 8;
  constexpr int ROWS = 4;                    // rows of a thread, all loaded before the first is stored
  constexpr int RSTEP = MOVE_THREADS / CH;
  griddep_launch_dependents();
  griddep_wait();
  const int hk = blockIdx.y, b = blockIdx.z;
  const int c = threadIdx.x % CH;
  const int n_new = min(rows_of(p, b, nullptr), p.keep);
  const int j0 = blockIdx.x * (ROWS * RSTEP) + threadIdx.x / CH;
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
      *reinterpret_cast<uint4*>(kd + 16 * c) = kr[i];
      *reinterpret_cast<uint4*>(vd + 16 * c) = vr[i];
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
  p.sums = sums;
  p.sums_sb = sums_sb; p.sums_sh = sums_sh;
  p.new_sums = new_sums; p.new_cap = new_cap;
  p.kept = kept; p.new_lens = new_lens;
  p.keep = keep; p.n_sink = n_sink; p.n_recent = n_recent;
  p.dst_table = dst_table; p.dst_stride = dst_stride; p.dst_width = dst_width;
  p.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (launch_dependent(evict::select_kernel, dim3(p.pool.Hkv, cache->B), dim3(evict::THREADS), 0, st, p) !=
      cudaSuccess)
    return RW_ERR_CUDA;
  const int rows = 4 * evict::MOVE_THREADS / (cache->D / 8);
  const dim3 grid((keep + rows - 1) / rows, p.pool.Hkv, cache->B);
  auto kernel = cache->D == 128 ? evict::move_kernel<128> : evict::move_kernel<64>;
  return launch_dependent(kernel, grid, dim3(evict::MOVE_THREADS), 0, st, p) == cudaSuccess ? RW_OK : RW_ERR_CUDA;
}
