// Attention of chunks of new tokens over a paged cache on the tensor cores: o =
// softmax(q k^T * scale) v for a ragged batch, with shared key heads and causal order.
//
// A unit is the 256 rows (head dim 128) or 128 rows (head dim 64) of one sequence that
// share a key head: the G query heads of the group by consecutive tokens, row = token *
// G + head, so that a key tile is used by all heads that share it.  With G not a power of
// two a tile of 128 holds floor(128 / G) * G rows.
//
// Head dim 128 runs on CTA pairs as attn_pair.cu does (2-SM tcgen05.mma, every CTA loads
// half of each key and value tile): one CTA alone would need 64 KB of k and v for every
// 128 x 128 scores, about twice what L2 delivers to all SMs at that rate.  With head dim
// 64 the tiles are half as large and the time a tile takes is the same (the 128 x 128
// exponentials), so one CTA reads what a pair's CTA does there; it runs alone.
//   TMEM columns  O [0, D)  S0 [128, 256)  S1 [256, 384)  S2 [384, 512)
// Key tile j lands in S buffer j mod 3 and its weights P (16-bit) overwrite the buffer's
// first 64 columns; the tensor pipe runs QK up to three tiles ahead of the softmax.
// Warps: two softmax warpgroups (tiles j even / odd, a row a thread), warp 8 loads q and keys,
// warp 9 issues the MMAs, warp 10 loads the values, warp 11 plans.
//
// Pages: a tile is gathered by one TMA box a page (and, of the values, 64 channels); page
// indices are read one tile ahead.  Of the page that a sequence ends in, the rows behind
// the end may hold anything.  Keys that a row does not see are masked by selection; of the
// values of tiles that not every row sees whole, warp 11 zeroes the rows behind the end and
// takes out what is not finite (paged.cuh) before the MMA warp gets them.
//
// Work: lengths are device data, so every CTA sums the key tiles of all units itself
// (a few microseconds' latency, no host, no extra launch).  Where it ends about as early, pairs take
// whole units, in rounds, the longest first and every other round backwards.  Otherwise they first take
// whole units in waves (pairs at work at the same time then share heads, and k and v come from L2),
// if the units are about equal; what does not fill a wave, or all of it if they are not,
// is one sequence of tiles of which every pair takes an equal share, and the parts of
// units that more than one pair worked on are joined by join_kernel.
//
// The weights P are rounded to the values' 16-bit type (an MMA's operands have one type); totals are
// sums of the unrounded ones, and O is fp32 until the output's one rounding.
//
// 2640 tokens over 34320 rows, 24 heads of 128: 0.88 ms (1.22 PFLOP/s) in a short run, 1.03 ms when the power
// limit holds the clock down; without the causal mask, which has 4 % more to do, 1.06 (the contiguous kernel 1.00).
#include <algorithm>

#include "paged.cuh"
#include "paged_chunk.h"
#include "paged_tiles.cuh"

namespace rw {
namespace chunk {

using paged::Num;
using paged::Pool;
using paged::Seq;
using namespace tiles;

constexpr int BN = 128;                      // keys of a tile
constexpr int NSBUF = 3;
constexpr int NSTAGE = 4;
constexpr int HALF_TILE = 16384;             // a CTA's part of a key or value tile
constexpr int PRE_BYTES = NSBUF * HALF_TILE; // keys of tiles 0-2
constexpr int STAGE_BYTES = 2 * HALF_TILE;   // stage j: values of tile j, then keys of tile j + 3
constexpr int NWG = 2;
constexpr int NUM_THREADS = 128 * (NWG + 1);
constexpr int WARP_LOAD = 8, WARP_MMA = 9, WARP_V = 10, WARP_PLAN = 11;
constexpr int SOFTMAX_THREADS = 256;
constexpr int REG_SOFTMAX = 208, REG_OTHER = 88;
static_assert(NWG * 128 * REG_SOFTMAX + 128 * REG_OTHER <= NUM_THREADS * 168, "register split exceeds the launch's");
constexpr float RESCALE_THRESHOLD = 8.0f;    // log2 units
// fp16 weights are exp2(s - base + 7), 2^15 at most: a row that gives one key nearly everything still has weights of
// 2^-14 to 2^-24 of that one, which fp16 would hold to a few bits or none, and a long cache has enough of them to be
// seen (4.5 * 2^-24 from each of 60000 keys is 1.6 % of a row, 11 % of it lost).  Totals have the factor too.
template <bool HALF> constexpr float UP_LOG2 = HALF ? 7.0f : 0.0f;
template <bool HALF> constexpr float DOWN = HALF ? 1.0f / 128 : 1.0f;
// What a score has added before the exponential.  For fp16 it is rounded down: scores of some 10^7 have it in steps of 2
// and more, and half a step up would take weights of 2^15 out of fp16.
template <bool HALF>
__device__ __forceinline__ float minus_base(float m, float sl2) {
  return HALF ? __fmaf_rd(-m, sl2, UP_LOG2<HALF>) : -m * sl2;
}
// What work dealt out in equal shares costs more than whole units: the starts of parts, and their joining.  Whole units
// against shares: 8 units of 12 tiles 25.1 and 30.6 us, of 16 tiles 28.2 and 31.4, of 32 tiles 39.9 and 36.1 (74 pairs); 64
// units of 35 tiles 46.5 and 56.5; head dim 64 (148 CTAs) 4 units of 8 tiles 20.3 and 22.2, of 20 tiles 26.9 and 23.8; 344
// units of 1 to 12 tiles 41.8 and 51.2.
template <int D> constexpr int JOIN_COST = D == 128 ? 17 : 13;
constexpr int MIN_SHARE = 12;                // cost of a share, where there is little work
// What a unit costs beside its key tiles, in tiles: filling and draining the pipeline (q and the first keys, the last
// softmax, the output) takes 5 to 8 us, a tile 0.75 to 0.9.  4 ragged chunks of up to 701 tokens 140.5 us dealt out with
// 3, 131.8 with 7, 131.7 with 11; 16 of up to 300 tokens 233, 198 and 196; 3 prompts of head dim 64 53.1, 51.2 and 50.5.
constexpr int UNIT_COST = 10;

template <int D>
struct Shape {
  static constexpr int NCTA = D == 128 ? 2 : 1;
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int KROWS = BN / NCTA;    // a CTA's keys of a tile
  static constexpr int SMEM = Q_BYTES + PRE_BYTES + NSTAGE * STAGE_BYTES + 1024;
  static constexpr long long SLOT_FLOATS = (long long)NCTA * BM * (D + 2);
};

// What a segment (the key tiles [kv0, kv0 + n) of one unit) needs.
struct Seg {
  int n;                 // 0: no more work
  int kv0;
  int slot;              // -1: the whole unit
  int b, hk, tok0;       // unit's first token within the sequence
  int s0, lq, kv;
  int all;               // keys that every token of the unit sees
};

struct Params {
  Pool pool;
  int T, Hq, G, causal;
  int tpc;               // tokens of a CTA: floor(128 / G)
  int C;                 // pairs (or CTAs) in the grid
  float scale_log2;
  uint8_t* out;
  long long o_sl, o_sh;  // byte strides
  float* lse;            // [T, Hq] or null
  float* row_b;          // [T, Hq]: -(m + log2 l) for the weight sums, or null
  float* scratch;        // [2 C] slots
  int* dirty;            // [CTAs]: whether the CTA took out values that are not finite (join_kernel puts them back)
  int4* header;          // [C]: the unit that the pair began and did not end: b, hk, tok0, parts (0: none)
  int kbox, vbox;        // rows of a TMA box: min(page, keys of a CTA), min(page, 128)
  int k_head, k_page;    // strides of head and page in the key map's last dimension
  int* status;
};

struct __align__(8) Barriers {
  uint64_t pre_full, q_full, o_done, drain, planned;
  uint64_t v_land[NSTAGE], v_ok[NSTAGE];
  uint64_t stage_full[NSTAGE], stage_free[NSTAGE];
  uint64_t s_full[NSBUF], p_ready[NSBUF], m_ready[NSBUF];
  uint32_t tmem_base;
  int abort_flag;
};

struct Ctx {
  Barriers* sb;
  uint32_t peer_abort;
  bool pair;
  int* status;
};

__device__ __forceinline__ bool pwait(uint64_t* bar, uint32_t parity, const Ctx& c, int err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 15u) == 0u) {
      if (*(volatile int*)&c.sb->abort_flag) return false;
      if (globaltimer_ns() - t0 > RW_WAIT_TIMEOUT_NS) {
        c.sb->abort_flag = 1;
        if (c.pair) st_shared_cluster_u32(c.peer_abort, 1u);
        report_status(c.status, err);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool pwait_warp(uint64_t* bar, uint32_t parity, const Ctx& c, int err) {
  return __all_sync(0xffffffffu, pwait(bar, parity, c, err));
}

template <int NCTA>
__device__ __forceinline__ void mma_ss_n(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if constexpr (NCTA == 2) mma_ss_pair(d, a, b, id, acc); else mma_ss(d, a, b, id, acc);
}
template <int NCTA>
__device__ __forceinline__ void mma_ts_n(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if constexpr (NCTA == 2) mma_ts_pair(d, a, b, id, acc); else mma_ts(d, a, b, id, acc);
}
template <int NCTA>
__device__ __forceinline__ void commit_n(uint64_t* bar) {  // arrives on every CTA's barrier
  if constexpr (NCTA == 2) tc_commit_pair_mc(bar, 0x3); else tc_commit(bar);
}

// ---------------------------------------------------------------- work
__device__ __forceinline__ int units_of(const Params& p, const Seq& s, int upt) { return (s.lq + upt - 1) / upt; }

// Key tiles of unit rt of a sequence (at least one: rows that see nothing are written too).
__device__ __forceinline__ int tiles_of(const Params& p, const Seq& s, int rt, int upt, int* keys) {
  const int end = min(s.lq, (rt + 1) * upt);
  const int k = p.causal ? max(0, s.kv - s.lq + end) : s.kv;
  *keys = k;
  return max(1, (k + BN - 1) / BN);
}

// The work is dealt out by cost: a unit of n tiles is UNIT_COST + n long.
struct Plan {
  long long cost[MAX_BATCH + 1];   // cost of the units of the sequences before each
  int units[MAX_BATCH + 1];        // units before each
  int longest;
};

// Filled by all threads; the caller synchronises.  cost[b + 1], units[b + 1] first hold
// the sequence's own numbers, then warp 0 sums them up.
__device__ __forceinline__ void plan_own(const Params& p, Plan& pl, int upt, int warp, int lane, int nwarps,
                                         bool report) {
  for (int b = warp; b < p.pool.B; b += nwarps) {
    const Seq s = paged::load_seq(p.pool, b, p.T, report && lane == 0 ? p.status : nullptr);
    const int nu = units_of(p, s, upt);
    long long sum = 0;
    int top = 0, keys;
    for (int rt = lane; rt < nu; rt += 32) {
      const int n = UNIT_COST + tiles_of(p, s, rt, upt, &keys);
      sum += n;
      top = max(top, n);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) {
      pl.cost[b + 1] = sum * p.pool.Hkv;
      pl.units[b + 1] = (int)min(0x7fffffffll, (long long)nu * p.pool.Hkv);
      atomicMax(&pl.longest, top);
    }
  }
}
// Number of units.  Sequences whose starts go up have far fewer than an int counts; others are reported (load_seq).
__device__ __forceinline__ long long plan_sum(const Params& p, Plan& pl, int lane) {
  long long ct = 0, cu = 0;
  for (int b0 = 0; b0 < p.pool.B; b0 += 32) {
    const int b = b0 + lane;
    long long t = b < p.pool.B ? pl.cost[b + 1] : 0;
    long long u = b < p.pool.B ? pl.units[b + 1] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, t, o);
      const long long z = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) { t += y; u += z; }
    }
    if (b < p.pool.B) {
      pl.cost[b + 1] = ct + t;
      pl.units[b + 1] = (int)(cu + u);
    }
    ct += __shfl_sync(0xffffffffu, t, 31);
    cu += __shfl_sync(0xffffffffu, u, 31);
  }
  if (lane == 0) { pl.cost[0] = 0; pl.units[0] = 0; }
  __syncwarp();
  return cu;
}

// Where a walker over the units in the order (sequence, head, row tile) stands.
struct Walk {
  int b, hk, rt, n, nu, keys;
  Seq s;
};

__device__ __forceinline__ void enter(const Params& p, Walk& w, int upt) {
  w.s = paged::load_seq(p.pool, w.b, p.T, nullptr);
  w.nu = units_of(p, w.s, upt);
}

// Whole warp: the unit with index u.
__device__ __forceinline__ Walk walk_to_unit(const Params& p, const Plan& pl, int u, int upt) {
  Walk w;
  int lo = 0, hi = p.pool.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pl.units[mid] <= u) lo = mid; else hi = mid - 1;
  }
  w.b = lo;
  enter(p, w, upt);
  const int r = u - pl.units[lo];
  w.hk = r / w.nu;
  w.rt = r - w.hk * w.nu;
  w.n = tiles_of(p, w.s, w.rt, upt, &w.keys);
  return w;
}
// Row tiles of a sequence with at most n key tiles: they are its first ones.
__device__ __forceinline__ int tiles_upto(const Params& p, const Seq& s, int nu, int n, int upt) {
  if (n < 1) return 0;
  if (s.kv <= (long long)n * BN) return nu;
  return p.causal ? paged::clampi((int)((long long)n * BN - (s.kv - s.lq)) / upt, 0, nu) : 0;
}
// The units ordered by their key tiles, the longest first: lane b's sequence has the row tiles [from, upto) of n key
// tiles, and `before` units are longer.
struct Ranks {
  Seq s;
  int nu, n, from, upto, before;
};
__device__ __forceinline__ Ranks ranks(const Params& p, int longest, int upt, int lane) {
  Ranks k{};
  if (lane < p.pool.B) {
    k.s = paged::load_seq(p.pool, lane, p.T, nullptr);
    k.nu = units_of(p, k.s, upt);
  }
  k.n = longest;
  k.upto = k.nu;
  k.from = tiles_upto(p, k.s, k.nu, longest - 1, upt);
  return k;
}
// Whole warp: the unit with index u in that order, no smaller than in the last call.
__device__ __forceinline__ Walk walk_to_rank(const Params& p, Ranks& k, int u, int upt, int lane) {
  for (int all; k.n > 1 && u >= k.before + (all = p.pool.Hkv * __reduce_add_sync(0xffffffffu, k.upto - k.from));) {
    k.before += all;
    --k.n;
    k.upto = k.from;
    k.from = tiles_upto(p, k.s, k.nu, k.n - 1, upt);
  }
  const int count = k.upto - k.from;
  int x = count * p.pool.Hkv;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  const int f = __ffs(__ballot_sync(0xffffffffu, k.before + x > u)) - 1;
  const int r = u - k.before - __shfl_sync(0xffffffffu, x - count * p.pool.Hkv, f);
  const int each = __shfl_sync(0xffffffffu, count, f);
  Walk w;
  w.b = f;
  enter(p, w, upt);
  w.hk = r / each;
  w.rt = __shfl_sync(0xffffffffu, k.from, f) + r - w.hk * each;
  w.n = tiles_of(p, w.s, w.rt, upt, &w.keys);
  return w;
}
// Whole warp: cost of the units before that one.
__device__ __forceinline__ long long cost_before(const Params& p, const Plan& pl, const Walk& w, int upt, int lane) {
  long long sum = 0, all = paged::div_count(pl.cost[w.b + 1] - pl.cost[w.b], p.pool.Hkv);
  int keys;
  for (int rt = lane; rt < w.rt; rt += 32) sum += UNIT_COST + tiles_of(p, w.s, rt, upt, &keys);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return pl.cost[w.b] + all * w.hk + sum;
}
// Whole warp: the unit in which the work before reaches cost t, and the cost before that unit.
__device__ __forceinline__ Walk walk_to_cost(const Params& p, const Plan& pl, long long t, int upt, int lane,
                                             long long* before) {
  Walk w;
  int lo = 0, hi = p.pool.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pl.cost[mid] <= t) lo = mid; else hi = mid - 1;
  }
  w.b = lo;
  enter(p, w, upt);
  const long long each = paged::div_count(pl.cost[lo + 1] - pl.cost[lo], p.pool.Hkv);
  w.hk = (int)paged::div_count(t - pl.cost[lo], each);
  long long at = pl.cost[lo] + each * w.hk;
  for (int r0 = 0; r0 < w.nu; r0 += 32) {
    int keys;
    const int n = r0 + lane < w.nu ? UNIT_COST + tiles_of(p, w.s, r0 + lane, upt, &keys) : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, at + x > t);  // lanes whose unit ends behind t
    if (behind) {
      const int f = __ffs(behind) - 1;
      w.rt = r0 + f;
      at += __shfl_sync(0xffffffffu, x - n, f);
      break;
    }
    at += __shfl_sync(0xffffffffu, x, 31);
  }
  w.n = tiles_of(p, w.s, w.rt, upt, &w.keys);
  *before = at;
  return w;
}
__device__ __forceinline__ void next_unit(const Params& p, Walk& w, int upt) {
  if (++w.rt == w.nu) {
    w.rt = 0;
    if (++w.hk == p.pool.Hkv) {
      w.hk = 0;
      do {
        ++w.b;
        enter(p, w, upt);
      } while (w.nu == 0 && w.b + 1 < p.pool.B);   // there is another unit: the caller has tiles left
    }
  }
  w.n = tiles_of(p, w.s, w.rt, upt, &w.keys);
}

template <bool HALF, int D>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p) {
  constexpr int NCTA = Shape<D>::NCTA;
  constexpr int Q_BYTES = Shape<D>::Q_BYTES;
  constexpr int Q_BOX = BM * 128;              // 128 rows x 64 channels
  constexpr int KROWS = Shape<D>::KROWS;
  // A key tile in shared memory: groups of 8 rows, in each the D / 64 blocks of 64 channels (8 x 128 bytes,
  // swizzled), so that one TMA box brings all channels of a page's rows.
  constexpr int K_GROUP = 1024 * (D / 64);
  extern __shared__ uint8_t dsmem_raw[];
  __shared__ Barriers sb;
  __shared__ Plan pl;
  __shared__ Seg seg_sh[2];
  __shared__ float m_sh[NSBUF][BM];
  __shared__ float fin[2 * NWG][BM];
  __shared__ uint8_t* row_out[BM];

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_q = smem;
  uint8_t* pre = smem + Q_BYTES;
  uint8_t* stages = pre + PRE_BYTES;
  const uint32_t rank = NCTA == 2 ? cluster_ctarank() : 0;
  const bool even = rank == 0;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0);
  const int lane = threadIdx.x & 31;
  const int pid = blockIdx.x / NCTA;
  const int upt = NCTA * p.tpc;                // tokens of a unit
  const int used = p.tpc * p.G;                // rows of a CTA that hold tokens

  if (threadIdx.x == WARP_LOAD * 32) {
    mbar_init(&sb.pre_full, 1);
    mbar_init(&sb.q_full, 1);
    mbar_init(&sb.o_done, 1);
    mbar_init(&sb.drain, 1);
    mbar_init(&sb.planned, 1);
    for (int t = 0; t < NSTAGE; ++t) {
      mbar_init(&sb.v_land[t], 1);
      mbar_init(&sb.v_ok[t], 32 * NCTA);
      mbar_init(&sb.stage_full[t], 1);
      mbar_init(&sb.stage_free[t], 1);
    }
    for (int b = 0; b < NSBUF; ++b) {
      mbar_init(&sb.s_full[b], 1);
      mbar_init(&sb.p_ready[b], NCTA * BM);
      mbar_init(&sb.m_ready[b], BM);
    }
    sb.abort_flag = 0;
    pl.longest = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == WARP_MMA) {
    if constexpr (NCTA == 2) {
      tmem_alloc_pair(&sb.tmem_base, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&sb.tmem_base, 512);
      tmem_relinquish();
    }
  }
  // rows of the Q tile that hold no token stay zero: no load reaches them
  for (int i = threadIdx.x; i < (BM - used) * (D / 8); i += NUM_THREADS) {
    const int r = used + i / (D / 8), c = i % (D / 8);
    *reinterpret_cast<uint4*>(smem_q + (c >> 3) * Q_BOX + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  griddep_wait();   // launched as a dependent: the cache and the lengths are written from here on
  __syncthreads();  // pl.longest
  plan_own(p, pl, upt, warp, lane, NUM_THREADS / 32, blockIdx.x == 0);
  __syncthreads();

  // ---- the planner's state (warp 11): its waves, then its share of the rest
  long long t = 0, t1 = 0, before = 0, t_base = 0, share = 1;  // pair c has [t_base + c share, t_base + (c + 1) share)
  int waves = 0, wave = 0, C = p.C;
  Walk wk{};
  Ranks rk{};
  bool in_tail = false, whole = false, sorted = false;
  auto plan_next = [&](int i) {
    Seg s{};
    if (whole) {
      // every other wave backwards: who has had a long unit gets a short one
      const int u = wave * C + ((wave & 1) ? C - 1 - pid : pid);
      if (wave < waves && u < pl.units[p.pool.B]) {
        wk = sorted ? walk_to_rank(p, rk, u, upt, lane) : walk_to_unit(p, pl, u, upt);
        ++wave;
        s.n = wk.n;
        s.slot = -1;
      }
    } else if (wave < waves) {
      wk = walk_to_unit(p, pl, wave * C + pid, upt);
      ++wave;
      s.n = wk.n;
      s.slot = -1;
    } else {
      while (t < t1 && s.n == 0) {
        if (!in_tail) {
          wk = walk_to_cost(p, pl, t, upt, lane, &before);
          in_tail = true;
        } else {
          before += UNIT_COST + wk.n;
          next_unit(p, wk, upt);
        }
        // a unit's own cost comes before its first tile: a share that begins or ends in it has none of its tiles
        const long long e = min(t1, before + UNIT_COST + wk.n);
        s.kv0 = (int)max(0ll, t - before - UNIT_COST);
        s.n = (int)max(0ll, e - before - UNIT_COST) - s.kv0;
        // a part: the unit's first one goes to the second slot of its pair (its share ends there), the others to the
        // first slot of theirs (their shares begin inside the unit)
        s.slot = s.n == wk.n ? -1 : (s.kv0 > 0 ? 2 * pid : 2 * pid + 1);
        t = e;
        if (even && lane == 0 && s.n > 0 && s.slot == 2 * pid + 1) {
          // the last pair whose share meets the unit
          const int c = (int)paged::div_count(before + UNIT_COST + wk.n - 1 - t_base, share);
          p.header[pid] = make_int4(wk.b, wk.hk, wk.rt * upt, c - pid + 1);
        }
      }
    }
    if (s.n) {
      s.b = wk.b;
      s.hk = wk.hk;
      s.tok0 = wk.rt * upt;
      s.s0 = wk.s.s0;
      s.lq = wk.s.lq;
      s.kv = wk.s.kv;
      s.all = p.causal ? max(0, min(s.kv, s.kv - s.lq + s.tok0 + 1)) : s.kv;
    }
    if (lane == 0) {
      seg_sh[i & 1] = s;
      mbar_arrive(&sb.planned);                // segment i is known (the loading warp reads it before the boundary)
    }
    __syncwarp();
  };
  if (warp == WARP_PLAN) {
    const long long U = plan_sum(p, pl, lane);
    const long long N = pl.cost[p.pool.B];       // of all work
    if (even && lane == 0) p.header[pid] = make_int4(0, 0, 0, 0);
    // about equal: no unit is over 1/8 longer than their mean
    const bool equal = (long long)pl.longest * U * 8 <= N * 9;
    int rounds = 1;
    if (U > 0 && U <= 0x7fffffffll) {
      if (U > C) rounds = ((unsigned)U + C - 1) / (unsigned)C;
      const float all = (float)N;            // (estimates: no division of integers for them)
      whole = fmaxf((float)pl.longest, rounds * __fdividef(all, (float)U)) <=
              fmaxf((float)MIN_SHARE, __fdividef(all, (float)C)) + JOIN_COST<D>;
      // (a lane a sequence.  With 12 ragged sequences of up to 600 tokens the order takes 88 us to 65 with head dim 64
      // and 99 to 96 with 128; with 32, when a CTA has many units, 177 to 175 and nothing: more go as they come)
      sorted = rounds > 1 && !equal && p.pool.B <= 32;
      if (sorted) rk = ranks(p, pl.longest - UNIT_COST, upt, lane);
    }
    if (whole)
      C = (int)min((long long)C, U);
    else if (N < (long long)C * MIN_SHARE)
      C = (int)min((long long)C, max(U, paged::div_count(N + MIN_SHARE - 1, MIN_SHARE)));
    if (whole) {
      if (pid < C) waves = rounds;
    } else if (pid < C && U <= 0x7fffffffll) {
      if (equal) waves = (int)paged::div_count(U, C);
      if (waves > 0 && waves * C < U) {
        const Walk f = walk_to_unit(p, pl, waves * C, upt);
        t_base = cost_before(p, pl, f, upt, lane);
      } else if (waves > 0) {
        t_base = N;
      }
      share = max(1ll, paged::div_count(N - t_base + C - 1, C));
      t = min(N, t_base + share * pid);
      t1 = min(N, t + share);
    }
    plan_next(0);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (NCTA == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sb.tmem_base;
  const Ctx cx{&sb, NCTA == 2 ? mapa_shared(smem_u32(&sb.abort_flag), rank ^ 1u) : 0u, NCTA == 2, p.status};
  auto aborted = [&]() { return *(volatile int*)&sb.abort_flag != 0; };
  // all threads, between two segments
  auto boundary = [&]() {
    tc_fence_before();
    if constexpr (NCTA == 2) cluster_sync(); else __syncthreads();
    tc_fence_after();
  };
  auto even_addr = [&](uint64_t* bar) { return NCTA == 2 ? mapa_shared(smem_u32(bar), 0) : smem_u32(bar); };
  // whether warp 11 looks through the values of tile j (of the unit): some row does not see all of it
  auto checked = [&](const Seg& sg, int j) { return (j + 1) * BN > sg.all; };

  if (warp == WARP_LOAD) {
    setmaxnreg_dec<REG_OTHER>();
    // a key tile: KROWS / kbox boxes; lane i holds page i's index, one lane issues
    const int nkp = KROWS / p.kbox;
    const int mask = (1 << p.pool.page_shift) - 1;
    const int koff = NCTA == 2 ? KROWS * (int)rank : 0;
    auto page_at = [&](const Seg& sg, int j) {
      const int row = (sg.kv0 + j) * BN + koff + lane * p.kbox;
      return lane < nkp && j < sg.n && row < sg.kv ? paged::raw_page_of(p.pool, sg.b, row) : 0;
    };
    auto load_k = [&](const Seg& sg, uint32_t dst, uint32_t bar, int j, int pages) {
      const int row0 = nkp == 1 ? ((sg.kv0 + j) * BN + koff) & mask : 0;  // within a page that holds several boxes
      pages = paged::checked_page(p.pool, pages, p.status);
      const int head = sg.hk * p.k_head;
      for_pages(head + pages * p.k_page, nkp, [&](int i, int line) {
        load_5d<NCTA>(dst + i * p.kbox * 2 * D, &tm_k, bar, 0, 0, 0, row0 >> 3, line);
      });
    };
    // q and the keys of the first tiles: for the next segment already while this one's output is written
    auto begin = [&](const Seg& sg) {
      int pk[NSBUF];
#pragma unroll
      for (int j = 0; j < NSBUF; ++j) pk[j] = page_at(sg, j);
      const int n_pre = min(sg.n, NSBUF);
      if (even && lane == 0) {
        mbar_expect_tx(&sb.q_full, NCTA * (D / 64) * used * 128);
        mbar_expect_tx(&sb.pre_full, NCTA * HALF_TILE * n_pre);
      }
      __syncwarp();
      if (lane < D / 64)
        load_3d<NCTA>(smem_u32(smem_q) + lane * Q_BOX, &tm_q, even_addr(&sb.q_full), 64 * lane, sg.hk * p.G,
                      sg.s0 + sg.tok0 + (int)rank * p.tpc);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NSBUF; ++j)
        if (j < n_pre) load_k(sg, smem_u32(pre) + j * HALF_TILE, even_addr(&sb.pre_full), j, pk[j]);
    };
    int J0 = 0;
    bool begun = false;
    for (int si = 0;; ++si) {
      const Seg sg = seg_sh[si & 1];
      if (sg.n == 0) break;
      const uint32_t sph = (uint32_t)si & 1u;
      if (!begun && !aborted()) {
        begin(sg);
        begun = true;
      }
      if (begun) {
        int kp = page_at(sg, NSBUF);                 // page indices one tile ahead
        bool ok = true;
        for (int j = 0; j < sg.n; ++j) {
          const int J = J0 + j, st = J % NSTAGE;
          const bool has_k = j + NSBUF < sg.n, has_v = !checked(sg, sg.kv0 + j);
          const int kn = page_at(sg, j + 1 + NSBUF);
          if (J >= NSTAGE &&
              !(ok = pwait_warp(&sb.stage_free[st], (uint32_t)(J / NSTAGE - 1) & 1u, cx, RW_STATUS_TIMEOUT_LOAD)))
            break;
          if (even && lane == 0)
            mbar_expect_tx(&sb.stage_full[st], NCTA * HALF_TILE * ((has_k ? 1 : 0) + (has_v ? 1 : 0)));
          __syncwarp();
          if (has_k)
            load_k(sg, smem_u32(stages) + st * STAGE_BYTES + HALF_TILE, even_addr(&sb.stage_full[st]), j + NSBUF, kp);
          kp = kn;
        }
        // every copy has landed and every stage is released before the barriers are set up for the next segment
        if (lane == 0) {
          const int tail = sg.n > NSTAGE ? sg.n - NSTAGE : 0;
          if (even) {
            mbar_wait_drain(&sb.pre_full, sph);
            for (int J = J0 + tail; J < J0 + sg.n; ++J)
              mbar_wait_drain(&sb.stage_full[J % NSTAGE], (uint32_t)(J / NSTAGE) & 1u);
            mbar_wait_drain(&sb.q_full, sph);
          }
          if (ok)
            for (int J = J0 + tail; J < J0 + sg.n; ++J)
              mbar_wait_drain(&sb.stage_free[J % NSTAGE], (uint32_t)(J / NSTAGE) & 1u);
        }
        __syncwarp();
        // (the last release follows every MMA of the segment: q and the first key tiles are read no more)
        begun = false;
        if (ok && pwait_warp(&sb.planned, (uint32_t)(si + 1) & 1u, cx, RW_STATUS_TIMEOUT_LOAD)) {
          const Seg nx = seg_sh[(si + 1) & 1];
          if (nx.n > 0 && !__any_sync(0xffffffffu, aborted())) {
            begin(nx);
            begun = true;
          }
        }
      }
      J0 += sg.n;
      boundary();
    }
  } else if (warp == WARP_MMA) {
    setmaxnreg_dec<REG_OTHER>();
    int J0 = 0;
    uint32_t phases = 0;                       // of v_ok
    for (int si = 0;; ++si) {
      const Seg sg = seg_sh[si & 1];
      if (sg.n == 0) break;
      const uint32_t sph = (uint32_t)si & 1u;
      if (even && !aborted()) {
        constexpr uint32_t ID_QK = idesc<HALF>(NCTA * BM, BN, 0);
        constexpr uint32_t ID_PV = idesc<HALF>(NCTA * BM, D, 1);
        const uint64_t dq = umma_desc(smem_u32(smem_q), 16, 1024);
        const uint64_t dk_pre = umma_desc(smem_u32(pre), 16, K_GROUP);
        const uint64_t dv_st = umma_desc(smem_u32(stages), 16384, 1024);
        const uint64_t dk_st = umma_desc(smem_u32(stages + HALF_TILE), 16, K_GROUP);
        constexpr uint64_t PRE_DESC = HALF_TILE >> 4, STAGE_DESC = STAGE_BYTES >> 4;
        auto issue_qk = [](uint32_t ts, uint64_t a, uint64_t b) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss_n<NCTA>(ts, a + (uint64_t)(((kk >> 2) * Q_BOX + (kk & 3) * 32) >> 4),
                           b + (uint64_t)(((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), ID_QK, kk > 0 ? 1u : 0u);
        };
        auto issue_pv = [](uint32_t to, uint32_t ts, uint64_t b, bool acc) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_ts_n<NCTA>(to, ts + kk * 8, b + (uint64_t)((kk * 2048) >> 4), ID_PV, (acc || kk > 0) ? 1u : 0u);
        };
        bool ok = pwait_warp(&sb.q_full, sph, cx, RW_STATUS_TIMEOUT_MMA) &&
                  pwait_warp(&sb.pre_full, sph, cx, RW_STATUS_TIMEOUT_MMA);
        tc_fence_after();
        if (ok) {
          const int n_pre = min(sg.n, NSBUF);
          if (elect_one()) {
            for (int j = 0; j < n_pre; ++j) {
              const int bk = (J0 + j) % NSBUF;
              issue_qk(tmem + 128u + 128u * bk, dq, dk_pre + j * PRE_DESC);
              commit_n<NCTA>(&sb.s_full[bk]);
            }
          }
          __syncwarp();
        }
        int b = J0 % NSBUF, st = J0 % NSTAGE, J = J0, j = 0;
        // The tiles that have a QK to issue behind them and whose values nobody looks through: this thread has about
        // 1000 clocks a tile, and waits and commits take 100 each, so their loop asks nothing else (with the questions
        // of the last tiles in it, 2640 tokens over 34320 rows took 5 % longer).
        const int plain = min(sg.n - NSBUF, sg.all / BN - sg.kv0);
        uint32_t pb = (uint32_t)(J0 / NSBUF) & 1u, ps = (uint32_t)(J0 / NSTAGE) & 1u;
        for (; j < plain && ok; ++j, ++J) {
          if (!(ok = pwait_warp(&sb.p_ready[b], pb, cx, RW_STATUS_TIMEOUT_MMA))) break;
          if (!(ok = pwait_warp(&sb.stage_full[st], ps, cx, RW_STATUS_TIMEOUT_MMA))) break;
          tc_fence_after();
          if (elect_one()) {
            issue_pv(tmem, tmem + 128u + 128u * b, dv_st + st * STAGE_DESC, j > 0);
            issue_qk(tmem + 128u + 128u * b, dq, dk_st + st * STAGE_DESC);
            commit_n<NCTA>(&sb.s_full[b]);
            commit_n<NCTA>(&sb.stage_free[st]);
          }
          __syncwarp();
          if (++b == NSBUF) { b = 0; pb ^= 1u; }
          if (++st == NSTAGE) { st = 0; ps ^= 1u; }
        }
#pragma unroll 1
        for (; j < sg.n && ok; ++j, ++J) {
          if (!(ok = pwait_warp(&sb.p_ready[b], (uint32_t)(J / NSBUF) & 1u, cx, RW_STATUS_TIMEOUT_MMA))) break;
          if (!(ok = pwait_warp(&sb.stage_full[st], (uint32_t)(J / NSTAGE) & 1u, cx, RW_STATUS_TIMEOUT_MMA))) break;
          if (checked(sg, sg.kv0 + j)) {
            if (!(ok = pwait_warp(&sb.v_ok[st], (phases >> st) & 1u, cx, RW_STATUS_TIMEOUT_MMA))) break;
            phases ^= 1u << st;
          }
          tc_fence_after();
          if (elect_one()) {
            issue_pv(tmem, tmem + 128u + 128u * b, dv_st + st * STAGE_DESC, j > 0);
            if (j == sg.n - 1) commit_n<NCTA>(&sb.o_done);
            if (j + NSBUF < sg.n) {
              issue_qk(tmem + 128u + 128u * b, dq, dk_st + st * STAGE_DESC);
              commit_n<NCTA>(&sb.s_full[b]);
            }
            commit_n<NCTA>(&sb.stage_free[st]);
          }
          __syncwarp();
          if (++b == NSBUF) b = 0;
          if (++st == NSTAGE) st = 0;
        }
        if (elect_one()) {
          if constexpr (NCTA == 2) tc_commit_pair_mc(&sb.drain, 0x1); else tc_commit(&sb.drain);
          mbar_wait_drain(&sb.drain, sph);
        }
        __syncwarp();
      }
      J0 += sg.n;
      boundary();
    }
  } else if (warp == WARP_V) {
    setmaxnreg_dec<REG_OTHER>();
    int J0 = 0;
    for (int si = 0;; ++si) {
      const Seg sg = seg_sh[si & 1];
      if (sg.n == 0) break;
      // values: 128 / vbox boxes a tile
      if (!aborted()) {
        const int nvp = BN / p.vbox;
        const int mask = (1 << p.pool.page_shift) - 1;
        auto page_at = [&](int j) {
          const int row = (sg.kv0 + j) * BN + lane * p.vbox;
          return lane < nvp && j < sg.n && row < sg.kv ? paged::raw_page_of(p.pool, sg.b, row) : 0;
        };
        int vp = page_at(0);
        for (int j = 0; j < sg.n; ++j) {
          const int J = J0 + j, st = J % NSTAGE;
          const int vn = page_at(j + 1);
          if (J >= NSTAGE &&
              !pwait_warp(&sb.stage_free[st], (uint32_t)(J / NSTAGE - 1) & 1u, cx, RW_STATUS_TIMEOUT_LOAD))
            break;
          // a tile that is looked through lands on this CTA's own barrier
          const bool look = checked(sg, sg.kv0 + j);
          const uint32_t bar = look ? smem_u32(&sb.v_land[st]) : even_addr(&sb.stage_full[st]);
          const uint32_t dst = smem_u32(stages) + st * STAGE_BYTES;
          if (look && lane == 0) mbar_expect_tx(&sb.v_land[st], HALF_TILE);
          const int row0 = ((sg.kv0 + j) * BN) & mask;
          vp = paged::checked_page(p.pool, vp, p.status);
          __syncwarp();
          for_pages(vp, nvp, [&](int i, int pg) {
            load_4d<NCTA>(dst + i * p.vbox * 128, &tm_v, bar, 64 * (int)rank, sg.hk, nvp == 1 ? row0 : 0, pg);
          });
          vp = vn;
        }
      }
      J0 += sg.n;
      boundary();
    }
  } else if (warp == WARP_PLAN) {
    setmaxnreg_dec<REG_OTHER>();
    int J0 = 0;
    uint32_t phases = 0;                       // of v_land
    bool dirty = false;
    for (int si = 0;; ++si) {
      const Seg sg = seg_sh[si & 1];
      if (sg.n == 0) break;
      plan_next(si + 1);
      // the values of the tiles that not every row sees whole: zeros behind the sequence's end, nothing that is not
      // finite
      for (int j = max(0, sg.all / BN - sg.kv0); j < sg.n; ++j) {
        const int st = (J0 + j) % NSTAGE;
        if (!pwait_warp(&sb.v_land[st], (phases >> st) & 1u, cx, RW_STATUS_TIMEOUT_LOAD)) break;
        phases ^= 1u << st;
        uint8_t* v = stages + st * STAGE_BYTES;
        // rows of the tile that the sequence has (a checked tile need not be its last)
        const int rows = min(BN, max(0, sg.kv - (sg.kv0 + j) * BN)), r0 = lane >> 3;
        auto at = [&](int r) { return reinterpret_cast<uint4*>(v + r * 128 + (((lane & 7) ^ (r & 7)) << 4)); };
#pragma unroll 1
        for (int r = r0 + (max(0, rows - r0) + 3) / 4 * 4; r < BN; r += 4) *at(r) = make_uint4(0, 0, 0, 0);
        uint32_t found = 0;
        if (rows >= BN) {
// (unrolled further, this loop cost the softmax loop 7 %: the kernel's code no longer fits where it did)
#pragma unroll 2
          for (int r = r0; r < BN; r += 4) found |= paged::has_nonfinite<HALF>(*at(r));
        } else {
#pragma unroll 1
          for (int r = r0; r < rows; r += 4) found |= paged::has_nonfinite<HALF>(*at(r));
        }
        if (found & paged::SIGNS) {
          dirty = true;
#pragma unroll 1
          for (int r = r0; r < rows; r += 4) {
            uint4 x = *at(r);
            if (paged::take_nonfinite<HALF>(x)) *at(r) = x;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive_cluster(even_addr(&sb.v_ok[st]));
      }
      __syncwarp();
      J0 += sg.n;
      boundary();
    }
    dirty = __any_sync(0xffffffffu, dirty);
    if (lane == 0) p.dirty[blockIdx.x] = dirty;
  } else {
    // ------------------------------------------------------------ softmax, then the output
    setmaxnreg_inc<REG_SOFTMAX>();
    const int w = warp >> 2;
    const int r = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_base;
    const float sl2 = p.scale_log2;
    const uint32_t p_ready0 = even_addr(&sb.p_ready[0]);
    int J0 = 0;
    for (int si = 0;; ++si) {
      // Only what the tiles' loop needs is held through it; the rest is read, or worked out, again behind it (held
      // in registers it was spilled, inside the loop).
      const Seg& sg = seg_sh[si & 1];
      const int n = sg.n, kv0 = sg.kv0;
      if (n == 0) break;
      const uint32_t sph = (uint32_t)si & 1u;
      int lim, all;
      {
        const int rtok = r / p.G, tok = sg.tok0 + (int)rank * p.tpc + rtok;
        // keys of the row; a row without a token takes them all (its values go nowhere)
        lim = p.causal && r < used && tok < sg.lq ? max(0, sg.kv - sg.lq + tok + 1) : sg.kv;
        // keys that every row of the CTA sees
        all = p.causal ? max(0, min(sg.kv, sg.kv - sg.lq + sg.tok0 + (int)rank * p.tpc + 1)) : sg.kv;
      }
      bool ok = !aborted();
      float m_base = -INFINITY;
      uint64_t l2 = 0ull;
      for (int j = w; j < n && ok; j += NWG) {
        const int J = J0 + j;
        const int b = J % NSBUF;
        const uint32_t tS = tmem + lane_base + 128u + 128u * b;
        if (!(ok = pwait_warp(&sb.s_full[b], (uint32_t)(J / NSBUF) & 1u, cx, RW_STATUS_TIMEOUT_SOFTMAX))) break;
        tc_fence_after();
        const int key0 = (kv0 + j) * BN;
        const bool masked = key0 + BN > all;
        const int cut = lim - key0;              // columns from here on are not seen
        auto load_half = [&](int h, uint32_t (&v)[2][32], const bool mask) {
          tmem_ld32(tS + 64 * h, v[0]);
          tmem_ld32(tS + 64 * h + 32, v[1]);
          tmem_wait_ld();
          reg_fence32(v[0]);
          reg_fence32(v[1]);
          if (mask) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (64 * h + 32 * c + e >= cut) v[c][e] = __float_as_uint(-INFINITY);
          }
        };
        auto quarter_max = [](const uint32_t (&v)[32], float row_max) -> float {
          float a[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t* x = &v[g * 8];
            float u = fmax3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
            u = fmax3(u, __uint_as_float(x[3]), __uint_as_float(x[4]));
            u = fmax3(u, __uint_as_float(x[5]), __uint_as_float(x[6]));
            a[g] = fmaxf(u, __uint_as_float(x[7]));
          }
          return fmax3(row_max, fmax3(a[0], a[1], a[2]), a[3]);
        };
        auto quarter_exp = [](const uint32_t (&v)[32], uint64_t s2, uint64_t nm2, uint32_t (&pk)[32], const int o,
                              uint64_t (&lacc)[2]) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t xv = ffma2(f2_pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), s2, nm2);
            float x0, x1;
            f2_unpack(xv, x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            lacc[e & 1] = fadd2(lacc[e & 1], f2_pack(p0, p1));
            pk[o + e] = Num<HALF>::pack(p0, p1);
          }
        };
        const uint64_t s2 = f2_pack(sl2, sl2);
        // One pass over S where nothing is masked, against the exponent base of this
        // warpgroup's previous tile; it stands when tile j - 1 kept that base and this
        // tile does not ask for a new one.  Otherwise S is read a second time.
        float row_max = -INFINITY, m_prev = -INFINITY;
        bool fast = false;
        const bool one_pass = j >= NWG && !masked;
        if (one_pass) {
          uint32_t pk[2][32];
          uint64_t l2f = l2;
          const float nm0 = minus_base<HALF>(m_base, sl2);
          const uint64_t nm02 = f2_pack(nm0, nm0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[2][32];
            load_half(h, v, false);
            uint64_t lacc[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              row_max = quarter_max(v[c], row_max);
              quarter_exp(v[c], s2, nm02, pk[h], 16 * c, lacc);
            }
            l2f = fadd2(l2f, fadd2(lacc[0], lacc[1]));
          }
          const int Jp = J - 1;
          if (!(ok = pwait_warp(&sb.m_ready[Jp % NSBUF], (uint32_t)(Jp / NSBUF) & 1u, cx, RW_STATUS_TIMEOUT_SOFTMAX)))
            break;
          m_prev = m_sh[Jp % NSBUF][r];
          const float m_new = fmaxf(m_prev, row_max);
          // (a base of -inf has made P NaN: it never stands)
          fast = __all_sync(0xffffffffu, m_prev == m_base && m_base != -INFINITY &&
                                             !((m_new - m_prev) * sl2 > RESCALE_THRESHOLD));
          if (fast) {
            m_sh[b][r] = m_base;
            mbar_arrive(&sb.m_ready[b]);
            l2 = l2f;
            tmem_st32(tS, pk[0]);
            tmem_st32(tS + 32, pk[1]);
          }
        }
        if (!fast) {
          if (!one_pass) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t v[2][32];
              load_half(h, v, masked);
              row_max = quarter_max(v[1], quarter_max(v[0], row_max));
            }
            if (j > 0) {
              const int Jp = J - 1;
              if (!(ok = pwait_warp(&sb.m_ready[Jp % NSBUF], (uint32_t)(Jp / NSBUF) & 1u, cx,
                                    RW_STATUS_TIMEOUT_SOFTMAX)))
                break;
              m_prev = m_sh[Jp % NSBUF][r];
            }
          }
          const float m_new = fmaxf(m_prev, row_max);
          const bool need = (m_new - m_prev) * sl2 > RESCALE_THRESHOLD;  // false where both are -inf
          const float m_use = need ? m_new : m_prev;
          m_sh[b][r] = m_use;
          mbar_arrive(&sb.m_ready[b]);
          if (j > 0 && __any_sync(0xffffffffu, need)) {
            const float alpha = need ? fast_exp2((m_prev - m_use) * sl2) : 1.f;
            if (!(ok = pwait_warp(&sb.stage_free[(J - 1) % NSTAGE], (uint32_t)((J - 1) / NSTAGE) & 1u, cx,
                                  RW_STATUS_TIMEOUT_SOFTMAX)))
              break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + 32 * c, o);
              tmem_wait_ld();
              reg_fence32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(tO + 32 * c, o);
            }
          }
          if (m_base != m_use) {
            float lo, hi;
            f2_unpack(l2, lo, hi);
            const float f = fast_exp2((m_base - m_use) * sl2);
            l2 = f2_pack(lo * f, hi * f);
            m_base = m_use;
          }
          const float nm = m_use == -INFINITY ? 0.f : minus_base<HALF>(m_use, sl2);  // nothing seen yet: weights of exp2(-inf) = 0
          const uint64_t nm2 = f2_pack(nm, nm);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pk[32];
            uint64_t lacc[2] = {0ull, 0ull};
            uint32_t v[2][32];
            load_half(h, v, masked);
#pragma unroll
            for (int c = 0; c < 2; ++c) quarter_exp(v[c], s2, nm2, pk, 16 * c, lacc);
            l2 = fadd2(l2, fadd2(lacc[0], lacc[1]));
            tmem_st32(tS + 32 * h, pk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_cluster(p_ready0 + 8u * (uint32_t)b);
      }
      {
        float lo, hi;
        f2_unpack(l2, lo, hi);
        fin[2 * w][r] = m_base;
        fin[2 * w + 1][r] = lo + hi;
      }
      named_bar_sync(1, SOFTMAX_THREADS);
      const float m_fin = fmaxf(fin[0][r], fin[2][r]);
      float l_row = 0.f;
#pragma unroll
      for (int g = 0; g < NWG; ++g) {
        const float lg = fin[2 * g + 1][r];
        // an empty sum adds nothing; anything else, NaN included, counts
        if (lg != 0.f) l_row += lg * fast_exp2((fin[2 * g][r] - m_fin) * sl2);
      }
      ok = __all_sync(0xffffffffu, ok) && !aborted();
      if (ok) ok = pwait_warp(&sb.o_done, sph, cx, RW_STATUS_TIMEOUT_SOFTMAX);
      tc_fence_after();
      constexpr int CW = D / NWG;                  // channels of a warpgroup
      int r_again = r;
      asm volatile("" : "+r"(r_again));
      const int rtok = r_again / p.G, rg = r_again - rtok * p.G;  // the row's token (of the CTA's) and head (of the group's)
      const int tok = sg.tok0 + (int)rank * p.tpc + rtok;         // within the sequence
      const bool there = r < used && tok < sg.lq;
      if (ok && sg.slot >= 0) {
        float* base = p.scratch + (long long)sg.slot * Shape<D>::SLOT_FLOATS;
        constexpr int R = NCTA * BM;
        const int row = (int)rank * BM + r;
#pragma unroll 1
        for (int c = 0; c < CW / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + CW * w + 32 * c, o);
          tmem_wait_ld();
          reg_fence32(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) base[(long long)(CW * w + 32 * c + e) * R + row] = __uint_as_float(o[e]);
        }
        if (w == 0) {
          base[(long long)D * R + row] = m_fin;
          base[(long long)D * R + R + row] = l_row;
        }
      } else if (sg.slot < 0) {
        // O / l in the type -> shared memory (the first stage, which no MMA reads any more and no load
        // reaches before the boundary) -> whole rows
        uint8_t* staged = stages;
        const float inv = l_row != 0.f ? 1.f / l_row : 0.f;
        if (ok && (warp & 3) * 32 < used) {         // a warp without a token has nothing to store
#pragma unroll 1
          for (int c = 0; c < CW / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + CW * w + 32 * c, o);
            tmem_wait_ld();
            reg_fence32(o);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int ch = (CW * w + 32 * c) / 8 + q;
              uint4 v;
              v.x = Num<HALF>::pack(__uint_as_float(o[8 * q + 0]) * inv, __uint_as_float(o[8 * q + 1]) * inv);
              v.y = Num<HALF>::pack(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv);
              v.z = Num<HALF>::pack(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv);
              v.w = Num<HALF>::pack(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv);
              if (r < used)
                *reinterpret_cast<uint4*>(staged + (ch >> 3) * Q_BOX + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
            }
          }
        }
        if (w == 0)
          row_out[r] = there ? p.out + (long long)(sg.s0 + tok) * p.o_sl + (long long)(sg.hk * p.G + rg) * p.o_sh
                             : nullptr;
        if (ok && w == 0 && there) {
          const long long at = (long long)(sg.s0 + tok) * p.Hq + sg.hk * p.G + rg;
          const float l = l_row * DOWN<HALF>;
          if (p.lse) p.lse[at] = l != 0.f ? (m_fin * sl2 + log2f(l)) * 0.6931471805599453f : -INFINITY;
          if (p.row_b) p.row_b[at] = l != 0.f ? -(m_fin * sl2 + log2f(l)) : -INFINITY;
        }
        named_bar_sync(1, SOFTMAX_THREADS);
        constexpr int CH = D / 8;
        for (int i = threadIdx.x; ok && i < used * CH; i += SOFTMAX_THREADS) {
          const int rr = i / CH, ch = i % CH;
          uint8_t* dst = row_out[rr];
          if (dst != nullptr)
            *reinterpret_cast<uint4*>(dst + 16 * ch) = *reinterpret_cast<const uint4*>(
                staged + (ch >> 3) * Q_BOX + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4));
        }
        fence_proxy_async_smem();                  // read before the next segment's loads go there
      }
      J0 += n;
      boundary();
    }
  }

  if (warp == WARP_LOAD && lane == 0 && aborted()) {
    // after a timeout some copies may be in flight without a wait for them: time to land
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
  }
  if (threadIdx.x == 0) griddep_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if constexpr (NCTA == 2) cluster_sync();
  if (warp == WARP_MMA) {
    tc_fence_after();
    if constexpr (NCTA == 2) tmem_dealloc_pair(tmem, 512); else tmem_dealloc(tmem, 512);
  }
}

// Row r of CTA `rank` of the unit of sequence b, key head hk and first token tok0: adds the values that are not finite
// and that the row sees, of the tiles that chunk_kernel looked through, to channels [c0, c0 + 32) of its output.
template <bool HALF, int D>
__device__ __noinline__ void mend_row(const Params& p, const Seq& sq, int b, int hk, int tok0, int tok, int head, int c0) {
  const int all = p.causal ? max(0, min(sq.kv, sq.kv - sq.lq + tok0 + 1)) : sq.kv;
  const int lim = p.causal ? max(0, sq.kv - sq.lq + tok + 1) : sq.kv;
  uint16_t* out = reinterpret_cast<uint16_t*>(p.out + (long long)(sq.s0 + tok) * p.o_sl + (long long)head * p.o_sh);
  paged::for_nonfinite<HALF>(p.pool, b, hk, all / BN * BN, min(lim, sq.kv), c0, 32, [&](int c, float x) {
    out[c] = (uint16_t)Num<HALF>::pack(Num<HALF>::wide(out[c]).x + x, 0.f);
  });
}

constexpr int MEND_BLOCKS = 64;

// Joins the parts of a unit that more than one pair worked on: the block of the pair that
// began it, in the order of the keys.  A thread has one row and 32 channels.  If values
// that are not finite were taken out somewhere, MEND_BLOCKS more go through all units and
// put them back (otherwise they leave at once); the rows of joined units get theirs here.
template <bool HALF, int D>
__global__ void __launch_bounds__(BM) join_kernel(const __grid_constant__ Params p) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int NCTA = Shape<D>::NCTA;
  constexpr int R = NCTA * BM;
  constexpr long long SLOT = Shape<D>::SLOT_FLOATS;
  const int pid = blockIdx.x, r = threadIdx.x;
  const int rank = blockIdx.y, row = rank * BM + r, c0 = 32 * blockIdx.z;
  const int rtok = r / p.G, g = r - rtok * p.G;
  auto any_dirty = [&]() {
    int d = 0;
    for (int i = r; i < NCTA * p.C; i += BM) d |= __ldcg(p.dirty + i);
    return __syncthreads_or(d) != 0;
  };
  if (pid >= p.C) {
    if (!any_dirty()) return;
    const int upt = NCTA * p.tpc;
    int u = 0;
    for (int b = 0; b < p.pool.B; ++b) {
      const Seq sq = paged::load_seq(p.pool, b, p.T, nullptr);
      const int nu = units_of(p, sq, upt);
      for (int i = 0; i < nu * p.pool.Hkv; ++i, ++u) {
        if (u % MEND_BLOCKS != pid - p.C) continue;
        const int hk = i / nu, tok0 = (i - hk * nu) * upt, tok = tok0 + rank * p.tpc + rtok;
        int joined = 0;
        for (int c = r; c < p.C; c += BM) {
          const int4 h = __ldcg(p.header + c);
          joined |= h.w > 0 && h.x == b && h.y == hk && h.z == tok0;
        }
        if (__syncthreads_or(joined)) continue;
        if (r < p.tpc * p.G && tok < sq.lq) mend_row<HALF, D>(p, sq, b, hk, tok0, tok, hk * p.G + g, c0);
      }
    }
    return;
  }
  const int4 h = __ldcg(p.header + pid);
  const int n = min(h.w, p.C - pid);
  if (n <= 0) return;
  const bool mend = any_dirty();
  const Seq sq = paged::load_seq(p.pool, h.x, p.T, nullptr);
  const int tok = h.z + rank * p.tpc + rtok;
  if (r >= p.tpc * p.G || tok >= sq.lq) return;
  // part i: slot 2 pid + 1, then 2 (pid + 1), 2 (pid + 2), ...
  auto slot = [&](int i) { return p.scratch + (2LL * (pid + i) + (i == 0)) * SLOT + row; };
  float m = -INFINITY;
#pragma unroll 8
  for (int i = 0; i < n; ++i) m = fmaxf(m, __ldcg(slot(i) + (long long)D * R));
  float acc[32], l = 0.f;
#pragma unroll
  for (int e = 0; e < 32; ++e) acc[e] = 0.f;
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const float* sl = slot(i);
    const float f = fast_exp2((__ldcg(sl + (long long)D * R) - base) * p.scale_log2);
    l += f * __ldcg(sl + (long long)D * R + R);
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[e] += f * __ldcg(sl + (long long)(c0 + e) * R);
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int head = h.y * p.G + g;
  uint4* dst = reinterpret_cast<uint4*>(p.out + (long long)(sq.s0 + tok) * p.o_sl + (long long)head * p.o_sh + 2 * c0);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 v;
    v.x = Num<HALF>::pack(acc[8 * q + 0] * inv, acc[8 * q + 1] * inv);
    v.y = Num<HALF>::pack(acc[8 * q + 2] * inv, acc[8 * q + 3] * inv);
    v.z = Num<HALF>::pack(acc[8 * q + 4] * inv, acc[8 * q + 5] * inv);
    v.w = Num<HALF>::pack(acc[8 * q + 6] * inv, acc[8 * q + 7] * inv);
    dst[q] = v;
  }
  if (c0 == 0) {
    const long long at = (long long)(sq.s0 + tok) * p.Hq + head;
    l *= DOWN<HALF>;
    if (p.lse) p.lse[at] = l != 0.f ? (m * p.scale_log2 + log2f(l)) * 0.6931471805599453f : -INFINITY;
    if (p.row_b) p.row_b[at] = l != 0.f ? -(m * p.scale_log2 + log2f(l)) : -INFINITY;
  }
  if (mend) mend_row<HALF, D>(p, sq, h.x, h.y, h.z, tok, head, c0);
}

// ---------------------------------------------------------------- host
// The value pool as (D, Hkv, page_size, num_pages), boxes of 64 channels x 1 head x `rows` rows of a page.
int value_map(CUtensorMap* m, const rw_paged_t* c, int rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return RW_ERR_DRIVER;
  // strides of dimensions of one are never used, but have to be valid
  const long long sp = c->num_pages == 1 ? 8 : c->v_sp, sh = c->Hkv == 1 ? 8 : c->v_sh;
  cuuint64_t dims[4] = {(cuuint64_t)c->D, (cuuint64_t)c->Hkv, (cuuint64_t)c->page_size, (cuuint64_t)c->num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)sh * 2, (cuuint64_t)c->v_sl * 2, (cuuint64_t)sp * 2};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, dt(c->dtype), 4, c->v, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? RW_OK : RW_ERR_DRIVER;
}

bool supported(const rw_paged_t* c) {
  // coordinates are 32-bit, and a row's stride of 16 has to fit a map's
  return key_lines(c).lines < (1ll << 31) && c->k_sl < (1ll << 35);
}

int grid_size(int D) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return D == 128 ? sms / 2 : sms;
}

long long workspace_bytes(int D) {
  const long long C = grid_size(D);
  return C * (2 * 4 * (D == 128 ? Shape<128>::SLOT_FLOATS : Shape<64>::SLOT_FLOATS) + 32);
}

template <bool HALF, int D>
int launch_one(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Params& p, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int NCTA = Shape<D>::NCTA;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(chunk_kernel<HALF, D>), Shape<D>::SMEM, &done))
    return RW_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(NCTA * p.C);
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = Shape<D>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = NCTA;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = NCTA == 2 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, chunk_kernel<HALF, D>, mq, mk, mv, p) != cudaSuccess) return RW_ERR_CUDA;
  return launch_dependent(join_kernel<HALF, D>, dim3(p.C + MEND_BLOCKS, NCTA, D / 32), dim3(BM), 0, st, p) == cudaSuccess
             ? RW_OK : RW_ERR_CUDA;
}

int launch(const rw_paged_t* cache, const Pool& pool, const Call& c, void* workspace, cudaStream_t st) {
  Params p{};
  p.pool = pool;
  p.T = c.T; p.Hq = c.Hq; p.G = c.Hq / pool.Hkv; p.causal = c.causal;
  p.tpc = BM / p.G;
  p.C = grid_size(cache->D);
  if (p.C < 1) return RW_ERR_CUDA;
  // no more CTAs than the work can be dealt to: units by the tokens, tiles by the table's width
  const long long upt = (cache->D == 128 ? Shape<128>::NCTA : Shape<64>::NCTA) * p.tpc;
  const long long units = pool.Hkv * std::min(pool.B * ((c.longest + upt - 1) / upt), c.T / upt + pool.B);
  const long long tiles = ((long long)cache->table_width * cache->page_size + BN - 1) / BN;
  const long long cost = units * (UNIT_COST + std::max(1ll, tiles));
  p.C = (int)std::max(1ll, std::min((long long)p.C, std::max(units, (cost + MIN_SHARE - 1) / MIN_SHARE)));
  p.scale_log2 = c.scale_log2;
  p.out = static_cast<uint8_t*>(c.out);
  p.o_sl = 2 * c.o_sl; p.o_sh = 2 * c.o_sh;
  p.lse = c.lse;
  p.row_b = c.row_b;
  p.header = static_cast<int4*>(workspace);
  p.dirty = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + 16LL * p.C);
  p.scratch = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 32LL * p.C);
  const int krows = cache->D == 128 ? Shape<128>::KROWS : Shape<64>::KROWS;
  p.kbox = cache->page_size < krows ? cache->page_size : krows;
  p.vbox = cache->page_size < BN ? cache->page_size : BN;
  const KeyLines kl = key_lines(cache);
  p.k_head = cache->Hkv == 1 ? 0 : (int)(cache->k_sh / kl.step);
  p.k_page = cache->num_pages == 1 ? 0 : (int)(cache->k_sp / kl.step);
  p.status = c.status;
  CUtensorMap mq, mk, mv;
  if (q_map(&mq, c.q, cache->dtype, c.T, c.Hq, cache->D, c.q_sl, c.q_sh, p.G, p.tpc) ||
      key_map(&mk, cache, p.kbox) || value_map(&mv, cache, p.vbox))
    return RW_ERR_DRIVER;
  if (cache->dtype == RW_DTYPE_FP16)
    return cache->D == 128 ? launch_one<true, 128>(mq, mk, mv, p, st) : launch_one<true, 64>(mq, mk, mv, p, st);
  return cache->D == 128 ? launch_one<false, 128>(mq, mk, mv, p, st) : launch_one<false, 64>(mq, mk, mv, p, st);
}

}  // namespace chunk
}  // namespace rw
