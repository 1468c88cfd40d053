// Attention of few new tokens over a paged cache: o = softmax(q k^T * scale) v for the
// rows of a sequence that share a key head (tokens x heads of the group), 16 at most (over
// short tables blocks of 16), with the keys split over the whole device.
//
// Such a call is bound by memory: every cached row of k and v is read once for 4 * 16
// products an element at most.  What decides is that all SMs read all the time, however
// ragged the lengths are.  So the work is one sequence of key tiles (64 keys of one
// sequence and key head), in the order (sequence, head, tile), and CTA c of C
// takes the c-th share of ceil(N / C) of its N tiles; lengths are read on the
// device, nothing is planned on the host.  A share covers the end of one unit (the
// tiles of one sequence and head), whole units, and the beginning of another.
// Units that lie in one share are written out directly; the others leave their
// unnormalised O, m and l in scratch, and join_kernel joins them, in the order of the keys.
// The first tiles of a CTA's next segment are on their way while one is written out.
//
// In a CTA each of the 4 warps takes 16 keys of a 64-key tile with a running maximum and
// sum of its own (mma.sync m16n8k16 feeds far more than memory delivers here: a tile of
// 32 KB costs a warp 32 MMAs), so the warps only meet for the loads; the 4 states are
// joined when the unit's tiles are done.
//
// A short call is bound by its launches and the loads that wait for one another.  Where the
// device holds a cluster of CTAs for every unit, and a CTA then has few tiles of the longest
// unit there can be, the cluster joins its parts through distributed shared memory, and adds
// the weights, whose scores it still has: one launch, no plan and no scratch.
//
// Keys and values come through a ring of 3 stages
// of 16-byte cp.async; rows behind the last visible one are filled with zeros, never
// read, so what a page holds there (NaN included) does not matter.
//
// 32 tokens over up to 8191 rows (ragged), 8 key heads of 128: 105 us, 5.7 TB/s, start and join included; 2 tokens over
// up to 131072 rows, 2 key heads: 48.6 us, 5.0 TB/s; 1 token over 511 rows, by clusters: 5.1 us.
#include <algorithm>

#include "paged.cuh"
#include "paged_chunk.h"

namespace rw {
namespace rows {

using paged::Num;
using paged::Pool;
using paged::Seq;

constexpr int TILE = 64;
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int RT = 16;          // rows of a unit
constexpr int STAGES = 3;

struct Params {
  Pool pool;
  const uint8_t* q;
  uint8_t* out;
  float* lse;                   // [T, Hq] natural logarithm, or null
  long long q_sl, q_sh, o_sl, o_sh;  // byte strides
  int T, Hq, G, causal;
  int cs, pitch;                // CLUSTER: CTAs of a unit, keys of a CTA at most
  int rows_most;                // rows of a sequence and key head at most
  float scale_log2;
  float* part;                  // [2 C][16 * D + 32]: O, then m, then l
  int2* header;                 // [B * Hkv]: first slot and parts of every unit (0: written whole)
  // raw scores (log2 units) and (m, 1 / l) of every row, for the weight sums; null otherwise
  float* scores;                // [B * Hkv * rows_most][cap]
  float2* row_ml;               // [B * Hkv * rows_most]
  float* sums;
  long long sums_sb, sums_sh;
  long long cap;
  float* block_sums;            // [blocks of 16 rows][B * Hkv][cap]: what each block adds, if there are several
  int* status;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // 0: the 16 bytes are zeroed and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

template <bool HALF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A sequence, its rows of a key head, and what the last of them sees.
struct Entry {
  Seq s;
  int rows;   // 0..rows_most (a sequence with more is one with more than max_q_len tokens)
  int keys;   // keys that any of the rows sees
};

// (of the rows from row0 on, 16 at most)
__device__ __forceinline__ Entry load_entry(const Params& p, int b, int* status, int row0 = 0) {
  Entry n;
  n.s = paged::load_seq(p.pool, b, p.T, status);
  n.rows = max(0, min(RT, (int)min((long long)p.rows_most, (long long)n.s.lq * p.G) - row0));
  n.keys = 0;
  if (n.rows > 0) n.keys = p.causal ? max(0, n.s.kv - n.s.lq + (row0 + n.rows - 1) / p.G + 1) : n.s.kv;
  return n;
}

// A segment: the tiles [k0, k0 + n) of a unit of n_tiles, which is tile u0 of all.
struct Seg {
  Entry en;
  int n, k0, n_tiles, b, hk, all;
  long long u0;
};

// Keys that every row from row0 on sees: tiles behind them are looked through for values that are not finite.
__device__ __forceinline__ int keys_of_all(const Params& p, const Entry& n, int row0) {
  return p.causal ? min(n.keys, max(0, n.s.kv - n.s.lq + row0 / p.G + 1)) : n.keys;
}

// Tiles of an entry: at least one while it has rows, so that rows that see nothing are written too.
__device__ __forceinline__ int tiles_of(const Entry& n) {
  return n.rows > 0 ? max(1, (n.keys + TILE - 1) / TILE) : 0;
}

// Channels c, c + 1 of row r of a unit: O / l, and with channel 0 the row's lse and (m, 1 / l).
template <bool HALF>
__device__ __forceinline__ void put_row(const Params& p, const Entry& en, int b, int hk, int r, int c, float2 v,
                                        float mm, float ll) {
  const int tok = r / p.G, g = r - tok * p.G;
  const float inv = ll != 0.f ? 1.f / ll : 0.f;
  uint8_t* dst = p.out + (long long)(en.s.s0 + tok) * p.o_sl + (long long)(hk * p.G + g) * p.o_sh;
  *reinterpret_cast<uint32_t*>(dst + 2 * c) = Num<HALF>::pack(v.x * inv, v.y * inv);
  if (c == 0) {
    if (p.lse)
      p.lse[(long long)(en.s.s0 + tok) * p.Hq + hk * p.G + g] =
          ll != 0.f ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
    if (p.row_ml) {
      const long long line = ((long long)b * p.pool.Hkv + hk) * p.rows_most + r;
      p.row_ml[line] = make_float2(mm == -INFINITY ? 0.f : mm, inv);
    }
  }
}

__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// What a score weighs, by its row's m and 1 / l.  One of -inf (a key that the row does not see, above all) weighs nothing,
// also where the row's total is NaN.
__device__ __forceinline__ float weight_of(float score, float2 ml) {
  return score == -INFINITY ? 0.f : fast_exp2(score - ml.x) * ml.y;
}

constexpr int MAX_CLUSTER = 16;
constexpr int CLUSTER_TILES = 16;  // of a CTA at most

// CLUSTER: the CTAs of a cluster share the tiles of one unit.
template <bool HALF, int D, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 2) rows_kernel(const __grid_constant__ Params p) {
  constexpr int PITCH = 2 * D;               // bytes of a row in shared memory
  constexpr int CH = D / 8;                  // 16-byte chunks of a row
  constexpr int STAGE = 2 * TILE * PITCH;    // k, then v
  constexpr int SLOT = RT * D + 2 * RT;      // floats of a part
  constexpr int LOADS = TILE * CH / THREADS; // cp.async of k (and of v) a thread
  constexpr int RSTEP = THREADS / CH;        // rows between two of them
  constexpr float UP = HALF ? 32768.f : 1.f; // factor of the weights in the second product
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ long long base[THREADS + 1];
  __shared__ Seg seg[2];
  __shared__ struct { long long t, ebase; Entry en; int e; } plan;
  __shared__ float sm_m[WARPS][RT], sm_l[WARPS][RT];
  __shared__ float2 ml[CLUSTER ? RT : 1];  // m and 1 / l of every row
  __shared__ int dirty;         // 1: the segment has values that are not finite (paged.cuh)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int grp = lane >> 2, quad = lane & 3;
  griddep_launch_dependents();
  griddep_wait();

  const int cta = blockIdx.x;
  const int rank = CLUSTER ? cta % p.cs : 0;
  int row0 = 0;         // CLUSTER: the unit's first row
  long long share = 1, t1 = 0;
  if constexpr (CLUSTER) {
    const int head = cta / p.cs;
    row0 = RT * blockIdx.y;
    Seg s;
    s.b = head / p.pool.Hkv;
    s.hk = head - s.b * p.pool.Hkv;
    s.en = load_entry(p, s.b, blockIdx.y == 0 && cta % (p.cs * p.pool.Hkv) == 0 && tid == 0 ? p.status : nullptr, row0);
    if (s.en.rows == 0) return;              // (with the whole cluster)
    s.n_tiles = tiles_of(s.en);
    const int per = (s.n_tiles + p.cs - 1) / p.cs;
    s.k0 = min(rank * per, s.n_tiles);
    s.n = min(per, s.n_tiles - s.k0);
    s.all = keys_of_all(p, s.en, row0);
    s.u0 = 0;
    if (tid == 0) {
      seg[0] = s;
      seg[1].n = 0;
      dirty = 0;
    }
  } else {
    // ---- tiles before every thread's run of entries, and of all
    const int NE = p.pool.B;
    const int run = (NE + THREADS - 1) / THREADS;
    {
      long long mine = 0;
      for (int e = tid * run; e < min(NE, (tid + 1) * run); ++e)
        mine += (long long)tiles_of(load_entry(p, e, blockIdx.x == 0 ? p.status : nullptr)) * p.pool.Hkv;
      long long x = mine;
  #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __shared__ long long wsum[WARPS];
      if (lane == 31) wsum[warp] = x;
      __syncthreads();
      for (int w = 0; w < warp; ++w) x += wsum[w];
      base[tid] = x - mine;
      if (tid == THREADS - 1) base[THREADS] = x;
      __syncthreads();
    }
    const long long N = base[THREADS];
    const int C = (int)max(1ll, min((long long)gridDim.x, N));  // (no share without a tile)
    if (cta >= C) return;
    share = paged::div_count(N + C - 1, C);
    if (share * cta >= N) return;  // (the last CTAs may find nothing left)
    t1 = min(N, share * (cta + 1));
  }
  // The segments of the share, one ahead, by thread 0: seg[i & 1] is segment i (n == 0: there is none).
  auto advance = [&](int i) {
    Seg s;
    s.n = 0;
    if (plan.t < t1) {
      while (plan.t >= plan.ebase + (long long)tiles_of(plan.en) * p.pool.Hkv) {
        plan.ebase += (long long)tiles_of(plan.en) * p.pool.Hkv;
        plan.en = load_entry(p, ++plan.e, p.status);
      }
      s.en = plan.en;
      s.n_tiles = tiles_of(s.en);
      s.b = plan.e;
      s.hk = (int)paged::div_count(plan.t - plan.ebase, s.n_tiles);
      s.u0 = plan.ebase + (long long)s.hk * s.n_tiles;
      s.k0 = (int)(plan.t - s.u0);
      s.n = (int)(min(t1, s.u0 + s.n_tiles) - plan.t);
      s.all = keys_of_all(p, s.en, 0);
      plan.t += s.n;
    }
    seg[i & 1] = s;
  };
  if (!CLUSTER && tid == 0) {
    const long long t0 = share * cta;
    const int run = (p.pool.B + THREADS - 1) / THREADS;
    int lo = 0, hi = THREADS - 1;
    while (lo < hi) {   // last thread whose run of entries begins at or before t0
      const int mid = (lo + hi + 1) >> 1;
      if (base[mid] <= t0) lo = mid; else hi = mid - 1;
    }
    plan.t = t0;
    plan.e = lo * run;
    plan.ebase = base[lo];
    plan.en = load_entry(p, plan.e, p.status);
    advance(0);
    dirty = 0;
  }
  __syncthreads();

  const uint32_t sbase = smem_u32(smem);
  const int slot_mask = (1 << p.pool.page_shift) - 1;
  // Page indices of tile k of a segment (lane i < 8 holds rows 8 i ..), and its loads into stage J mod STAGES.
  auto pages = [&](const Seg& s, int k) {
    const int row = (s.k0 + k) * TILE + 8 * (lane & 7);
    return (k < s.n && row < s.en.keys) ? paged::raw_page_of(p.pool, s.b, row) : 0;
  };
  auto load = [&](const Seg& s, int k, int J, int pg) {
    if (k < s.n) {
      const uint32_t st = sbase + (uint32_t)(J % STAGES) * STAGE;
      const int c = tid % CH, r0 = tid / CH, keys = s.en.keys, row0 = (s.k0 + k) * TILE;
      const uint8_t* kb = p.pool.k + (long long)s.hk * p.pool.k_sh + 16 * c;
      const uint8_t* vb = p.pool.v + (long long)s.hk * p.pool.v_sh + 16 * c;
      pg = paged::checked_page(p.pool, pg, p.status);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int r = r0 + i * RSTEP, row = row0 + r;
        const long long pi = __shfl_sync(0xffffffffu, pg, r >> 3);
        const bool there = row < keys;
        const int sl = there ? (row & slot_mask) : 0;
        const uint32_t d = st + r * PITCH + ((c ^ (r & 7)) << 4);
        cp16(d, kb + pi * p.pool.k_sp + sl * p.pool.k_sl, there);
        cp16(d + TILE * PITCH, vb + pi * p.pool.v_sp + sl * p.pool.v_sl, there);
      }
    }
    cp_commit();
  };
  int J0 = 0;           // tiles of the share before the current segment
  {
    const int pg0 = pages(seg[0], 0), pg1 = pages(seg[0], 1);
    load(seg[0], 0, 0, pg0);
    load(seg[0], 1, 1, pg1);
  }
  for (int si = 0;; ++si) {
    const Seg& sg = seg[si & 1];
    const int n = sg.n;
    if (!CLUSTER && n == 0) break;
    if (!CLUSTER && tid == 0) advance(si + 1);  // (read behind the barriers below)
    const Entry en = sg.en;
    const Seq s = en.s;
    const int hk = sg.hk, b = sg.b, k0 = sg.k0, all = sg.all;

    // ---- q fragments: rows grp and grp + 8, channels 16 kk + 2 quad (+ 8)
    uint32_t qf[D / 16][4];
    int lim[2];          // keys that the thread's two rows see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + grp + 8 * i;
      const int tok = r / p.G, g = r - tok * p.G;
      const bool there = grp + 8 * i < en.rows;
      lim[i] = there ? (p.causal ? max(0, s.kv - s.lq + tok + 1) : s.kv) : 0;
      const uint8_t* src = p.q + (long long)(s.s0 + tok) * p.q_sl + (long long)(hk * p.G + g) * p.q_sh;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][i] = there ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * kk + 4 * quad)) : 0u;
        qf[kk][2 + i] = there ? __ldg(reinterpret_cast<const uint32_t*>(src + 32 * kk + 16 + 4 * quad)) : 0u;
      }
    }
    int pg = pages(sg, STAGES - 1), npg0 = 0, npg1 = 0;
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int k = 0; k < n; ++k) {
      const int j = k0 + k;                  // of the unit
      cp_wait<STAGES - 2>();
      __syncthreads();                       // tile k is there, tile k - 1 is done with
      {
        const int nx = pages(sg, k + STAGES);
        load(sg, k + STAGES - 1, J0 + k + STAGES - 1, pg);
        pg = nx;
      }
      if (k == n - 1) {                      // the next segment's first page indices
        npg0 = pages(seg[(si + 1) & 1], 0);
        npg1 = pages(seg[(si + 1) & 1], 1);
      }
      const uint32_t ks = sbase + (uint32_t)((J0 + k) % STAGES) * STAGE;
      const uint32_t vs = ks + TILE * PITCH;
      const int kw = warp * 16;              // this warp's keys of the tile
      if (all < en.keys && (j + 1) * TILE > all) {
        bool found = false;
        for (int i = lane; i < 16 * CH; i += 32) {
          uint4* at = reinterpret_cast<uint4*>(smem + (vs - sbase) + (kw + i / CH) * PITCH + 16 * (i % CH));
          uint4 x = *at;
          if (paged::take_nonfinite<HALF>(x)) {
            *at = x;
            found = true;
          }
        }
        if (found) dirty = 1;
        __syncwarp();
      }
      float sc[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        // matrices: keys 0-7 / 8-15 (lane bit 4) x channels 0-7 / 8-15 (lane bit 3)
        const int r = kw + (lane & 7) + ((lane >> 4) << 3);
        const int c = 2 * kk + ((lane >> 3) & 1);
        uint32_t kf[4];
        ldm4(kf, ks + r * PITCH + ((c ^ (r & 7)) << 4));
        mma<HALF>(sc[0], qf[kk], kf[0], kf[1]);
        mma<HALF>(sc[1], qf[kk], kf[2], kf[3]);
      }
      const int key0 = j * TILE + kw + 2 * quad;
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = key0 + 8 * i + (x & 1);
          // selected, not added: whatever the product is, a key that is not seen has no weight
          const float v = key < lim[x >> 1] ? sc[i][x] * p.scale_log2 : -INFINITY;
          sc[i][x] = v;
          mx[x >> 1] = fmaxf(mx[x >> 1], v);
        }
      if (CLUSTER && p.sums) {
        float* sc_sh = reinterpret_cast<float*>(smem + STAGES * STAGE) + k * TILE + kw + 2 * quad;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (grp + 8 * x < en.rows)
              *reinterpret_cast<float2*>(sc_sh + (grp + 8 * x) * p.pitch + 8 * i) =
                  make_float2(sc[i][2 * x], sc[i][2 * x + 1]);
      }
      if (!CLUSTER && p.scores) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = grp + 8 * x;
            const long long line = ((long long)b * p.pool.Hkv + hk) * p.rows_most + r;
            if (r < en.rows && key0 + 8 * i < p.cap)
              *reinterpret_cast<float2*>(p.scores + line * p.cap + key0 + 8 * i) =
                  make_float2(sc[i][2 * x], sc[i][2 * x + 1]);
          }
      }
      float base_[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
        base_[x] = mx[x] == -INFINITY ? 0.f : mx[x];
      }
      if (__any_sync(0xffffffffu, mx[0] != m[0] || mx[1] != m[1])) {
        const float f0 = fast_exp2(m[0] - base_[0]), f1 = fast_exp2(m[1] - base_[1]);
        l[0] *= f0;
        l[1] *= f1;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= f0; o[i][1] *= f0;
          o[i][2] *= f1; o[i][3] *= f1;
        }
        m[0] = mx[0];
        m[1] = mx[1];
      }
      // weights in fp32 for the sum, rounded to the values' type for the product (its operands' type); fp16 ones 2^15 times
      // as large, so that a key with 2^-24 of the largest weight still has all its bits.  What the rounding leaves off
      // as a second operand, the weights whole, took 107.5 us instead of 105.0 (32 ragged tokens), 27.8 instead of 24.3
      // (up to 1000 rows), 22.8 instead of 20.3 (20 rows over 6005 keys): not worth half a step of a 16-bit output.
      uint32_t pf[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a0 = fast_exp2(sc[i][0] - base_[0]), a1 = fast_exp2(sc[i][1] - base_[0]);
        const float b0 = fast_exp2(sc[i][2] - base_[1]), b1 = fast_exp2(sc[i][3] - base_[1]);
        l[0] += a0 + a1;
        l[1] += b0 + b1;
        pf[2 * i] = Num<HALF>::pack(UP * a0, UP * a1);
        pf[2 * i + 1] = Num<HALF>::pack(UP * b0, UP * b1);
      }
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) {
        const int r = kw + (lane & 15);
        const int c = 2 * dd + (lane >> 4);
        uint32_t vf[4];
        ldm4t(vf, vs + r * PITCH + ((c ^ (r & 7)) << 4));
        mma<HALF>(o[2 * dd], pf, vf[0], vf[1]);
        mma<HALF>(o[2 * dd + 1], pf, vf[2], vf[3]);
      }
    }
    // The next segment's first two tiles go to the two stages that are free, while this one is written out.
    load(seg[(si + 1) & 1], 0, J0 + n, npg0);
    load(seg[(si + 1) & 1], 1, J0 + n + 1, npg1);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    __syncthreads();                         // the last tile's stage is free: it takes the warps' states

    // ---- join the warps: fo[warp][16][D], 16-byte chunks of a row in another order for every row
    float* fo = reinterpret_cast<float*>(smem + (CLUSTER ? 0 : ((J0 + n - 1) % STAGES) * STAGE));
    auto at = [&](int w, int r, int c) { return fo + (w * RT + r) * D + (((c >> 2) ^ (r & 7)) << 2) + (c & 3); };
    if (quad == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sm_m[warp][grp + 8 * x] = m[x];
        sm_l[warp][grp + 8 * x] = l[x];
      }
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float2*>(at(warp, grp + 8 * x, 8 * i + 2 * quad)) =
            make_float2(o[i][2 * x] * (1.f / UP), o[i][2 * x + 1] * (1.f / UP));
    __syncthreads();

    const bool whole = !CLUSTER && n == sg.n_tiles;
    // the parts of a unit: the first in the second slot of its CTA if that has a segment before it, the others in the
    // first slots of the CTAs that follow
    const int my_slot = 2 * cta + (si > 0 ? 1 : 0);
    if (!CLUSTER && k0 == 0 && tid == 0) {
      int parts = 0;
      if (!whole) {
        // up to the CTA that has the unit's last tile
        const int c = (int)paged::div_count(sg.u0 + sg.n_tiles - 1, share);
        parts = c - cta + 1;
      }
      p.header[(long long)b * p.pool.Hkv + hk] = make_int2(my_slot, parts);
    }
    float* slot = CLUSTER ? reinterpret_cast<float*>(smem + STAGE) : p.part + (long long)my_slot * SLOT;
    auto put = [&](int r, int c, float2 v, float mm, float ll) { put_row<HALF>(p, en, b, hk, row0 + r, c, v, mm, ll); };
    // 2 channels of a row a thread and step
    for (int i = tid; i < en.rows * (D / 2); i += THREADS) {
      const int r = i / (D / 2), c = 2 * (i % (D / 2));
      float mm = sm_m[0][r];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) mm = fmaxf(mm, sm_m[w][r]);
      const float bs = mm == -INFINITY ? 0.f : mm;
      float2 v = make_float2(0.f, 0.f);
      float ll = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = fast_exp2(sm_m[w][r] - bs);
        const float2 x = *reinterpret_cast<const float2*>(at(w, r, c));
        v.x += f * x.x;
        v.y += f * x.y;
        ll += f * sm_l[w][r];
      }
      if (dirty) {
        // taken-out values go to the rows that see them
        const int lim = p.causal ? max(0, s.kv - s.lq + (row0 + r) / p.G + 1) : s.kv;
        paged::for_nonfinite<HALF>(p.pool, b, hk, max(all / TILE, k0) * TILE, min(lim, (k0 + n) * TILE), c, 2,
                                   [&](int ch, float x) { (ch == c ? v.x : v.y) += x; });
      }
      if (whole) {
        put(r, c, v, mm, ll);
      } else {
        *reinterpret_cast<float2*>(slot + r * D + c) = v;
        if (c == 0) {
          slot[RT * D + r] = mm;
          slot[RT * D + RT + r] = ll;
        }
      }
    }
    if constexpr (CLUSTER) {
      constexpr int KEYS = CLUSTER_TILES * TILE / THREADS;   // of a thread, whose sums are read meanwhile
      float* dst = nullptr;
      const int keys = min(n * TILE, en.keys - k0 * TILE) - tid;
      float old[KEYS];
      if (p.sums) {
        dst = p.sums + b * p.sums_sb + hk * p.sums_sh;
        if (p.block_sums) dst = p.block_sums + (((long long)blockIdx.y * p.pool.B + b) * p.pool.Hkv + hk) * p.cap;
        dst += k0 * TILE + tid;
#pragma unroll
        for (int i = 0; i < KEYS; ++i) old[i] = !p.block_sums && i * THREADS < keys ? dst[i * THREADS] : 0.f;
      }
      cluster_sync();
      auto part = [&](int i, int at) { return mapa_shared(sbase + STAGE + 4 * at, (uint32_t)i); };
      // (m, l, and with them channels c, c + 1) of row r over the cluster, 8 parts' loads under way at once
      auto join = [&](int r, int c, bool with_o, float& mm, float& ll, float2& v) {
        mm = -INFINITY;
        ll = 0.f;
        v = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int w0 = 0; w0 < p.cs; w0 += 8) {
          float pm[8], pl[8];
          float2 px[8];
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            pm[w] = -INFINITY;
            pl[w] = 0.f;
            px[w] = make_float2(0.f, 0.f);
            if (w0 + w < p.cs) {
              pm[w] = ld_cluster(part(w0 + w, RT * D + r));
              pl[w] = ld_cluster(part(w0 + w, RT * D + RT + r));
              if (with_o) px[w] = ld_cluster2(part(w0 + w, r * D + c));
            }
          }
          float top = mm;
#pragma unroll
          for (int w = 0; w < 8; ++w) top = fmaxf(top, pm[w]);
          const float bs = top == -INFINITY ? 0.f : top, f0 = fast_exp2(mm - bs);
          v.x *= f0;
          v.y *= f0;
          ll *= f0;
          mm = top;
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const float f = fast_exp2(pm[w] - bs);
            v.x += f * px[w].x;
            v.y += f * px[w].y;
            ll += f * pl[w];
          }
        }
      };
      float mm, ll;
      float2 v;
      for (int i = rank * THREADS + tid; i < en.rows * (D / 2); i += p.cs * THREADS) {
        const int r = i / (D / 2), c = 2 * (i % (D / 2));
        join(r, c, true, mm, ll, v);
        put(r, c, v, mm, ll);
      }
      if (p.sums) {
        if (tid < en.rows) {
          join(tid, 0, false, mm, ll, v);
          ml[tid] = make_float2(mm == -INFINITY ? 0.f : mm, ll != 0.f ? 1.f / ll : 0.f);
        }
        __syncthreads();
        const float* sc_sh = reinterpret_cast<const float*>(smem + STAGES * STAGE) + tid;
#pragma unroll
        for (int i = 0; i < KEYS; ++i)
          if (i * THREADS < keys) {
            float add = 0.f;
            for (int r = 0; r < en.rows; ++r) add += weight_of(sc_sh[r * p.pitch + i * THREADS], ml[r]);
            dst[i * THREADS] = old[i] + add;
          }
      }
      cluster_sync();                        // no CTA leaves while another may read its part
      break;
    }
    J0 += n;
    __syncthreads();                         // the warps' states are read
    if (tid == 0) dirty = 0;
  }
}

// sums[b, hk, j] += what the blocks of rows added up, in their order.
constexpr int ADD_THREADS = 128;
__global__ void __launch_bounds__(ADD_THREADS) add_blocks_kernel(const __grid_constant__ Params p) {
  griddep_launch_dependents();
  griddep_wait();
  const int head = blockIdx.y, b = head / p.pool.Hkv, j = blockIdx.x * ADD_THREADS + threadIdx.x;
  const Seq s = paged::load_seq(p.pool, b, p.T, nullptr);
  const long long rows = min((long long)p.rows_most, (long long)s.lq * p.G), step = (long long)p.pool.B * p.pool.Hkv * p.cap;
  const float* src = p.block_sums + head * p.cap + j;
  float add = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 16 * RT) {
    float x[16];                             // all under way at once
#pragma unroll
    for (int i = 0; i < 16; ++i, src += step) {
      const int first = r0 + i * RT, last = (int)min(rows, (long long)first + RT) - 1;
      x[i] = first < rows && j < (p.causal ? s.kv - s.lq + last / p.G + 1 : s.kv) ? __ldcg(src) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) add += x[i];
  }
  if (j < s.kv && rows > 0) p.sums[b * p.sums_sb + (head - b * p.pool.Hkv) * p.sums_sh + j] += add;
}

// Joins the parts of the units that more than one CTA worked on: a block takes one row of
// one unit, its 8 groups of D / 4 threads every eighth part each.  (Joined by the last CTA
// that comes to a unit instead, without another launch, calls were slower
// throughout: 32 tokens of 2000 rows 54.3 us and 54.0, 2 of 131072 rows 86 and, at that time, 74; they take 49.6 now.)
constexpr int JOIN_GROUPS = 8;
constexpr int MAX_PARTS = 1024;  // CTAs of a launch: checked by the host

template <int D>
struct JoinShared {
  float fac[MAX_PARTS];
  float red[2][JOIN_GROUPS * D / 4 / 32];
  float4 acc[JOIN_GROUPS][D / 4];
};

// One row, by all threads of a block of JOIN_GROUPS * D / 4; h: the unit's header.
// PRE: parts of a thread whose values are loaded before the factors are known.
template <bool HALF, int D, int PRE>
__device__ __forceinline__ void join_row(const Params& p, const Entry& en, int b, int hk, int2 h, int r,
                                         JoinShared<D>& sh) {
  constexpr int SLOT = RT * D + 2 * RT;
  constexpr int NT = JOIN_GROUPS * D / 4;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = min(h.y, MAX_PARTS);
  // part 0 may be in its CTA's second slot, the others are in the first slots of the CTAs that follow
  auto slot = [&](int i) { return p.part + (i == 0 ? (long long)h.x : 2LL * (h.x / 2 + i)) * SLOT; };
  const int g = tid / (D / 4), c = 4 * (tid % (D / 4));
  // the first loads of everything at once
  float4 x[PRE];
#pragma unroll
  for (int j = 0; j < PRE; ++j)
    x[j] = g + j * JOIN_GROUPS < n ? __ldcg(reinterpret_cast<const float4*>(slot(g + j * JOIN_GROUPS) + r * D + c))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  const float m0 = tid < n ? __ldcg(slot(tid) + RT * D + r) : -INFINITY;
  const float l0 = tid < n ? __ldcg(slot(tid) + RT * D + RT + r) : 0.f;
  float mm = m0;
  for (int i = tid + NT; i < n; i += NT) {
    sh.fac[i] = __ldcg(slot(i) + RT * D + r);
    mm = fmaxf(mm, sh.fac[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (lane == 0) sh.red[0][warp] = mm;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) mm = fmaxf(mm, sh.red[0][i]);
  const float bs = mm == -INFINITY ? 0.f : mm;
  const float f0 = fast_exp2(m0 - bs);
  float ll = f0 * l0;
  if (tid < n) sh.fac[tid] = f0;
  for (int i = tid + NT; i < n; i += NT) {
    sh.fac[i] = fast_exp2(sh.fac[i] - bs);
    ll += sh.fac[i] * __ldcg(slot(i) + RT * D + RT + r);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
  if (lane == 0) sh.red[1][warp] = ll;
  __syncthreads();
  ll = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) ll += sh.red[1][i];
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float f, const float4& y) {
    v.x += f * y.x;
    v.y += f * y.y;
    v.z += f * y.z;
    v.w += f * y.w;
  };
#pragma unroll
  for (int j = 0; j < PRE; ++j)
    if (g + j * JOIN_GROUPS < n) add(sh.fac[g + j * JOIN_GROUPS], x[j]);
#pragma unroll 10
  for (int i = g + PRE * JOIN_GROUPS; i < n; i += JOIN_GROUPS)
    add(sh.fac[i], __ldcg(reinterpret_cast<const float4*>(slot(i) + r * D + c)));
  sh.acc[g][c / 4] = v;
  __syncthreads();
  if (g == 0) {
#pragma unroll
    for (int i = 1; i < JOIN_GROUPS; ++i) {
      const float4 x = sh.acc[i][c / 4];
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    put_row<HALF>(p, en, b, hk, r, c, make_float2(v.x, v.y), mm, ll);
    put_row<HALF>(p, en, b, hk, r, c + 2, make_float2(v.z, v.w), mm, ll);
  }
}

template <bool HALF, int D>
__global__ void __launch_bounds__(JOIN_GROUPS * D / 4) join_kernel(const __grid_constant__ Params p) {
  __shared__ JoinShared<D> sh;
  griddep_launch_dependents();
  griddep_wait();
  const int r = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int2 h = __ldcg(p.header + (long long)b * p.pool.Hkv + hk);  // (not written, and not used, without rows)
  const Entry en = load_entry(p, b, nullptr);
  if (r < en.rows && h.y > 0) join_row<HALF, D, 10>(p, en, b, hk, h, r, sh);  // (80 parts at once)
}

// join_kernel that also adds the weights: sums[b, hk, j] += sum over the rows, in their
// order, of exp2(score - m) / l.  A block takes every gridDim.x-th row to join, and keys.
template <bool HALF, int D>
__global__ void __launch_bounds__(JOIN_GROUPS * D / 4) join_sums_kernel(const __grid_constant__ Params p) {
  constexpr int SLOT = RT * D + 2 * RT;
  constexpr int NT = JOIN_GROUPS * D / 4;
  __shared__ JoinShared<D> sh;
  __shared__ float2 ml[RT];                  // m and 1 / l of every row
  griddep_launch_dependents();
  griddep_wait();
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31;
  const long long unit = (long long)b * p.pool.Hkv + hk;
  const int2 h = __ldcg(p.header + unit);
  const Entry en = load_entry(p, b, nullptr);
  const int rows = en.rows;
  if (rows == 0) return;
  for (int r = tid >> 5; r < rows; r += NT / 32) {
    float2 x;
    if (h.y == 0) {
      x = __ldcg(p.row_ml + unit * p.rows_most + r);
    } else {
      float mm = -INFINITY, ll = 0.f;
      const float* at = p.part + RT * D + r;
      auto slot = [&](int i) { return (i == 0 ? (long long)h.x : 2LL * (h.x / 2 + i)) * SLOT; };
      for (int i = lane; i < h.y; i += 32) mm = fmaxf(mm, __ldcg(at + slot(i)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
      mm = mm == -INFINITY ? 0.f : mm;
      for (int i = lane; i < h.y; i += 32) ll += fast_exp2(__ldcg(at + slot(i)) - mm) * __ldcg(at + slot(i) + RT);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
      x = make_float2(mm, ll != 0.f ? 1.f / ll : 0.f);
    }
    if (lane == 0) ml[r] = x;
  }
  __syncthreads();
  float* dst = p.sums + b * p.sums_sb + hk * p.sums_sh;
  const float* sc = p.scores + unit * p.rows_most * p.cap;
  // 4 keys a thread (a key tile's scores are there to its end): one wave of blocks
  for (int j = 4 * (blockIdx.x * NT + tid); j < en.keys; j += 4 * gridDim.x * NT) {
    float4 add = make_float4(0.f, 0.f, 0.f, 0.f);
    float old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = j + i < en.keys ? dst[j + i] : 0.f;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(sc + r * p.cap + j));
      const float2 m = ml[r];
      add.x += weight_of(x.x, m);
      add.y += weight_of(x.y, m);
      add.z += weight_of(x.z, m);
      add.w += weight_of(x.w, m);
    }
    const float a[4] = {add.x, add.y, add.z, add.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < en.keys) dst[j + i] = old[i] + a[i];
  }
  if (h.y > 0)
    // (the last blocks first: a sequence shorter than the table leaves them without keys)
    for (int r = gridDim.x - 1 - blockIdx.x; r < rows; r += gridDim.x) {
      __syncthreads();
      join_row<HALF, D, 1>(p, en, b, hk, h, r, sh);  // (with 10, 16 ragged tokens 48.1 -> 49.2 us: fewer blocks fit)
    }
}

// CTAs of a launch: as many as stay resident (2 an SM with a head of 128, 4 with 64).
inline int grid_size(int D) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms * (D == 128 ? 2 : 4);
}

// Which kernel: 16 rows of a sequence and key head are all that rows_kernel can use of a
// key tile it has read; where there may be more, the tiles of chunk_kernel, or blocks of 16 (clusters_for).
inline bool few_rows(long long rows) { return rows <= RT; }

struct Layout {
  long long part, header, ml, scores, total;  // byte offsets
};

inline Layout layout(int D, int C, int B, int Hkv, long long rows, long long cap, bool sums) {
  Layout l;
  l.part = 0;
  l.header = (2LL * C * (RT * D + 2 * RT) * 4 + 255) & ~255LL;
  l.ml = (l.header + 8LL * B * Hkv + 255) & ~255LL;
  const long long lines = (long long)B * Hkv * rows;
  l.scores = l.ml + (sums ? (lines * 8 + 255) & ~255LL : 0);
  l.total = l.scores + (sums ? lines * cap * 4 : 0);
  return l;
}

// Sequences of a launch by shares.  With weights every row's scores are kept for the second kernel, for as many keys as
// the table has room for: a batch whose scores would take more than SCORE_BYTES goes in slices that take no more (one
// sequence's, if that is more), so that a wide table cannot make a decoding step run out of memory.  A slice more is
// a start and a joining more: 256 sequences of 2154 rows on average, 32 heads, a table of 32768 (1 GB of scores) 549 us
// in one, 572 in two, 696 in eight slices; 64 of 2141 rows, 64 heads, a table of 131072 (2.1 GB) 312, 389 in four.
constexpr long long SCORE_BYTES = 1ll << 30;
inline int slice_of(int B, int Hkv, long long rows, long long cap, bool sums) {
  const long long each = 4 * Hkv * rows * cap;
  return sums && each > 0 ? (int)std::min((long long)B, std::max(1ll, SCORE_BYTES / each)) : B;
}

// A launch of the CLUSTER kernel: CTAs of a unit (0: units are shared out among all CTAs instead), keys of a CTA at most,
// dynamic shared memory.
//
// A cluster saves a second launch, the plan and what goes through scratch: 3 to 6 us, with weights 9.  What it may lose
// is that its CTAs have more tiles than an equal share of all CTAs would be, 0.6 to 0.9 us each with a head of 128, half
// of that with 64.  By cluster and by shares, us: 8 heads of 128, 500 rows 6.1 and 9.2, 4000 rows 10.6 and 14.1, 8000
// rows (8 tiles a CTA) 14.9 and 17.1, 16000 rows (16 tiles) 24.0 and 21.2; 2 heads of 64, 511 rows 5.1 and 8.2, 16000
// rows 14.9 and 19.2; 32 ragged sequences x 8 heads, up to 500 rows 15.4 and 26.5, up to 1000 rows 23.9 and 31.9; 128
// of them 68.8 and 79.5, with equal lengths 104 and 98.  With weights: 8 heads, 500 rows 7.2 and 17.2, 8000 rows 17.9
// and 21.3, 16000 rows 27.7 and 26.9.
//
// More than 16 rows are so many blocks of 16, which read the keys from L2 at the same time: while all CTAs are
// resident that is over before the tiles of chunk_kernel have filled their pipeline.  A tile takes a CTA 0.9 us, with two
// CTAs on an SM 1.6.  By blocks and by chunk_kernel, us: 8 heads x 20 rows over 505 keys 8.7 and 18.1, over 6005 20.3 and
// 38.9; x 64 rows over 516 keys 10.4 and 19.3; x 256 rows over 564 keys 14.9 and 20.0, over 2064 (2 CTAs an SM, 17 tiles
// each) 28.3 and 29.2; x 512 rows over 628 keys (10 tiles) 23.7 and 20.1. 
// What each block adds to the sums goes to scratch; add_blocks_kernel adds it up in the blocks' order: 8 heads x 64 rows
// over 516 keys with weights 14.1 us, by chunk_kernel and weigh_kernel 25.5; x 256 rows 26.1 and 27.4.
struct Clusters {
  int cs, pitch, bytes;
};
inline Clusters clusters_for(int D, long long heads, long long rows, long long cap, bool sums) {
  const long long tiles = std::max(1ll, (cap + TILE - 1) / TILE), blocks = (rows + RT - 1) / RT, units = heads * blocks;
  const int all = grid_size(D), sm = D == 128 ? 2 : 4, half = 128 / D;
  if (all == 0 || units >= (1 << 30)) return {0, 0, 0};
  for (int cs = MAX_CLUSTER; cs >= 1; cs /= 2) {
    const long long per = (tiles + cs - 1) / cs;
    const long long bytes = STAGES * 4 * TILE * D + (sums ? 4 * std::min(rows, (long long)RT) * per * TILE : 0);
    // as many CTAs as are resident together, by shared memory (4 KB of it is static, or the system's); not all
    // clusters of 16 fit that the SMs would hold (16 of them, two CTAs an SM, took two rounds)
    const long long fit = std::min((long long)sm, (220 << 10) / (bytes + 4096)) * (all / sm);
    if (cs > 1 && (cs / 2 >= tiles || per > CLUSTER_TILES * (sums ? 1 : 4) || units * cs > (cs > 8 ? fit * 3 / 4 : fit)))
      continue;
    long long most;
    if (blocks > 1) most = half * (units * cs * 2 > all ? std::min(20, 8 * cs) : 20);
    else most = std::min((long long)CLUSTER_TILES, half * 8 + units * tiles / all);
    if (sums) most = std::min(most, (long long)CLUSTER_TILES);
    if (blocks > 1 && units > fit) break;    // (with weights, 256 units of 6 tiles 40 us, by chunk_kernel 27)
    if (per <= most) return {cs, (int)per * TILE, (int)bytes};
    break;
  }
  return {0, 0, 0};
}
inline long long block_sums_bytes(long long heads, long long rows, long long cap, bool sums) {
  return sums && rows > RT ? 4 * ((rows + RT - 1) / RT) * heads * cap : 0;
}

template <bool HALF, int D>
int launch_cluster(const Params& p, int bytes, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0}, done_size{0};
  constexpr int MOST = STAGES * 4 * TILE * D + 4 * RT * CLUSTER_TILES * TILE;
  const void* kernel = reinterpret_cast<const void*>(rows_kernel<HALF, D, true>);
  if (!ensure_smem_attr(kernel, MOST, &done) || !ensure_cluster_attr(kernel, &done_size)) return RW_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.pool.B * p.pool.Hkv * p.cs), (unsigned)((p.rows_most + RT - 1) / RT));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, rows_kernel<HALF, D, true>, p) != cudaSuccess) return RW_ERR_CUDA;
  if (!p.block_sums) return RW_OK;
  return launch_dependent(add_blocks_kernel, dim3((unsigned)((p.cap + ADD_THREADS - 1) / ADD_THREADS), p.pool.B * p.pool.Hkv),
                          dim3(ADD_THREADS), 0, stream, p) == cudaSuccess ? RW_OK : RW_ERR_CUDA;
}

template <bool HALF, int D>
int launch_rows(const Params& p, int C, int cluster_bytes, cudaStream_t stream) {
  if (p.cs) return launch_cluster<HALF, D>(p, cluster_bytes, stream);
  static std::atomic<unsigned long long> done{0};
  const int bytes = STAGES * 2 * TILE * 2 * D;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(rows_kernel<HALF, D, false>), bytes, &done)) return RW_ERR_CUDA;
  if (launch_dependent(rows_kernel<HALF, D, false>, dim3(C), dim3(THREADS), bytes, stream, p) != cudaSuccess)
    return RW_ERR_CUDA;
  constexpr int NT = JOIN_GROUPS * D / 4;
  const unsigned bx = p.sums ? (unsigned)std::min(1024ll, (p.cap + 4 * NT - 1) / (4 * NT)) : (unsigned)p.rows_most;
  return launch_dependent(p.sums ? join_sums_kernel<HALF, D> : join_kernel<HALF, D>, dim3(bx, p.pool.Hkv, p.pool.B),
                          dim3(NT), 0, stream, p) == cudaSuccess ? RW_OK : RW_ERR_CUDA;
}

int run_rows(const rw_paged_t* cache, const Pool& pool, const chunk::Call& c, long long rows, float* sums,
             long long sums_sb, long long sums_sh, void* workspace, long long workspace_bytes, cudaStream_t st) {
  const long long cap = (long long)cache->table_width * cache->page_size;
  const int C = grid_size(cache->D);
  if (C == 0 || C > MAX_PARTS) return RW_ERR_CUDA;
  const Clusters cl = clusters_for(cache->D, (long long)cache->B * pool.Hkv, rows, cap, sums != nullptr);
  if (cap == 0) sums = nullptr;
  const long long need = cl.cs ? block_sums_bytes((long long)cache->B * pool.Hkv, rows, cap, sums != nullptr) : 0;
  if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return RW_ERR_INVALID_ARG;
  const int slice = cl.cs ? cache->B : slice_of(cache->B, pool.Hkv, rows, cap, sums != nullptr);
  const Layout lay = layout(cache->D, C, slice, pool.Hkv, rows, cap, sums != nullptr);
  if (cl.cs == 0 && (!workspace || !aligned16(workspace) || workspace_bytes < lay.total)) return RW_ERR_INVALID_ARG;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p{};
  p.pool = pool;
  p.q = static_cast<const uint8_t*>(c.q);
  p.out = static_cast<uint8_t*>(c.out);
  p.lse = c.lse;
  p.q_sl = 2 * c.q_sl; p.q_sh = 2 * c.q_sh; p.o_sl = 2 * c.o_sl; p.o_sh = 2 * c.o_sh;
  p.T = c.T; p.Hq = c.Hq; p.G = c.Hq / pool.Hkv; p.causal = c.causal;
  p.rows_most = (int)rows;
  p.cs = cl.cs;
  p.pitch = cl.pitch;
  p.scale_log2 = c.scale_log2;
  if (need) p.block_sums = static_cast<float*>(workspace);
  if (cl.cs == 0) {
    p.part = reinterpret_cast<float*>(ws + lay.part);
    p.header = reinterpret_cast<int2*>(ws + lay.header);
    p.scores = sums ? reinterpret_cast<float*>(ws + lay.scores) : nullptr;
    p.row_ml = sums ? reinterpret_cast<float2*>(ws + lay.ml) : nullptr;
  }
  p.sums_sb = sums_sb; p.sums_sh = sums_sh;
  p.cap = cap;
  p.status = c.status;
  const auto launch = cache->dtype == RW_DTYPE_FP16 ? (cache->D == 128 ? launch_rows<true, 128> : launch_rows<true, 64>)
                                                    : (cache->D == 128 ? launch_rows<false, 128> : launch_rows<false, 64>);
  for (int b = 0; b < cache->B; b += slice) {
    p.pool.B = std::min(slice, cache->B - b);
    p.pool.table = pool.table + b * pool.table_stride;
    p.pool.q_starts = pool.q_starts + b;
    p.pool.kv_lens = pool.kv_lens + b;
    p.sums = sums ? sums + b * sums_sb : nullptr;
    // no more CTAs than there can be tiles: the others would only cost their launch
    const long long most = (long long)p.pool.B * pool.Hkv * std::max(1ll, (cap + TILE - 1) / TILE);
    if (int e = launch(p, (int)std::min((long long)C, most), cl.bytes, st)) return e;
  }
  return RW_OK;
}

// The chunk kernels plan MAX_BATCH sequences a launch.
int run_tiles(const rw_paged_t* cache, const Pool& pool, chunk::Call c, float* sums, long long sums_sb,
              long long sums_sh, void* workspace, long long workspace_bytes, cudaStream_t st) {
  const long long parts = chunk::workspace_bytes(cache->D);
  if (!chunk::supported(cache)) return RW_ERR_UNSUPPORTED;
  if (!workspace || !aligned16(workspace) || workspace_bytes < parts + (sums ? 4LL * c.T * c.Hq : 0))
    return RW_ERR_INVALID_ARG;
  c.row_b = sums ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + parts) : nullptr;
  for (int b = 0; b < cache->B; b += chunk::MAX_BATCH) {
    Pool some = pool;
    some.B = std::min(chunk::MAX_BATCH, cache->B - b);
    some.table += b * pool.table_stride;
    some.q_starts += b;
    some.kv_lens += b;
    if (int e = chunk::launch(cache, some, c, workspace, st)) return e;
    if (sums)
      if (int e = weigh::launch(cache, some, c, sums + b * sums_sb, sums_sb, sums_sh, st)) return e;
  }
  return RW_OK;
}

}  // namespace rows
}  // namespace rw

extern "C" int rw_paged_attn(const rw_paged_t* cache, const void* q, void* out, float* lse, int T, int Hq,
                             int max_q_len, long long q_sl, long long q_sh, long long o_sl, long long o_sh, int causal,
                             float softmax_scale, float* sums, long long sums_sb, long long sums_sh, void* workspace,
                             long long workspace_bytes, int* status, void* stream) {
  using namespace rw;
  paged::Pool pool;
  if (int e = paged::make_pool(cache, &pool)) return e;
  if (T < 0 || Hq < 1 || Hq % pool.Hkv || max_q_len < 0 || !cache->q_starts) return RW_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f) || !(softmax_scale < 1e30f)) return RW_ERR_INVALID_ARG;
  if (Hq / pool.Hkv > 128) return RW_ERR_UNSUPPORTED;
  if (T == 0 || cache->B == 0 || max_q_len == 0) return RW_OK;
  if (!q || !out || !aligned16(q) || !aligned16(out) || !stride_ok(q_sl) || !stride_ok(q_sh) || !stride_ok(o_sl) ||
      !stride_ok(o_sh))
    return RW_ERR_INVALID_ARG;
  if (sums && (sums_sb < 0 || sums_sh < 0)) return RW_ERR_INVALID_ARG;
  const int longest = std::min(max_q_len, T);
  const long long rows = (long long)longest * (Hq / pool.Hkv);
  const chunk::Call c{q, out, lse, nullptr, T, Hq, longest, causal != 0, q_sl, q_sh, o_sl, o_sh,
                      softmax_scale * 1.4426950408889634f, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool few = rows::few_rows(rows) ||
                   rows::clusters_for(cache->D, (long long)cache->B * pool.Hkv, rows,
                                      (long long)cache->table_width * cache->page_size, sums != nullptr).cs != 0;
  return few ? rows::run_rows(cache, pool, c, rows, sums, sums_sb, sums_sh, workspace, workspace_bytes, st)
             : rows::run_tiles(cache, pool, c, sums, sums_sb, sums_sh, workspace, workspace_bytes, st);
}

extern "C" long long rw_paged_attn_workspace_bytes(int T, int Hq, int Hkv, int D, int B, int max_q_len,
                                                   long long cache_rows, int with_sums) {
  using namespace rw;
  if (T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || B < 1 || max_q_len < 1 || (D != 64 && D != 128) || cache_rows < 0)
    return 0;
  const long long rows = (long long)std::min(max_q_len, T) * (Hq / Hkv);
  if (rows::clusters_for(D, (long long)B * Hkv, rows, cache_rows, with_sums != 0).cs)
    return rows::block_sums_bytes((long long)B * Hkv, rows, cache_rows, with_sums != 0);
  if (rows::few_rows(rows))
    return rows::layout(D, rows::grid_size(D), rows::slice_of(B, Hkv, rows, cache_rows, with_sums != 0), Hkv, rows,
                        cache_rows, with_sums != 0).total;
  return chunk::workspace_bytes(D) + (with_sums ? 4LL * T * Hq : 0);
}
