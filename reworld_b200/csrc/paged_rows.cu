// Attention of few new tokens over a paged cache: o = softmax(q k^T * scale) v for the
// rows of a sequence that share a key head (tokens x heads of the group), 16 rows at a
// time, with the keys split over the whole device.
//
// Such a call is bound by memory: every cached row of k and v is read once for 4 * 16
// products an element at most.  What decides is that all SMs read all the time, however
// ragged the lengths are.  So the work is one sequence of key tiles (64 keys of one
// sequence and key head), in the order (sequence, row tile, head, tile), and CTA c of C
// takes the share [c N / C, (c + 1) N / C) of its N tiles; lengths are read on the
// device, nothing is planned on the host.  A share covers the end of one unit (the
// tiles of one sequence, row tile and head), whole units, and the beginning of another.
// Units that lie in one share are written out directly; the others leave their
// unnormalised O, m and l in scratch, and the CTA that comes last to a unit (a counter)
// joins its parts, always in the same order, so results do not depend on who is last.
//
// In a CTA each of the 4 warps takes 16 keys of a 64-key tile with a running maximum and
// sum of its own (mma.sync m16n8k16 feeds far more than memory delivers here: a tile of
// 32 KB costs a warp 32 MMAs), so the warps only meet for the loads; the 4 states are
// joined when the unit's tiles are done.  Keys and values come through a ring of 3 stages
// of 16-byte cp.async; rows behind the last visible one are filled with zeros, never
// read, so what a page holds there (NaN included) does not matter.
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
constexpr int RT = 16;          // rows of a row tile
constexpr int STAGES = 3;

struct Params {
  Pool pool;
  const uint8_t* q;
  uint8_t* out;
  float* lse;                   // [T, Hq] natural logarithm, or null
  long long q_sl, q_sh, o_sl, o_sh;  // byte strides
  int T, Hq, G, nrt, causal;    // nrt: row tiles of a sequence (by max_q_len)
  int min_tiles;                // tiles that a share has at least, where there are few
  float scale_log2;
  float* part;                  // [2 C][16 * D + 32]: O, then m, then l
  int* counters;                // [B * nrt * Hkv], zero before and after
  int2* header;                 // [B * nrt * Hkv]: first slot and parts of every unit (join_kernel joins); null: the last CTA joins
  // raw scores (log2 units) and (m, 1 / l) of every row, for the weight sums; null otherwise
  float* scores;                // [B * Hkv * nrt * 16][cap]
  float2* row_ml;               // [B * Hkv * nrt * 16]
  long long cap;
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

// Entry e = (sequence, row tile) and the rows that its last row sees.
struct Entry {
  Seq s;
  int rows;   // valid rows, 0..16
  int row0;   // first row of the tile within the sequence's lq * G
  int keys;   // keys that any of the rows sees
};

__device__ __forceinline__ Entry load_entry(const Params& p, int e, int* status) {
  Entry n;
  const int b = e / p.nrt, rt = e - b * p.nrt;
  n.s = paged::load_seq(p.pool, b, p.T, status);
  const long long all = (long long)n.s.lq * p.G;
  n.row0 = rt * RT;
  n.rows = (int)min((long long)RT, max(0ll, all - n.row0));
  n.keys = 0;
  if (n.rows > 0) {
    const int last = (n.row0 + n.rows - 1) / p.G;   // last token of the tile
    n.keys = p.causal ? max(0, n.s.kv - n.s.lq + last + 1) : n.s.kv;
  }
  return n;
}

// Tiles of an entry: at least one while it has rows, so that rows that see nothing are written too.
__device__ __forceinline__ int tiles_of(const Entry& n) {
  return n.rows > 0 ? max(1, (n.keys + TILE - 1) / TILE) : 0;
}

// Channels c, c + 1 of row r of a unit: O / l, and with channel 0 the row's lse and (m, 1 / l).
template <bool HALF>
__device__ __forceinline__ void put_row(const Params& p, const Entry& en, int b, int hk, int r, int c, float2 v,
                                        float mm, float ll) {
  const int rr = en.row0 + r, tok = rr / p.G, g = rr - tok * p.G;
  const float inv = ll != 0.f ? 1.f / ll : 0.f;
  uint8_t* dst = p.out + (long long)(en.s.s0 + tok) * p.o_sl + (long long)(hk * p.G + g) * p.o_sh;
  *reinterpret_cast<uint32_t*>(dst + 2 * c) = Num<HALF>::pack(v.x * inv, v.y * inv);
  if (c == 0) {
    if (p.lse)
      p.lse[(long long)(en.s.s0 + tok) * p.Hq + hk * p.G + g] =
          ll != 0.f ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
    if (p.row_ml) {
      const long long line = (((long long)b * p.pool.Hkv + hk) * p.nrt + en.row0 / RT) * RT + r;
      p.row_ml[line] = make_float2(mm == -INFINITY ? 0.f : mm, inv);
    }
  }
}

template <bool HALF, int D>
__global__ void __launch_bounds__(THREADS, 2) rows_kernel(const __grid_constant__ Params p) {
  constexpr int PITCH = 2 * D;               // bytes of a row in shared memory
  constexpr int CH = D / 8;                  // 16-byte chunks of a row
  constexpr int STAGE = 2 * TILE * PITCH;    // k, then v
  constexpr int SLOT = RT * D + 2 * RT;      // floats of a part
  constexpr int LOADS = TILE * CH / THREADS; // cp.async of k (and of v) a thread
  constexpr int RSTEP = THREADS / CH;        // rows between two of them
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ long long base[THREADS + 1];
  __shared__ int come;
  __shared__ float sm_m[WARPS][RT], sm_l[WARPS][RT];
  __shared__ int dirty;         // 1: the segment has values that are not finite (paged.cuh)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int grp = lane >> 2, quad = lane & 3;
  griddep_launch_dependents();
  griddep_wait();

  // ---- tiles before every thread's run of entries, and of all
  const int NE = p.pool.B * p.nrt;
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
  const int C = (int)max(1ll, min((long long)gridDim.x, N / p.min_tiles)), cta = blockIdx.x;
  if (cta >= C) return;
  const long long t0 = N * cta / C, t1 = N * (cta + 1) / C;
  if (t0 >= t1) return;

  // ---- the entry that holds tile t0
  int e;
  long long ebase;      // tiles before entry e
  {
    int lo = 0, hi = THREADS - 1;
    while (lo < hi) {   // last thread whose run begins at or before t0
      const int mid = (lo + hi + 1) >> 1;
      if (base[mid] <= t0) lo = mid; else hi = mid - 1;
    }
    e = lo * run;
    ebase = base[lo];
  }
  Entry en = load_entry(p, e, p.status);
  for (;;) {
    const long long n = (long long)tiles_of(en) * p.pool.Hkv;
    if (t0 < ebase + n) break;
    ebase += n;
    en = load_entry(p, ++e, p.status);
  }

  const uint32_t sbase = smem_u32(smem);
  long long t = t0;
  while (t < t1) {
    while (t >= ebase + (long long)tiles_of(en) * p.pool.Hkv) {
      ebase += (long long)tiles_of(en) * p.pool.Hkv;
      en = load_entry(p, ++e, p.status);
    }
    const int n_tiles = tiles_of(en);
    const int hk = (int)((t - ebase) / n_tiles);
    const long long u0 = ebase + (long long)hk * n_tiles, u1 = u0 + n_tiles;  // the unit's tiles
    const int k0 = (int)(t - u0), k1 = (int)(min(t1, u1) - u0);               // this segment's
    const int b = e / p.nrt;
    const Seq s = en.s;

    // ---- q fragments: rows grp and grp + 8, channels 16 kk + 2 quad (+ 8)
    uint32_t qf[D / 16][4];
    int lim[2];          // keys that the thread's two rows see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = en.row0 + grp + 8 * i;
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

    // ---- loads of key tile j: page indices one tile ahead (lane i < 8 holds rows 8i.. of a tile)
    const uint8_t* kb = p.pool.k + (long long)hk * p.pool.k_sh;
    const uint8_t* vb = p.pool.v + (long long)hk * p.pool.v_sh;
    const int slot_mask = (1 << p.pool.page_shift) - 1;
    auto pages = [&](int j) {
      const int row = j * TILE + 8 * (lane & 7);
      return (j < k1 && row < en.keys) ? paged::raw_page_of(p.pool, b, row) : 0;
    };
    auto load = [&](int j, int pg) {
      const uint32_t st = sbase + (uint32_t)((j - k0) % STAGES) * STAGE;
      const int c = tid % CH, r0 = tid / CH;
      pg = paged::checked_page(p.pool, pg, p.status);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int r = r0 + i * RSTEP;
        const int row = j * TILE + r;
        const long long pi = __shfl_sync(0xffffffffu, pg, r >> 3);
        const bool there = row < en.keys;
        const int sl = there ? (row & slot_mask) : 0;
        const uint32_t d = st + r * PITCH + ((c ^ (r & 7)) << 4);
        cp16(d, kb + pi * p.pool.k_sp + sl * p.pool.k_sl + 16 * c, there);
        cp16(d + TILE * PITCH, vb + pi * p.pool.v_sp + sl * p.pool.v_sl + 16 * c, there);
      }
    };
    int pg = pages(k0);
    for (int i = 0; i < STAGES - 1; ++i) {
      const int nx = pages(k0 + i + 1);
      if (k0 + i < k1) load(k0 + i, pg);
      cp_commit();
      pg = nx;
    }

    // keys that every row sees: tiles behind them are looked through for values that are not finite
    const int all = p.causal ? min(en.keys, max(0, s.kv - s.lq + en.row0 / p.G + 1)) : en.keys;
    if (tid == 0) dirty = 0;                 // (read after the barriers below)
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int j = k0; j < k1; ++j) {
      cp_wait<STAGES - 2>();
      __syncthreads();                       // tile j is there, tile j - 1 is done with
      {
        const int nx = pages(j + STAGES);
        if (j + STAGES - 1 < k1) load(j + STAGES - 1, pg);
        cp_commit();
        pg = nx;
      }
      const uint32_t ks = sbase + (uint32_t)((j - k0) % STAGES) * STAGE;
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
      if (p.scores) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = grp + 8 * x;
            const long long line = (((long long)b * p.pool.Hkv + hk) * p.nrt + en.row0 / RT) * RT + r;
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
      // weights in fp32 for the sum, rounded to the values' type for the product (its operands' type)
      uint32_t pf[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a0 = fast_exp2(sc[i][0] - base_[0]), a1 = fast_exp2(sc[i][1] - base_[0]);
        const float b0 = fast_exp2(sc[i][2] - base_[1]), b1 = fast_exp2(sc[i][3] - base_[1]);
        l[0] += a0 + a1;
        l[1] += b0 + b1;
        pf[2 * i] = Num<HALF>::pack(a0, a1);
        pf[2 * i + 1] = Num<HALF>::pack(b0, b1);
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
    cp_wait<0>();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    __syncthreads();                         // the stages are free: they take the warps' states

    // ---- join the warps: fo[warp][16][D + 4]
    constexpr int FP = D + 4;
    float* fo = reinterpret_cast<float*>(smem);
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
        *reinterpret_cast<float2*>(fo + ((warp * RT + grp + 8 * x) * FP + 8 * i + 2 * quad)) =
            make_float2(o[i][2 * x], o[i][2 * x + 1]);
    __syncthreads();

    const bool whole = k0 == 0 && k1 == n_tiles;
    // largest c with N c / C <= x: the CTA that has tile x
    auto owner = [&](long long x) {
      long long c = (x * C) / N;
      while (c + 1 < C && N * (c + 1) / C <= x) ++c;
      while (c > 0 && N * c / C > x) --c;
      return (int)c;
    };
    if (p.header && k0 == 0 && tid == 0)
      p.header[(long long)e * p.pool.Hkv + hk] =
          make_int2(2 * cta + (t == t0 ? 0 : 1), whole ? 0 : owner(u1 - 1) - cta + 1);
    float* slot = p.part + (long long)(2 * cta + (t == t0 ? 0 : 1)) * SLOT;
    auto put = [&](int r, int c, float2 v, float mm, float ll) { put_row<HALF>(p, en, b, hk, r, c, v, mm, ll); };
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
        const float2 x = *reinterpret_cast<const float2*>(fo + (w * RT + r) * FP + c);
        v.x += f * x.x;
        v.y += f * x.y;
        ll += f * sm_l[w][r];
      }
      if (dirty) {
        // taken-out values go to the rows that see them
        const int lim = p.causal ? max(0, s.kv - s.lq + (en.row0 + r) / p.G + 1) : s.kv;
        paged::for_nonfinite<HALF>(p.pool, b, hk, max(all / TILE, k0) * TILE, min(lim, k1 * TILE), c, 2,
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
    if (!whole && !p.header) {
      // the CTAs whose shares meet the unit: the one that holds tile u0 to the one that holds u1 - 1
      const int ca = owner(u0), cb = owner(u1 - 1);
      int* counter = p.counters + (long long)e * p.pool.Hkv + hk;
      __threadfence();
      __syncthreads();
      if (tid == 0) come = atomicAdd(counter, 1);
      __syncthreads();
      const int parts = cb - ca + 1;         // (C <= N: every share has a tile)
      if (come == parts - 1) {
        __threadfence();
        if (tid == 0) *counter = 0;          // ready for the next call
        // part i of the unit, from CTA ca + i: in that CTA's first slot unless its share began before the unit
        auto slot_of = [&](int i) {
          return p.part + (2LL * (ca + i) + (i == 0 && N * ca / C < u0 ? 1 : 0)) * SLOT;
        };
        // factor of every part and row, [parts][16], and the rows' m and l; a warp has 4 rows
        float* fac = reinterpret_cast<float*>(smem);
        for (int i = tid; i < parts * RT; i += THREADS) fac[i] = __ldcg(slot_of(i / RT) + RT * D + i % RT);
        __syncthreads();
        for (int r = warp * 4; r < warp * 4 + 4; ++r) {
          float mm = -INFINITY;
          for (int i = lane; i < parts; i += 32) mm = fmaxf(mm, fac[i * RT + r]);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
          const float bs = mm == -INFINITY ? 0.f : mm;
          float ll = 0.f;
          for (int i = lane; i < parts; i += 32) {
            const float f = fast_exp2(fac[i * RT + r] - bs);
            fac[i * RT + r] = f;
            ll += f * __ldcg(slot_of(i) + RT * D + RT + r);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
          if (lane == 0) {
            sm_m[0][r] = mm;
            sm_l[0][r] = ll;
          }
        }
        __syncthreads();
        // 4 channels of a row a thread and step; 16 parts' loads under way at once
        for (int i = tid; i < en.rows * (D / 4); i += THREADS) {
          const int r = i / (D / 4), c = 4 * (i % (D / 4));
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          auto add = [&](const float4& x, float f) {
            v.x += f * x.x;
            v.y += f * x.y;
            v.z += f * x.z;
            v.w += f * x.w;
          };
          // the first part may be in its CTA's second slot; the others lie 2 SLOT apart
          add(__ldcg(reinterpret_cast<const float4*>(slot_of(0) + r * D + c)), fac[r]);
          const float* at = p.part + 2LL * ca * SLOT + r * D + c;
#pragma unroll 16
          for (int k = 1; k < parts; ++k)
            add(__ldcg(reinterpret_cast<const float4*>(at + 2LL * k * SLOT)), fac[k * RT + r]);
          put(r, c, make_float2(v.x, v.y), sm_m[0][r], sm_l[0][r]);
          put(r, c + 2, make_float2(v.z, v.w), sm_m[0][r], sm_l[0][r]);
        }
      }
    }
    __syncthreads();                         // shared memory is free for the next segment
    t = u0 + k1;
  }
}

// Joins the parts of the units that more than one CTA worked on, where units are few and
// have many parts: a block takes one row of one unit, its 8 groups of D / 4 threads every
// eighth part each.  (One CTA joining 148 parts of 8 rows, 600 KB, took 35 us.)
constexpr int JOIN_GROUPS = 8;
// Parts a unit, above which this kernel joins: 2 units of 8 parts 18.4 us without and 20.5 with it, 24 units of 12
// parts 38.9 and 34.8 (4000 rows), 4 units of 74 parts 86 and 74, 1 unit of 296 parts 86 and 51.
constexpr int WIDE_JOIN = 10;
constexpr int MAX_PARTS = 1024;  // CTAs of a launch: checked by the host

template <bool HALF, int D>
__global__ void __launch_bounds__(JOIN_GROUPS * D / 4) join_kernel(const __grid_constant__ Params p) {
  constexpr int SLOT = RT * D + 2 * RT;
  constexpr int NT = JOIN_GROUPS * D / 4;
  __shared__ float fac[MAX_PARTS];
  __shared__ float red[2][NT / 32];
  __shared__ float4 acc[JOIN_GROUPS][D / 4];
  griddep_launch_dependents();
  griddep_wait();
  const int u = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int e = u / p.pool.Hkv, hk = u - e * p.pool.Hkv;
  const int2 h = __ldcg(p.header + u);         // (not written, and not used, where the unit has no rows)
  const Entry en = load_entry(p, e, nullptr);
  if (r >= en.rows) return;
  const int n = min(h.y, MAX_PARTS);
  if (n == 0) return;                          // one CTA did it all, and wrote it
  // part 0 may be in its CTA's second slot, the others are in the first slots of the CTAs that follow
  auto slot = [&](int i) { return p.part + (i == 0 ? (long long)h.x : 2LL * (h.x / 2 + i)) * SLOT; };
  float mm = -INFINITY;
  for (int i = tid; i < n; i += NT) {
    fac[i] = __ldcg(slot(i) + RT * D + r);
    mm = fmaxf(mm, fac[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (lane == 0) red[0][warp] = mm;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) mm = fmaxf(mm, red[0][i]);
  const float bs = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  for (int i = tid; i < n; i += NT) {
    fac[i] = fast_exp2(fac[i] - bs);
    ll += fac[i] * __ldcg(slot(i) + RT * D + RT + r);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
  if (lane == 0) red[1][warp] = ll;
  __syncthreads();
  ll = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) ll += red[1][i];
  const int g = tid / (D / 4), c = 4 * (tid % (D / 4));
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 10
  for (int i = g; i < n; i += JOIN_GROUPS) {
    const float4 x = __ldcg(reinterpret_cast<const float4*>(slot(i) + r * D + c));
    const float f = fac[i];
    v.x += f * x.x;
    v.y += f * x.y;
    v.z += f * x.z;
    v.w += f * x.w;
  }
  acc[g][c / 4] = v;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int i = 1; i < JOIN_GROUPS; ++i) {
    const float4 x = acc[i][c / 4];
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
  }
  const int b = e / p.nrt;
  put_row<HALF>(p, en, b, hk, r, c, make_float2(v.x, v.y), mm, ll);
  put_row<HALF>(p, en, b, hk, r, c + 2, make_float2(v.z, v.w), mm, ll);
}

// sums[b, hk, j] += sum over the rows of exp2(score - m) / l, rows in their order.
struct SumParams {
  Pool pool;
  const float* scores;
  const float2* row_ml;
  float* sums;
  long long sums_sb, sums_sh, cap;
  int T, G, nrt, causal;
};

__global__ void __launch_bounds__(256) row_sums_kernel(const __grid_constant__ SumParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int b = blockIdx.z, hk = blockIdx.y;
  const Seq s = paged::load_seq(p.pool, b, p.T, nullptr);
  const long long all = (long long)s.lq * p.G;
  const long long line0 = ((long long)b * p.pool.Hkv + hk) * p.nrt * RT;
  for (int j = blockIdx.x * 256 + threadIdx.x; j < s.kv; j += gridDim.x * 256) {
    float add = 0.f;
    for (int rt = 0; rt < p.nrt && (long long)rt * RT < all; ++rt) {
      const int rows = (int)min((long long)RT, all - (long long)rt * RT);
      const int last = (rt * RT + rows - 1) / p.G;
      if (p.causal && j >= s.kv - s.lq + last + 1) continue;   // behind the tile's last key: no score was written
      for (int r = 0; r < rows; ++r) {
        const long long line = line0 + (long long)rt * RT + r;
        const float2 ml = __ldg(p.row_ml + line);
        add += fast_exp2(__ldcs(p.scores + line * p.cap + j) - ml.x) * ml.y;
      }
    }
    p.sums[b * p.sums_sb + hk * p.sums_sh + j] += add;
  }
}

long long counters_needed(int B, int Hkv, int nrt) { return (long long)B * Hkv * nrt; }

// CTAs of a launch: as many as stay resident (2 an SM with a head of 128, 4 with 64).
inline int grid_size(int D) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms * (D == 128 ? 2 : 4);
}

// Which kernel: 16 rows of a sequence and key head are all that rows_kernel can use of a
// key tile it has read; with more, the tiles of chunk_kernel.
inline bool on_tensor_tiles(int B, long long nrt) { return nrt > 1 && B <= chunk::MAX_BATCH; }

struct Layout {
  long long part, header, ml, scores, total;  // byte offsets
};

inline Layout layout(int D, int C, int B, int Hkv, int nrt, long long cap, bool sums) {
  Layout l;
  l.part = 0;
  l.header = (2LL * C * (RT * D + 2 * RT) * 4 + 255) & ~255LL;
  l.ml = (l.header + 8LL * B * Hkv * nrt + 255) & ~255LL;
  const long long lines = (long long)B * Hkv * nrt * RT;
  l.scores = l.ml + (sums ? (lines * 8 + 255) & ~255LL : 0);
  l.total = l.scores + (sums ? lines * cap * 4 : 0);
  return l;
}

template <bool HALF, int D>
int launch_rows(const Params& p, int C, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const int bytes = STAGES * 2 * TILE * 2 * D;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(rows_kernel<HALF, D>), bytes, &done)) return RW_ERR_CUDA;
  if (launch_dependent(rows_kernel<HALF, D>, dim3(C), dim3(THREADS), bytes, stream, p) != cudaSuccess)
    return RW_ERR_CUDA;
  if (!p.header) return RW_OK;
  const dim3 grid(p.pool.B * p.nrt * p.pool.Hkv, std::min(RT, p.T * p.G));
  return launch_dependent(join_kernel<HALF, D>, grid, dim3(JOIN_GROUPS * D / 4), 0, stream, p) == cudaSuccess
             ? RW_OK : RW_ERR_CUDA;
}

}  // namespace rows
}  // namespace rw

extern "C" int rw_paged_attn(const rw_paged_t* cache, const void* q, void* out, float* lse, int T, int Hq,
                             int max_q_len, long long q_sl, long long q_sh, long long o_sl, long long o_sh, int causal,
                             float softmax_scale, float* sums, long long sums_sb, long long sums_sh, int* counters,
                             long long n_counters, void* workspace, long long workspace_bytes, int* status,
                             void* stream) {
  using namespace rw;
  rows::Params p{};
  if (int e = paged::make_pool(cache, &p.pool)) return e;
  if (T < 0 || Hq < 1 || Hq % p.pool.Hkv || max_q_len < 0 || !cache->q_starts) return RW_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f) || !(softmax_scale < 1e30f)) return RW_ERR_INVALID_ARG;
  if (Hq / p.pool.Hkv > 128) return RW_ERR_UNSUPPORTED;
  if (T == 0 || cache->B == 0 || max_q_len == 0) return RW_OK;
  if (!q || !out || !aligned16(q) || !aligned16(out) || !stride_ok(q_sl) || !stride_ok(q_sh) || !stride_ok(o_sl) ||
      !stride_ok(o_sh))
    return RW_ERR_INVALID_ARG;
  if (sums && (sums_sb < 0 || sums_sh < 0)) return RW_ERR_INVALID_ARG;
  const int G = Hq / p.pool.Hkv;
  const long long nrt = ((long long)(max_q_len < T ? max_q_len : T) * G + rows::RT - 1) / rows::RT;
  if (nrt * cache->B * p.pool.Hkv > (1ll << 30)) return RW_ERR_CAPACITY;
  const long long cap = (long long)cache->table_width * cache->page_size;
  const float scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows::on_tensor_tiles(cache->B, nrt) && chunk::supported(cache)) {
    const long long parts = chunk::workspace_bytes(cache->D);
    if (!workspace || !aligned16(workspace) || workspace_bytes < parts + (sums ? 4LL * T * Hq : 0))
      return RW_ERR_INVALID_ARG;
    float* rb = sums ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + parts) : nullptr;
    const chunk::Call c{q, out, lse, rb, T, Hq, max_q_len < T ? max_q_len : T, causal != 0, q_sl, q_sh, o_sl, o_sh, scale_log2, status};
    const int rc = chunk::launch(cache, p.pool, c, workspace, st);
    return rc != RW_OK || !sums ? rc : weigh::launch(cache, p.pool, c, sums, sums_sb, sums_sh, st);
  }
  // (a pool of over 2^31 lines of its strides' common divisor takes no tensor map; the rows kernel reads it, but
  // would need a workspace for a chunk's scores)
  if (rows::on_tensor_tiles(cache->B, nrt) && sums) return RW_ERR_UNSUPPORTED;
  const int C = rows::grid_size(cache->D);
  if (C == 0 || C > rows::MAX_PARTS) return RW_ERR_CUDA;
  const rows::Layout lay = rows::layout(cache->D, C, cache->B, p.pool.Hkv, (int)nrt, cap, sums != nullptr);
  if (!workspace || !aligned16(workspace) || workspace_bytes < lay.total || !counters ||
      n_counters < rows::counters_needed(cache->B, p.pool.Hkv, (int)nrt))
    return RW_ERR_INVALID_ARG;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.q = static_cast<const uint8_t*>(q);
  p.out = static_cast<uint8_t*>(out);
  p.lse = lse;
  p.q_sl = 2 * q_sl; p.q_sh = 2 * q_sh; p.o_sl = 2 * o_sl; p.o_sh = 2 * o_sh;
  p.T = T; p.Hq = Hq; p.G = G; p.nrt = (int)nrt; p.causal = causal != 0;
  p.min_tiles = 1;
  // no more CTAs than there can be tiles: the others would only cost their launch
  const long long most = nrt * cache->B * p.pool.Hkv * std::max(1ll, (cap + rows::TILE - 1) / rows::TILE);
  const int ctas = (int)std::min((long long)C, most);
  p.scale_log2 = scale_log2;
  p.part = reinterpret_cast<float*>(ws + lay.part);
  p.counters = counters;
  // Where a unit can have many parts (CTAs a unit, tiles of a unit), they are joined by a kernel of their own; where
  // it has few, by the last CTA that comes to it, without another launch.
  if (std::min((long long)C / (cache->B * p.pool.Hkv * nrt), cap / rows::TILE) > rows::WIDE_JOIN)
    p.header = reinterpret_cast<int2*>(ws + lay.header);
  p.scores = sums ? reinterpret_cast<float*>(ws + lay.scores) : nullptr;
  p.row_ml = sums ? reinterpret_cast<float2*>(ws + lay.ml) : nullptr;
  p.cap = cap;
  p.status = status;
  int rc;
  if (cache->dtype == RW_DTYPE_FP16)
    rc = cache->D == 128 ? rows::launch_rows<true, 128>(p, ctas, st) : rows::launch_rows<true, 64>(p, ctas, st);
  else
    rc = cache->D == 128 ? rows::launch_rows<false, 128>(p, ctas, st) : rows::launch_rows<false, 64>(p, ctas, st);
  if (rc != RW_OK || !sums || cap == 0) return rc;
  rows::SumParams sp{};
  sp.pool = p.pool;
  sp.scores = p.scores;
  sp.row_ml = p.row_ml;
  sp.sums = sums;
  sp.sums_sb = sums_sb; sp.sums_sh = sums_sh; sp.cap = cap;
  sp.T = T; sp.G = G; sp.nrt = (int)nrt; sp.causal = causal != 0;
  const long long bx = (cap + 255) / 256;
  const dim3 grid((unsigned)(bx < 1024 ? bx : 1024), p.pool.Hkv, cache->B);
  return launch_dependent(rows::row_sums_kernel, grid, dim3(256), 0, st, sp) == cudaSuccess ? RW_OK : RW_ERR_CUDA;
}

extern "C" long long rw_paged_attn_workspace_bytes(int T, int Hq, int Hkv, int D, int B, int max_q_len,
                                                   long long cache_rows, int with_sums, long long* n_counters) {
  using namespace rw;
  if (n_counters) *n_counters = 0;
  if (T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || B < 1 || max_q_len < 1 || (D != 64 && D != 128) || cache_rows < 0)
    return 0;
  const long long nrt = ((long long)(max_q_len < T ? max_q_len : T) * (Hq / Hkv) + rows::RT - 1) / rows::RT;
  if (nrt * B * Hkv > (1ll << 30)) return 0;
  if (n_counters) *n_counters = rows::counters_needed(B, Hkv, (int)nrt);
  if (rows::on_tensor_tiles(B, nrt)) {
    const long long tiles = chunk::workspace_bytes(D) + (with_sums ? 4LL * T * Hq : 0);
    // (a pool whose strides no tensor map takes falls back to the rows kernel, which needs no more without sums)
    return with_sums ? tiles : std::max(tiles, rows::layout(D, rows::grid_size(D), B, Hkv, (int)nrt, 0, false).total);
  }
  return rows::layout(D, rows::grid_size(D), B, Hkv, (int)nrt, cache_rows, with_sums != 0).total;
}
