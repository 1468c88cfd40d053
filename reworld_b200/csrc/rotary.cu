// Rotary positions of packed tokens [T, heads, D], and the write of new keys and
// values into a paged cache with the keys rotated on the way.
//
// A pair (a, b) of a head at position p becomes (a c - b s, a s + b c) with
// (c, s) = table[p][i]; the pairs of the first `rot` channels are (2i, 2i + 1)
// (interleaved) or (i, i + rot / 2) (halves), the channels behind them pass through.
// The table is fp32, made from fp64 angles (far positions lose nothing); products and
// sums are fp32, one rounding at the store.
//
// HBM-bound: q, k and v are read and written once, 16 bytes at a time.  A thread's
// work item is two 16-byte chunks of one head that hold 8 whole pairs (chunks i and
// i + rot / 16, or 2i and 2i + 1), so both layouts need the same 64 bytes of table,
// and 128 / (D / 16) heads are under way in a CTA at once; a thread keeps its place in
// the head, so the table is read once a token.
//
// 4 x 2640 tokens of 24 + 48 heads of 128: 65.9 us, 5.9 TB/s; 8 single tokens of 32 + 16 heads: 3.6 us.
#include <algorithm>

#include "paged.cuh"

namespace rw {
namespace rotary {

using paged::Num;
using paged::Pool;

constexpr int THREADS = 128;
constexpr int NB = 3;  // heads that a thread has under way at once

struct Side {
  const uint8_t* in;
  uint8_t* out;
  long long i_sl, i_sh, o_sl, o_sh;  // byte strides: token, head
};

struct Params {
  Side q, k, v;  // k, v: `out` strides unused (rows go to the pool)
  int Hq, T, D, rot, interleaved, max_pos;
  int run;  // consecutive tokens of a CTA
  const float4* table;  // [max_pos][rot / 2] (cos, sin) pairs, two to a float4; null: no rotation
  const int* positions;
  int with_pool;
  Pool pool;
  int* status;
};

template <bool HALF>
__device__ __forceinline__ void turn(uint32_t& x, uint32_t& y, float2 cs0, float2 cs1, bool inter) {
  // interleaved: x holds one pair, y another (cs0, cs1); halves: x holds the first members of two pairs, y the second
  const float2 a = Num<HALF>::wide(x), b = Num<HALF>::wide(y);
  if (inter) {
    x = Num<HALF>::pack(a.x * cs0.x - a.y * cs0.y, a.x * cs0.y + a.y * cs0.x);
    y = Num<HALF>::pack(b.x * cs1.x - b.y * cs1.y, b.x * cs1.y + b.y * cs1.x);
  } else {
    x = Num<HALF>::pack(a.x * cs0.x - b.x * cs0.y, a.y * cs1.x - b.y * cs1.y);
    y = Num<HALF>::pack(a.x * cs0.y + b.x * cs0.x, a.y * cs1.y + b.y * cs1.x);
  }
}

template <bool HALF>
__device__ __forceinline__ void turn_item(uint4& x, uint4& y, const float4 (&cs)[4], bool inter) {
  if (inter) {  // chunk x: pairs 0-3, chunk y: pairs 4-7
    turn<HALF>(x.x, x.y, make_float2(cs[0].x, cs[0].y), make_float2(cs[0].z, cs[0].w), true);
    turn<HALF>(x.z, x.w, make_float2(cs[1].x, cs[1].y), make_float2(cs[1].z, cs[1].w), true);
    turn<HALF>(y.x, y.y, make_float2(cs[2].x, cs[2].y), make_float2(cs[2].z, cs[2].w), true);
    turn<HALF>(y.z, y.w, make_float2(cs[3].x, cs[3].y), make_float2(cs[3].z, cs[3].w), true);
  } else {
    turn<HALF>(x.x, y.x, make_float2(cs[0].x, cs[0].y), make_float2(cs[0].z, cs[0].w), false);
    turn<HALF>(x.y, y.y, make_float2(cs[1].x, cs[1].y), make_float2(cs[1].z, cs[1].w), false);
    turn<HALF>(x.z, y.z, make_float2(cs[2].x, cs[2].y), make_float2(cs[2].z, cs[2].w), false);
    turn<HALF>(x.w, y.w, make_float2(cs[3].x, cs[3].y), make_float2(cs[3].z, cs[3].w), false);
  }
}

template <bool HALF>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const __grid_constant__ Params p) {
  griddep_launch_dependents();
  griddep_wait();
  if (p.with_pool && blockIdx.x == gridDim.x - 1) {
    // The last CTA has no token: it looks at every sequence's start and length, also of those that no token finds.
    for (int b = threadIdx.x; b < p.pool.B; b += THREADS) paged::load_seq(p.pool, b, p.T, p.status);
    return;
  }
  const int ipt = p.D / 16;              // items of a head
  const int item = threadIdx.x % ipt;
  const int h0 = threadIdx.x / ipt, hstep = THREADS / ipt;
  const int lane = threadIdx.x & 31;
  const bool inter = p.interleaved != 0;
  const bool rotates = p.table != nullptr && item < p.rot / 16;
  // byte offsets of the item's two chunks in the head
  int c0, c1;
  if (p.table != nullptr && !inter && rotates) {
    c0 = 16 * item;
    c1 = c0 + p.rot;                     // rot / 2 elements of 2 bytes
  } else {
    c0 = 32 * item;                      // behind `rot` too: items rot/16.. hold chunks rot/8..
    c1 = c0 + 16;
  }
  const int Hk = p.with_pool ? p.pool.Hkv : 0;
  const int vectors = p.Hq + 2 * Hk;     // heads of q, then of k, then of v
  const long long t_end = min((long long)p.T, (long long)(blockIdx.x + 1) * p.run);
  int b = -1;
  paged::Seq sq{0, 0, 0};
  for (int t = blockIdx.x * p.run; t < t_end; ++t) {
    int pos = p.positions ? __ldg(p.positions + t) : 0;
    const uint8_t* kd = nullptr;
    const uint8_t* vd = nullptr;
    if (p.with_pool) {
      if (b < 0 || t >= sq.s0 + sq.lq) {
        // sequences that end at or before t; the sequence of t follows them
        b = 0;
        for (int i = 1; i <= p.pool.B; i += 32) {
          const int e = i + lane <= p.pool.B ? __ldg(p.pool.q_starts + i + lane) : 0x7fffffff;
          b += __popc(__ballot_sync(0xffffffffu, e <= t));
        }
        if (b >= p.pool.B) break;        // tokens behind the last sequence stay as they were,
        sq = paged::load_seq(p.pool, b, p.T, nullptr);
      }
      if (t < sq.s0 || t >= sq.s0 + sq.lq) continue;   // and those before the first one or where starts fall
      const int row = sq.kv - sq.lq + (t - sq.s0);
      if (!p.positions) pos = row;
      if (row >= 0) {
        const int pg = __ldg(p.pool.table + b * p.pool.table_stride + (row >> p.pool.page_shift));
        const int slot = row & ((1 << p.pool.page_shift) - 1);
        if ((unsigned)pg < (unsigned)p.pool.num_pages) {
          kd = p.pool.k + pg * p.pool.k_sp + slot * p.pool.k_sl;
          vd = p.pool.v + pg * p.pool.v_sp + slot * p.pool.v_sl;
        } else {
          report_status(p.status, RW_STATUS_BAD_SLOT);
        }
      } else {
        report_status(p.status, RW_STATUS_BAD_SLOT);  // more new tokens than rows
      }
    }
    float4 cs[4];
    if (rotates) {
      const int at = paged::clampi(pos, 0, p.max_pos - 1);
      if (at != pos) report_status(p.status, RW_STATUS_BAD_SLOT);
      const float4* tp = p.table + ((long long)at * p.rot + 16 * item) / 4;  // rot floats a position, 16 an item
#pragma unroll
      for (int j = 0; j < 4; ++j) cs[j] = __ldg(tp + j);
    }
    for (int hb = h0; hb < vectors; hb += hstep * NB) {
      uint4 x[NB], y[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int h = hb + j * hstep;
        if (h >= vectors) continue;
        const Side& s = h < p.Hq ? p.q : (h < p.Hq + Hk ? p.k : p.v);
        const int hh = h < p.Hq ? h : (h < p.Hq + Hk ? h - p.Hq : h - p.Hq - Hk);
        const uint8_t* src = s.in + t * s.i_sl + hh * s.i_sh;
        // plain loads: the output may be the input (in-place rotation)
        x[j] = *reinterpret_cast<const uint4*>(src + c0);
        y[j] = *reinterpret_cast<const uint4*>(src + c1);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int h = hb + j * hstep;
        if (h >= vectors) continue;
        if (rotates && h < p.Hq + Hk) turn_item<HALF>(x[j], y[j], cs, inter);
        uint8_t* dst;
        if (h < p.Hq) dst = p.q.out + t * p.q.o_sl + h * p.q.o_sh;
        else if (h < p.Hq + Hk) dst = const_cast<uint8_t*>(kd ? kd + (h - p.Hq) * p.pool.k_sh : nullptr);
        else dst = const_cast<uint8_t*>(vd ? vd + (h - p.Hq - Hk) * p.pool.v_sh : nullptr);
        if (dst == nullptr) continue;
        *reinterpret_cast<uint4*>(dst + c0) = x[j];
        *reinterpret_cast<uint4*>(dst + c1) = y[j];
      }
    }
  }
}

inline int check_table(const float* table, int max_pos, int rot, int D) {
  if (!table) return RW_OK;
  if (!aligned16(table) || max_pos < 1 || rot < 16 || rot > D || rot % 16) return RW_ERR_INVALID_ARG;
  return RW_OK;
}

inline int launch(Params& p, int dtype, void* stream) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return RW_ERR_CUDA;
  // A token a CTA: the SMs' scheduler covers one token's chain of loads (sequence, page, table) with others.  Where
  // there are many tokens, three, so that they share the search for the sequence: 4 x 2640 tokens of 24 + 48 heads
  // 65.9 us with 1, 65.3 with 2, 65.6 with 3, 70.0 with 4 (72 with one wave of CTAs), of 24 + 8 heads 37.2, 34.6,
  // 32.9, 35.9; 4 x 700 tokens of 24 + 48 heads 20.5, 23.1, 21.6, 25.7.
  p.run = std::min(3, std::max(1, p.T / (sms * 16)));
  const int grid = (p.T + p.run - 1) / p.run + (p.with_pool ? 1 : 0);
  auto kernel = dtype == RW_DTYPE_FP16 ? rotary_kernel<true> : rotary_kernel<false>;
  return launch_dependent(kernel, dim3(grid), dim3(THREADS), 0, static_cast<cudaStream_t>(stream), p) == cudaSuccess
             ? RW_OK : RW_ERR_CUDA;
}

}  // namespace rotary
}  // namespace rw

extern "C" int rw_rotary(const void* x, void* out, int T, int H, int D, int dtype, long long x_sl, long long x_sh,
                         long long o_sl, long long o_sh, const float* table, int max_pos, int rot, int interleaved,
                         const int* positions, int* status, void* stream) {
  using namespace rw;
  if ((D != 64 && D != 128) || (dtype != RW_DTYPE_BF16 && dtype != RW_DTYPE_FP16)) return RW_ERR_UNSUPPORTED;
  if (T < 0 || H < 0 || !table || !positions) return RW_ERR_INVALID_ARG;
  if (int e = rotary::check_table(table, max_pos, rot, D)) return e;
  if (T == 0 || H == 0) return RW_OK;
  if (!x || !out || !aligned16(x) || !aligned16(out) || !stride_ok(x_sl) || !stride_ok(x_sh) || !stride_ok(o_sl) ||
      !stride_ok(o_sh))
    return RW_ERR_INVALID_ARG;
  rotary::Params p{};
  p.q = {static_cast<const uint8_t*>(x), static_cast<uint8_t*>(out), 2 * x_sl, 2 * x_sh, 2 * o_sl, 2 * o_sh};
  p.Hq = H; p.T = T; p.D = D; p.rot = rot; p.interleaved = interleaved; p.max_pos = max_pos;
  p.table = reinterpret_cast<const float4*>(table);
  p.positions = positions;
  p.status = status;
  return rotary::launch(p, dtype, stream);
}

extern "C" int rw_paged_rotary_store(const rw_paged_t* cache, const void* k, const void* v, const void* q, void* q_out,
                                     int T, int Hq, long long k_sl, long long k_sh, long long v_sl, long long v_sh,
                                     long long q_sl, long long q_sh, long long qo_sl, long long qo_sh,
                                     const float* table, int max_pos, int rot, int interleaved, const int* positions,
                                     int* status, void* stream) {
  using namespace rw;
  rotary::Params p{};
  if (int e = paged::make_pool(cache, &p.pool)) return e;
  if (T < 0 || Hq < 0 || !cache->q_starts) return RW_ERR_INVALID_ARG;
  if (int e = rotary::check_table(table, max_pos, rot, cache->D)) return e;
  if (T == 0 || cache->B == 0) return RW_OK;
  if (!k || !v || !aligned16(k) || !aligned16(v) || !stride_ok(k_sl) || !stride_ok(k_sh) || !stride_ok(v_sl) ||
      !stride_ok(v_sh))
    return RW_ERR_INVALID_ARG;
  if ((q == nullptr) != (q_out == nullptr)) return RW_ERR_INVALID_ARG;
  if (q && (Hq < 1 || !aligned16(q) || !aligned16(q_out) || !stride_ok(q_sl) || !stride_ok(q_sh) || !stride_ok(qo_sl) ||
            !stride_ok(qo_sh)))
    return RW_ERR_INVALID_ARG;
  p.q = {static_cast<const uint8_t*>(q), static_cast<uint8_t*>(q_out), 2 * q_sl, 2 * q_sh, 2 * qo_sl, 2 * qo_sh};
  p.k = {static_cast<const uint8_t*>(k), nullptr, 2 * k_sl, 2 * k_sh, 0, 0};
  p.v = {static_cast<const uint8_t*>(v), nullptr, 2 * v_sl, 2 * v_sh, 0, 0};
  p.Hq = q ? Hq : 0;
  p.T = T; p.D = cache->D; p.rot = rot; p.interleaved = interleaved; p.max_pos = max_pos;
  p.table = reinterpret_cast<const float4*>(table);
  p.positions = positions;
  p.with_pool = 1;
  p.status = status;
  return rotary::launch(p, cache->dtype, stream);
}
