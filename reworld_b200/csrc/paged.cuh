// What the kernels over a paged KV cache share: the pools and the batch as they
// travel to a kernel, the bounds that every kernel puts on what it reads from
// device memory (page indices, lengths, starts), and the 16-bit types.
//
// The pools are [num_pages, page_size, Hkv, D] with free strides of page, row and
// head.  Row r of sequence b lies in page block_table[b][r / page_size] at row
// r % page_size.  Lengths and starts are device data, so a call needs no
// synchronisation and can be captured and replayed with new values; a value out of
// range is brought into range, and RW_STATUS_BAD_SLOT is reported.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "host_util.h"

namespace rw {
namespace paged {

struct Pool {
  const uint8_t* k;
  const uint8_t* v;
  long long k_sp, k_sl, k_sh, v_sp, v_sl, v_sh;  // byte strides: page, row, head
  int num_pages, page_shift, Hkv, B, width;
  const int* table;
  long long table_stride;
  const int* q_starts;
  const int* kv_lens;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// a / b of counts: in 32 bits where they fit (a 64-bit division is a subroutine of some 100 dependent
// instructions, which a plan made by one warp shows).
__device__ __forceinline__ long long div_count(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// Tokens [s0, s0 + lq) and cached rows of a sequence, within the call's T tokens and
// the table's width.
struct Seq {
  int s0, lq, kv;
};

__device__ __forceinline__ Seq load_seq(const Pool& p, int b, int T, int* status) {
  const int a = __ldg(p.q_starts + b), e = __ldg(p.q_starts + b + 1), n = __ldg(p.kv_lens + b);
  Seq s;
  s.s0 = clampi(a, 0, T);
  s.lq = clampi(e, s.s0, T) - s.s0;
  s.kv = (int)min((long long)max(n, 0), (long long)p.width << p.page_shift);
  if (s.s0 != a || s.s0 + s.lq != e || s.kv != n) report_status(status, RW_STATUS_BAD_SLOT);
  return s;
}

// Page of a sequence's row; a page outside the pool becomes page 0 (its rows are
// then wrong, and said to be) so that no address leaves the pool.
__device__ __forceinline__ int raw_page_of(const Pool& p, int b, int row) {
  return __ldg(p.table + b * p.table_stride + (row >> p.page_shift));
}
// (apart from the load, so that a page index fetched ahead is waited for only where it is used)
__device__ __forceinline__ int checked_page(const Pool& p, int pg, int* status) {
  if ((unsigned)pg >= (unsigned)p.num_pages) {
    report_status(status, RW_STATUS_BAD_SLOT);
    return 0;
  }
  return pg;
}
__device__ __forceinline__ int page_of(const Pool& p, int b, int row, int* status) {
  return checked_page(p, raw_page_of(p, b, row), status);
}

// The two 16-bit types.  Values are widened to fp32 exactly and rounded once, to
// nearest, when they are stored.
template <bool HALF>
struct Num;

template <>
struct Num<false> {
  static constexpr uint32_t EXP = 0x7F807F80u;  // exponent bits: all set in an infinity or NaN
  static constexpr uint32_t ULP = 0x00800080u;  // their lowest ones
  static __device__ __forceinline__ float2 wide(uint32_t v) { return make_float2(bf16_lo(v), bf16_hi(v)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};

template <>
struct Num<true> {
  static constexpr uint32_t EXP = 0x7C007C00u;
  static constexpr uint32_t ULP = 0x04000400u;
  static __device__ __forceinline__ float2 wide(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

// Values of keys that only some rows of a tile see.  The weight of a key that a row does
// not see is 0, but 0 times an infinity or NaN is NaN, and a token's value must not reach
// the tokens before it.  So tiles with such keys are looked through before the second
// product: values that are not finite are taken out (0), and, if there were any, added to
// the rows that do see them afterwards (an infinity or NaN whatever its weight).
//
// has_nonfinite: sign bits of a word are set where its values are not finite (the magnitude
// and one step of the exponent carry into the sign's place); other bits mean nothing.
template <bool HALF>
__device__ __forceinline__ uint32_t has_nonfinite(const uint4& v) {
  const uint32_t u = Num<HALF>::ULP, m = 0x7FFF7FFFu;
  return ((v.x & m) + u) | ((v.y & m) + u) | ((v.z & m) + u) | ((v.w & m) + u);
}
constexpr uint32_t SIGNS = 0x80008000u;

template <bool HALF>
__device__ __forceinline__ bool take_nonfinite(uint4& v) {
  const uint32_t e = Num<HALF>::EXP;
  const uint32_t a = __vcmpeq2(v.x & e, e), b = __vcmpeq2(v.y & e, e), c = __vcmpeq2(v.z & e, e),
                 d = __vcmpeq2(v.w & e, e);
  v.x &= ~a;
  v.y &= ~b;
  v.z &= ~c;
  v.w &= ~d;
  return (a | b | c | d) != 0u;
}

// add(c, x) for every value x that is not finite in channels [c0, c0 + n) of rows [from, to); n a multiple of 2.
template <bool HALF, typename F>
__device__ __forceinline__ void for_nonfinite(const Pool& p, int b, int hk, int from, int to, int c0, int n, F add) {
#pragma unroll 1
  for (int row = from; row < to; ++row) {
    const long long pg = page_of(p, b, row, nullptr);
    const uint8_t* src = p.v + pg * p.v_sp + (row & ((1 << p.page_shift) - 1)) * p.v_sl + hk * p.v_sh;
#pragma unroll 1
    for (int c = c0; c < c0 + n; c += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(src + 2 * c), e = Num<HALF>::EXP;
      const uint32_t m = __vcmpeq2(w & e, e);
      const float2 x = Num<HALF>::wide(w);
      if (m & 0xffffu) add(c, x.x);
      if (m & 0xffff0000u) add(c + 1, x.y);
    }
  }
}

// Host: checks a rw_paged_t and makes the kernels' form of it.  RW_OK, or what is wrong.
inline int make_pool(const rw_paged_t* a, Pool* p) {
  if (!a) return RW_ERR_INVALID_ARG;
  if ((a->D != 64 && a->D != 128) || (a->dtype != RW_DTYPE_BF16 && a->dtype != RW_DTYPE_FP16))
    return RW_ERR_UNSUPPORTED;
  if (!a->k || !a->v || !a->block_table || !a->kv_lens || !aligned16(a->k) || !aligned16(a->v))
    return RW_ERR_INVALID_ARG;
  if (a->num_pages < 1 || a->Hkv < 1 || a->Hkv > 65535 || a->B < 0 || a->B > 65535 || a->table_width < 0 ||
      a->table_stride < a->table_width)
    return RW_ERR_INVALID_ARG;
  if (a->page_size < 8 || a->page_size > (1 << 20) || (a->page_size & (a->page_size - 1))) return RW_ERR_UNSUPPORTED;
  // rows are counted in 32 bits, with room for a tile behind the last one
  if ((long long)a->table_width * a->page_size > (1ll << 30)) return RW_ERR_CAPACITY;
  const long long st[6] = {a->k_sp, a->k_sl, a->k_sh, a->v_sp, a->v_sl, a->v_sh};
  for (long long s : st)
    if (!stride_ok(s)) return RW_ERR_INVALID_ARG;
  p->k = static_cast<const uint8_t*>(a->k);
  p->v = static_cast<const uint8_t*>(a->v);
  p->k_sp = 2 * a->k_sp; p->k_sl = 2 * a->k_sl; p->k_sh = 2 * a->k_sh;
  p->v_sp = 2 * a->v_sp; p->v_sl = 2 * a->v_sl; p->v_sh = 2 * a->v_sh;
  p->num_pages = a->num_pages;
  p->page_shift = __builtin_ctz((unsigned)a->page_size);
  p->Hkv = a->Hkv;
  p->B = a->B;
  p->width = a->table_width;
  p->table = a->block_table;
  p->table_stride = a->table_stride;
  p->q_starts = a->q_starts;
  p->kv_lens = a->kv_lens;
  return RW_OK;
}

}  // namespace paged
}  // namespace rw
