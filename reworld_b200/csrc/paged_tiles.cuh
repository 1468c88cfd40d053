// What the tensor-core kernels over a paged cache share: the TMA maps of q and of the key
// pool, their loads, and the instruction descriptor of the two 16-bit types.
#pragma once

#include "paged.cuh"

namespace rw {
namespace tiles {

constexpr int BM = 128;  // rows of a tile in tensor memory

// Tiled load into this CTA's shared memory, bytes counted on the barrier at the
// shared::cluster address `bar` (the even CTA's for a pair).  No multicast.
template <int NCTA>
__device__ __forceinline__ void load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2,
                                        int c3) {
  if constexpr (NCTA == 2)
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "r"(c3) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "r"(c3) : "memory");
}
template <int NCTA>
__device__ __forceinline__ void load_5d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2,
                                        int c3, int c4) {
  if constexpr (NCTA == 2)
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "r"(c3), "r"(c4) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2), "r"(c3), "r"(c4) : "memory");
}
template <int NCTA>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (NCTA == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0),
        "r"(c1), "r"(c2) : "memory");
}
// f(i, x of lane i) for i < n, by one lane, 8 at a time: an election for every box made
// the loading warps, which have 12 boxes a tile with pages of 16, the slowest part.
template <typename F>
__device__ __forceinline__ void for_pages(int x, int n, F f) {
  for (int i0 = 0; i0 < n; i0 += 8) {
    int y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x, i0 + i);
    if (elect_one()) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < n) f(i0 + i, y[i]);
    }
    __syncwarp();
  }
}

template <bool HALF>
constexpr uint32_t idesc(int M, int N, int b_mn) {
  return HALF ? (idesc_bf16_f32(M, N, 0, b_mn) & ~((1u << 7) | (1u << 10))) : idesc_bf16_f32(M, N, 0, b_mn);
}

// ---------------------------------------------------------------- host
inline CUtensorMapDataType dt(int dtype) {
  return dtype == RW_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// The key pool's head and page are one dimension of the map, in steps of the strides'
// greatest common divisor (a map has five dimensions).
struct KeyLines {
  long long step, lines;  // elements; lines of the dimension
};
inline KeyLines key_lines(const rw_paged_t* c) {
  long long a = c->num_pages == 1 ? 0 : c->k_sp, b = c->Hkv == 1 ? 0 : c->k_sh;
  const long long last = (c->num_pages - 1) * a + (c->Hkv - 1) * b;
  while (b) {
    const long long r = a % b;
    a = b;
    b = r;
  }
  if (a == 0) a = 8;  // one page, one head
  return {a, last / a + 1};
}

// The key pool as (64 channels, 8 rows, D / 64, page_size / 8, head and page), boxes of all
// channels of `rows` rows of a page.
inline int key_map(CUtensorMap* m, const rw_paged_t* c, int rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return RW_ERR_DRIVER;
  const KeyLines kl = key_lines(c);
  cuuint64_t dims[5] = {64, 8, (cuuint64_t)(c->D / 64), (cuuint64_t)(c->page_size / 8), (cuuint64_t)kl.lines};
  cuuint64_t strides[4] = {(cuuint64_t)c->k_sl * 2, 128, (cuuint64_t)c->k_sl * 16, (cuuint64_t)kl.step * 2};
  cuuint32_t box[5] = {64, 8, (cuuint32_t)(c->D / 64), (cuuint32_t)(rows / 8), 1};
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  return enc(m, dt(c->dtype), 5, c->k, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? RW_OK : RW_ERR_DRIVER;
}

// q as (D, Hq, T), boxes of 64 channels x `heads` heads x `tokens` tokens.
inline int q_map(CUtensorMap* m, const void* q, int dtype, int T, int Hq, int D, long long sl, long long sh, int heads,
          int tokens) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return RW_ERR_DRIVER;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)Hq, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)sh * 2, (cuuint64_t)sl * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens};
  cuuint32_t es[3] = {1, 1, 1};
  return enc(m, dt(dtype), 3, const_cast<void*>(q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? RW_OK : RW_ERR_DRIVER;
}

}  // namespace tiles
}  // namespace rw
