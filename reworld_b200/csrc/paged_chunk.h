// Host interface of paged_chunk.cu, and what decides between it and paged_rows.cu.
#pragma once

#include "paged.cuh"

namespace rw {
namespace chunk {

// Sequences of a call whose plan fits the kernel's shared memory.
constexpr int MAX_BATCH = 1024;

struct Call {
  const void* q;
  void* out;
  float* lse;
  float* row_b;
  int T, Hq, longest, causal;         // longest: the most new tokens of a sequence
  long long q_sl, q_sh, o_sl, o_sh;  // element strides
  float scale_log2;
  int* status;
};

int launch(const rw_paged_t* cache, const paged::Pool& pool, const Call& c, void* workspace, cudaStream_t st);
long long workspace_bytes(int D);
bool supported(const rw_paged_t* cache);

}  // namespace chunk

namespace weigh {

// Adds the weights of a chunk::launch that filled c.row_b.
int launch(const rw_paged_t* cache, const paged::Pool& pool, const chunk::Call& c, float* sums, long long sums_sb,
           long long sums_sh, cudaStream_t st);

}  // namespace weigh
}  // namespace rw
