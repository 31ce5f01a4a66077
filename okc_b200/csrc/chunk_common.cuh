// Ragged batches shared by the multi-axis RoPE append (rope_axes.cu) and the chunk attention
// (attention_chunk*.cu): request b owns the token rows cu_q[b] .. cu_q[b+1]-1, and row t sits at
// the cache position seq_lens[b] - (cu_q[b+1] - t).
#pragma once

#include "kernels.cuh"

namespace okc {

constexpr int kMaxChunkRequests = 2048;  // the per-request prefix sums live in shared memory

// The request of token row t, by one warp: the number of requests that end at or before t, found
// 32 ways at a time (cu_q ascending).  -1 for a row behind the last request.
__device__ __forceinline__ int find_request(const int32_t* cu_q, int B, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = B;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step + step - 1;
    const bool ended = i < hi && cu_q[i + 1] <= t;
    const int k = __popc(__ballot_sync(0xffffffffu, ended));
    lo += k * step;
    hi = min(hi, lo + step - 1);
  }
  return lo < B ? lo : -1;
}

}  // namespace okc
