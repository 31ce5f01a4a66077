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

// 2^x; ex2(-inf) = 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(x) from exp(2x) given x * 2 log2(e): 1 - 2 / (1 + e^2x); off by 1.2e-7 absolute, which the cap multiplies: by
// 6e-6 of a score at a cap of 50, by 1.2e-4 at kPlainCap.
__device__ __forceinline__ float tanh_from_2l2e(float x) { return 1.f - __fdividef(2.f, 1.f + ex2(x)); }
constexpr float kPlainCap = 1024.f;
// How scores are capped: up to kPlainCap, and above it.  A kernel variant each: chosen within the kernel, the second cost the
// first 4 to 10% (128 requests of one token 219 and 234 us, of four 419 and 459).
constexpr int kCapNone = 0, kCapPlain = 1, kCapFine = 2;
inline int cap_form(float softcap) { return softcap > kPlainCap ? kCapFine : softcap > 0.f ? kCapPlain : kCapNone; }

// tanh(x) / x over |x| <= 1 as a polynomial in x^2 of the least relative error: 1.5e-7 in fp32.
constexpr int kTanhTerms = 7;
__host__ __device__ constexpr float tanh_term(int k) {
  return k == 0   ? 0.99999994f
         : k == 1 ? -0.3333284f
         : k == 2 ? 0.13325204f
         : k == 3 ? -0.053457007f
         : k == 4 ? 0.020289943f
         : k == 5 ? -0.0062033492f
                  : 0.0010410136f;
}
// The same within 2^-21 of itself however small: for caps above kPlainCap, whose scores of a few units are a tanh of
// next to nothing.
__device__ __forceinline__ float tanh_fine_from_2l2e(float v) {
  const float x = v * 0.34657359027997264f, w = x * x;
  float p = tanh_term(kTanhTerms - 1);
#pragma unroll
  for (int k = kTanhTerms - 2; k >= 0; --k) p = fmaf(w, p, tanh_term(k));
  return w <= 1.f ? x * p : tanh_from_2l2e(v);
}

__device__ __forceinline__ uint32_t e4m3x2_h2(uint32_t two) {
  uint32_t h;
  asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(h) : "r"(two));
  return h;
}

__device__ __forceinline__ uint32_t h2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The page of a position.
__device__ __forceinline__ int page_of(const ChunkArgs& a, int position) {
  return (int)((uint64_t)(uint32_t)position * a.page_mul >> a.page_shift);
}

// The first position that the window leaves a row at position p, which is negative where a request has more new
// tokens than cached ones (those rows see nothing, whatever the window).
__device__ __forceinline__ int window_start(const ChunkArgs& a, int p) {
  return a.window > 0 ? max(0, max(0, p + 1) - a.window) : 0;
}

// A request: its rows' key intervals all lie in [lo, hi).
struct Req {
  int n, len, lo, hi, prefix;  // new tokens, cached tokens, union of the rows' key intervals
};

__device__ __forceinline__ Req request(const ChunkArgs& a, int b) {
  Req r;
  r.n = max(0, a.cu_q[b + 1] - a.cu_q[b]);
  r.len = max(0, a.seq_lens[b]);
  r.prefix = a.prefix_lens ? a.prefix_lens[b] : 0;
  r.lo = window_start(a, r.len - r.n);
  r.hi = min(r.len, a.max_keys);  // positions past the table's columns do not exist
  return r;
}

// One query row: its position and the interval [lo, hi) that it sees (hi <= lo: nothing).
struct RowSpan {
  int pos, lo, hi;
};
__device__ __forceinline__ RowSpan row_span(const ChunkArgs& a, const Req& rq, int row0, int i) {
  RowSpan r;
  r.pos = rq.len - rq.n + i;
  r.lo = window_start(a, r.pos);
  if (a.doc_start) r.lo = max(r.lo, a.doc_start[row0 + i]);
  r.hi = min(rq.hi, max(r.pos + 1, rq.prefix));
  return r;
}

// The power of two that brings a bf16 row whose largest magnitude has the bits `top` into
// [2^13, 2^14): the row is then exact in f16 down to 2^-27 of that magnitude.
__device__ __forceinline__ int f16_shift(uint32_t top) { return max(-100, (int)(top >> 7) - 127 - 13); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// A piece of the workspace.
inline size_t up(size_t n) { return (n + 255) / 256 * 256; }

// A kernel of this file family serves the requests of at most / more than this many rows a KV
// head (new tokens x query heads of one KV head).  128 requests of 64 / 8 heads, the short chunks' kernel against the
// tensor-memory one: 32 rows 416 and 637 us, 64 rows 676 and 767; one request of 64 rows 35 and 35.
constexpr int kSplitRows = 64;

// The tensor-memory kernel (attention_chunk_tc.cu) for the requests of more than `above` rows (kSplitRows, or 0
// where the only request may have more than kSplitRows).  `sums` [T * Hq][D] and `origins` [T * Hq][2]: scratch of very
// long contexts, which may be what the short chunks' kernel takes behind it.
size_t attn_chunk_tc_ws_bytes(int T, int B, int Hq, int Hkv, int D);
int launch_attn_chunk_tc(const ChunkArgs& a, int above, void* ws, float* sums, float* origins, cudaStream_t stream);

}  // namespace okc
