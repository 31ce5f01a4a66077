// Residual add + RMSNorm with an e4m3 output and one scale per row:
//   s = round(x + r)              (r bf16 or fp32; s is stored in r's type, the next residual)
//   y = s * rsqrt(mean(s^2) + eps) * g,  g = w or 1 + w     (s as it is stored)
//   scale = max|y| / 448 (1 for a row of zeros),  q = e4m3(y / scale)
// without r: s = x.
//
// HBM-bound: 2H (x) + 2..4H (r) + 2..4H (s) + H (q) bytes a row.  The row stays in registers
// between its two reductions (sum of squares, then the largest magnitude), so each byte moves
// once.  A row takes 32 threads up to H = 1024 (eight rows a block, no block barrier) and 128,
// 256 or 512 threads beyond, so that a thread holds at most four 8-element vectors, in 64 registers (16384 wide in bf16 74 us
// for 4096 rows; 98 with the 70 that the compiler would take, one block an SM).
// 8192 rows of 8192 with an fp32 residual: 110 us, 6.7 TB/s (a device copy runs at 6.55), a bf16 one 70, none 52; one row
// 3.2 us, which is the launch and one trip to memory.
//
// The sum of squares, the norm and the scale are fp32; q is the one rounding to 8 bits.  The
// largest magnitude is an integer maximum of the absolute bit patterns, which orders finite
// values as floats and puts infinities and NaN above them: a row that holds either, or whose squares
// overflow, gets a NaN scale instead of a finite scale that hides it.
#include "kernels.cuh"

namespace okc {

namespace {

constexpr float kE4m3Max = 448.f;

struct NormFp8Args {
  const __nv_bfloat16* x;
  long long ldx;
  const void* res;
  long long ldr;
  const __nv_bfloat16* w;
  void* res_out;
  long long ldo;
  uint8_t* q;
  long long ldq;
  float* scale;
  int T, H;
  float eps;
  int unit_offset;
};

__device__ __forceinline__ uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// RES: 0 none, 1 bf16, 2 fp32.  TPR threads a row, V vectors of 8 elements a thread.
template <int RES, int TPR, int V>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, V == 4 && TPR > 32 ? 1024 / TPR : 1) add_rmsnorm_fp8_kernel(NormFp8Args a) {
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;  // rows a block
  constexpr int WPR = TPR / 32;                    // warps a row
  __shared__ float red_s[ROWS][WPR];
  __shared__ uint32_t red_m[ROWS][WPR];
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x / TPR, tid = threadIdx.x % TPR;
  const int row = blockIdx.x * ROWS + sub;
  const bool live = row < a.T;
  const size_t t = live ? row : 0;
  float h[V][8];
  uint4 gw[V];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = (j * TPR + tid) * 8;
    const bool on = live && i < a.H;
    uint4 xv = make_uint4(0, 0, 0, 0);
    float4 r0 = make_float4(0, 0, 0, 0), r1 = r0;
    uint4 rb = make_uint4(0, 0, 0, 0);
    gw[j] = xv;
    if (on) {
      xv = *reinterpret_cast<const uint4*>(a.x + t * a.ldx + i);
      if (RES == 1) rb = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.res) + t * a.ldr + i);
      if (RES == 2) {
        const float* r = reinterpret_cast<const float*>(a.res) + t * a.ldr + i;
        r0 = *reinterpret_cast<const float4*>(r);
        r1 = *reinterpret_cast<const float4*>(r + 4);
      }
      gw[j] = *reinterpret_cast<const uint4*>(a.w + i);
    }
    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w}, rw[4] = {rb.x, rb.y, rb.z, rb.w};
    const float rf[8] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[j][2 * k] = bf16_lo(xw[k]);
      h[j][2 * k + 1] = bf16_hi(xw[k]);
      if (RES == 1) {
        const uint32_t s = pack_bf16x2(h[j][2 * k] + bf16_lo(rw[k]), h[j][2 * k + 1] + bf16_hi(rw[k]));
        h[j][2 * k] = bf16_lo(s);
        h[j][2 * k + 1] = bf16_hi(s);
      } else if (RES == 2) {
        h[j][2 * k] += rf[2 * k];
        h[j][2 * k + 1] += rf[2 * k + 1];
      }
      ss += h[j][2 * k] * h[j][2 * k] + h[j][2 * k + 1] * h[j][2 * k + 1];
    }
  }
  // the stream goes out while the reductions run
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = (j * TPR + tid) * 8;
    if (!live || i >= a.H) break;
    if (RES == 1) {
      uint4 o;
      o.x = pack_bf16x2(h[j][0], h[j][1]);
      o.y = pack_bf16x2(h[j][2], h[j][3]);
      o.z = pack_bf16x2(h[j][4], h[j][5]);
      o.w = pack_bf16x2(h[j][6], h[j][7]);
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.res_out) + t * a.ldo + i) = o;
    } else if (RES == 2) {
      float* o = reinterpret_cast<float*>(a.res_out) + t * a.ldo + i;
      *reinterpret_cast<float4*>(o) = make_float4(h[j][0], h[j][1], h[j][2], h[j][3]);
      *reinterpret_cast<float4*>(o + 4) = make_float4(h[j][4], h[j][5], h[j][6], h[j][7]);
    }
  }
  ss = warp_sum(ss);
  if (WPR > 1) {
    if ((tid & 31) == 0) red_s[sub][tid >> 5] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += red_s[sub][i];
  }
  float inv = rsqrtf(ss / (float)a.H + a.eps);
  if (ss == 0.f && a.eps == 0.f) inv = 0.f;                // a row of zeros
  if (!(ss < INFINITY)) inv = __uint_as_float(0x7fffffffu);  // no number of its own, whatever 1 / inf would make of it
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const uint32_t g4[4] = {gw[j].x, gw[j].y, gw[j].z, gw[j].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float g0 = bf16_lo(g4[k]), g1 = bf16_hi(g4[k]);
      if (a.unit_offset) {
        g0 += 1.f;
        g1 += 1.f;
      }
      h[j][2 * k] = h[j][2 * k] * inv * g0;
      h[j][2 * k + 1] = h[j][2 * k + 1] * inv * g1;
      // elements past H are 0 * inv * (0 or 1): NaN only if inv is, and then the row is NaN anyway
      top = max(top, max(__float_as_uint(h[j][2 * k]) & 0x7fffffffu, __float_as_uint(h[j][2 * k + 1]) & 0x7fffffffu));
    }
  }
  top = warp_umax(top);
  if (WPR > 1) {
    if ((tid & 31) == 0) red_m[sub][tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; ++i) top = max(top, red_m[sub][i]);
  }
  const float amax = __uint_as_float(top);
  float scale = __fdiv_rn(amax, kE4m3Max);
  if (scale == 0.f) scale = 1.f;
  if (!live) return;
  if (tid == 0) a.scale[row] = scale;
  // one reciprocal a row, each quotient as a division rounds it
  const bool held = Quotient::holds(scale);
  const Quotient by(scale);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = (j * TPR + tid) * 8;
    if (i >= a.H) break;
    uint32_t o[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float2 e[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float x = h[j][4 * k + 2 * m], y = h[j][4 * k + 2 * m + 1];
        e[m] = held ? by(x, y) : make_float2(__fdiv_rn(x, scale), __fdiv_rn(y, scale));
      }
      o[k] = (uint32_t)f2_to_e4m3x2_sat(e[0].x, e[0].y) | ((uint32_t)f2_to_e4m3x2_sat(e[1].x, e[1].y) << 16);
    }
    *reinterpret_cast<uint2*>(a.q + t * a.ldq + i) = make_uint2(o[0], o[1]);
  }
}

template <int RES>
int launch_res(const NormFp8Args& a, cudaStream_t stream) {
  const int nv = a.H / 8;
#define OKC_NORM(TPR, V)                                                                                     \
  return okc_host::launch_k(add_rmsnorm_fp8_kernel<RES, TPR, V>, dim3((a.T + (TPR < 256 ? 256 / TPR : 1) - 1) / \
                                                                      (TPR < 256 ? 256 / TPR : 1)),          \
                            dim3(TPR < 256 ? 256 : TPR), 0, stream, dim3(1), a)
  if (nv <= 32) OKC_NORM(32, 1);
  if (nv <= 64) OKC_NORM(32, 2);
  if (nv <= 128) OKC_NORM(32, 4);
  if (nv <= 256) OKC_NORM(128, 2);
  if (nv <= 512) OKC_NORM(256, 2);
  if (nv <= 1024) OKC_NORM(256, 4);
  OKC_NORM(512, 4);
#undef OKC_NORM
}

}  // namespace

int launch_add_rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldr, int res_fp32, const void* w,
                           void* res_out, long long ldo, void* q, long long ldq, float* scale, int T, int H, float eps,
                           int unit_offset, cudaStream_t stream) {
  NormFp8Args a;
  a.x = reinterpret_cast<const __nv_bfloat16*>(x);
  a.ldx = ldx;
  a.res = res;
  a.ldr = ldr;
  a.w = reinterpret_cast<const __nv_bfloat16*>(w);
  a.res_out = res_out;
  a.ldo = ldo;
  a.q = reinterpret_cast<uint8_t*>(q);
  a.ldq = ldq;
  a.scale = scale;
  a.T = T;
  a.H = H;
  a.eps = eps;
  a.unit_offset = unit_offset;
  if (!res) return launch_res<0>(a, stream);
  return res_fp32 ? launch_res<2>(a, stream) : launch_res<1>(a, stream);
}

}  // namespace okc
