// What the projection kernels with an epilogue share (linear.cu: tall token blocks, linear_split.cu:
// few tokens): tensor maps over 8- and 16-bit rows, the instruction descriptors and the epilogue's
// arithmetic.  A K step is 128 bytes of a row for either type (128 e4m3 or 64 bf16 values: one
// swizzle atom), an MMA 32 bytes of it, so the kernels differ only in kind and descriptor.
#pragma once

#include <type_traits>

#include "kernels.cuh"
#include "tcgen05.cuh"

namespace okc {

constexpr int LIN_KB = 128;  // bytes of a row per K block

// Both kernels take K in stages of 256 bytes a row.
inline int lin_stages(const LinearArgs& a) { return (int)(((long long)a.K * (a.e4m3 ? 1 : 2) + 255) / 256); }

// Stages that the K-split kernel (linear_split.cu) runs one after the other for this projection.
int linear_split_stages(const LinearArgs& a);

// D fp32, both operands K-major, M x N; e4m3 (kind::f8f6f4, type code 0) or bf16 (kind::f16, type code 1).
__host__ __device__ constexpr uint32_t lin_idesc(bool e4m3, int m, int n) {
  return (1u << 4) | (e4m3 ? 0u : ((1u << 7) | (1u << 10))) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <bool E4M3>
__device__ __forceinline__ void lin_mma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (E4M3)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    umma_bf16(tmem_d, a, b, idesc, acc);
}

enum { LIN_ACT_NONE = 0, LIN_ACT_RELU = 1, LIN_ACT_SILU = 2, LIN_ACT_GELU = 3, LIN_ACT_GELU_TANH = 4 };

// Activations in fp32.  tanh and the logistic function go through one exponential:
// 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2u)).  A NaN stays a NaN (relu included: fmaxf would drop it).
// FINE, for an fp32 output: the exponential's argument in two parts, since one rounding of it (what a bf16 output does not
// see) is |v| units of the result.
template <bool FINE>
__device__ __forceinline__ float lin_exp(float u) {
  if (!FINE) return __expf(u);
  constexpr float hi = 1.4426950216293335f, lo = 1.9259629911266175e-8f;  // log2(e)
  const float t = u * hi, rest = fmaf(u, lo, fmaf(u, hi, -t));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fabsf(t) < 128.f ? fmaf(e, rest * 0.6931471805599453f, e) : e;  // at either end it is 0 or infinite
}
template <int ACT, bool FINE>
__device__ __forceinline__ float lin_act(float v) {
  auto over = [](float n, float u) { return __fdividef(n, 1.f + lin_exp<FINE>(u)); };
  if constexpr (ACT == LIN_ACT_RELU) return v < 0.f ? 0.f : v;
  if constexpr (ACT == LIN_ACT_SILU) return over(v, -v);
  if constexpr (ACT == LIN_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.7071067811865476f));
  if constexpr (ACT == LIN_ACT_GELU_TANH) return over(v, -1.5957691216057308f * (v + 0.044715f * v * v * v));
  return v;
}

// Calls f(integral_constant<ACT>) for the run-time activation.
template <typename F>
__device__ __forceinline__ void lin_act_switch(int act, F&& f) {
  switch (act) {
    case LIN_ACT_RELU: f(std::integral_constant<int, LIN_ACT_RELU>()); break;
    case LIN_ACT_SILU: f(std::integral_constant<int, LIN_ACT_SILU>()); break;
    case LIN_ACT_GELU: f(std::integral_constant<int, LIN_ACT_GELU>()); break;
    case LIN_ACT_GELU_TANH: f(std::integral_constant<int, LIN_ACT_GELU_TANH>()); break;
    default: f(std::integral_constant<int, LIN_ACT_NONE>()); break;
  }
}

template <bool OUT32>
__device__ __forceinline__ void lin_put(uint8_t* p, float v) {
  if constexpr (OUT32)
    *reinterpret_cast<float*>(p) = v;
  else
    *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
}

// A bf16, or 0 where !on, without a branch: so that a row's load does not wait for the one before.
__device__ __forceinline__ float ld_bf16_if(const uint8_t* p, bool on) {
  uint16_t w;
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n mov.b16 %0, 0;\n @p ld.global.u16 %0, [%1];\n}"
               : "=h"(w) : "l"(p), "r"((uint32_t)on) : "memory");
  return __uint_as_float((uint32_t)w << 16);
}

__device__ __forceinline__ float lin_row_scale(const LinearArgs& a, int m) { return a.x_scale ? a.x_scale[m] : 1.f; }
__device__ __forceinline__ float lin_col_scale(const LinearArgs& a, int n) {
  return a.w_scale ? a.w_scale[a.w_scale_one ? 0 : n] : 1.f;
}

// 32 consecutive TMEM columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  tm_ld32(taddr, r);
  tm_wait_ld(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Host: a 2-D map over [rows][inner] of 8- or 16-bit elements, boxes of LIN_KB bytes x box_rows rows.
inline bool lin_make_map(CUtensorMap* m, const void* base, int inner, int rows, long long ld, int box_rows, bool e4m3) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  const int es = e4m3 ? 1 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * es};
  cuuint32_t box[2] = {(cuuint32_t)(LIN_KB / es), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base),
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace okc
