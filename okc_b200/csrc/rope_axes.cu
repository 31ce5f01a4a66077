// Rotary positions with several axes (time, height, width) and the FP8 KV-append of a ragged
// batch.  Token t of request b (cu_q[b] <= t < cu_q[b+1]) sits at the cache position
// seq_lens[b] - (cu_q[b+1] - t), which its rotary positions need not equal; pair i turns by
//   angle = positions[axis(i)][t] * inv_freq[i],   i < R,
// with pair i = (2i, 2i+1), or (i, i + R) in the half-split form; elements from 2R on pass through.
//
// The angle is a product and a reduction to [-pi, pi] in 64 bits: in 32 bits the product alone is
// off by half a unit of its last place, 0.03 rad at position 10^6.  One angle serves every head of
// the token, so this costs R 64-bit reductions a token against (Hq + Hkv) D / 2 rotations.
// Rotations are fp32; q is rounded once to bf16 and k, v once to e4m3 (RNE, overflow -> NaN).
//
// 2 (Hq + 2 Hkv) D bytes in, 2 Hq D + 2 Hkv D bytes out per token, in 16-byte vectors.  The instructions
// (about 110 a vector, more for e4m3) weigh more than the bytes, and for few tokens the chain to the page id: row
// vectors are fetched before it, and a thread fetches its next vector before it turns one.
// 3614 tokens of 28 + 4 heads of 128, 96 elements turned: 15.4 us, 4.1 TB/s (18.7 with the inputs out of L2); 128 tokens of
// 64 + 8 heads: 5 us.
#include "chunk_common.cuh"

namespace okc {

namespace {

constexpr int kRopeThreads = 256;  // at most
constexpr int kMaxPairs = 128;

// Four values to e4m3, to the nearest even one, overflow -> NaN.  The hardware's conversion saturates: it is
// right up to 464, half a step above the largest number, where the tie goes to the even 448.
__device__ __forceinline__ uint32_t e4m3x4_nosat(float a, float b, float c, float d) {
  uint32_t w;
  asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n"
      " mov.b32 %0, {l, h};\n}"
      : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
  if (fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d))) > 464.f) {
    if (fabsf(a) > 464.f) w |= 0x7fu;
    if (fabsf(b) > 464.f) w |= 0x7f00u;
    if (fabsf(c) > 464.f) w |= 0x7f0000u;
    if (fabsf(d) > 464.f) w |= 0x7f000000u;
  }
  return w;
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = bf16_lo(w[k]);
    f[2 * k + 1] = bf16_hi(w[k]);
  }
}

__device__ __forceinline__ void store8_bf16(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// The quotients are those of an fp32 division; one that overflows ends as NaN either way.
__device__ __forceinline__ void store8_e4m3(uint8_t* p, const float (&f)[8], float scale) {
  float e[8];
  if (Quotient::holds(scale)) {
    const Quotient by(scale);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = by(f[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = __fdiv_rn(f[k], scale);
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(e4m3x4_nosat(e[0], e[1], e[2], e[3]), e4m3x4_nosat(e[4], e[5], e[6], e[7]));
}

// n / d from ceil(2^31 / d): exact for n < 2^31 / d.
__device__ __forceinline__ int over(int n, uint32_t by) { return (int)((uint64_t)(uint32_t)n * by >> 31); }

// A block takes TB tokens: a warp each finds their places, all threads share their angles and their items.
template <int TB>
__global__ void __launch_bounds__(kRopeThreads) rope_axes_append_kernel(RopeAxesArgs a) {
  __shared__ __align__(16) float cs[TB][kMaxPairs], sn[TB][kMaxPairs];
  __shared__ int req[TB];
  __shared__ long long slot_of[TB];
  pdl_trigger();
  pdl_wait();
  const int t0 = blockIdx.x * TB, nt = min(TB, a.T - t0);
  const int D = a.D, R = a.R;
  // items: 8 pairs of a q or k head, then 8 passed elements of a q or k head, then 8 of a v head
  const int rp = R / 8, pp = (D - 2 * R) / 8, vp = D / 8, hqk = a.Hq + a.Hkv;
  const int n_rot = hqk * rp, n_pass = hqk * pp, n_all = n_rot + n_pass + a.Hkv * vp;
  struct Item {
    int tk, it, head, u0, u1;  // elements u0 .. + 8 and, of pairs, u1 .. + 8
    uint4 x, y;
  };
  auto fetch = [&](int tk, int it) {
    while (it >= n_all) {
      it -= n_all;
      ++tk;
    }
    Item m = {};
    m.tk = tk;
    m.it = it;
    if (tk >= nt) return m;
    const __nv_bfloat16* row = a.qkv + (size_t)(t0 + tk) * a.ldqkv;
    if (it < n_rot) {
      m.head = over(it, a.by_rp);
      const int i0 = (it - m.head * rp) * 8;
      m.u0 = a.half ? i0 : 2 * i0;
      m.u1 = a.half ? i0 + R : 2 * i0 + 8;
      m.y = *reinterpret_cast<const uint4*>(row + (size_t)m.head * D + m.u1);
    } else {
      const bool is_v = it - n_rot >= n_pass;
      const int per = is_v ? vp : pp, k = it - n_rot - (is_v ? n_pass : 0), h = over(k, is_v ? a.by_vp : a.by_pp);
      m.u0 = (k - h * per) * 8 + (is_v ? 0 : 2 * R);
      m.head = is_v ? hqk + h : h;
    }
    m.x = *reinterpret_cast<const uint4*>(row + (size_t)m.head * D + m.u0);
    return m;
  };
  Item next = fetch(0, threadIdx.x);  // on its way while the block finds its places in the cache

  const int warp = threadIdx.x >> 5;
  for (int tk = warp; tk < nt; tk += blockDim.x >> 5) {
    const int t = t0 + tk, b = find_request(a.cu_q, a.B, t);
    if ((threadIdx.x & 31) == 0) {
      long long slot = -1;
      if (b >= 0) {
        const long long pos = (long long)a.seq_lens[b] - a.cu_q[b + 1] + t;
        if (pos >= 0 && pos <= 0x7fffffff && (uint32_t)pos / (uint32_t)a.P < (uint32_t)a.max_pages) {
          const uint32_t in_row = (uint32_t)pos / (uint32_t)a.P;
          const int page = a.page_table[(size_t)b * a.table_ld + in_row];
          if (page >= 0 && page < a.num_pages) slot = (long long)page * a.P + ((uint32_t)pos - in_row * a.P);
        }
        if (slot < 0) atomicOr(a.err, OKC_DEVERR_PAGE);
      }
      req[tk] = b;
      slot_of[tk] = slot;
    }
  }
  // the last threads first: the first warps are still looking
  for (int k = blockDim.x - 1 - threadIdx.x; k < nt * R; k += blockDim.x) {
    const int tk = TB == 1 ? 0 : over(k, a.by_r), i = k - tk * R;
    const int axis = (int)((a.axis_bits[i >> 5] >> (2 * (i & 31))) & 3u);
    const double ang = (double)a.positions[(size_t)axis * a.ld_pos + t0 + tk] * (double)a.inv_freq[i];
    const double turns = ang * 0.15915494309189535;  // 1 / (2 pi)
    sincospif(2.f * (float)(turns - rint(turns)), &sn[tk][i], &cs[tk][i]);
  }
  __syncthreads();
  while (next.tk < nt) {
    const Item m = next;
    next = fetch(m.tk, m.it + blockDim.x);
    const int t = t0 + m.tk, it = m.it;
    if (req[m.tk] < 0) continue;  // a row behind the last request
    const long long slot = slot_of[m.tk];
    __nv_bfloat16* qo = a.q_out + (size_t)t * a.ldq;
    const size_t kv_row = slot < 0 ? 0 : (size_t)slot * a.Hkv * D;
    const int head = m.head;
    float x[8];
    unpack8(m.x, x);
    if (it < n_rot) {
      const int i0 = a.half ? m.u0 : m.u0 / 2;
      float y[8], p[8], q[8], c[8], s[8];
      unpack8(m.y, y);
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        *reinterpret_cast<float4*>(c + k) = *reinterpret_cast<const float4*>(cs[m.tk] + i0 + k);
        *reinterpret_cast<float4*>(s + k) = *reinterpret_cast<const float4*>(sn[m.tk] + i0 + k);
      }
      if (a.half) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          p[k] = x[k] * c[k] - y[k] * s[k];
          q[k] = x[k] * s[k] + y[k] * c[k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          p[2 * k] = x[2 * k] * c[k] - x[2 * k + 1] * s[k];
          p[2 * k + 1] = x[2 * k] * s[k] + x[2 * k + 1] * c[k];
          q[2 * k] = y[2 * k] * c[4 + k] - y[2 * k + 1] * s[4 + k];
          q[2 * k + 1] = y[2 * k] * s[4 + k] + y[2 * k + 1] * c[4 + k];
        }
      }
      if (head < a.Hq) {
        store8_bf16(qo + (size_t)head * D + m.u0, p);
        store8_bf16(qo + (size_t)head * D + m.u1, q);
      } else if (slot >= 0) {
        uint8_t* dst = a.k_cache + kv_row + (size_t)(head - a.Hq) * D;
        store8_e4m3(dst + m.u0, p, a.k_scale[head - a.Hq]);
        store8_e4m3(dst + m.u1, q, a.k_scale[head - a.Hq]);
      }
    } else if (head < a.Hq) {
      store8_bf16(qo + (size_t)head * D + m.u0, x);
    } else if (slot >= 0) {
      const bool is_v = head >= hqk;
      const int kh = is_v ? head - hqk : head - a.Hq;
      store8_e4m3((is_v ? a.v_cache : a.k_cache) + kv_row + (size_t)kh * D + m.u0, x,
                  is_v ? a.v_scale[kh] : a.k_scale[kh]);
    }
  }
}

}  // namespace

int launch_rope_axes_append(const RopeAxesArgs& args, cudaStream_t stream) {
  RopeAxesArgs a = args;
  auto by = [](int d) { return d > 0 ? (uint32_t)(((1ull << 31) + d - 1) / d) : 0u; };
  a.by_rp = by(a.R / 8);
  a.by_pp = by((a.D - 2 * a.R) / 8);
  a.by_vp = by(a.D / 8);
  a.by_r = by(a.R);
  // 3614 tokens of 28 + 4 heads 16.7 us, a token a block 19.4; 1806 tokens 10.5 and 11.8; 903 tokens 7.1 either way
  if (a.T >= 1024)
    return okc_host::launch_k(rope_axes_append_kernel<4>, dim3((a.T + 3) / 4), dim3(kRopeThreads), 0, stream, dim3(1), a);
  // a thread for each item (see the kernel), within two to eight warps
  const int items = (a.Hq + a.Hkv) * (a.D / 8 - a.R / 8) + a.Hkv * (a.D / 8);
  const int threads = items <= 64 ? 64 : items >= kRopeThreads ? kRopeThreads : (items + 31) / 32 * 32;
  return okc_host::launch_k(rope_axes_append_kernel<1>, dim3(a.T), dim3(threads), 0, stream, dim3(1), a);
}

}  // namespace okc
