// Projection with an epilogue, tall token blocks: y = act(x w^T * x_scale[m] * w_scale[n] + bias[n]) + residual,
// e4m3 or bf16 operands, fp32 accumulation in tensor memory.
//
// Compute-bound from a few hundred tokens on (2MNK operations against (M + N) K bytes in).
//  * a CTA owns a 128-token x BN-channel tile; persistent grid, one CTA per SM; tiles are taken
//    in groups of 16 token tiles per channel column so that the CTAs in flight share operands in L2;
//  * warp 0 streams K blocks of 128 bytes a row of both operands with TMA into a ring, warp 1 issues
//    the MMAs into one of two TMEM accumulators, warps 2-5 drain the other one;
//  * the epilogue turns each 32 x 32 block through shared memory, so that a warp reads the residual
//    and writes y a row at a time whatever their strides and alignment.
#include "linear.cuh"

namespace okc {

namespace {

template <int BN, int STAGES>
struct LinCfg {
  static constexpr int A_BYTES = 128 * LIN_KB;
  static constexpr int B_BYTES = BN * LIN_KB;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int TURN = 4 * 32 * 33 * 4;  // a 32 x 32 fp32 block per epilogue warp
  static constexpr int BODY = STAGE * STAGES + TURN;
  static constexpr int SMEM = 1024 + BODY + 256;
  static constexpr int TMEM_COLS = 2 * BN;
};

// Tile order: groups of 16 token tiles, channel tiles outer within a group.
__device__ __forceinline__ void lin_tile(int u, int mt, int nt, int& tm, int& tn) {
  constexpr int GM = 16;
  const int per = GM * nt, g = u / per, first = g * GM, rows = min(GM, mt - first);
  const int r = u - g * per;
  tn = r / rows;
  tm = first + r - tn * rows;
}

template <bool E4M3, int BN, int STAGES>
__global__ void __launch_bounds__(192) linear_tall_kernel(const __grid_constant__ CUtensorMap map_x,
                                                          const __grid_constant__ CUtensorMap map_w, LinearArgs a) {
  using C = LinCfg<BN, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* turn = reinterpret_cast<float*>(smem + C::STAGE * STAGES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BODY);
  uint64_t* empty = full + STAGES;
  uint64_t* accf = empty + STAGES;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int KE = E4M3 ? LIN_KB : LIN_KB / 2;  // K elements per block
  const int nkb = (a.K + KE - 1) / KE;
  const int mt = (a.M + 127) / 128, nt = (a.N + BN - 1) / BN, tiles = mt * nt;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accf[i], 1);
      mbar_init(&acce[i], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < tiles && ok; u += gridDim.x) {
        int tm, tn;
        lin_tile(u, mt, nt, tm, tn);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty[s], ((uint32_t)(it / STAGES) & 1u) ^ 1u, a.err, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], C::STAGE);
          uint8_t* sa = smem + s * C::STAGE;
          tma_load_2d(sa, &map_x, kb * KE, tm * 128, &full[s]);
          tma_load_2d(sa + C::A_BYTES, &map_w, kb * KE, tn * BN, &full[s]);
        }
      }
      if (!ok) *abort_flag = 1;
      // no copy may be in flight when the block ends
      for (int i = max(0, it - STAGES); i < it; ++i)
        if (!mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u, a.err)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = lin_idesc(E4M3, 128, BN);
      int it = 0, seg = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < tiles && ok; u += gridDim.x, ++seg) {
        const int buf = seg & 1;
        if (!mbar_wait(&acce[buf], ((uint32_t)(seg >> 1) & 1u) ^ 1u, a.err, abort_flag)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full[s], (uint32_t)(it / STAGES) & 1u, a.err, abort_flag)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sa = smem_u32(smem + s * C::STAGE);
          const uint64_t da = umma_desc_sw128(sa), db = umma_desc_sw128(sa + C::A_BYTES);
#pragma unroll
          for (int j = 0; j < LIN_KB / 32; ++j)
            lin_mma<E4M3>(tmem + buf * BN, da + 2 * j, db + 2 * j, idesc, (kb | j) != 0);
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&accf[buf]);
      }
      if (!ok) *abort_flag = 1;
      umma_commit(drain);  // no MMA may be in flight when the tensor memory is released
      mbar_wait(drain, 0, a.err);
    }
  } else {
    const int q4 = warp & 3;
    float* st = turn + q4 * 32 * 33;
    int seg = 0;
    for (int u = blockIdx.x; u < tiles; u += gridDim.x, ++seg) {
      int tm, tn;
      lin_tile(u, mt, nt, tm, tn);
      const int buf = seg & 1;
      const bool ok = mbar_wait(&accf[buf], (uint32_t)(seg >> 1) & 1u, a.err, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int m0 = tm * 128 + q4 * 32;
      const float my_sx = m0 + lane < a.M ? lin_row_scale(a, m0 + lane) : 0.f;
      const int rows = min(32, a.M - m0);
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += 32) {
        const int n = tn * BN + c0 + lane;
        if (tn * BN + c0 >= a.N || rows <= 0) break;
        float v[32];
        tmem_ld32(tmem + ((uint32_t)(q4 * 32) << 16) + buf * BN + c0, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) st[lane * 33 + j] = v[j];
        __syncwarp();
        const bool on = n < a.N;
        const float sw = on ? lin_col_scale(a, n) : 0.f;
        const float bias = on && a.bias ? __bfloat162float(a.bias[n]) : 0.f;
#pragma unroll 8
        for (int i = 0; i < rows; ++i) {
          const float sx = __shfl_sync(0xffffffffu, my_sx, i);
          if (on) lin_store(a, m0 + i, n, st[i * 33 + lane], sx, sw, bias);
        }
        __syncwarp();
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acce[buf]);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
  }
}

template <bool E4M3, int BN, int STAGES>
int launch_tall(const LinearArgs& a, cudaStream_t stream) {
  using C = LinCfg<BN, STAGES>;
  CUtensorMap mx, mw;
  if (!lin_make_map(&mx, a.x, a.K, a.M, a.ldx, 128, E4M3) || !lin_make_map(&mw, a.w, a.K, a.N, a.ldw, BN, E4M3))
    return OKC_ERR_INVALID;
  static okc_host::PerDevice configured;
  if (int st = configured.smem(linear_tall_kernel<E4M3, BN, STAGES>, C::SMEM)) return st;
  const long long tiles = (long long)((a.M + 127) / 128) * ((a.N + BN - 1) / BN);
  if (tiles > 0x7fffffff) return OKC_ERR_TOO_LARGE;
  const int grid = (int)(tiles < okc_host::num_sms() ? tiles : okc_host::num_sms());
  return okc_host::launch_k(linear_tall_kernel<E4M3, BN, STAGES>, dim3(grid), dim3(192), C::SMEM, stream, dim3(1), mx,
                            mw, a);
}

}  // namespace

int launch_linear(const LinearArgs& a, cudaStream_t stream) {
  return a.e4m3 ? launch_tall<true, 256, 4>(a, stream) : launch_tall<false, 256, 4>(a, stream);
}

}  // namespace okc
