// Projection with an epilogue, few tokens: the weight is the MMA's 128-row operand and the tokens its N
// side, so one CTA tile covers 128 channels x up to BN tokens and the weight is read once.
//
// HBM-bound on the weight stream (N K bytes in e4m3): one token x 10240 x 8192 17.5 us (4.8 TB/s), of which about 4 are
// the launch and the pipeline's ends; 8192 x 8192 with a residual (67 MB, half of it in L2 from call to call) 9.8 us at 2
// tokens, 14 at 32, 18 at 128, in bf16 24, 30 and 35; with L2 flushed between the calls 19, 23 and 27, in bf16 32, 38 and 43.
//  * K is split over the S = 1, 2, 4 or 8 CTAs of a cluster, chosen so that the waves of resident clusters
//    times a CTA's stages (and ends) are fewest: the whole card reads whatever N is;
//  * warp 0 streams K blocks of 256 bytes a weight row with TMA into a ring, warp 1 issues the
//    MMAs, warps 2-9 drain the accumulator; for an fp32 output every kSplitSegment stages, summed in
//    registers, because the MMA truncates as it accumulates;
//  * each CTA leaves its fp32 sums in its shared memory; the cluster's CTAs take the tokens in turn, add
//    the S sums in rank order over distributed shared memory (the result repeats bit for bit), apply
//    the epilogue and write y 128 channels a row: no workspace, no second launch.
#include "linear.cuh"

namespace okc {

namespace {

constexpr int kSplitPanels = 2;
constexpr int kSplitSegment = 4;
constexpr int kSplitDrain = 8;
constexpr int kSplitThreads = 64 + 32 * kSplitDrain;

template <int BN>
struct SplitCfg {
  static constexpr int A_PANEL = 128 * LIN_KB;
  static constexpr int B_PANEL = BN * LIN_KB;
  static constexpr int STAGE = kSplitPanels * (A_PANEL + B_PANEL);
  // up to 16 tokens two CTAs an SM of three stages each, beyond one of as many as fit
  static constexpr int STAGES = BN <= 16 ? 3 : BN <= 32 ? 5 : BN <= 64 ? 4 : 3;
  static constexpr int BODY = STAGE * STAGES;
  static constexpr int SMEM = 1024 + BODY + 256;
  static constexpr int ACC = BN < 32 ? 32 : BN;  // TMEM columns of an accumulator
  static_assert(BODY >= BN * 128 * 4, "the sums reuse the ring");
};

// A float of CTA `rank`'s shared memory at this CTA's address `local`; 0 where !on.
__device__ __forceinline__ float ld_cluster(uint32_t local, uint32_t rank, bool on) {
  float v;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b32 a;\n setp.ne.b32 p, %3, 0;\n mov.f32 %0, 0f00000000;\n"
      " mapa.shared::cluster.u32 a, %1, %2;\n @p ld.shared::cluster.f32 %0, [a];\n}\n"
      : "=f"(v)
      : "r"(local), "r"(rank), "r"((uint32_t)on)
      : "memory");
  return v;
}

template <bool E4M3, bool OUT32, int BN>
__global__ void __launch_bounds__(kSplitThreads) linear_split_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                     const __grid_constant__ CUtensorMap map_w,
                                                                     const __grid_constant__ LinearArgs a) {
  using C = SplitCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BODY);
  uint64_t* empty = full + C::STAGES;
  uint64_t* accf = empty + C::STAGES;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int KE = E4M3 ? LIN_KB : LIN_KB / 2;
  const int S = gridDim.x, rank = blockIdx.x;
  const int nkb = (a.K + KE * kSplitPanels - 1) / (KE * kSplitPanels);
  const int per = nkb / S, rest = nkb % S;  // this CTA's stages [k_first, k_first + k_n)
  const int k_first = rank * per + min(rank, rest), k_n = per + (rank < rest ? 1 : 0);
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * BN;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accf[i], 1);
      mbar_init(&acce[i], kSplitDrain);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * C::ACC));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  constexpr int COLS = BN >= 64 ? BN / 2 : BN < 32 ? 16 : 32;  // a draining warp's tokens
  const int q4 = warp & 3, half = (warp - 2) >> 2;
  const bool drains = warp >= 2 && half * COLS < BN;
  float acc[COLS];
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (; it < k_n; ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&empty[s], ((uint32_t)(it / C::STAGES) & 1u) ^ 1u, a.err, abort_flag)) {
          *abort_flag = 1;
          break;
        }
        mbar_arrive_expect_tx(&full[s], C::STAGE);
        uint8_t* sa = smem + s * C::STAGE;
#pragma unroll
        for (int p = 0; p < kSplitPanels; ++p) {
          const int k = ((k_first + it) * kSplitPanels + p) * KE;
          tma_load_2d(sa + p * C::A_PANEL, &map_w, k, n0, &full[s]);
          tma_load_2d(sa + kSplitPanels * C::A_PANEL + p * C::B_PANEL, &map_x, k, m0, &full[s]);
        }
      }
      // no copy may be in flight when the block ends or reuses the ring
      for (int i = max(0, it - C::STAGES); i < it; ++i)
        if (!mbar_wait(&full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, a.err)) break;
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = lin_idesc(E4M3, 128, BN);
      int seg = 0;
      bool ok = true;
      for (int it = 0; it < k_n; ++it) {
        const int buf = OUT32 ? seg & 1 : 0;
        const bool begin = OUT32 ? it % kSplitSegment == 0 : it == 0;
        if (OUT32 && begin) ok = mbar_wait(&acce[buf], ((uint32_t)(seg >> 1) & 1u) ^ 1u, a.err, abort_flag);
        const int s = it % C::STAGES;
        ok = ok && mbar_wait(&full[s], (uint32_t)(it / C::STAGES) & 1u, a.err, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sa = smem_u32(smem + s * C::STAGE);
        const uint64_t da = umma_desc_sw128(sa), db = umma_desc_sw128(sa + kSplitPanels * C::A_PANEL);
#pragma unroll
        for (int p = 0; p < kSplitPanels; ++p)
#pragma unroll
          for (int j = 0; j < LIN_KB / 32; ++j)
            lin_mma<E4M3>(tmem + buf * C::ACC, da + ((p * C::A_PANEL + 32 * j) >> 4), db + ((p * C::B_PANEL + 32 * j) >> 4),
                          idesc, !(begin && p == 0 && j == 0));
        umma_commit(&empty[s]);
        if (it == k_n - 1 || (OUT32 && it % kSplitSegment == kSplitSegment - 1)) {
          umma_commit(&accf[buf]);
          ++seg;
        }
      }
      if (!ok) *abort_flag = 1;
      umma_commit(drain);  // no MMA may be in flight when the tensor memory is released
      mbar_wait(drain, 0, a.err);
    }
  } else {
    if (a.res) {  // the rows of the residual that this CTA will add, into L2 while the weight streams
                  // (128 tokens: 22.1 us, without 23.3)
      const int re = a.res_fp32 ? 4 : 2, lines = re, t = threadIdx.x - 64;  // 128 channels are `re` lines
      for (int i = t; i < (min(BN, a.M - m0) - rank + S - 1) / S * lines; i += 32 * kSplitDrain) {
        const int m = m0 + rank + i / lines * S, n = n0 + i % lines * (128 / re);
        if (n < a.N)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(a.res) +
                                                         ((size_t)m * a.ldr + n) * re));
      }
    }
#pragma unroll
    for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
    const int nseg = k_n == 0 ? 0 : OUT32 ? (k_n + kSplitSegment - 1) / kSplitSegment : 1;
    for (int seg = 0; seg < nseg; ++seg) {
      const int buf = OUT32 ? seg & 1 : 0;
      const bool ok = mbar_wait(&accf[buf], (uint32_t)(seg >> 1) & 1u, a.err, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        *abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (drains) {
#pragma unroll
        for (int h = 0; h < COLS; h += 16) {
          float v[16];
          tmem_ld16(tmem + ((uint32_t)(q4 * 32) << 16) + buf * C::ACC + half * COLS + h, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[h + j] += v[j];
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acce[buf]);
    }
  }

  // ---- this CTA's sums [token][channel] into the ring, which nothing uses any more ----
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
  if (drains) {
#pragma unroll
    for (int j = 0; j < COLS; ++j) sums[(half * COLS + j) * 128 + q4 * 32 + lane] = acc[j];
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  // ---- tokens rank, rank + S, ..: thread = (channel, every second of them) ----
  if (warp >= 2) {
    const int t = threadIdx.x - 64, ch = t & 127, n = n0 + ch;
    const int live = min(BN, a.M - m0);
    const float sw = n < a.N ? lin_col_scale(a, n) : 0.f;
    const float bias = n < a.N && a.bias ? __bfloat162float(a.bias[n]) : 0.f;
    // a thread's tokens in flight; few for small tiles, whose time is the cold fetch of this code
    // (1 x 10240 x 8192: 16.9 us with short code, 20.4 us with eight tokens unrolled)
    constexpr int U = BN / 16, oe = OUT32 ? 4 : 2;
    for (int m1 = rank + (t >> 7) * S; m1 < live; m1 += 2 * U * S) {
      float v[U], r[U], sx[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int m = m1 + 2 * i * S;
        sx[i] = m < live ? lin_row_scale(a, m0 + m) : 0.f;
        v[i] = r[i] = 0.f;
      }
      if (a.res && a.res_fp32) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int m = m1 + 2 * i * S;
          if (m < live && n < a.N) r[i] = reinterpret_cast<const float*>(a.res)[(size_t)(m0 + m) * a.ldr + n];
        }
      } else if (a.res) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int m = m1 + 2 * i * S;
          r[i] = ld_bf16_if(reinterpret_cast<const uint8_t*>(a.res) + ((size_t)(m0 + m) * a.ldr + n) * 2, m < live && n < a.N);
        }
      }
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int m = m1 + 2 * i * S;
          v[i] += ld_cluster(smem_u32(sums) + (m * 128 + ch) * 4, (uint32_t)s, m < live);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = fmaf(v[i] * sx[i], sw, bias);
      lin_act_switch(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = lin_act<decltype(act)::value, OUT32>(v[i]);
      });
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int m = m1 + 2 * i * S;
        if (m < live && n < a.N)
          lin_put<OUT32>(reinterpret_cast<uint8_t*>(a.y) + ((size_t)(m0 + m) * a.ldy + n) * oe, v[i] + r[i]);
      }
    }
  }
  if (S > 1) cluster_sync();  // the others have read this CTA's sums
  else __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * C::ACC));
  }
}

// Clusters of S CTAs that this device holds at once, asked once per kernel, S and device.  The query
// answers for one CTA an SM (148 for S = 1); the tiles of up to 16 tokens fit twice.
template <bool E4M3, bool OUT32, int BN>
int resident_clusters(int S) {
  static int known[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  if (known[dev][S] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S, 1024);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = SplitCfg<BN>::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = S;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, linear_split_kernel<E4M3, OUT32, BN>, &cfg) != cudaSuccess) cudaGetLastError();
    constexpr int layers = 2 * (SplitCfg<BN>::SMEM + 1024) <= 228 * 1024 ? 2 : 1;
    known[dev][S] = n > 0 ? n * layers : 1;
  }
  return known[dev][S];
}

// The K split of `tiles` tiles of `stages` stages: fewest stages in a row, a CTA's ends counted as
// eight (one token, 28672 x 8192: 40 us as one wave of whole tiles, 52 us as four of a fifth each).
// Powers of two only: clusters of 3, 5 and 7 left SMs idle (1 x 1280 x 8192: 6.2 us with 8, 11.9 with 7).
template <bool E4M3, bool OUT32, int BN>
int split_plan(long long tiles, int stages, int& S) {
  long long best = -1;
  for (int s = 1; s <= 8 && s <= stages; s *= 2) {
    const long long n = resident_clusters<E4M3, OUT32, BN>(s);
    const long long row = (tiles + n - 1) / n * ((stages + s - 1) / s + 8);
    if (best < 0 || row < best) {
      best = row;
      S = s;
    }
  }
  return best > 0x7fffffff ? 0x7fffffff : (int)best;
}

template <bool E4M3, bool OUT32, int BN>
int launch_split_bn(const LinearArgs& a, int* stages_in_a_row, cudaStream_t stream) {
  using C = SplitCfg<BN>;
  static okc_host::PerDevice configured;
  if (int st = configured.smem(linear_split_kernel<E4M3, OUT32, BN>, C::SMEM)) return st;
  const long long tiles = ((long long)a.N + 127) / 128, mt = (a.M + BN - 1) / BN;
  if (tiles > 65535 || mt > 65535) return OKC_ERR_TOO_LARGE;
  int S = 1;
  const int row = split_plan<E4M3, OUT32, BN>(tiles * mt, lin_stages(a), S);
  if (stages_in_a_row) {
    *stages_in_a_row = row;
    return OKC_OK;
  }
  CUtensorMap mx, mw;
  if (!lin_make_map(&mx, a.x, a.K, a.M, a.ldx, BN, E4M3) || !lin_make_map(&mw, a.w, a.K, a.N, a.ldw, 128, E4M3))
    return OKC_ERR_INVALID;
  return okc_host::launch_k(linear_split_kernel<E4M3, OUT32, BN>, dim3(S, (unsigned)tiles, (unsigned)mt),
                            dim3(kSplitThreads), C::SMEM, stream, dim3(S), mx, mw, a);
}

template <bool E4M3, bool OUT32>
int launch_split_t(const LinearArgs& a, int* row, cudaStream_t stream) {
  if (a.M <= 16) return launch_split_bn<E4M3, OUT32, 16>(a, row, stream);
  if (a.M <= 32) return launch_split_bn<E4M3, OUT32, 32>(a, row, stream);
  if (a.M <= 64) return launch_split_bn<E4M3, OUT32, 64>(a, row, stream);
  return launch_split_bn<E4M3, OUT32, 128>(a, row, stream);
}

int dispatch(const LinearArgs& a, int* row, cudaStream_t stream) {
  if (a.out_fp32) return a.e4m3 ? launch_split_t<true, true>(a, row, stream) : launch_split_t<false, true>(a, row, stream);
  return a.e4m3 ? launch_split_t<true, false>(a, row, stream) : launch_split_t<false, false>(a, row, stream);
}

}  // namespace

int linear_split_stages(const LinearArgs& a) {
  int row = 0x7fffffff;
  return dispatch(a, &row, nullptr) == OKC_OK ? row : 0x7fffffff;
}

int launch_linear_split(const LinearArgs& a, cudaStream_t stream) { return dispatch(a, nullptr, stream); }

}  // namespace okc
