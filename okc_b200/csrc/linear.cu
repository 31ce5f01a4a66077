// Projection with an epilogue, tall token blocks: y = act(x w^T * x_scale[m] * w_scale[n] + bias[n]) + residual,
// e4m3 or bf16 operands, fp32 accumulation in tensor memory.
//
// Compute-bound from a few hundred tokens on (2MNK operations against (M + N) K bytes in).  8192 x 10240 x 8192 in
// e4m3 with a gelu: 478 to 568 us by the card's temperature, 2.4 to 2.9 PFLOP/s under the power cap.  777 x 4099 x 4104 in
// bf16 to fp32 with a silu and a residual: 47 us (36 us at 4096 x 4096 without the silu): 4 token tiles on 148 SMs, and the ends of a tile in the open.
//  * a CTA pair owns a tile of 256 tokens x bn channels (tcgen05 cta_group::2): each CTA loads its 128
//    token rows and half of the channel rows, 32 KB a K block for 256 x 256 x 128 bytes of products,
//    so shared-memory traffic stays below what the 8-bit MMA rate takes (a single CTA's 128 x 256 tile
//    needs 48 KB for half the products);
//  * persistent grid of pairs; tiles are taken in groups of 8 token tiles per channel column, so that the
//    pairs in flight share operands in L2; bn (a multiple of 32) is chosen so that the last
//    wave is full;
//  * warp 0 streams K blocks of 256 bytes a row with TMA into a ring, warp 1 of the leading CTA issues
//    the MMAs, warps 4-11 of both CTAs drain the accumulators;
//  * the MMA truncates as it accumulates (3e-6 relative over K = 4104 in bf16).  A bf16 output does
//    not see that; for an fp32 output an accumulator takes kSegment K blocks only, and the draining warps
//    add the segments in fp32 registers while the next one runs in the other accumulator: 3e-7.
//    A thread holds 128 sums then, with the registers that the first warpgroup gives up;
//  * the epilogue turns each 32 x 32 block through shared memory, so that a warp reads the residual
//    and writes y a row at a time whatever their strides and alignment.
#include "linear.cuh"

namespace okc {

namespace {

constexpr int kMaxStages = 4;
constexpr int kRing = 192 * 1024;  // as many stages as fit: 3 of 256 channels, 4 of up to 128
constexpr int kPanels = 2;       // 128-byte K panels of a stage: one barrier and one commit for eight MMAs
constexpr int kSegment = 4;      // stages an accumulator takes, for an fp32 output
constexpr int kDrainWarps = 8;   // a CTA's
constexpr int kFirstDrain = 4;   // warps 0 and 1 load and issue; 2 and 3 fill their warpgroup
constexpr int kTallThreads = 32 * (kFirstDrain + kDrainWarps);
// Registers a thread: the launch's, and how fp32 outputs split them over the three warpgroups.
constexpr int kLaunchRegs = 168, kIssueRegs = 40, kDrainRegs = 232;
static_assert(128 * kIssueRegs + 256 * kDrainRegs <= kTallThreads * kLaunchRegs, "the split must fit the launch");
static_assert(kIssueRegs < kLaunchRegs && kDrainRegs > kLaunchRegs,
              "setmaxnreg.dec lowers and .inc raises; the other way round is an illegal instruction");
constexpr int kGroup = 8;        // token tiles of a group
constexpr uint16_t kLeader = 1, kBoth = 3;  // of a pair

struct TallSmem {
  static constexpr int A_PANEL = 128 * LIN_KB;       // this CTA's 128 token rows
  static constexpr int B_PANEL = 128 * LIN_KB;       // its channel rows, at most
  static_assert(kRing >= 3 * kPanels * (A_PANEL + B_PANEL), "three of the widest stages");
  static constexpr int BLOCK = 32 * 32;              // a 32 x 32 fp32 block per draining warp
  static constexpr int TURN = kDrainWarps * BLOCK * 4;
  static constexpr int BAR0 = kRing + TURN;
  static constexpr int TOTAL = 1024 + BAR0 + 256;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The shared-memory address of `bar` in the pair's leading CTA.
__device__ __forceinline__ uint32_t in_leader(uint64_t* bar) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
  return r;
}
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
template <bool E4M3>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (E4M3)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Arrives on `bar` of the CTAs in `who` (bit = rank) when every MMA issued so far is done.  A CTA waits for all that is
// signalled to it before it leaves: its shared memory may be another block's by the time a later signal lands.
__device__ __forceinline__ void pair_commit(uint64_t* bar, uint16_t who) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(who)
      : "memory");
}

// Tile order: groups of kGroup token tiles, channel tiles outer within a group.
__device__ __forceinline__ void lin_tile(int u, int mt, int nt, int& tm, int& tn) {
  const int per = kGroup * nt, g = u / per, first = g * kGroup, rows = min(kGroup, mt - first);
  const int r = u - g * per;
  tn = r / rows;
  tm = first + r - tn * rows;
}

// A lane's row into a 32 x 32 block, two columns at a time; the pairs of a row are permuted by it, so
// that rows are written and read without bank conflicts.
__device__ __forceinline__ void block_put(float* block, int row, int pair, float x, float y) {
  reinterpret_cast<float2*>(block)[row * 16 + (pair ^ (row & 15))] = make_float2(x, y);
}

// Writes a 32 x 32 block of y whose rows take aligned accesses of two columns: a lane has two neighbouring
// columns of every second row.  Residual rows are fetched ahead of the stores, which may overwrite them.
template <bool OUT32>
__device__ __forceinline__ void tall_block(const float* block, float my_sx, const LinearArgs& a, int m0, int n0) {
  constexpr int B = 8;  // a lane's rows in flight
  const int lane = threadIdx.x & 31, odd = lane >> 4, pair = lane & 15;
  const int oe = OUT32 ? 4 : 2, re = a.res_fp32 ? 4 : 2;
  float sw[2], bias[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = n0 + 2 * pair + i;
    sw[i] = lin_col_scale(a, n);
    bias[i] = a.bias ? __bfloat162float(a.bias[n]) : 0.f;
  }
  uint8_t* y = reinterpret_cast<uint8_t*>(a.y) + ((size_t)(m0 + odd) * a.ldy + n0 + 2 * pair) * oe;
  const uint8_t* res = reinterpret_cast<const uint8_t*>(a.res) + ((size_t)(m0 + odd) * a.ldr + n0 + 2 * pair) * re;
  const long long y_step = 2 * a.ldy * oe, r_step = 2 * a.ldr * re;
#pragma unroll 1
  for (int i0 = 0; i0 < 16; i0 += B) {
    float2 r[B], v[B];
    if (a.res) {
      if (a.res_fp32) {
#pragma unroll
        for (int i = 0; i < B; ++i) r[i] = *reinterpret_cast<const float2*>(res + i * r_step);
      } else {
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const uint32_t b = *reinterpret_cast<const uint32_t*>(res + i * r_step);
          r[i] = make_float2(bf16_lo(b), bf16_hi(b));
        }
      }
      res += B * r_step;
    } else {
#pragma unroll
      for (int i = 0; i < B; ++i) r[i] = make_float2(0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int row = 2 * (i0 + i) + odd;
      v[i] = reinterpret_cast<const float2*>(block)[row * 16 + (pair ^ (row & 15))];
      const float sx = __shfl_sync(0xffffffffu, my_sx, row);
      v[i].x = fmaf(v[i].x * sx, sw[0], bias[0]);
      v[i].y = fmaf(v[i].y * sx, sw[1], bias[1]);
    }
    lin_act_switch(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < B; ++i) {
        v[i].x = lin_act<decltype(act)::value, OUT32>(v[i].x);
        v[i].y = lin_act<decltype(act)::value, OUT32>(v[i].y);
      }
    });
#pragma unroll
    for (int i = 0; i < B; ++i) {
      v[i].x += r[i].x;
      v[i].y += r[i].y;
      if (OUT32)
        *reinterpret_cast<float2*>(y + i * y_step) = v[i];
      else
        *reinterpret_cast<uint32_t*>(y + i * y_step) = pack_bf16x2(v[i].x, v[i].y);
    }
    y += B * y_step;
  }
}

// A whole bf16 block without a residual, whose rows take 16-byte accesses: finished by the lanes that have its rows, so
// that it is turned as bf16 in 16-byte vectors (5957 x 25904 x 480 in e4m3: 150 us, through tall_block 181;
// with a gelu 272 and 337).
__device__ __forceinline__ void packed_block(uint8_t* block, const float (&v)[32], float my_sx, const LinearArgs& a, int m0,
                                             int n0) {
  const int lane = threadIdx.x & 31;
  float2* column = reinterpret_cast<float2*>(block + 2048);  // scale and bias of each
  column[lane] = make_float2(lin_col_scale(a, n0 + lane), a.bias ? __bfloat162float(a.bias[n0 + lane]) : 0.f);
  __syncwarp();
  float z[32];
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float4 c = *reinterpret_cast<const float4*>(column + j);
    z[j] = fmaf(v[j] * my_sx, c.x, c.y);
    z[j + 1] = fmaf(v[j + 1] * my_sx, c.z, c.w);
  }
  lin_act_switch(a.act, [&](auto act) {
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = lin_act<decltype(act)::value, false>(z[j]);
  });
  // rows of 64 bytes; the chunks of two neighbouring rows are permuted by them, against bank conflicts
#pragma unroll
  for (int k = 0; k < 4; ++k)
    *reinterpret_cast<uint4*>(block + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16)) =
        make_uint4(pack_bf16x2(z[8 * k], z[8 * k + 1]), pack_bf16x2(z[8 * k + 2], z[8 * k + 3]),
                   pack_bf16x2(z[8 * k + 4], z[8 * k + 5]), pack_bf16x2(z[8 * k + 6], z[8 * k + 7]));
  __syncwarp();
  __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(a.y) + (size_t)(m0 + lane / 4) * a.ldy + n0 + lane % 4 * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + lane / 4;
    *reinterpret_cast<uint4*>(y + i * 8 * a.ldy) =
        *reinterpret_cast<const uint4*>(block + row * 64 + (((lane % 4) ^ ((row >> 1) & 3)) * 16));
  }
}

// The same for any block, of which `rows` x `cols` exist: a lane has one column, so that a row takes one access
// whatever its alignment (777 x 4095 x 4104 in bf16, fp32 out, bf16
// residual: 45 us; two columns a lane and a branch at each load 57).
template <bool OUT32>
__device__ __forceinline__ void ragged_block(const float* block, int rows, int cols, float my_sx, const LinearArgs& a,
                                             int m0, int n0) {
  constexpr int B = 16;  // rows in flight
  const int lane = threadIdx.x & 31;
  const bool on = lane < cols;
  const int oe = OUT32 ? 4 : 2, re = a.res_fp32 ? 4 : 2;
  const float sw = on ? lin_col_scale(a, n0 + lane) : 0.f;
  const float bias = on && a.bias ? __bfloat162float(a.bias[n0 + lane]) : 0.f;
  uint8_t* y = reinterpret_cast<uint8_t*>(a.y) + ((size_t)m0 * a.ldy + n0 + lane) * oe;
  const uint8_t* res = reinterpret_cast<const uint8_t*>(a.res) + ((size_t)m0 * a.ldr + n0 + lane) * re;
  const long long y_step = a.ldy * oe, r_step = a.ldr * re;
#pragma unroll 1
  for (int i0 = 0; i0 < rows; i0 += B) {
    float v[B], r[B];
#pragma unroll
    for (int i = 0; i < B; ++i) r[i] = 0.f;
    if (a.res) {
      if (a.res_fp32) {
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (on && i0 + i < rows) r[i] = *reinterpret_cast<const float*>(res + i * r_step);
      } else {
#pragma unroll
        for (int i = 0; i < B; ++i) r[i] = ld_bf16_if(res + i * r_step, on && i0 + i < rows);
      }
      res += B * r_step;
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int row = i0 + i;
      const float sx = __shfl_sync(0xffffffffu, my_sx, row);
      v[i] = fmaf(block[row * 32 + 2 * ((lane >> 1) ^ (row & 15)) + (lane & 1)] * sx, sw, bias);
    }
    lin_act_switch(a.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < B; ++i) v[i] = lin_act<decltype(act)::value, OUT32>(v[i]);
    });
#pragma unroll
    for (int i = 0; i < B; ++i)
      if (on && i0 + i < rows) lin_put<OUT32>(y + i * y_step, v[i] + r[i]);
    y += B * y_step;
  }
}

template <bool E4M3, bool OUT32>
__global__ void __launch_bounds__(kTallThreads, 1) linear_tall_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                      const __grid_constant__ CUtensorMap map_w,
                                                                      const __grid_constant__ LinearArgs a, int bn) {
  using C = TallSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* turn = reinterpret_cast<float*>(smem + kRing);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR0);  // the leader's count both CTAs' bytes
  uint64_t* empty = full + kMaxStages;
  uint64_t* accf = empty + kMaxStages;
  uint64_t* acce = accf + 2;  // the leader's count both CTAs' draining warps
  uint64_t* drain = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  constexpr int KE = E4M3 ? LIN_KB : LIN_KB / 2;  // K elements of a panel
  const int nkb = (a.K + KE * kPanels - 1) / (KE * kPanels);
  const int mt = (a.M + 255) / 256, nt = (a.N + bn - 1) / bn, tiles = mt * nt;
  const int b_panel = bn / 2 * LIN_KB, stage = kPanels * (C::A_PANEL + b_panel), stages = min(kMaxStages, kRing / stage);
  const int u_first = blockIdx.x >> 1, u_step = gridDim.x >> 1;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&accf[i], 1);
      mbar_init(&acce[i], 2 * kDrainWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // both CTAs' barriers and tensor memory are there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp < kFirstDrain) {
    if constexpr (OUT32) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 0 && lane == 0) {
      const int half = bn / 2;
      int it = 0, s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = u_first; u < tiles && ok; u += u_step) {
        int tm, tn;
        lin_tile(u, mt, nt, tm, tn);
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          if (!mbar_wait(&empty[s], ph ^ 1u, a.err, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * stage);
          uint8_t* sa = smem + s * stage;
          const uint32_t bar = in_leader(&full[s]);
#pragma unroll
          for (int p = 0; p < kPanels; ++p) {
            const int k = (kb * kPanels + p) * KE;
            tma_load_pair(sa + p * C::A_PANEL, &map_x, k, tm * 256 + (int)rank * 128, bar);
            tma_load_pair(sa + kPanels * C::A_PANEL + p * b_panel, &map_w, k, tn * bn + (int)rank * half, bar);
          }
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // a stage is left once its MMAs are done, so no copy is in flight after these waits (where a
      // role gave up, it waited for longer than any copy takes)
      for (int i = max(0, it - stages); i < it; ++i)
        if (!mbar_wait(&empty[i % stages], (uint32_t)(i / stages) & 1u, a.err, abort_flag)) break;
    } else if (warp == 1 && lane == 0 && rank == 0) {
      const uint32_t idesc = lin_idesc(E4M3, 256, bn);
      int s = 0, seg = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = u_first; u < tiles && ok; u += u_step) {
        for (int kb = 0; kb < nkb; ++kb) {
          const int buf = seg & 1;
          const bool begin = OUT32 ? kb % kSegment == 0 : kb == 0;
          if (begin) {
            ok = mbar_wait(&acce[buf], ((uint32_t)(seg >> 1) & 1u) ^ 1u, a.err, abort_flag);
            if (!ok) break;
          }
          ok = mbar_wait(&full[s], ph, a.err, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sa = smem_u32(smem + s * stage);
          const uint64_t da = umma_desc_sw128(sa), db = umma_desc_sw128(sa + kPanels * C::A_PANEL);
#pragma unroll
          for (int p = 0; p < kPanels; ++p)
#pragma unroll
            for (int j = 0; j < LIN_KB / 32; ++j)
              pair_mma<E4M3>(tmem + buf * 256, da + ((p * C::A_PANEL + 32 * j) >> 4),
                             db + ((p * b_panel + 32 * j) >> 4), idesc, !(begin && p == 0 && j == 0));
          pair_commit(&empty[s], kBoth);
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
          if (kb == nkb - 1 || (OUT32 && kb % kSegment == kSegment - 1)) {
            pair_commit(&accf[buf], kBoth);
            ++seg;
          }
        }
      }
      if (!ok) *abort_flag = 1;
      pair_commit(drain, kLeader);  // no MMA may be in flight when the tensor memory is released
      mbar_wait(drain, 0, a.err);
    }
  } else {
    if constexpr (OUT32) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kDrainRegs));
    const int q4 = warp & 3, half = (warp - kFirstDrain) >> 2;
    const int chunks = bn / 32, c_first = half * ((chunks + 1) / 2), c_n = half ? chunks / 2 : (chunks + 1) / 2;
    const int nseg = OUT32 ? (nkb + kSegment - 1) / kSegment : 1;
    const uint32_t lanes = tmem + ((uint32_t)(q4 * 32) << 16) + c_first * 32;
    float* st = turn + (warp - kFirstDrain) * C::BLOCK;
    int seg = 0;
    bool ok = true;
    auto wait_acc = [&](int buf) {
      ok = __all_sync(0xffffffffu, mbar_wait(&accf[buf], (uint32_t)(seg >> 1) & 1u, a.err, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return ok;
    };
    auto free_acc = [&](int buf) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(&acce[buf])) : "memory");
    };
    for (int u = u_first; u < tiles; u += u_step) {
      int tm, tn;
      lin_tile(u, mt, nt, tm, tn);
      const int m0 = tm * 256 + (int)rank * 128 + q4 * 32, rows = min(32, a.M - m0);
      const float my_sx = lane < rows ? lin_row_scale(a, m0 + lane) : 0.f;
      if (a.res && lane < rows) {  // this lane's row of the residual, into L2 while the products run (777 x 4095: 1 to 4 us)
        const int re = a.res_fp32 ? 4 : 2, n0 = tn * bn + c_first * 32, cols = min(c_n * 32, a.N - n0);
        const uint8_t* p = reinterpret_cast<const uint8_t*>(a.res) + ((size_t)(m0 + lane) * a.ldr + n0) * re;
        for (int i = 0; cols > 0 && i < cols * re + 128; i += 128)  // a row may begin inside a line
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p + min(i, cols * re - 1)));
      }
      auto emit = [&](int c) {
        const int n0 = tn * bn + (c_first + c) * 32;
        __syncwarp();
        if (a.pairs && rows == 32 && a.N - n0 >= 32) tall_block<OUT32>(st, my_sx, a, m0, n0);
        else ragged_block<OUT32>(st, rows, a.N - n0, my_sx, a, m0, n0);
        __syncwarp();
      };
      const int c_live = rows > 0 ? min(c_n, (a.N - tn * bn + 31) / 32 - c_first) : 0;
      if constexpr (OUT32) {
        float acc[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] = 0.f;
        for (int i = 0; i < nseg; ++i, ++seg) {
          if (!wait_acc(seg & 1)) break;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c >= c_n) break;
            float v[32];
            tmem_ld32(lanes + (seg & 1) * 256 + c * 32, v);
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c][j] += v[j];
          }
          free_acc(seg & 1);
        }
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < c_live; ++c) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k != c) continue;
#pragma unroll
            for (int j = 0; j < 16; ++j) block_put(st, lane, j, acc[k][2 * j], acc[k][2 * j + 1]);
          }
          emit(c);
        }
      } else {
        if (!wait_acc(seg & 1)) break;
#pragma unroll 1
        for (int c = 0; c < c_live; ++c) {
          float v[32];
          tmem_ld32(lanes + (seg & 1) * 256 + c * 32, v);
          if (c == c_live - 1) free_acc(seg & 1);
          const int n0 = tn * bn + (c_first + c) * 32;
          if (a.packed && rows == 32 && a.N - n0 >= 32) {
            packed_block(reinterpret_cast<uint8_t*>(st), v, my_sx, a, m0, n0);
            __syncwarp();
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) block_put(st, lane, j, v[2 * j], v[2 * j + 1]);
            emit(c);
          }
        }
        if (c_live <= 0) free_acc(seg & 1);
        ++seg;
      }
    }
    if (!ok) *abort_flag = 1;
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may signal it or use its shared memory
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Channels a tile: the multiple of 32 from 64 to 256 whose waves cost least.  A stage's time goes with the rows it
// loads, 256 and bn of them (1024 x 8192 x 8192 in e4m3, a wave of 32 stages: 16.9, 18.9, 21, 26.9, 27 us at 64, 128,
// 160, 224 and 256 channels), not with its products.
int tall_bn(int M, int N, int pairs) {
  int best = 256;
  long long cost = -1;
  for (int bn = 256; bn >= 64; bn -= 32) {
    const long long tiles = (long long)((M + 255) / 256) * ((N + bn - 1) / bn);
    const long long c = (tiles + pairs - 1) / pairs * (bn + 256);
    if (cost < 0 || c < cost) {
      cost = c;
      best = bn;
    }
  }
  return best;
}

template <bool E4M3, bool OUT32>
int launch_tall(const LinearArgs& a, cudaStream_t stream) {
  const int pairs = okc_host::num_sms() / 2;
  const int bn = tall_bn(a.M, a.N, pairs);
  CUtensorMap mx, mw;
  if (!lin_make_map(&mx, a.x, a.K, a.M, a.ldx, 128, E4M3) || !lin_make_map(&mw, a.w, a.K, a.N, a.ldw, bn / 2, E4M3))
    return OKC_ERR_INVALID;
  static okc_host::PerDevice configured;
  if (int st = configured.smem(linear_tall_kernel<E4M3, OUT32>, TallSmem::TOTAL, OUT32 ? kLaunchRegs : 0)) return st;
  const long long tiles = (long long)((a.M + 255) / 256) * ((a.N + bn - 1) / bn);
  if (tiles > 0x7fffffff) return OKC_ERR_TOO_LARGE;
  const int grid = 2 * (int)(tiles < pairs ? tiles : pairs);
  return okc_host::launch_k(linear_tall_kernel<E4M3, OUT32>, dim3(grid), dim3(kTallThreads), TallSmem::TOTAL, stream, dim3(2),
                            mx, mw, a, bn);
}

}  // namespace

// Up to 128 tokens the K-split kernel; beyond, the kernel whose estimate is shorter.  A stage of the
// K-split kernel's 128 x 128 tiles takes 0.68 us (its ends count as eight), one of a pair's tiles 0.46 us
// up to 128 channels and 0.58 us at 256, besides 4.5 us at the ends (measured from 192 to 1024 tokens, N 256 to 8192,
// K 1024 to 8192: the estimate picks the faster one or is within 10%.  256 tokens, N = 256,
// K = 8192 in bf16: 34.6 us on pairs, 11.5 us split; 512 x 8192 x 8192: 57 and 88 us).
int launch_linear(const LinearArgs& a, cudaStream_t stream) {
  if (a.M <= 128) return launch_linear_split(a, stream);
  const int pairs = okc_host::num_sms() / 2, bn = tall_bn(a.M, a.N, pairs);
  const long long tiles = (long long)((a.M + 255) / 256) * ((a.N + bn - 1) / bn);
  const double tall = 4.5 + (double)((tiles + pairs - 1) / pairs) * lin_stages(a) * (bn <= 128 ? 0.46 : 0.34 + 0.00094 * bn);
  if (tiles <= pairs && 0.68 * linear_split_stages(a) < tall) return launch_linear_split(a, stream);
  if (a.out_fp32) return a.e4m3 ? launch_tall<true, true>(a, stream) : launch_tall<false, true>(a, stream);
  return a.e4m3 ? launch_tall<true, false>(a, stream) : launch_tall<false, false>(a, stream);
}

}  // namespace okc
