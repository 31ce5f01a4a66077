// Attention of ragged chunks over the paged e4m3 cache for chunks of many rows: both products on the
// tensor cores with scores, probabilities and outputs in tensor memory.  The masks and the scores
// are those of attention_chunk.cu, which serves the short chunks.
//
// Compute-bound: 4 D operations per (row, visible key) against 2 D cache bytes per key and 256 rows.
// A block takes 256 rows (token-major, the G query heads of one KV head side by side) as two tiles
// of 128 and streams the keys that any of them sees in blocks of 64:
//  * a softmax warpgroup per tile, one thread a row: P goes back over S as f16 and is the next product's A
//    operand there.  S has two buffers a tile, so that a block's scores are formed while the one
//    before is in the softmax, and a row's sums never leave its thread;
//  * four warps fetch key and value rows by page, turn e4m3 into f16 (exact) and store both as the
//    swizzled rows that the MMAs read (keys K-major, values MN-major: no transpose), four blocks deep;
//  * a thread per tile issues its MMAs;
//  * a block's exponentials are taken against the origin so far, in one pass over S, and done again with
//    O rescaled only where a P exceeds 2^8 of the origin's: rare after a row's first blocks.
// The special-function unit bounds it: 256 x 64 exponentials take 1024 cycles of it a block, where the tensor
// cores need 1024 too, and a block takes 1960 (the softmax warps' other instructions and latencies overlap
// only in part; a third of the exponentials as polynomials on the fused-operation pipe made it slower).
// 4096 tokens behind 4096 cached, 64 / 8 heads of 128: 825 us (1000 TFLOP/s), capped 1004 us, under a bias 855.  A CTA of one key block
// takes 11 us (finding its rows, their keys and the query 3, the first keys 2, the first block's two passes 2, the
// output 2): short spans are bound by that.
// Blocks of a request are taken from its last rows on: the longest causal spans start first.  With few
// blocks the keys are split over several, which leave fp32 partial sums for a merge.
#include <type_traits>

#include "chunk_common.cuh"
#include "tcgen05.cuh"

namespace okc {

namespace {

constexpr int kTile = 128;                 // rows of a tile
constexpr int kKeys = 64;                  // keys of a block
constexpr int kDepth = 4;                  // blocks of keys and values in shared memory
constexpr int kPair = 2 * kTile;           // rows of a CTA
constexpr int kSoftmaxThreads = 256;
constexpr int kLoadThreads = 128;
constexpr int kIssueWarp = (kSoftmaxThreads + kLoadThreads) / 32;          // and the next; the others of their warpgroup idle
constexpr int kTcThreads = kSoftmaxThreads + kLoadThreads + 128;
// Registers a thread: the launch's, and how the four warpgroups split them.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 168, kLoadRegs = 120, kIssueRegs = 56;
static_assert(2 * kSoftmaxRegs + kLoadRegs + kIssueRegs <= 4 * kLaunchRegs, "the split must fit the launch");
static_assert(kSoftmaxRegs > kLaunchRegs && kLoadRegs < kLaunchRegs && kIssueRegs < kLaunchRegs,
              "setmaxnreg.inc raises and .dec lowers; the other way round is an illegal instruction");
constexpr int kHigh = 0, kLow = 1, kExact = 2;  // how a block's exponentials are taken
constexpr int kSlack = 8;                  // log2 growth of the maximum that O tolerates
// log2 of the largest P at the origin of the exponentials: f16 keeps P down to 2^-25, so that keys are lost from the sum only
// 2^-(25 + kLift) below the largest score that the origin was taken from, and reaches 2^16.
constexpr int kLift = 7;
static_assert(kLift + kSlack <= 15, "P stays finite in f16");

template <int D>
struct TcCfgA {
  static constexpr int PANELS = D / 64;                // swizzled panels of 64 f16 columns
  static constexpr int QSUB = kTile * 128;             // a panel of a query tile
  static constexpr int QTILE = QSUB * PANELS;
  static constexpr int SUB = kKeys * 128;              // a panel of a key or value block
  static constexpr int BLOCK = SUB * PANELS;
  static constexpr int Q0 = 0;
  static constexpr int K0 = 2 * QTILE;
  static constexpr int V0 = K0 + kDepth * BLOCK;
  static constexpr int OFF0 = V0 + kDepth * BLOCK;     // [2][kKeys] cache rows of the keys
  static constexpr int BAR0 = OFF0 + 2 * kKeys * 4;
  static constexpr int SMEM = 1024 + BAR0 + 512;
};

// The tensor core truncates as it adds to O: 1e-7 of it for 16 keys, always towards zero (0.06% over 131072 keys, 0.6% over
// 2^20).  After so many blocks a row's O goes into its fp32 sums in the workspace, and starts again.
constexpr int kFold = 2048;

struct TcPlanA {
  int splits;
  int above;   // requests of more rows than this are served
  float* acc;  // [splits][T * Hq][D]: a split's sums, or what has been folded
  float* ml;   // [splits][T * Hq][2]: their origin, and the sum of P
};

// f16 operands, fp32 sums, 128 x n.
__device__ __forceinline__ uint32_t umma_idesc_f16(int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// A from shared memory, K-major.
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// A from tensor memory: lane = row, column = two consecutive k.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// MN-major SWIZZLE_128B: 64-element panels `panel` bytes apart (LBO), 8-row groups 1024 B apart (SBO).
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t saddr, uint32_t panel) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ f32x2 bits2(uint32_t x, uint32_t y) { return pair2(__uint_as_float(x), __uint_as_float(y)); }

// tanh(x) / x as a polynomial in x^2: the seven terms of tanh_term over |x| <= 1, or three of the least |x * error|
// (1.2e-6, 1.5e-4 of a score at kLowCap) over |x| <= 0.4: fused operations where the exponential and the reciprocal
// of the exact form occupy the special-function unit twice.
constexpr float kTanhRange2 = 1.f, kTanhLowRange2 = 0.16f;  // squares of the ranges
constexpr float kLowCap = 128.f;
template <bool LOW>
__device__ __forceinline__ f32x2 tanh2(int k) {
  const float c = !LOW ? tanh_term(k) : k == 0 ? 0.99997884f : k == 1 ? -0.33225426f : 0.11942387f;
  return pair2(c, c);
}

__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Barriers and words shared by the roles.
struct TcShared {
  uint64_t plan, q_full, k_full[kDepth], v_full[kDepth], kv_empty[kDepth], drain[2];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][buffer]
  uint32_t tmem;
  int abort;
  int b, tile, row0;       // the block's request (-1: none), its row tile pair, the request's first row
  Req rq;
  int lo, hi;              // union of its rows' intervals
  int full_lo, full_hi;    // intersection: keys in it need no mask
  uint32_t nan[kDepth][kKeys / 32];  // per V block: its keys that hold a NaN that was taken out
};

template <int D, int CAP, bool BIAS, bool FOLD>
__global__ void __launch_bounds__(kTcThreads, 1) attn_chunk_tc_kernel(ChunkArgs a, TcPlanA pl) {
  using C = TcCfgA<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared& sh = *reinterpret_cast<TcShared*>(smem + C::BAR0);
  static_assert(sizeof(TcShared) <= 512, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  if (threadIdx.x == 0) {
    mbar_init(&sh.plan, kSoftmaxThreads / 32);
    mbar_init(&sh.q_full, kSoftmaxThreads / 32);
    for (int i = 0; i < kDepth; ++i) {
      mbar_init(&sh.k_full[i], kLoadThreads / 32);
      mbar_init(&sh.v_full[i], kLoadThreads / 32);
      mbar_init(&sh.kv_empty[i], 2);  // one per tile
      for (int w = 0; w < kKeys / 32; ++w) sh.nan[i][w] = 0;
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.drain[t], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.s_full[t][i], 1);
        mbar_init(&sh.p_full[t][i], kSoftmaxThreads / 64);
      }
    }
    sh.abort = 0;
    sh.lo = 0x7fffffff;
    sh.hi = 0;
    sh.full_lo = 0;
    sh.full_hi = 0x7fffffff;
    fence_mbar_init();
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  const int head = blockIdx.x % a.Hkv, split = blockIdx.x / a.Hkv;
  if (warp == 0) {  // the blockIdx.y-th tile pair of the requests it serves
    int before = 0, found = -1, tile = 0;
    for (int base = 0; base < a.B && found < 0; base += 32) {
      const int b = base + lane;
      int n = 0;
      Req r = {};
      if (b < a.B) {
        r = request(a, b);
        const int rows = r.n * a.G;
        if (rows > pl.above) n = (rows + kPair - 1) / kPair;
        if (r.len > a.max_keys && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(a.err, OKC_DEVERR_PAGE);
      }
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      const bool here = before + sum > (int)blockIdx.y;
      const uint32_t who = __ballot_sync(0xffffffffu, here);
      if (who) {
        const int l = __ffs(who) - 1;
        found = base + l;
        // from the request's last tile pair on
        tile = __shfl_sync(0xffffffffu, before + sum, l) - 1 - (int)blockIdx.y;
        if (lane == l) {
          sh.rq = r;
          sh.row0 = a.cu_q[b];
        }
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
      sh.b = found;
      sh.tile = tile;
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  const int b = sh.b;
  volatile int* abort_flag = &sh.abort;
  // The union of the rows' intervals, once the softmax threads have published it, gives the keys: this
  // split's first one, and its blocks.  The j-th block taken is key0 + block_at(j).  Under a distance bias the
  // nearest keys come first, so that a row meets its largest scores at once (front to back every block raises
  // the maximum: 1770 us against 915 for 4096 tokens behind 4096): from the last row's block down, then the
  // blocks ahead of it, which only a prefix has.  Without a bias a row's first block is better a whole one than
  // its diagonal.
  struct Plan {
    int key0, k_hi, nb, near;
  };
  auto plan = [&]() -> Plan {
    if (!mbar_wait(&sh.plan, 0, a.err, abort_flag)) *abort_flag = 1;
    const int k_lo = *reinterpret_cast<volatile int*>(&sh.lo);
    Plan p;
    p.k_hi = *reinterpret_cast<volatile int*>(&sh.hi);
    int first = 0;
    p.nb = p.k_hi > k_lo ? (p.k_hi - k_lo + kKeys - 1) / kKeys : 0;
    if (pl.splits > 1) {
      const int per = (p.nb + pl.splits - 1) / pl.splits;
      first = min(p.nb, split * per);
      p.nb = min(p.nb, first + per) - first;
    }
    p.key0 = k_lo + first * kKeys;
    p.near = 0;
    if (BIAS && p.nb > 0) {
      const int last = min(sh.rq.n - 1, (int)((uint64_t)(uint32_t)(sh.tile * kPair + kPair - 1) * a.group_mul >> a.group_shift));
      p.near = min(p.nb - 1, max(0, sh.rq.len - sh.rq.n + last - p.key0) / kKeys);
    }
    return p;
  };
  auto block_at = [](const Plan& p, int j) { return (BIAS && j <= p.near ? p.near - j : j) * kKeys; };

  if (warp < kSoftmaxThreads / 32) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax
    const int w = warp >> 2, lr = (warp & 3) * 32 + lane;  // tile, row of it
    const int r = sh.tile * kPair + w * kTile + lr;
    Req rq = {};
    int row0 = 0;
    if (b >= 0) {
      rq = sh.rq;
      row0 = sh.row0;
    }
    const int rows = rq.n * a.G, my_tok = (int)((uint64_t)(uint32_t)r * a.group_mul >> a.group_shift);
    const bool live = r < rows, on = sh.tile * kPair + w * kTile < rows;
    const int tok = live ? row0 + my_tok : 0, hq = live ? head * a.G + r - my_tok * a.G : 0;
    // The warp's 32 query rows, on their way while the keys are found: a lane has chunk qc of 16 bytes of every
    // QR-th row from qr on, so that an access takes whole rows.
    constexpr int QC = D / 8, QR = 32 / QC, QN = 32 / QR;
    const int qr = lane / QC, qc = lane % QC;
    auto at_row = [&](long long mine, int row) {  // a value of the lane that has the row
      return (long long)__shfl_sync(0xffffffffu, (unsigned long long)mine, row);
    };
    const long long q_at = live ? (long long)tok * a.ldq + (long long)hq * D : -1;
    auto q_slot = [&](int row, int chunk) {  // of the warp's rows, in a swizzled panel
      const int r128 = (warp & 3) * 32 + row;
      return smem + C::Q0 + w * C::QTILE + (chunk / 8) * C::QSUB + r128 * 128 + ((chunk % 8) ^ (r128 & 7)) * 16;
    };
#pragma unroll 4
    for (int i = 0; i < QN; ++i) {
      const long long at = at_row(q_at, i * QR + qr);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(q_slot(i * QR + qr, qc))),
                   "l"(a.q + (at >= 0 ? at + qc * 8 : 0)), "r"(at >= 0 ? 16 : 0)
                   : "memory");
    }
    RowSpan me = {0, 0, 0};
    if (live) me = row_span(a, rq, row0, my_tok);
    {
      const int lo = __reduce_min_sync(0xffffffffu, live && me.lo < me.hi ? me.lo : 0x7fffffff);
      const int hi = __reduce_max_sync(0xffffffffu, live && me.lo < me.hi ? me.hi : 0);
      const int flo = __reduce_max_sync(0xffffffffu, live ? me.lo : 0);
      const int fhi = __reduce_min_sync(0xffffffffu, live ? me.hi : 0x7fffffff);
      if (lane == 0) {
        atomicMin(&sh.lo, lo);
        atomicMax(&sh.hi, hi);
        atomicMax(&sh.full_lo, flo);
        atomicMin(&sh.full_hi, fhi);
        mbar_arrive(&sh.plan);
      }
      __syncwarp();
    }
    const Plan keys = plan();
    const int nb = keys.nb;
    const int f_lo = sh.full_lo, f_hi = sh.full_hi;
    const uint32_t lanes = sh.tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = lanes + 2 * kTile + w * D;
    float fac = 0.f, slope = 0.f, m_ref = -INFINITY, l = 0.f;
    uint32_t nan_d[D / 32];  // output columns that a visible NaN value reaches
#pragma unroll
    for (int i = 0; i < D / 32; ++i) nan_d[i] = 0;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (nb > 0 && on) {
      // the row in f16, scaled by a power of two, in place; a lane has one row, whose chunks the swizzle puts
      // into different banks than its neighbours'
      uint4 v[D / 8];
      uint32_t two = 0;  // the largest magnitudes of the even and of the odd elements
#pragma unroll
      for (int i = 0; i < D / 8; ++i) v[i] = *reinterpret_cast<const uint4*>(q_slot(lane, i));
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        two = __vmaxu2(__vmaxu2(two, __vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu)),
                       __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
      const uint32_t top = max(two & 0xffffu, two >> 16);
      const int shf = f16_shift(top);
      fac = a.k_scale[head] * a.sm_scale * (CAP ? 2.f / a.softcap : 1.f) * 1.4426950408889634f * pow2(shf);
      // a negative factor goes into the query, so that the largest score is the largest sum
      const float down = fac < 0.f ? -pow2(-shf) : pow2(-shf);
      fac = fabsf(fac);
      if (BIAS && live) slope = a.slopes[hq] * 1.4426950408889634f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = h2(bf16_lo(u[k]) * down, bf16_hi(u[k]) * down);
        *reinterpret_cast<uint4*>(q_slot(lane, i)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.q_full);

    const float cap2 = CAP ? a.softcap * 1.4426950408889634f : 0.f;
    const float f = CAP ? cap2 : fac;
    auto s_ready = [&](int j) {  // block j's scores are there, and with them every product up to P V of block j - 2
      return mbar_wait(&sh.s_full[w][j & 1], (uint32_t)(j >> 1) & 1u, a.err, abort_flag);
    };
    bool ok = true;
    bool low = a.softcap <= kLowCap;  // ... and no score so far has left the three-term range
    auto part_of = [&] { return (size_t)split * a.T * a.Hq + (size_t)tok * a.Hq + hq; };  // the row in the workspace
    // O of the blocks before j0 into the row's sums in the workspace, which are brought to its origin.
    auto fold = [&](int j0) {
      const size_t part = part_of();
      if (!s_ready(j0 + 1)) *abort_flag = 1;  // P V of the block before is done, and the next waits for its P
      tc_after();
      const float was = j0 > kFold && live ? pl.ml[part * 2] : -INFINITY, down = was == -INFINITY ? 0.f : ex2(was - m_ref);
      float* sums = pl.acc + part * D;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 16) {
        uint32_t v[16];
        tm_ld16(to + c0, v);
        tm_wait_ld(v);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          if (!live) continue;
          const float o = __uint_as_float(v[c]);
          sums[c0 + c] = j0 > kFold ? fmaf(sums[c0 + c], down, o) : o;
        }
      }
      if (live) pl.ml[part * 2] = m_ref;
      tc_before();
    };
#pragma unroll 1
    for (int j = 0; j < nb && on; ++j) {
      if (FOLD && j > 0 && j % kFold == 0) fold(j);
      const int kb = keys.key0 + block_at(keys, j);
      const uint32_t ts = lanes + w * kTile + (j & 1) * kKeys;  // S, and P over its first half
      ok = __all_sync(0xffffffffu, s_ready(j));
      if (!ok) {
        *abort_flag = 1;
        break;
      }
      tc_after();
      const bool edge = !__all_sync(0xffffffffu, !live || (me.lo <= kb && me.hi >= kb + kKeys));
      // visible columns [vis_lo, vis_hi)
      const int vis_lo = me.lo - kb, vis_hi = me.hi - kb;
      auto seen = [&](int c) { return c >= vis_lo && c < vis_hi; };
      // The log2 score of raw sum v at key kb + c is u * f, u = v or its capped form, with a bias less
      // slope * |ahead - c|.  Where the visible keys of all rows lie on one side of them, no absolute value is
      // needed: the bias is toward * (c - ahead).
      const float ahead = (float)(me.pos - kb);
      const bool behind = BIAS && __all_sync(0xffffffffu, !live || min(me.hi, kb + kKeys) - 1 <= me.pos);
      const bool beyond = BIAS && !behind && __all_sync(0xffffffffu, !live || max(me.lo, kb) >= me.pos);
      const float toward = beyond ? -slope : slope;
      auto exact_unit = [&](float v) -> float {
        return CAP == kCapFine ? tanh_fine_from_2l2e(v * fac) : CAP ? tanh_from_2l2e(v * fac) : v;
      };
      auto bias = [&](int c) -> float { return -slope * fabsf(ahead - (float)c); };

      // Raises m_ref to kLift below the row's maximum over the block, with O and l scaled down to it.
      auto raise = [&]() {
        float mx = -INFINITY;
#pragma unroll 1
        for (int c0 = 0; c0 < kKeys; c0 += 16) {
          uint32_t v[16];
          tm_ld16(ts + c0, v);
          tm_wait_ld(v);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x = __uint_as_float(v[c]);
            if (BIAS) x = fmaf(exact_unit(x), f, bias(c0 + c));
            if (!seen(c0 + c)) x = -INFINITY;
            mx = fmaxf(mx, x);
          }
        }
        // without a bias the score grows with the raw sum; rounded up, so that no fused u * f - org is positive
        if (!BIAS && mx != -INFINITY) mx = __fmul_ru(exact_unit(mx), f);
        mx = __fadd_ru(mx, -(float)kLift);  // the origin, rounded up so that P is 2^kLift at most
        const bool grow = mx > m_ref;
        const bool scale = m_ref != -INFINITY && grow;  // from -infinity: O and l are zero
        const float down = scale ? ex2(m_ref - mx) : 1.f;
        if (grow) m_ref = mx;
        if (!__any_sync(0xffffffffu, scale)) return;
        l *= down;
        if (!s_ready(j + 1)) *abort_flag = 1;  // P V of the block before is done, and the next waits for this P
        tc_after();
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 16) {
          uint32_t v[16];
          tm_ld16(to + c0, v);
          tm_wait_ld(v);
#pragma unroll
          for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * down);
          tm_st16(to + c0, v);
        }
      };

      // P = 2^(score - org) as f16 and its sum.  MODE kExact: after raise(); else against an m_ref that the
      // block may exceed and with a polynomial for the cap: `top` (the largest P) and `reach` (the largest
      // square of tanh's argument) tell whether that was right.
      uint32_t o[kKeys / 2];
      float sum = 0.f, reach = 0.f;
      __half2 top = __floats2half2_rn(0.f, 0.f);
      auto exponentials = [&](auto masked, auto mode) {
        constexpr bool MASK = decltype(masked)::value, EXACT = decltype(mode)::value == kExact;
        constexpr bool LOW = decltype(mode)::value == kLow;
        const float org = m_ref == -INFINITY ? 0.f : m_ref;
        const f32x2 org2 = pair2(-org, -org), f2 = pair2(f, f), step2 = pair2(2.f * toward, 2.f * toward);
        const float z1 = fac * 0.34657359027997264f;  // fac carries 2 log2(e)
        f32x2 sum2 = pair2(0.f, 0.f);
        auto columns = [&](const uint32_t(&v)[32], int c0) {
          f32x2 b2 = org2;
          if (BIAS && !EXACT) {
            const float b1 = fmaf(toward, (float)c0 - ahead, -org);
            b2 = pair2(b1, b1 + toward);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            f32x2 x2;
            if constexpr (EXACT || (CAP && BIAS)) {
              const f32x2 u2 = pair2(exact_unit(__uint_as_float(v[c])), exact_unit(__uint_as_float(v[c + 1])));
              if constexpr (BIAS)
                x2 = add2(fma2(u2, f2, pair2(bias(c0 + c), bias(c0 + c + 1))), org2);
              else
                x2 = fma2(u2, f2, org2);
            } else if constexpr (BIAS) {
              x2 = fma2(bits2(v[c], v[c + 1]), f2, b2);
              b2 = add2(b2, step2);
            } else if constexpr (CAP) {
              const f32x2 z = mul2(bits2(v[c], v[c + 1]), pair2(z1, z1)), w2 = mul2(z, z);
              constexpr int N = LOW ? 3 : kTanhTerms;
              f32x2 h = fma2(w2, tanh2<LOW>(N - 1), tanh2<LOW>(N - 2));
#pragma unroll
              for (int k = N - 3; k >= 0; --k) h = fma2(w2, h, tanh2<LOW>(k));
              x2 = fma2(mul2(z, f2), h, org2);
              const float2 ww = split2(w2);
              reach = fmaxf(reach, fmaxf(ww.x, ww.y));
            } else {
              x2 = fma2(bits2(v[c], v[c + 1]), f2, org2);
            }
            float2 p = split2(x2);
            p.x = ex2(p.x);
            p.y = ex2(p.y);
            if (MASK) {
              p.x = seen(c0 + c) ? p.x : 0.f;
              p.y = seen(c0 + c + 1) ? p.y : 0.f;
            }
            sum2 = add2(sum2, pair2(p.x, p.y));
            const __half2 h = __floats2half2_rn(p.x, p.y);
            o[(c0 + c) / 2] = *reinterpret_cast<const uint32_t*>(&h);
            if (!EXACT) top = __hmax2(top, h);
          }
        };
        uint32_t va[32], vb[32];
        tm_ld32(ts, va);
        tm_ld32(ts + 32, vb);
        tm_wait_ld(va);
        tm_wait_ld(vb);
        columns(va, 0);
        columns(vb, 32);
        const float2 s2 = split2(sum2);
        sum = s2.x + s2.y;
      };
      // The first block that a row sees sets its m_ref.  Later ones rarely exceed it by 2^kSlack: they are
      // tried against the old one, and done again where some row of the warp does.
      bool again = (BIAS && !CAP && !behind && !beyond) ||
                   __any_sync(0xffffffffu, live && m_ref == -INFINITY && me.lo < min(me.hi, kb + kKeys) && me.hi > kb);
      if (!again) {
        if (edge)
          exponentials(std::true_type(), std::integral_constant<int, kHigh>());
        else if (CAP && !BIAS && low)
          exponentials(std::false_type(), std::integral_constant<int, kLow>());
        else
          exponentials(std::false_type(), std::integral_constant<int, kHigh>());
        const __half2 most = __float2half2_rn((float)(1 << (kLift + kSlack)));
        const float range = low && !edge ? kTanhLowRange2 : kTanhRange2;
        if (CAP && __any_sync(0xffffffffu, live && reach > kTanhLowRange2)) low = false;
        again = __any_sync(0xffffffffu, live && (!__hble2(top, most) || reach > range));
      }
      if (again) {
        raise();
        exponentials(std::true_type(), std::integral_constant<int, kExact>());
      }
      l += sum;
      tm_st16(ts, o);
      tm_st16(ts + 16, o + 16);
      tm_wait_st();
      if (kb < f_lo || kb + kKeys > f_hi) {  // as the loading warps decide it
        // NaN values of keys that some rows do not see were taken out of V: put them into the rows that do
        const int st = j % kDepth;
        if (!mbar_wait(&sh.v_full[st], (uint32_t)(j / kDepth) & 1u, a.err, abort_flag)) *abort_flag = 1;
        for (int q = 0; q < kKeys / 32; ++q) {
          for (uint32_t bits = *reinterpret_cast<volatile uint32_t*>(&sh.nan[st][q]); bits; bits &= bits - 1) {
            const int key = kb + 32 * q + __ffs(bits) - 1;
            if (!live || key < me.lo || key >= me.hi) continue;
            const int page = a.page_table[(size_t)b * a.table_ld + page_of(a, key)];
            const uint8_t* vr = a.v_cache + (((size_t)page * a.P + key - page_of(a, key) * a.P) * a.Hkv + head) * D;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
              for (int c = 0; c < 32; ++c) nan_d[i] |= (uint32_t)((vr[32 * i + c] & 0x7f) == 0x7f) << c;
          }
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[w][j & 1]);
    }
    // ---- output ----
    const bool have = nb > 0 && on && __all_sync(0xffffffffu, ok && s_ready(nb + 1));
    tc_after();
    const float inv = l == 0.f ? 0.f : __fdividef(a.v_scale[head], l);
    // The warp's rows are turned in its share of the query tile (2 D bytes a row) and leave as whole rows: all of a bf16
    // row at once, an fp32 one in halves.  That share holds other warps' queries, too: the products that `have` tells of
    // waited for every warp's, and are done with them.  Without them (no keys: the other warps' copies may still be
    // landing) zeros leave straight from registers.
    uint8_t* turn = smem + C::Q0 + w * C::QTILE + (warp & 3) * 32 * 2 * D;
    const size_t part = part_of();
    const bool folded = FOLD && nb > kFold && live;
    const float was = folded ? pl.ml[part * 2] : -INFINITY, down = was == -INFINITY ? 0.f : ex2(was - m_ref);
    if (pl.splits > 1 && live) *reinterpret_cast<float2*>(pl.ml + part * 2) = make_float2(m_ref, l);
    auto columns = [&](int c0, uint32_t (&v)[32]) {
      tm_ld32(to + c0, v);
      tm_wait_ld(v);
      if (FOLD && folded) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(fmaf(pl.acc[part * D + c0 + c], down, __uint_as_float(v[c])));
      }
      const uint32_t nan = nan_d[c0 / 32];
      if (nan) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if ((nan >> c) & 1u) v[c] = 0x7fffffffu;
      }
    };
    auto put = [&](int chunk, uint4 x) { *reinterpret_cast<uint4*>(turn + lane * 2 * D + (chunk ^ (lane % QC)) * 16) = x; };
    auto leave = [&](uint8_t* base, long long at) {  // `at`: bytes to this lane's row from base, -1: none
      __syncwarp();
#pragma unroll 4
      for (int i = 0; i < QN; ++i) {
        const int row = i * QR + qr;
        const long long to_row = at_row(at, row);
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (have) x = *reinterpret_cast<const uint4*>(turn + row * 2 * D + (qc ^ (row % QC)) * 16);
        if (to_row >= 0) *reinterpret_cast<uint4*>(base + to_row + qc * 16) = x;
      }
      __syncwarp();
    };
    if (pl.splits > 1) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c0 = 0; c0 < D / 2; c0 += 32) {
          if (!have) break;
          uint32_t v[32];
          columns(half * (D / 2) + c0, v);
#pragma unroll
          for (int c = 0; c < 32; c += 4) put((c0 + c) / 4, make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]));
        }
        leave(reinterpret_cast<uint8_t*>(pl.acc) + half * 2 * D, live ? (long long)(part * D * 4) : -1);
      }
    } else {
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        if (!have) break;
        uint32_t v[32];
        columns(c0, v);
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = pack_bf16x2(__uint_as_float(v[c + 2 * k]) * inv, __uint_as_float(v[c + 2 * k + 1]) * inv);
          put((c0 + c) / 8, make_uint4(o[0], o[1], o[2], o[3]));
        }
      }
      leave(reinterpret_cast<uint8_t*>(a.out), live ? ((long long)tok * a.ldo + (long long)hq * D) * 2 : -1);
    }
  } else if (warp < kIssueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    // ------------------------------------------------------------------ keys and values
    const int lt = threadIdx.x - kSoftmaxThreads;  // 0 .. 127
    const Plan keys = plan();
    const int nb = keys.nb;
    const int f_lo = sh.full_lo, f_hi = sh.full_hi;
    // Threads 0 .. 63: the cache row (of D bytes) of the block's key lt; kNoRow: reads zeros.
    constexpr uint32_t kNoRow = 0xffffffffu;
    uint32_t* offs = reinterpret_cast<uint32_t*>(smem + C::OFF0);
    auto offset = [&](int j) {
      if (lt >= kKeys || j >= nb) return;
      const int key = keys.key0 + block_at(keys, j) + lt;
      uint32_t off = kNoRow;
      if (key < keys.k_hi) {
        const int page = a.page_table[(size_t)b * a.table_ld + page_of(a, key)];
        if (page >= 0 && page < a.num_pages)
          off = (uint32_t)(((long long)page * a.P + key - page_of(a, key) * a.P) * a.Hkv + head);
        else
          atomicOr(a.err, OKC_DEVERR_PAGE);
      }
      offs[(j & 1) * kKeys + lt] = off;
    };
    // the loading warps' barrier: whether any of them gave up (they leave together)
    auto sync_any = [&](bool bad) {
      uint32_t any;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n"
          " selp.b32 %0, 1, 0, q;\n}\n"
          : "=r"(any)
          : "r"((uint32_t)bad)
          : "memory");
      return any != 0;
    };
    // A thread's 16-byte chunks: chunk `ch` of every KSTEP-th key from `kf` on.  Eight lanes take four
    // chunks of two neighbouring keys, which the swizzle puts into different banks.
    constexpr int NCH = D / 16, PER = kKeys * NCH / kLoadThreads, KSTEP = kKeys / PER;
    const int ch = NCH == 8 ? (lt & 3) + 4 * ((lt >> 3) & 1) : lt & 3;
    const int kf = 2 * (lt / (2 * NCH)) + ((lt >> 2) & 1);
    static_assert(KSTEP % 8 == 0, "a thread's keys share a swizzle");
    const int at0 = (ch / 4) * C::SUB + kf * 128 + (((2 * (ch % 4)) ^ (kf & 7)) * 16);
    const int at1 = (ch / 4) * C::SUB + kf * 128 + (((2 * (ch % 4) + 1) ^ (kf & 7)) * 16);
    auto store = [&](uint8_t* base, const uint4 (&r)[PER]) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t x[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = e4m3x2_h2(x[k] & 0xffffu);
          o[2 * k + 1] = e4m3x2_h2(x[k] >> 16);
        }
        *reinterpret_cast<uint4*>(base + at0 + i * KSTEP * 128) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(base + at1 + i * KSTEP * 128) = make_uint4(o[4], o[5], o[6], o[7]);
      }
    };
    // a block's K and V chunks of this thread, in flight while the block before is converted
    struct Chunks {
      uint4 k[PER], v[PER];
    };
    auto fetch = [&](int j, Chunks& c) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t row = offs[(j & 1) * kKeys + kf + i * KSTEP];
        const size_t at = (size_t)row * D + ch * 16;
        c.k[i] = c.v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row != kNoRow) {
          c.k[i] = *reinterpret_cast<const uint4*>(a.k_cache + at);
          c.v[i] = *reinterpret_cast<const uint4*>(a.v_cache + at);
        }
      }
    };
    bool ok = true;
    auto block = [&](int j, Chunks& now, Chunks& next) {  // false: given up
      // the offsets of block j + 1 are there, and those of block j are read
      if (sync_any(!ok)) return false;
      if (j + 1 < nb) fetch(j + 1, next);
      offset(j + 2);
      const int st = j % kDepth, kb = keys.key0 + block_at(keys, j);
      ok = mbar_wait(&sh.kv_empty[st], ((uint32_t)(j / kDepth) & 1u) ^ 1u, a.err, abort_flag);
      store(smem + C::K0 + st * C::BLOCK, now.k);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.k_full[st]);
      if (kb < f_lo || kb + kKeys > f_hi) {
        if (lt < kKeys / 32) sh.nan[st][lt] = 0;
        sync_any(false);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int key = kf + i * KSTEP;
          uint32_t x[4] = {now.v[i].x, now.v[i].y, now.v[i].z, now.v[i].w}, bad = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t nan = ((x[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            bad |= nan;
            x[k] &= ~((nan >> 7) * 0xffu);
          }
          if (bad) atomicOr(&sh.nan[st][key >> 5], 1u << (key & 31));
          now.v[i] = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      store(smem + C::V0 + st * C::BLOCK, now.v);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.v_full[st]);
      return true;
    };
    offset(0);
    offset(1);
    sync_any(false);
    Chunks c0, c1;
    if (nb > 0) fetch(0, c0);
    for (int j = 0; j < nb; j += 2) {
      if (!block(j, c0, c1) || (j + 1 < nb && !block(j + 1, c1, c0))) {
        *abort_flag = 1;
        break;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    // ------------------------------------------------------------------ MMA issue, a warp per tile
    const int w = warp - kIssueWarp;
    if (w < 2 && lane == 0) {
      const int nb = plan().nb;
      const bool two = b >= 0 && (a.cu_q[b + 1] - a.cu_q[b]) * a.G - sh.tile * kPair > kTile;
      const uint32_t t_s = sh.tmem + w * kTile, t_o = sh.tmem + 2 * kTile + w * D;
      const uint32_t id_s = umma_idesc_f16(kKeys, false), id_o = umma_idesc_f16(D, true);
      const uint64_t qa = umma_desc_sw128(smem_u32(smem + C::Q0 + w * C::QTILE));
      auto scores = [&](int j) {  // S of block j
        const uint64_t ka = umma_desc_sw128(smem_u32(smem + C::K0 + j % kDepth * C::BLOCK));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(t_s + (j & 1) * kKeys, qa + (((k / 4) * C::QSUB + (k % 4) * 32) >> 4),
                  ka + (((k / 4) * C::SUB + (k % 4) * 32) >> 4), id_s, k != 0);
      };
      bool ok = true;
      if (nb > 0 && (w == 0 || two)) {
        ok = mbar_wait(&sh.q_full, 0, a.err, abort_flag);
        for (int j = 0; ok && j < 2 && j < nb; ++j) {
          ok = mbar_wait(&sh.k_full[j], 0, a.err, abort_flag);
          if (!ok) break;
          tc_after();
          scores(j);
          umma_commit(&sh.s_full[w][j]);
        }
        for (int j = 0; ok && j < nb; ++j) {
          const int st = j % kDepth;
          ok = mbar_wait(&sh.v_full[st], (uint32_t)(j / kDepth) & 1u, a.err, abort_flag) &&
               mbar_wait(&sh.p_full[w][j & 1], (uint32_t)(j >> 1) & 1u, a.err, abort_flag);
          if (!ok) break;
          tc_after();
          const uint64_t va = umma_desc_mn(smem_u32(smem + C::V0 + st * C::BLOCK), C::SUB);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            umma_ts(t_o, t_s + (j & 1) * kKeys + 8 * k, va + k * (2048 >> 4), id_o, ((FOLD ? j % kFold : j) | k) != 0);
          umma_commit(&sh.kv_empty[st]);
          if (!two) umma_commit(&sh.kv_empty[st]);  // (the barrier counts both tiles)
          if (j + 2 < nb) {
            ok = mbar_wait(&sh.k_full[(j + 2) % kDepth], (uint32_t)((j + 2) / kDepth) & 1u, a.err, abort_flag);
            if (!ok) break;
            tc_after();
            scores(j + 2);  // over P: the tensor core takes a thread's MMAs in order, and the ones above read it
          }
          umma_commit(&sh.s_full[w][j & 1]);  // behind the last block: that P V of block j is done
        }
        if (!ok) *abort_flag = 1;
        umma_commit(&sh.drain[w]);  // no MMA may be in flight when the tensor memory is released
        mbar_wait(&sh.drain[w], 0, a.err);
      }
    }
  }

  tc_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem));
  }
}

// Joins the key splits of a row (token, query head), one warp a row.
template <int D>
__global__ void __launch_bounds__(256) attn_chunk_tc_merge_kernel(ChunkArgs a, TcPlanA pl) {
  constexpr int E = D / 32;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), all = (long long)a.T * a.Hq;
  if (item >= all) return;
  const int t = (int)(item / a.Hq), hq = (int)(item - (long long)t * a.Hq);
  const int b = find_request(a.cu_q, a.B, t);
  if (b < 0 || (a.cu_q[b + 1] - a.cu_q[b]) * a.G <= pl.above) return;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < pl.splits) ml = *reinterpret_cast<const float2*>(pl.ml + ((size_t)lane * all + item) * 2);
  const float M = warp_max(ml.x), org = M == -INFINITY ? 0.f : M;
  const float w = ex2(ml.x - org), L = warp_sum(w * ml.y);
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s = 0; s < pl.splits; ++s) {
    const float ws = __shfl_sync(0xffffffffu, w, s);
    if (__shfl_sync(0xffffffffu, ml.y, s) == 0.f) continue;  // no key of this segment is the row's
    const float* src = pl.acc + ((size_t)s * all + item) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + e);
      o[e] += ws * v.x;
      o[e + 1] += ws * v.y;
    }
  }
  const float inv = L == 0.f ? 0.f : __fdividef(a.v_scale[hq / a.G], L);
  __nv_bfloat16* dst = a.out + (size_t)t * a.ldo + (size_t)hq * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(o[e] * inv, o[e + 1] * inv);
}

// Tile pairs of the requests above kSplitRows, at most.
long long tc_tiles(int T, int B, int G) {
  const long long rows = (long long)T * G, big = rows / (kSplitRows + 1);
  return rows / kPair + (big < B ? big : B);
}

int tc_splits(int T, int B, int Hq, int Hkv, long long max_keys) {
  const long long ctas = tc_tiles(T, B, Hq / Hkv) * Hkv;
  if (ctas <= 0) return 1;
  long long s = okc_host::num_sms() / ctas;
  const long long most = max_keys / 512;  // at least four key blocks a split
  if (s > most) s = most;
  return s < 1 ? 1 : s > 32 ? 32 : (int)s;
}

template <int D, int CAP, bool BIAS, bool FOLD>
int launch_tc_as(const ChunkArgs& a, const TcPlanA& pl, cudaStream_t stream) {
  using C = TcCfgA<D>;
  static okc_host::PerDevice configured;
  if (int st = configured.smem(attn_chunk_tc_kernel<D, CAP, BIAS, FOLD>, C::SMEM, kLaunchRegs)) return st;
  const long long tiles = tc_tiles(a.T, a.B, a.G);
  if (tiles > 65535) return OKC_ERR_TOO_LARGE;
  if (int st = okc_host::launch_k(attn_chunk_tc_kernel<D, CAP, BIAS, FOLD>, dim3(a.Hkv * pl.splits, (unsigned)tiles),
                                  dim3(kTcThreads), C::SMEM, stream, dim3(1), a, pl))
    return st;
  if (pl.splits == 1) return OKC_OK;
  return okc_host::launch_k(attn_chunk_tc_merge_kernel<D>, dim3((unsigned)(((long long)a.T * a.Hq + 7) / 8)), dim3(256),
                            0, stream, dim3(1), a, pl);
}

// The variant with sums set aside where the table is wide enough for it: within one kernel it cost 1 to 4% (4096 tokens
// behind 4096 at heads of 64, capped, 902 and 937 us).
template <int D, int CAP, bool BIAS>
int launch_tc(const ChunkArgs& a, const TcPlanA& pl, cudaStream_t stream) {
  return a.max_keys / pl.splits > kFold * kKeys ? launch_tc_as<D, CAP, BIAS, true>(a, pl, stream)
                                                : launch_tc_as<D, CAP, BIAS, false>(a, pl, stream);
}

template <int CAP>
int launch_tc_cap(const ChunkArgs& a, const TcPlanA& pl, cudaStream_t stream) {
  const bool bias = a.slopes != nullptr;
  if (a.D == 64) return bias ? launch_tc<64, CAP, true>(a, pl, stream) : launch_tc<64, CAP, false>(a, pl, stream);
  return bias ? launch_tc<128, CAP, true>(a, pl, stream) : launch_tc<128, CAP, false>(a, pl, stream);
}

}  // namespace

size_t attn_chunk_tc_ws_bytes(int T, int B, int Hq, int Hkv, int D) {
  const int s = tc_splits(T, B, Hq, Hkv, 1ll << 31);
  if (s == 1) return 0;
  const size_t rows = (size_t)s * T * Hq;
  return up(rows * D * 4) + up(rows * 8);
}

int launch_attn_chunk_tc(const ChunkArgs& a, int above, void* ws, float* sums, float* origins, cudaStream_t stream) {
  TcPlanA pl;
  pl.above = above;
  pl.splits = tc_splits(a.T, a.B, a.Hq, a.Hkv, a.max_keys);
  pl.acc = sums;
  pl.ml = origins;
  if (pl.splits > 1) {
    pl.acc = reinterpret_cast<float*>(ws);
    pl.ml = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(ws) + up((size_t)pl.splits * a.T * a.Hq * a.D * 4));
  }
  switch (cap_form(a.softcap)) {
    case kCapFine: return launch_tc_cap<kCapFine>(a, pl, stream);
    case kCapPlain: return launch_tc_cap<kCapPlain>(a, pl, stream);
    default: return launch_tc_cap<kCapNone>(a, pl, stream);
  }
}

}  // namespace okc
