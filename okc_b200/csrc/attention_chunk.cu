// Attention of ragged chunks of new tokens over the paged e4m3 cache, for chunks of few rows
// (decode tokens, verify blocks): split over the keys, joined by a log-sum-exp merge.
//
// Query row (token t, head h) of request b, at position p, sees the positions [lo, hi) with
//   lo = max(0, doc_start[t], p + 1 - window),   hi = min(seq_len, max(p + 1, prefix_len)),
// so every mask here (causal, sliding window, packed documents, a prefix that all tokens see) is one
// interval per row.  Its scores are
//   s_j = cap * tanh(q.k_j * sm_scale / cap) - slope[h] * |p - j|,   o = sum_j softmax(s)_j v_j,
// and a row that sees nothing is zero.
//
// Bound by the cache read (2 D bytes a key and KV head), nearly: 128 requests of 64 / 8 heads of 128 behind 1050 to
// 8192 positions take 218 us (5.7 TB/s; capped, the loads alone 198), uncapped 214; 4 tokens each (32 rows: two
// tiles, the keys converted for each) 417.  One token behind 81919 positions, 16 / 2 heads of 64: 21.7 us, of which
// the two launches and the chains to the first key and through the merge are 9.  The rows of one KV head's query group
// (token-major, G heads a token) fill the 16 rows of mma.sync tiles, or, where no request has more than 8,
// their 8 columns with keys and outputs as the rows: half the MMAs and half the accumulators.  e4m3 keys and
// values are exact in f16, the query too once its row is scaled by a power of two, and P is rounded to f16 (2^-11; the
// sum that divides takes it unrounded).
//  * units of 32 keys x (8 / nh) subgroups of a (request, row tile, nh heads) are numbered in order
//    and split evenly over a persistent grid (ragged contexts stay balanced); the nh heads of a
//    key lie side by side in the cache, so the block's warps read whole token rows together;
//  * a warp owns a ring of key blocks in shared memory that it fills with cp.async and reads as MMA
//    fragments: no block barrier in the loop.  Page ids are fetched a block ahead.  Positions outside the
//    tile's interval, or on a page outside the pool, are zero-filled, never read;
//  * a K fragment's k slots and a V fragment's columns are permuted so that each lane's share is
//    whole 16-byte chunks (a sum over k does not depend on its order).
// Partial sums go to the workspace as fp32 with their running maximum and sum; segments are joined
// in block order, so results repeat bit for bit.  mma.sync truncates as it adds to the output, 1.4e-7 of it for 16 keys of a
// warp: 6e-5 for one request behind 2^20 positions, 0.5% at most, where the keys fill the whole card (594000 of them a
// warp).  Summed outside of the instruction that goes, and the kernel takes 1 to 4% longer.
#include "chunk_common.cuh"

#include <type_traits>

namespace okc {

namespace {

constexpr int kStep = 32;      // keys of a warp's step: a lane looks one up
constexpr int kWarps = 8;
// log2 of the largest P: f16 keeps P down to 2^-25, so that keys are lost from the sum only 2^-(25 + kLift) below the
// row's largest (from an origin at the largest, a million keys at e^-18 of it lost 1.5% of the weight).
constexpr int kLift = 14;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

template <int D>
struct ChunkCfg {
  static constexpr int STAGE = 2 * kStep * D;  // K and V of a step
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGE * STAGES;
  static constexpr int SMEM = RING * kWarps;
};

struct SplitPlan {
  int nh, nsub, hg;   // heads side by side in a block, key subgroups, head groups
  int step_keys;      // keys of a unit
  int rows;           // rows of a tile: 16, or 8 where no request has more
  int ctas, few;      // CTAs of the grid, and those that share little work (shared_by)
  int* pre_u;         // [B + 1] units before a request
  int* pre_t;         // [B + 1] row tiles (times head groups) before a request
  float* ml;          // [slot][nh][16][2]
  float* acc;         // [slot][nh][16][D]
  int most_rows;      // requests of more rows are served by the tensor-memory kernel
  int merge_tokens;   // > 0: requests have at most this many tokens here; 0: rows are looked up
};

__device__ __forceinline__ void unit_split(int U, int C, int c, int& u0, int& u1) {
  const int q = U / C, r = U % C;
  u0 = c * q + min(c, r);
  u1 = u0 + q + (c < r ? 1 : 0);
}
__device__ __forceinline__ int unit_owner(int U, int C, int u) {
  const int q = U / C, r = U % C, big = r * (q + 1);
  return u < big ? u / (q + 1) : r + (u - big) / q;
}

// How many of the CTAs share U units.  A second one an SM (heads of 64) hides the first's latency where each has some
// units, and costs the merge twice the segments where not: 128 requests 131 us against 208, 16 requests 31 and 40; one token
// behind 81919 (4 units an SM) 24.2 and 21.6, behind 2000 11.1 and 10.6.
__device__ __forceinline__ int shared_by(const SplitPlan& pl, int U) { return U > 6 * pl.few ? pl.ctas : pl.few; }

// Units and row tiles before each request, by one warp.
__device__ __forceinline__ void split_prefix(const ChunkArgs& a, const SplitPlan& pl, int* pre_u, int* pre_t) {
  const int lane = threadIdx.x & 31;
  int cu = 0, ct = 0;
  for (int base = 0; base < a.B; base += 32) {
    const int b = base + lane;
    int u = 0, t = 0;
    if (b < a.B) {
      const Req r = request(a, b);
      const int rows = r.n * a.G;
      if (r.len > a.max_keys && blockIdx.x == 0) atomicOr(a.err, OKC_DEVERR_PAGE);
      if (rows <= pl.most_rows) {
        t = (rows + pl.rows - 1) / pl.rows * pl.hg;
        u = t * ((max(0, r.hi - r.lo) + pl.step_keys - 1) / pl.step_keys);
      }
    }
    int su = u, st = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, su, o), y = __shfl_up_sync(0xffffffffu, st, o);
      if (lane >= o) {
        su += x;
        st += y;
      }
    }
    if (b < a.B) {
      pre_u[b] = cu + su - u;
      pre_t[b] = ct + st - t;
    }
    cu += __shfl_sync(0xffffffffu, su, 31);
    ct += __shfl_sync(0xffffffffu, st, 31);
  }
  if (lane == 0) {
    pre_u[a.B] = cu;
    pre_t[a.B] = ct;
  }
}

template <int D, int CAP, int R>
__global__ void __launch_bounds__(32 * kWarps, D == 64 ? 2 : 1) attn_chunk_split_kernel(ChunkArgs a, SplitPlan pl) {
  using C = ChunkCfg<D>;
  constexpr int KS = D / 16;   // k16 steps of QK
  constexpr int ND = R == 16 ? D / 8 : D / 16;  // PV blocks: 8 columns, or 16 rows, of the output
  constexpr int GAP = R == 16 ? 8 : 1;          // a lane's two rows in the softmax: first and first + GAP
  constexpr int NCH = D / 16;  // 16-byte chunks of a key
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre_u = reinterpret_cast<int*>(smem + C::SMEM);
  int* pre_t = pre_u + a.B + 1;

  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  if (warp == 0) split_prefix(a, pl, pre_u, pre_t);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x) {
      pl.pre_u[i] = pre_u[i];
      pl.pre_t[i] = pre_t[i];
    }
  const int share = shared_by(pl, pre_u[a.B]);
  int u0 = 0, u1 = 0;
  if ((int)blockIdx.x < share) unit_split(pre_u[a.B], share, blockIdx.x, u0, u1);
  const int hw = warp % pl.nh, sub = warp / pl.nh;
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_s = smem_u32(ring);

  while (u0 < u1) {
    int b, hi_b = a.B - 1;
    for (b = 0; b < hi_b;) {  // largest b with pre_u[b] <= u0 (requests without units share a prefix)
      const int mid = (b + hi_b + 1) >> 1;
      if (pre_u[mid] <= u0) b = mid; else hi_b = mid - 1;
    }
    const Req rq = request(a, b);
    const int nc = (max(0, rq.hi - rq.lo) + pl.step_keys - 1) / pl.step_keys;
    const int in_b = u0 - pre_u[b], tile = in_b / nc, c0 = in_b - tile * nc;
    const int c1 = min(nc, c0 + (u1 - u0));
    const int rt = tile / pl.hg, head = (tile - rt * pl.hg) * pl.nh + hw;
    const int slot = blockIdx.x + pre_t[b] + tile;
    u0 += c1 - c0;

    // ---- the lane's two rows ----
    const int rows = rq.n * a.G, r0 = rt * R;
    const int first = R == 16 ? g : 2 * c;
    const int row0 = a.cu_q[b];
    int lo[2], hi[2], pos[2], tok[2], hq[2];
    bool live[2];
    const bool two = R == 8 || rows - r0 > 8;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + first + GAP * e;
      live[e] = r < rows;
      tok[e] = live[e] ? r / a.G : 0;
      hq[e] = head * a.G + (live[e] ? r - tok[e] * a.G : 0);
      pos[e] = lo[e] = hi[e] = 0;
      if (live[e]) {
        const RowSpan sp = row_span(a, rq, row0, tok[e]);
        pos[e] = sp.pos;
        lo[e] = sp.lo;
        hi[e] = sp.hi;
      }
    }
    // keys that every live row sees need no mask; keys outside [t_lo, t_hi) are not read
    int full_lo = max(live[0] ? lo[0] : 0, live[1] ? lo[1] : 0);
    int full_hi = min(live[0] ? hi[0] : 0x7fffffff, live[1] ? hi[1] : 0x7fffffff);
    const bool sees[2] = {live[0] && lo[0] < hi[0], live[1] && lo[1] < hi[1]};
    int t_lo = min(sees[0] ? lo[0] : 0x7fffffff, sees[1] ? lo[1] : 0x7fffffff);
    int t_hi = max(sees[0] ? hi[0] : 0, sees[1] ? hi[1] : 0);
    full_lo = __reduce_max_sync(0xffffffffu, full_lo);
    full_hi = __reduce_min_sync(0xffffffffu, full_hi);
    t_lo = __reduce_min_sync(0xffffffffu, t_lo);
    t_hi = __reduce_max_sync(0xffffffffu, t_hi);

    // ---- the warp's steps: keys [k0 + s * step_keys, + 32), those that meet [t_lo, t_hi) ----
    const int k0 = rq.lo + c0 * pl.step_keys + sub * kStep;
    int s_lo = 0, s_hi = c1 - c0;
    if (t_lo >= t_hi) {
      s_hi = 0;  // no row of the tile sees a key
    } else {
      if (t_lo > k0 + kStep - 1) s_lo = (t_lo - (k0 + kStep - 1) + pl.step_keys - 1) / pl.step_keys;
      if (t_hi < k0 + (s_hi - 1) * pl.step_keys + 1) s_hi = t_hi <= k0 ? 0 : (t_hi - k0 + pl.step_keys - 1) / pl.step_keys;
    }
    const int32_t* trow = a.page_table + (size_t)b * a.table_ld;
    auto fetch_page = [&](int s) -> int {  // of this lane's key of step s; what it is, issue() checks
      const int key = k0 + s * pl.step_keys + lane;
      return s < s_hi && key >= t_lo && key < t_hi ? trow[page_of(a, key)] : -1;
    };
    auto issue = [&](int s, int page) {
      if (s < s_hi) {
        const int key = k0 + s * pl.step_keys + lane;
        const bool on = page >= 0 && page < a.num_pages;
        if (!on && key >= t_lo && key < t_hi) atomicOr(a.err, OKC_DEVERR_PAGE);
        // rows of D bytes, below 2^32
        const uint32_t row = on ? ((uint32_t)page * a.P + key - page_of(a, key) * a.P) * a.Hkv + head : 0u;
        const uint32_t mask = __ballot_sync(0xffffffffu, on);
        constexpr int KI = 32 / NCH;  // keys of an instruction
        const int kl = lane / NCH, ch = lane % NCH;
        const uint32_t st = ring_s + (uint32_t)((s - s_lo) % C::STAGES) * C::STAGE + kl * D;
        const uint32_t kd = st + (D == 128 ? ch ^ (4 * (kl & 1)) : ch) * 16, vd = st + kStep * D;
        const uint8_t* kp = a.k_cache + ch * 16;
        const uint8_t* vp = a.v_cache + ch * 16;
        auto copy = [&](auto whole) {
#pragma unroll
          for (int i = 0; i < kStep / KI; ++i) {
            const size_t src = (size_t)__shfl_sync(0xffffffffu, row, i * KI + kl) * D;
            const bool in = decltype(whole)::value || (mask >> (i * KI + kl) & 1u);
            cp16(kd + i * KI * D, kp + src, in);
            cp16(vd + i * KI * D + (D == 128 ? ch ^ (2 * (i & 3)) : ch) * 16, vp + src, in);
          }
        };
        if (mask == 0xffffffffu) copy(std::true_type{});
        else copy(std::false_type{});
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    int page = fetch_page(s_lo);
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) {
      const int next = fetch_page(s_lo + i + 1);
      issue(s_lo + i, page);
      page = next;
    }
    // ---- the query, while the first keys are on their way ----
    // R = 16: rows g and g + 8 as the A operand.  R = 8: row g as the B operand, whose scale the lanes that
    // have the row in the softmax fetch from it.
    float slope[2], fac[2];
    uint32_t qf[KS][R == 16 ? 4 : 2];
    float up[2];  // what undoes the row's scale
#pragma unroll
    for (int e = 0; e < R / 8; ++e) {
      const int r = r0 + g + 8 * e, t = r / a.G;
      uint2 qv[KS];
#pragma unroll
      for (int k = 0; k < KS; ++k) qv[k] = make_uint2(0u, 0u);
      if (r < rows) {
        const __nv_bfloat16* qp = a.q + (size_t)(row0 + t) * a.ldq + (size_t)(head * a.G + r - t * a.G) * D;
#pragma unroll
        for (int k = 0; k < KS; ++k)  // the four elements of step k's slots
          qv[k] = *reinterpret_cast<const uint2*>(qp + 64 * (k >> 2) + 16 * c + 4 * (k & 3));
      }
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        top = max(max(top, max(qv[k].x & 0x7fffu, (qv[k].x >> 16) & 0x7fffu)),
                  max(qv[k].y & 0x7fffu, (qv[k].y >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int sh = f16_shift(top);
      const float down = pow2(-sh);
      up[e] = pow2(sh);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[k][e] = h2(bf16_lo(qv[k].x) * down, bf16_hi(qv[k].x) * down);
        qf[k][R / 8 + e] = h2(bf16_lo(qv[k].y) * down, bf16_hi(qv[k].y) * down);
      }
    }
    if (R == 8) {
      const float mine = up[0];
      up[0] = __shfl_sync(0xffffffffu, mine, 8 * c);
      up[1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      slope[e] = live[e] && a.slopes ? a.slopes[hq[e]] * 1.4426950408889634f : 0.f;
      // without a cap: log2 units; with one: the argument of tanh times 2 log2(e)
      fac[e] = a.k_scale[head] * a.sm_scale * (CAP ? 2.f / a.softcap : 1.f) * 1.4426950408889634f * up[e];
    }
    const float cap2 = CAP ? a.softcap * 1.4426950408889634f : 0.f;

    float o_acc[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n) o_acc[n][0] = o_acc[n][1] = o_acc[n][2] = o_acc[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int s = s_lo; s < s_hi; ++s) {
      const int next = fetch_page(s + C::STAGES);
      __syncwarp();  // every lane has read the stage that is filled now
      issue(s + C::STAGES - 1, page);
      page = next;
      asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
      __syncwarp();
      const uint8_t* ks = ring + ((s - s_lo) % C::STAGES) * C::STAGE;
      const uint8_t* vs = ks + kStep * D;
      const int kb0 = k0 + s * pl.step_keys;

      // S, keys permuted: within 16 of them, block h's n-th is 4 (n / 2) + n % 2 + 2 h.
      // R = 16: sc[2 kb + h], rows g and g + 8, column n = key.  R = 8: sc[2 kb] and sc[2 kb + 1] are the halves
      // h of a 16-key tile, row n = key g, columns 2 c, 2 c + 1 the lane's two rows.
      float sc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      auto key_words = [&](int n, int v) {  // the lane's chunk of its key of block n
        const int k = 16 * (n >> 1) + 4 * (g >> 1) + (g & 1) + 2 * (n & 1);
        int ch = c + 4 * v;
        if (D == 128) ch ^= 4 * (k & 1);
        return *reinterpret_cast<const uint4*>(ks + k * D + ch * 16);
      };
      if constexpr (R == 16) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int v = 0; v < D / 64; ++v) {
            const uint4 kv = key_words(n, v);
            const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma_f16_16816(sc[n], qf[4 * v + i][0], qf[4 * v + i][1], qf[4 * v + i][R / 8], qf[4 * v + i][R / 8 + 1],
                            e4m3x2_h2(w[i] & 0xffffu), e4m3x2_h2(w[i] >> 16));
          }
      } else {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < D / 64; ++v) {
            const uint4 k0v = key_words(2 * kb, v), k1v = key_words(2 * kb + 1, v);
            const uint32_t w0[4] = {k0v.x, k0v.y, k0v.z, k0v.w}, w1[4] = {k1v.x, k1v.y, k1v.z, k1v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma_f16_16816(sc[2 * kb], e4m3x2_h2(w0[i] & 0xffffu), e4m3x2_h2(w1[i] & 0xffffu), e4m3x2_h2(w0[i] >> 16),
                            e4m3x2_h2(w1[i] >> 16), qf[4 * v + i][0], qf[4 * v + i][1]);
          }
        // to the order of the other form: sc[2 kb + h][i], i = the lane's row
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          sc[2 * kb + 1][0] = sc[2 * kb][2];
          sc[2 * kb + 1][1] = sc[2 * kb][3];
        }
      }
      // scores, running maximum, P
      const bool edge = kb0 < full_lo || kb0 + kStep > full_hi;
      constexpr int X = R == 16 ? 8 : 4;  // a lane's keys of a row
      auto key_of = [&](int i) {          // its i-th
        return R == 16 ? kb0 + 16 * (i >> 2) + 4 * c + (i & 1) + 2 * ((i >> 1) & 1)
                       : kb0 + 16 * (i >> 1) + 4 * (g >> 1) + (g & 1) + 2 * (i & 1);
      };
      float x[2][X];
      float corr[2] = {1.f, 1.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e == 1 && !two) {
#pragma unroll
          for (int i = 0; i < X; ++i) x[1][i] = 0.f;
          break;
        }
#pragma unroll
        for (int i = 0; i < X; ++i) {
          // rounded here: fused into the subtraction below, a large score could exceed the maximum
          float v = __fmul_rn(R == 16 ? sc[i >> 1][2 * e + (i & 1)] : sc[i][e], fac[e]);
          if (CAP) v = __fmul_rn(cap2, CAP == kCapFine ? tanh_fine_from_2l2e(v) : tanh_from_2l2e(v));
          x[e][i] = v;
        }
        if (a.slopes) {
#pragma unroll
          for (int i = 0; i < X; ++i) x[e][i] -= slope[e] * fabsf((float)(pos[e] - kb0) - (float)(key_of(i) - kb0));
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < X; ++i)
            if (key_of(i) < lo[e] || key_of(i) >= hi[e]) x[e][i] = -INFINITY;
        }
        float top = x[e][0];
#pragma unroll
        for (int i = 1; i < X; ++i) top = fmaxf(top, x[e][i]);
        // over the lanes that have the row: c, or g
#pragma unroll
        for (int s = R == 16 ? 1 : 4; s < (R == 16 ? 4 : 32); s *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
        // the origin of the exponentials, kLift below the largest score and rounded up: P reaches 2^kLift
        const float nm = fmaxf(m[e], __fadd_ru(top, -(float)kLift));
        const float org = nm == -INFINITY ? 0.f : nm;  // nothing seen yet: any finite origin
        corr[e] = ex2(m[e] - org);
        m[e] = nm;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < X; ++i) {
          x[e][i] = ex2(x[e][i] - org);
          sum += x[e][i];
        }
        l[e] = l[e] * corr[e] + sum;
      }
      // P: the A operand (R = 16), or turned into the B operand, block by block
      uint32_t pf[2][R == 16 ? 4 : 2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        if constexpr (R == 16) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            pf[kb][e] = h2(x[e][4 * kb], x[e][4 * kb + 1]);
            pf[kb][R / 8 + e] = h2(x[e][4 * kb + 2], x[e][4 * kb + 3]);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t own = h2(x[0][2 * kb + h], x[1][2 * kb + h]);
            asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pf[kb][h]) : "r"(own));
          }
        }
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          o_acc[n][0] *= corr[0];
          o_acc[n][1] *= corr[R == 16 ? 0 : 1];
          o_acc[n][2] *= corr[R == 16 ? 1 : 0];
          o_acc[n][3] *= corr[1];
        }
      }
      // O += P V.  R = 16: column n of block nb <-> d = (D / 8) n + nb.  R = 8, transposed: rows n and n + 8 of block nb
      // <-> d = (D / 8) n + 2 nb and the next.
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        constexpr int W = D / 32;  // words of a lane's share of a key
        uint32_t vw[4][W];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 16 * kb + 4 * c + i;
          if (D == 128) {
            const uint4 t4 = *reinterpret_cast<const uint4*>(vs + k * D + (g ^ (2 * ((k >> 2) & 3))) * 16);
            vw[i][0] = t4.x;
            vw[i][1] = t4.y;
            vw[i][W - 2] = t4.z;
            vw[i][W - 1] = t4.w;
          } else {
            const uint2 t2 = *reinterpret_cast<const uint2*>(vs + k * D + g * 8);
            vw[i][0] = t2.x;
            vw[i][1] = t2.y;
          }
        }
        // A NaN value in a position that a row does not see must not reach it through 0 * NaN: on a step
        // with such positions NaN values are taken out of the product and put into the rows that see them.
        if (edge) {
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const uint32_t nan = ((vw[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
              bad |= nan;
              vw[i][w] &= ~((nan >> 7) * 0xffu);
            }
          if (__any_sync(0xffffffffu, bad != 0)) {
            for (int k = 0; k < 16; ++k)
#pragma unroll
              for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const int kk = 16 * kb + k, key = kb0 + kk;
                  const int d = R == 16 ? (D / 8) * (2 * c + i) + n : (D / 8) * g + 2 * n + i;
                  int ch = d / 16;
                  if (D == 128) ch ^= 2 * ((kk >> 2) & 3);
                  if ((vs[kk * D + ch * 16 + d % 16] & 0x7f) == 0x7f) {
                    if (key >= lo[0] && key < hi[0]) o_acc[n][R == 16 ? i : 2 * i] = __uint_as_float(0x7fffffffu);
                    if (key >= lo[1] && key < hi[1]) o_acc[n][R == 16 ? 2 + i : 2 * i + 1] = __uint_as_float(0x7fffffffu);
                  }
                }
          }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t a01 = prmt(vw[0][w], vw[1][w], 0x5140), b01 = prmt(vw[0][w], vw[1][w], 0x7362);
          const uint32_t a23 = prmt(vw[2][w], vw[3][w], 0x5140), b23 = prmt(vw[2][w], vw[3][w], 0x7362);
          if constexpr (R == 16) {
            auto col = [&](int n, uint32_t b0, uint32_t b1) {
              mma_f16_16816(o_acc[4 * w + n], pf[kb][0], pf[kb][1], pf[kb][R / 8], pf[kb][R / 8 + 1], e4m3x2_h2(b0),
                            e4m3x2_h2(b1));
            };
            col(0, a01 & 0xffffu, a23 & 0xffffu);
            col(1, a01 >> 16, a23 >> 16);
            col(2, b01 & 0xffffu, b23 & 0xffffu);
            col(3, b01 >> 16, b23 >> 16);
          } else {
            mma_f16_16816(o_acc[2 * w], e4m3x2_h2(a01 & 0xffffu), e4m3x2_h2(a01 >> 16), e4m3x2_h2(a23 & 0xffffu),
                          e4m3x2_h2(a23 >> 16), pf[kb][0], pf[kb][1]);
            mma_f16_16816(o_acc[2 * w + 1], e4m3x2_h2(b01 & 0xffffu), e4m3x2_h2(b01 >> 16), e4m3x2_h2(b23 & 0xffffu),
                          e4m3x2_h2(b23 >> 16), pf[kb][0], pf[kb][1]);
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int s = R == 16 ? 1 : 4; s < (R == 16 ? 4 : 32); s *= 2) l[e] += __shfl_xor_sync(0xffffffffu, l[e], s);
    }

    // Row first + GAP e of the tile: this lane's part of its outputs, from d0 on, is part(e, 0 .. NP - 1).
    constexpr int NP = R == 16 ? D / 4 : D / 8;
    const int d0 = R == 16 ? (D / 4) * c : (D / 8) * g;
    auto part = [&](int e, int i) -> float& {
      if constexpr (R == 16) return o_acc[i % ND][2 * e + i / ND];
      else return o_acc[i / 2][2 * (i % 2) + e];
    };
    const bool leads = R == 16 ? c == 0 : g == 0;  // the lane that tells a row's maximum and sum

    // ---- join the key subgroups of a head in shared memory, in order ----
    if (pl.nsub > 1) {
      float* mine = reinterpret_cast<float*>(ring);  // [R][D] and [R][2]
      __syncwarp();
      if (sub > 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = first + GAP * e;
#pragma unroll
          for (int i = 0; i < NP; ++i) mine[r * D + d0 + i] = part(e, i);
          if (leads) {
            mine[R * D + 2 * r] = m[e];
            mine[R * D + 2 * r + 1] = l[e];
          }
        }
      }
      __syncthreads();
      if (sub == 0) {
        for (int s2 = 1; s2 < pl.nsub; ++s2) {
          const float* from = reinterpret_cast<const float*>(smem + (warp + s2 * pl.nh) * C::RING);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = first + GAP * e;
            const float om = from[R * D + 2 * r], ol = from[R * D + 2 * r + 1];
            const float nm = fmaxf(m[e], om), org = nm == -INFINITY ? 0.f : nm;
            const float fa = ex2(m[e] - org), fb = ex2(om - org);
            m[e] = nm;
            l[e] = l[e] * fa + ol * fb;
#pragma unroll
            for (int i = 0; i < NP; ++i) part(e, i) = part(e, i) * fa + from[r * D + d0 + i] * fb;
          }
        }
      }
      __syncthreads();
    }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (!live[e]) continue;
        const size_t r = ((size_t)slot * pl.nh + hw) * R + first + GAP * e;
        float4* dst = reinterpret_cast<float4*>(pl.acc + r * D + d0);
#pragma unroll
        for (int i = 0; i < NP; i += 4) dst[i / 4] = make_float4(part(e, i), part(e, i + 1), part(e, i + 2), part(e, i + 3));
        if (leads) *reinterpret_cast<float2*>(pl.ml + r * 2) = make_float2(m[e], l[e]);
      }
    }
    __syncwarp();  // the ring is refilled
  }
}

// Joins the segments of one output row (token, query head): WPR warps take its segments in turn, then
// the first the warps' sums.  o = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.
template <int D, int WPR>
__global__ void __launch_bounds__(256) attn_chunk_merge_kernel(ChunkArgs a, SplitPlan pl) {
  constexpr int E = D / 32;  // elements a lane
  __shared__ float part[8][D + 2];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (8 / WPR) + warp / WPR;
  const int sub = warp % WPR;
  int t = (int)(item / a.Hq), b = -1;
  const int hq = (int)(item - (long long)t * a.Hq);
  if (pl.merge_tokens > 0) {  // the first merge_tokens tokens of every request
    b = t / pl.merge_tokens;
    const int i = t - b * pl.merge_tokens;
    if (b >= a.B || i >= a.cu_q[b + 1] - a.cu_q[b]) b = -1;
    else t = a.cu_q[b] + i;
  } else if (t < a.T) {
    b = find_request(a.cu_q, a.B, t);
  }
  bool mine = false;
  float M = -INFINITY, L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  if (b >= 0) {
    const Req rq = request(a, b);
    mine = rq.n * a.G <= pl.most_rows;
    const int nc = (max(0, rq.hi - rq.lo) + pl.step_keys - 1) / pl.step_keys;
    if (mine && nc > 0) {
      const int h = hq / a.G, r = (t - a.cu_q[b]) * a.G + hq - h * a.G;
      const int in_t = (r / pl.rows) * pl.hg + h / pl.nh, tile = pl.pre_t[b] + in_t;
      const int U = pl.pre_u[a.B], first = pl.pre_u[b] + in_t * nc;
      const int share = shared_by(pl, U);
      const int s0 = unit_owner(U, share, first), s1 = unit_owner(U, share, first + nc - 1) + 1;
      const size_t in_slot = (size_t)(h % pl.nh) * pl.rows + r % pl.rows, per = (size_t)pl.nh * pl.rows;
      for (int base = s0 + sub; base < s1; base += 32 * WPR) {  // segments base, base + WPR, ..: a lane each
        const int mine_at = base + lane * WPR;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (mine_at < s1) ml = *reinterpret_cast<const float2*>(pl.ml + ((size_t)(mine_at + tile) * per + in_slot) * 2);
        const float nm = fmaxf(M, warp_max(ml.x)), org = nm == -INFINITY ? 0.f : nm;
        const float old = ex2(M - org), w = ex2(ml.x - org);
        M = nm;
        L = L * old + warp_sum(w * ml.y);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= old;
        const int cnt = min(32, (s1 - base + WPR - 1) / WPR);
#pragma unroll 8
        for (int i = 0; i < cnt; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w, i);
          const float* src = pl.acc + ((size_t)(base + i * WPR + tile) * per + in_slot) * D + lane * E;
          if (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            o[0] += wi * v.x;
            o[1] += wi * v.y;
            o[E - 2] += wi * v.z;
            o[E - 1] += wi * v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            o[0] += wi * v.x;
            o[1] += wi * v.y;
          }
        }
      }
    }
  }
  if (WPR > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane * E + e] = o[e];
    if (lane == 0) {
      part[warp][D] = M;
      part[warp][D + 1] = L;
    }
    __syncthreads();
    if (sub != 0) return;
    for (int w = 1; w < WPR; ++w) {
      const float om = part[warp + w][D], ol = part[warp + w][D + 1];
      const float nm = fmaxf(M, om), org = nm == -INFINITY ? 0.f : nm;
      const float fa = ex2(M - org), fb = ex2(om - org);
      M = nm;
      L = L * fa + ol * fb;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * fa + part[warp + w][lane * E + e] * fb;
    }
  }
  if (!mine) return;
  const float inv = L == 0.f ? 0.f : __fdividef(a.v_scale[hq / a.G], L);
  __nv_bfloat16* dst = a.out + (size_t)t * a.ldo + (size_t)hq * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(o[e] * inv, o[e + 1] * inv);
}

int heads_a_block(int Hkv) { return Hkv % 8 == 0 ? 8 : Hkv % 4 == 0 ? 4 : Hkv % 2 == 0 ? 2 : 1; }

// CTAs at most: as many as are resident at once.
int split_ctas(int D) { return okc_host::num_sms() * (D == 64 ? 2 : 1); }

size_t split_slots(int T, int B, int Hq, int Hkv, int D, int rows) {
  const size_t hg = Hkv / heads_a_block(Hkv);
  return split_ctas(D) + (((size_t)T * (Hq / Hkv) + rows - 1) / rows + B) * hg;
}

template <int D, int CAP, int R>
int launch_split(const ChunkArgs& a, const SplitPlan& pl, cudaStream_t stream) {
  using C = ChunkCfg<D>;
  const int smem = C::SMEM + 2 * (a.B + 1) * 4;
  static okc_host::PerDevice configured;
  if (int st = configured.smem(attn_chunk_split_kernel<D, CAP, R>, C::SMEM + 2 * (kMaxChunkRequests + 1) * 4)) return st;
  if (int st = okc_host::launch_k(attn_chunk_split_kernel<D, CAP, R>, dim3(pl.ctas), dim3(32 * kWarps), smem, stream,
                                  dim3(1), a, pl))
    return st;
  const long long items = (long long)(pl.merge_tokens > 0 ? (long long)a.B * pl.merge_tokens : a.T) * a.Hq;
  // few rows: eight warps share a row's segments
  if (items <= 1024)
    return okc_host::launch_k(attn_chunk_merge_kernel<D, 8>, dim3((unsigned)items), dim3(256), 0, stream, dim3(1), a, pl);
  return okc_host::launch_k(attn_chunk_merge_kernel<D, 1>, dim3((unsigned)((items + 7) / 8)), dim3(256), 0, stream,
                            dim3(1), a, pl);
}

template <int CAP>
int launch_split_cap(const ChunkArgs& a, const SplitPlan& pl, cudaStream_t stream) {
  if (a.D == 64)
    return pl.rows == 8 ? launch_split<64, CAP, 8>(a, pl, stream) : launch_split<64, CAP, 16>(a, pl, stream);
  return pl.rows == 8 ? launch_split<128, CAP, 8>(a, pl, stream) : launch_split<128, CAP, 16>(a, pl, stream);
}

}  // namespace

size_t attn_chunk_ws_bytes(int T, int B, int Hq, int Hkv, int D) {
  // 16-row tiles need the more: up to B tiles more of twice the rows
  const size_t rows = split_slots(T, B, Hq, Hkv, D, 16) * heads_a_block(Hkv) * 16;
  return 2 * up((size_t)(B + 1) * 4) + up(rows * 8) + up(rows * D * 4) + attn_chunk_tc_ws_bytes(T, B, Hq, Hkv, D);
}

namespace {

// How a call is served, but for the workspace's pieces.
struct Served {
  SplitPlan split;
  bool split_only, tc_only;
  long long units;  // that the short chunks' kernel may number, as far as T and the table's width tell
};

Served serve(const ChunkArgs& a) {
  Served how;
  SplitPlan& pl = how.split;
  pl.nh = heads_a_block(a.Hkv);
  pl.nsub = kWarps / pl.nh;
  pl.hg = a.Hkv / pl.nh;
  pl.step_keys = kStep * pl.nsub;
  pl.few = okc_host::num_sms();

  // Every request short: this kernel alone.  Also where all of them make few tiles and steps (as far as T and the
  // table's width tell), since two kernels and two merges in a row take longer: 8 chunks of up to 44 tokens behind 325
  // positions, 8 / 1 heads, 19 us against 37, behind 2000 36 and 45; 16 / 8 heads 22 and 36; at 64 / 8 heads (295000 rows
  // of tiles times keys) 37 either way.  One long request: the tensor-memory kernel alone.  Else each serves its own.
  const long long longest = a.max_q > 0 && a.max_q < a.T ? a.max_q : a.T;
  const long long tiles16 = ((long long)a.T * a.G - a.B) / 16 + a.B;
  how.split_only = longest * a.G <= kSplitRows ||
                   (tiles16 * pl.hg <= okc_host::num_sms() &&
                    tiles16 * a.max_keys * a.Hkv * a.D / 128 <= (a.B == 1 ? 20000 : 300000));
  how.tc_only = !how.split_only && a.B == 1;
  pl.most_rows = how.split_only ? 0x7fffffff : kSplitRows;
  pl.merge_tokens = how.split_only ? 0 : kSplitRows / a.G;
  pl.rows = how.split_only && longest * a.G <= 8 ? 8 : 16;
  // the grid by the units that the table's width allows; the kernels know how many there are
  const long long row_tiles = ((long long)a.T * a.G - a.B) / pl.rows + a.B;
  pl.ctas = row_tiles * pl.hg * (a.max_keys / pl.step_keys + 1) > 6 * pl.few ? split_ctas(a.D) : pl.few;

  // a request that is served beside the tensor-memory kernel has at most kSplitRows rows
  const long long most_tiles = (long long)a.B * (kSplitRows / 16);
  const long long tiles = how.split_only || row_tiles < most_tiles ? row_tiles : most_tiles;
  const bool launched = how.split_only || (!how.tc_only && pl.merge_tokens > 0);
  how.units = launched ? tiles * pl.hg * (((long long)a.max_keys + pl.step_keys - 1) / pl.step_keys) : 0;
  return how;
}

}  // namespace

long long attn_chunk_units(const ChunkArgs& a) { return serve(a).units; }

int launch_attn_chunk(const ChunkArgs& a, cudaStream_t stream) {
  const Served how = serve(a);
  SplitPlan pl = how.split;
  const size_t rows = split_slots(a.T, a.B, a.Hq, a.Hkv, a.D, pl.rows) * pl.nh * pl.rows;
  uint8_t* p = reinterpret_cast<uint8_t*>(a.ws);
  pl.pre_u = reinterpret_cast<int*>(p);
  p += up((size_t)(a.B + 1) * 4);
  pl.pre_t = reinterpret_cast<int*>(p);
  p += up((size_t)(a.B + 1) * 4);
  pl.ml = reinterpret_cast<float*>(p);
  p += up(rows * 8);
  pl.acc = reinterpret_cast<float*>(p);
  p += up(rows * a.D * 4);
  if (!how.split_only) {
    if (int st = launch_attn_chunk_tc(a, how.tc_only ? 0 : kSplitRows, p, pl.acc, pl.ml, stream)) return st;
    if (how.tc_only || pl.merge_tokens == 0) return OKC_OK;  // no request is short enough
  }
  switch (cap_form(a.softcap)) {
    case kCapFine: return launch_split_cap<kCapFine>(a, pl, stream);
    case kCapPlain: return launch_split_cap<kCapPlain>(a, pl, stream);
    default: return launch_split_cap<kCapNone>(a, pl, stream);
  }
}

}  // namespace okc
