// extern "C" entry points of the 8-bit projection path and of ragged batches: argument validation.
// Declarations and contracts: include/okc_b200.h.
#include "chunk_common.cuh"

using okc_host::aligned16;

namespace {

bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A finite float (the device math assumes it).
bool finite(float v) { return v - v == 0.f; }

// n / d = n * mul >> shift for 0 <= n < 2^31: with 2^(l-1) < d <= 2^l and mul = ceil(2^(31+l) / d), n * mul is
// above 2^(31+l) * n / d by less than 2^(31+l) / d, so the quotient is exact.
void divide_by(int d, uint32_t& mul, int& shift) {
  int l = 0;
  while (1ll << l < d) ++l;
  shift = 31 + l;
  mul = (uint32_t)(((1ull << shift) + d - 1) / d);
}

}  // namespace

extern "C" {

int okc_add_rmsnorm_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr, int residual_fp32,
                        const void* w, void* residual_out, int64_t ldo, void* q, int64_t ldq, float* scale, int T,
                        int H, float eps, int unit_offset, okc_stream_t stream) {
  if (T == 0) return OKC_OK;
  if (!x || !w || !q || !scale || T < 0 || H <= 0 || H % 16 || H > 16384 || !(eps >= 0.f)) return OKC_ERR_INVALID;
  if (!residual != !residual_out) return OKC_ERR_INVALID;
  if (ldx < H || ldq < H || (residual && (ldr < H || ldo < H))) return OKC_ERR_INVALID;
  const int re = residual_fp32 ? 4 : 8;  // elements of 16 bytes
  if (!aligned16(x) || !aligned16(w) || !aligned_to(q, 8) || !aligned_to(scale, 4) || ldx % 8 || ldq % 8)
    return OKC_ERR_ALIGNMENT;
  if (residual && (!aligned16(residual) || !aligned16(residual_out) || ldr % re || ldo % re)) return OKC_ERR_ALIGNMENT;
  return okc::launch_add_rmsnorm_fp8(x, ldx, residual, ldr, residual_fp32, w, residual_out, ldo, q, ldq, scale, T, H,
                                     eps, unit_offset, stream);
}

int okc_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, int e4m3, const float* x_scale,
               const float* w_scale, int w_scale_one, const void* bias, int act, const void* residual, int64_t ldr,
               int residual_fp32, void* y, int64_t ldy, int out_fp32, int M, int N, int K, int32_t* error,
               okc_stream_t stream) {
  if (M == 0) return OKC_OK;
  if (!x || !w || !y || !error || M < 0 || N <= 0 || K <= 0 || act < 0 || act > 4) return OKC_ERR_INVALID;
  const int es = e4m3 ? 1 : 2, ve = 16 / es;
  if (K % ve || ldx < K || ldw < K || ldy < N || (residual && ldr < N)) return OKC_ERR_INVALID;
  if (ldx > (1ll << 38) / es || ldw > (1ll << 38) / es) return OKC_ERR_INVALID;  // tensor-map strides
  if (!aligned16(x) || !aligned16(w) || ldx % ve || ldw % ve || !aligned_to(y, out_fp32 ? 4 : 2) ||
      !aligned_to(residual, residual_fp32 ? 4 : 2) || !aligned_to(bias, 2) || !aligned_to(x_scale, 4) ||
      !aligned_to(w_scale, 4))
    return OKC_ERR_ALIGNMENT;
  okc::LinearArgs a;
  a.x = x;
  a.w = w;
  a.ldx = ldx;
  a.ldw = ldw;
  a.y = y;
  a.ldy = ldy;
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.w_scale_one = w_scale_one;
  a.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  a.res = residual;
  a.ldr = ldr;
  a.res_fp32 = residual_fp32;
  a.out_fp32 = out_fp32;
  a.act = act;
  a.M = M;
  a.N = N;
  a.K = K;
  a.e4m3 = e4m3;
  a.pairs = ldy % 2 == 0 && aligned_to(y, out_fp32 ? 8 : 4) &&
            (!residual || (ldr % 2 == 0 && aligned_to(residual, residual_fp32 ? 8 : 4)));
  a.packed = !out_fp32 && !residual && ldy % 8 == 0 && aligned16(y);
  a.err = error;
  return okc::launch_linear(a, stream);
}

int okc_rope_axes_kv_append(const void* qkv, int64_t ldqkv, const int64_t* positions, int64_t ld_pos, int axes,
                            const uint8_t* axis_of_pair, const float* inv_freq, int pairs, int half_split,
                            const int32_t* cu_q, const int32_t* seq_lens, int B, const int32_t* page_table,
                            int64_t table_ld, int max_pages, const float* k_scale, const float* v_scale, void* q_out,
                            int64_t ldq, void* k_cache, void* v_cache, int T, int Hq, int Hkv, int D, int page_size,
                            int64_t num_pages, int32_t* error, okc_stream_t stream) {
  if (T == 0) return OKC_OK;
  if (!qkv || !positions || !axis_of_pair || !inv_freq || !cu_q || !seq_lens || !page_table || !k_scale || !v_scale ||
      !q_out || !k_cache || !v_cache || !error)
    return OKC_ERR_INVALID;
  if (T < 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || D % 8 || D > 256 || pairs <= 0 || pairs % 8 ||
      2 * pairs > D || axes < 1 || axes > 4 || page_size <= 0 || num_pages <= 0 || max_pages <= 0)
    return OKC_ERR_INVALID;
  if (table_ld < max_pages || ld_pos < T || ldqkv < (int64_t)(Hq + 2 * Hkv) * D || ldq < (int64_t)Hq * D)
    return OKC_ERR_INVALID;
  okc::RopeAxesArgs a = {};
  for (int i = 0; i < pairs; ++i) {
    if (axis_of_pair[i] >= axes) return OKC_ERR_INVALID;
    a.axis_bits[i >> 5] |= (unsigned long long)axis_of_pair[i] << (2 * (i & 31));
  }
  if (!aligned16(qkv) || !aligned16(q_out) || ldqkv % 8 || ldq % 8 || !aligned_to(k_cache, 8) ||
      !aligned_to(v_cache, 8) || !aligned_to(positions, 8))
    return OKC_ERR_ALIGNMENT;
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv);
  a.ldqkv = ldqkv;
  a.positions = positions;
  a.ld_pos = ld_pos;
  a.inv_freq = inv_freq;
  a.R = pairs;
  a.half = half_split;
  a.cu_q = cu_q;
  a.seq_lens = seq_lens;
  a.page_table = page_table;
  a.table_ld = table_ld;
  a.max_pages = max_pages;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
  a.ldq = ldq;
  a.k_cache = reinterpret_cast<uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<uint8_t*>(v_cache);
  a.T = T;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.P = page_size;
  a.num_pages = num_pages;
  a.err = error;
  return okc::launch_rope_axes_append(a, stream);
}

size_t okc_attn_chunk_workspace_bytes(int T, int B, int Hq, int Hkv, int D) {
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (D != 64 && D != 128)) return 0;
  return okc::attn_chunk_ws_bytes(T, B, Hq, Hkv, D);
}

int okc_attn_chunk_fp8(const void* q, int64_t ldq, const void* k_cache, const void* v_cache, const int32_t* page_table,
                       int64_t table_ld, int max_pages, const int32_t* cu_q, const int32_t* seq_lens,
                       const float* k_scale, const float* v_scale, const float* slopes, const int32_t* prefix_lens,
                       const int32_t* doc_start, void* out, int64_t ldo, int T, int B, int Hq, int Hkv, int D,
                       int page_size, int64_t num_pages, float sm_scale, float softcap, int window, int max_q,
                       void* workspace, size_t workspace_bytes, int32_t* error, okc_stream_t stream) {
  if (T == 0) return OKC_OK;
  if (!q || !k_cache || !v_cache || !page_table || !cu_q || !seq_lens || !k_scale || !v_scale || !out || !error)
    return OKC_ERR_INVALID;
  if (T < 0 || B <= 0 || B > okc::kMaxChunkRequests || Hq <= 0 || Hkv <= 0 || Hq % Hkv || (D != 64 && D != 128) ||
      page_size <= 0 || num_pages <= 0 || max_pages <= 0 || window < 0 || max_q < 0)
    return OKC_ERR_INVALID;
  if (!finite(sm_scale) || !(softcap == 0.f || (softcap >= 1e-6f && softcap <= 1e12f))) return OKC_ERR_INVALID;
  if (table_ld < max_pages || ldq < (int64_t)Hq * D || ldo < (int64_t)Hq * D) return OKC_ERR_INVALID;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || ldq % 8 || ldo % 8)
    return OKC_ERR_ALIGNMENT;
  if ((long long)T * Hq > 0x7fffffffll) return OKC_ERR_TOO_LARGE;  // output rows
  // row tile pairs are a grid's second dimension
  if ((long long)T * (Hq / Hkv) / 256 + B > 65535) return OKC_ERR_TOO_LARGE;
  // the cache's rows of D bytes are numbered in 32 bits: 256 GB of keys at D = 64
  if (num_pages > 0xfffffffell / page_size / Hkv) return OKC_ERR_TOO_LARGE;
  const long long most_keys = (1ll << 31) - (1ll << 17);
  const long long keys = (long long)max_pages * page_size < most_keys ? (long long)max_pages * page_size : most_keys;
  okc::ChunkArgs a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.ldq = ldq;
  a.k_cache = reinterpret_cast<const uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<const uint8_t*>(v_cache);
  a.page_table = page_table;
  a.table_ld = table_ld;
  a.max_keys = (int)keys;
  a.cu_q = cu_q;
  a.seq_lens = seq_lens;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.slopes = slopes;
  a.prefix_lens = prefix_lens;
  a.doc_start = doc_start;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  a.T = T;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.D = D;
  a.P = page_size;
  a.window = window;
  a.num_pages = num_pages;
  divide_by(page_size, a.page_mul, a.page_shift);
  divide_by(a.G, a.group_mul, a.group_shift);
  a.sm_scale = sm_scale;
  a.softcap = softcap;
  a.max_q = max_q;
  a.ws = workspace;
  a.err = error;
  if (okc::attn_chunk_units(a) > 0x7fffffffll) return OKC_ERR_TOO_LARGE;
  if (!workspace || workspace_bytes < okc::attn_chunk_ws_bytes(T, B, Hq, Hkv, D)) return OKC_ERR_WORKSPACE;
  if (!aligned16(workspace)) return OKC_ERR_ALIGNMENT;
  return okc::launch_attn_chunk(a, stream);
}

}  // extern "C"
