// attention_paged.cu -- attention over the paged 8-bit KV cache.
//
// Both entry points are one computation: query row t of sequence b sees the
// positions [0, last] of its slot.  With x_j = scale log2(e) ks_j (q . ck_j), where
// ck, cv are codes and ks, vs the scales of their page,
//   w_j = 2^(x_j + log2 vs_j - m),  out = sum_j w_j cv_j / sum_j (w_j / vs_j),
// m the running maximum of x_j + log2 vs_j.  Keeping the page's scale of V inside
// the weight leaves the products to the codes alone, and the weight is scaled by
// what it contributes.  A page whose values are all zero has scale 0: it counts
// with vs = 1 (its codes are zeros).
//
// First form: one warp per query row and head, FP32 on CUDA cores.
#include <cmath>

#include "kernels.cuh"
#include "kv_pages.cuh"

namespace b200 {
namespace {

struct ApParams {
  KvView c;
  const __half* q;
  int64_t q_pitch;
  const int32_t* slots;
  const int32_t* cu;  // null: one row per sequence, all keys
  __half* out;
  float* lse;
  int64_t n_seq, n_tokens;
  int n_heads;
  int causal;
  float scale_log2;
};

template <int D, bool E4M3>
__global__ void __launch_bounds__(128) attn_paged_simple_kernel(const ApParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (task >= p.n_tokens * p.n_heads) return;
  const int64_t t = task / p.n_heads;
  const int h = static_cast<int>(task % p.n_heads);
  int64_t b = -1, first = t;
  int n = 1;
  if (p.cu == nullptr) {
    b = t;
  } else {
    for (int64_t base = 0; base < p.n_seq && b < 0; base += 32) {
      const int64_t i = base + lane;
      if (i < p.n_seq) n = kv_rows(p.c, p.cu, i, p.n_tokens, &first);
      const bool mine = i < p.n_seq && first <= t && t < first + n;
      const unsigned hit = __ballot_sync(0xffffffffu, mine);
      if (hit != 0) b = base + __ffs(hit) - 1;
    }
    if (b < 0) return;
    n = kv_rows(p.c, p.cu, b, p.n_tokens, &first);
  }
  const int slot = kv_slot(p.c, p.slots, b);
  const int len = kv_length(p.c, slot);
  const int last = p.causal ? len - n + static_cast<int>(t - first) : len - 1;
  constexpr int E = D / 32;
  const int kvh = h / (p.n_heads / p.c.heads);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __half2float(p.q[t * p.q_pitch + static_cast<int64_t>(h) * D + lane * E + e]);
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  auto code = [](uint8_t v) {
    uint32_t lo, hi;
    codes_to_half4<E4M3>(v, lo, hi);
    return __half2float(__low2half(*reinterpret_cast<__half2*>(&lo)));
  };
  const int page = 1 << p.c.shift;
  for (int e0 = 0; e0 * page <= last; ++e0) {
    const int id = kv_page(p.c, slot, e0);
    if (id < 0) continue;
    const float ks = p.c.ks[kv_scale_at(p.c, id, kvh)] * p.scale_log2;
    float vs = p.c.vs[kv_scale_at(p.c, id, kvh)];
    if (vs == 0.0f) vs = 1.0f;
    const float lv = log2f(vs), iv = 1.0f / vs;
    const int64_t tile = kv_tile<D>(p.c, id, kvh);
    for (int j = 0; j < page && e0 * page + j <= last; ++j) {
      const uint8_t* kr = p.c.k + tile + j * D + lane * E;
      const uint8_t* vr = p.c.v + tile + j * D + lane * E;
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], code(kr[e]), s);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      const float x = fmaf(s, ks, lv);
      const float m_new = fmaxf(m, x);
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float a = exp2f(m - base), w = exp2f(x - base);
      l = fmaf(w, iv, l * a);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, code(vr[e]), o[e] * a);
      m = m_new;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < E; ++e)
    p.out[(t * p.n_heads + h) * D + lane * E + e] = __float2half_rn(o[e] * inv);
  if (p.lse != nullptr && lane == 0)
    p.lse[t * p.n_heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <int D, bool E4M3>
int launch_simple(const ApParams& p, cudaStream_t st) {
  const int64_t blocks = (p.n_tokens * p.n_heads + 3) / 4;
  B200_CUDA(launch_pdl(attn_paged_simple_kernel<D, E4M3>, dim3(static_cast<unsigned>(blocks)), dim3(128),
                       0, st, p));
  return ENGINE_OK;
}

int run_paged(const ApParams& p, const engine_kv_pages_t* kv, cudaStream_t st, const char* what) {
  const bool e4m3 = kv->type == ENGINE_KV_E4M3;
  int rc;
  if (kv->head_dim == 64) rc = e4m3 ? launch_simple<64, true>(p, st) : launch_simple<64, false>(p, st);
  else rc = e4m3 ? launch_simple<128, true>(p, st) : launch_simple<128, false>(p, st);
  if (rc != ENGINE_OK) return rc;
  return check_launch(what);
}

int check_paged(const engine_kv_pages_t* kv, int64_t layer, const void* q, int64_t q_pitch,
                const void* slots, const void* out, int64_t n_seq, int64_t n_tokens,
                int64_t n_heads, float scale, const char* what) {
  const std::string w(what);
  if (const int rc = kv_pages_check(kv, layer, what)) return rc;
  B200_REQUIRE(layer >= 0, w + ": layer out of range");
  B200_REQUIRE(n_seq >= 0 && n_tokens >= 0, w + ": n_seq and n_tokens must be non-negative");
  B200_REQUIRE(slots != nullptr || n_seq <= kv->n_slots, w + ": n_seq > n_slots");
  B200_REQUIRE(n_heads > 0, w + ": n_heads must be positive");
  B200_REQUIRE(n_heads % kv->n_kv_heads == 0, w + ": n_heads must be divisible by n_kv_heads");
  B200_REQUIRE(std::isfinite(scale) && scale > 0.0f, w + ": scale must be finite and positive");
  B200_REQUIRE(q_pitch >= n_heads * kv->head_dim, w + ": q_pitch < n_heads * head_dim");
  if (n_seq == 0 || n_tokens == 0) return ENGINE_OK;
  B200_REQUIRE(q != nullptr, w + ": q is null");
  B200_REQUIRE(out != nullptr, w + ": out is null");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0 ||
      q_pitch % 8 != 0)
    return set_error(ENGINE_ERR_UNSUPPORTED,
                     w + ": q and out must be 16-byte aligned, q_pitch a multiple of 8");
  if (n_tokens > 0x7fffff00 || n_seq > 0x7fffff00 || n_heads > 65535 ||
      n_tokens * n_heads > 0x7fffff00)
    return set_error(ENGINE_ERR_UNSUPPORTED, w + ": n_tokens * n_heads too large");
  return ENGINE_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int engine_cuda_attention_paged_decode(const engine_kv_pages_t* kv, int64_t layer,
                                       const engine_half_t* q, int64_t q_pitch,
                                       const int32_t* slots, engine_half_t* out, float* out_lse,
                                       int64_t n_seq, int64_t n_heads, float scale,
                                       engine_stream_t stream) {
  B200_ENTRY_BEGIN
  const char* what = "attention_paged_decode";
  if (const int rc = check_paged(kv, layer, q, q_pitch, slots, out, n_seq, n_seq, n_heads, scale, what))
    return rc;
  if (n_seq == 0) return ENGINE_OK;
  const ApParams p{kv_view(kv, layer),
                   reinterpret_cast<const __half*>(q),
                   q_pitch,
                   slots,
                   nullptr,
                   reinterpret_cast<__half*>(out),
                   out_lse,
                   n_seq,
                   n_seq,
                   static_cast<int>(n_heads),
                   0,
                   scale * 1.4426950408889634f};
  return run_paged(p, kv, static_cast<cudaStream_t>(stream), what);
  B200_ENTRY_END
}

int engine_cuda_attention_paged_prefill(const engine_kv_pages_t* kv, int64_t layer,
                                        const engine_half_t* q, int64_t q_pitch,
                                        const int32_t* slots, const int32_t* cu_q,
                                        engine_half_t* out, float* out_lse, int64_t n_seq,
                                        int64_t n_tokens, int64_t n_heads, float scale,
                                        int is_causal, engine_stream_t stream) {
  B200_ENTRY_BEGIN
  const char* what = "attention_paged_prefill";
  if (const int rc =
          check_paged(kv, layer, q, q_pitch, slots, out, n_seq, n_tokens, n_heads, scale, what))
    return rc;
  if (n_seq == 0 || n_tokens == 0) return ENGINE_OK;
  B200_REQUIRE(cu_q != nullptr, "attention_paged_prefill: cu_q is null");
  const ApParams p{kv_view(kv, layer),
                   reinterpret_cast<const __half*>(q),
                   q_pitch,
                   slots,
                   cu_q,
                   reinterpret_cast<__half*>(out),
                   out_lse,
                   n_seq,
                   n_tokens,
                   static_cast<int>(n_heads),
                   is_causal != 0 ? 1 : 0,
                   scale * 1.4426950408889634f};
  return run_paged(p, kv, static_cast<cudaStream_t>(stream), what);
  B200_ENTRY_END
}

}  // extern "C"
