// kv_pages.cuh -- the paged 8-bit KV cache as the kernels see it: one layer of
// an engine_kv_pages_t, its bounds-checked lookups and its code conversions.
//
// A page holds page_size tokens of every KV head, head-major
// ([n_kv_heads][page_size][head_dim] codes), so one head's part of a page is one
// contiguous tile; every (page, head) has one FP32 scale for K and one for V:
// value = scale * code.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

/// One layer of a cache (validated on the host: kv_pages_check).
struct KvView {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  const int32_t* table;
  int32_t* length;
  const int32_t* ref;
  int64_t n_pages;
  int max_pages;   // entries of a table row
  int n_slots;
  int heads;       // KV heads
  int shift;       // log2(page size)
  unsigned int* err;
};

constexpr float kQMaxI8 = 127.0f;
constexpr float kQMaxE4M3 = 448.0f;
/// What attention takes for a scale of V that is 0 (a page of zeros, whose weights count in
/// the denominator alone): below any that a write gives, so that w = p vs of such a page is
/// never what the others' weights are rounded against.
constexpr float kNoScale = 1.1641532182693481e-10f;  // 2^-33 < 2^-24 / 448

/// Validates the descriptor (and `layer`, unless it is -1: all layers); returns
/// ENGINE_OK or an error with the message recorded.  kv_pages.cu.
int kv_pages_check(const engine_kv_pages_t* kv, int64_t layer, const char* what);
/// The view of one layer of a validated descriptor.
KvView kv_view(const engine_kv_pages_t* kv, int64_t layer);

/// Slot of row b of a batch, or -1 (and error bit 2) outside the cache.
__device__ __forceinline__ int kv_slot(const KvView& c, const int32_t* slots, int64_t b) {
  const int64_t s = slots != nullptr ? slots[b] : b;
  if (s < 0 || s >= c.n_slots) {
    atomicOr(c.err, kErrBadArgument);
    return -1;
  }
  return static_cast<int>(s);
}

/// Length of a slot: 0 for slot -1, and (with error bit 2) for one that its table row cannot address.
__device__ __forceinline__ int kv_length(const KvView& c, int slot) {
  if (slot < 0) return 0;
  const int n = c.length[slot];
  const int64_t cap = static_cast<int64_t>(c.max_pages) << c.shift;
  if (n < 0 || n > cap) {
    atomicOr(c.err, kErrBadArgument);
    return 0;
  }
  return n;
}

/// Page of entry `e` of a slot's row, or -1 (and error bit 2) when it is none.
__device__ __forceinline__ int kv_page(const KvView& c, int slot, int e) {
  const int p = c.table[static_cast<int64_t>(slot) * c.max_pages + e];
  if (p < 0 || p >= c.n_pages) {
    atomicOr(c.err, kErrBadArgument);
    return -1;
  }
  return p;
}

/// Rows [*first, *first + n) of sequence b in a batch of n_tokens rows: cu[b] to
/// cu[b + 1], or row b where cu is null.  Returns n; 0 (and error bit 2) where the
/// entries are not an ascending pair within the rows.
__device__ __forceinline__ int kv_rows(const KvView& c, const int32_t* cu, int64_t b,
                                       int64_t n_tokens, int64_t* first) {
  *first = b;
  if (cu == nullptr) return 1;
  const int a = cu[b], e = cu[b + 1];
  *first = a;
  if (a < 0 || e < a || e > n_tokens) {
    atomicOr(c.err, kErrBadArgument);
    return 0;
  }
  return e - a;
}

/// Sum of v >= 0 over the warp, which may pass 32 bits.
__device__ __forceinline__ int64_t kv_wide_sum(int v) {
  return (static_cast<int64_t>(__reduce_add_sync(0xffffffffu, v >> 16)) << 16) +
         __reduce_add_sync(0xffffffffu, v & 0xffff);
}
/// Steps of a launch from their exact sum.  The host has bounded those of sequences that share
/// no rows; entries of cu that go back and forth can pass 32 bits: nothing is done then.
__device__ __forceinline__ int kv_total(const KvView& c, int64_t all) {
  if (all <= 0x7fffffff) return static_cast<int>(all);
  atomicOr(c.err, kErrBadArgument);
  return 0;
}

/// First code of (page, head, row 0) for head_dim D, and the index of its scale.
template <int D>
__device__ __forceinline__ int64_t kv_tile(const KvView& c, int page, int head) {
  return ((static_cast<int64_t>(page) * c.heads + head) << c.shift) * D;
}
__device__ __forceinline__ int64_t kv_scale_at(const KvView& c, int page, int head) {
  return static_cast<int64_t>(page) * c.heads + head;
}

/// Four codes (one 32-bit word, lowest byte first) as two FP16 pairs, exactly:
/// both 8-bit types are subsets of FP16.  int8: the byte with its sign bit
/// flipped is q + 128, and 0x6400 | byte is the FP16 number 1024 + byte, so
/// subtracting 1152 gives q -- a byte permute and one packed subtraction per
/// pair, where an integer conversion would take one quarter-rate instruction per
/// element.
template <bool E4M3>
__device__ __forceinline__ void codes_to_half4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t bias = 0x64806480u;  // 1152, twice
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(bias));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(bias));
  }
}

/// One code of value y (already divided by the scale), to nearest, ties to even.
template <bool E4M3>
__device__ __forceinline__ uint32_t to_code(float y) {
  if constexpr (E4M3) {
    return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  } else {
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(y, -kQMaxI8), kQMaxI8))) & 0xffu;
  }
}

}  // namespace b200
