// kv_pages.cu -- the paged 8-bit KV cache: quantising writes, and the pages'
// bookkeeping (extend, fork, free, compact) on the device, so that a decode loop
// needs no host round trip and can be captured whole.
#include <algorithm>
#include <cmath>

#include "kernels.cuh"
#include "kv_pages.cuh"

namespace b200 {

int kv_pages_check(const engine_kv_pages_t* kv, int64_t layer, const char* what) {
  const std::string w(what);
  B200_REQUIRE(kv != nullptr, w + ": kv is null");
  B200_REQUIRE(kv->k != nullptr && kv->v != nullptr, w + ": k/v is null");
  B200_REQUIRE(kv->k_scale != nullptr && kv->v_scale != nullptr, w + ": k_scale/v_scale is null");
  B200_REQUIRE(kv->table != nullptr && kv->length != nullptr && kv->ref != nullptr,
               w + ": table/length/ref is null");
  B200_REQUIRE(kv->type == ENGINE_KV_I8 || kv->type == ENGINE_KV_E4M3,
               w + ": type must be ENGINE_KV_I8 or ENGINE_KV_E4M3");
  B200_REQUIRE(kv->page_size == 16 || kv->page_size == 32 || kv->page_size == 64 ||
                   kv->page_size == 128,
               w + ": page_size must be 16, 32, 64 or 128");
  B200_REQUIRE(kv->head_dim == 64 || kv->head_dim == 128, w + ": head_dim must be 64 or 128");
  B200_REQUIRE(kv->n_layers > 0 && kv->n_pages > 0 && kv->n_kv_heads > 0 && kv->n_slots > 0 &&
                   kv->max_pages > 0,
               w + ": n_layers, n_pages, n_kv_heads, n_slots and max_pages must be positive");
  B200_REQUIRE(layer >= -1 && layer < kv->n_layers, w + ": layer out of range");
  const uintptr_t a = reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v);
  B200_REQUIRE(a % 16 == 0, w + ": k/v must be 16-byte aligned");
  // Row indexes of one layer's pool and positions of one slot are 32-bit.
  constexpr int64_t kMost = 0x7fffff00;
  if (kv->n_pages > kMost || kv->n_kv_heads > 65535 || kv->n_slots > kMost ||
      kv->n_layers > 65535 || kv->n_pages * kv->n_kv_heads > kMost / kv->page_size ||
      kv->max_pages > kMost / kv->page_size)
    return set_error(ENGINE_ERR_UNSUPPORTED, w + ": cache dimensions too large");
  return ENGINE_OK;
}

KvView kv_view(const engine_kv_pages_t* kv, int64_t layer) {
  KvView c;
  const int64_t sc = layer * kv->n_pages * kv->n_kv_heads;
  const int64_t codes = sc * kv->page_size * kv->head_dim;
  c.k = static_cast<uint8_t*>(kv->k) + codes;
  c.v = static_cast<uint8_t*>(kv->v) + codes;
  c.ks = kv->k_scale + sc;
  c.vs = kv->v_scale + sc;
  c.table = kv->table;
  c.length = kv->length;
  c.ref = kv->ref;
  c.n_pages = kv->n_pages;
  c.max_pages = static_cast<int>(kv->max_pages);
  c.n_slots = static_cast<int>(kv->n_slots);
  c.heads = static_cast<int>(kv->n_kv_heads);
  c.shift = kv->page_size == 16 ? 4 : kv->page_size == 32 ? 5 : kv->page_size == 64 ? 6 : 7;
  c.err = device_error_word();
  return c;
}

namespace {

// ---------------------------------------------------------------- write
//
// A (page, KV head, K | V) tile's new rows come in once, 8 halves a thread and pass, and
// stay in registers between the maximum and the rounding: 2 bytes read and 1 written
// per element, which is what bounds a prompt.  The maximum is taken on the bit patterns
// with the sign cleared: for FP16 these order as the magnitudes do, and anything from
// 0x7c00 up is an infinity or NaN.

constexpr int kWrThreads = 128;

struct WrParams {
  KvView c;
  const __half* k_new;
  const __half* v_new;
  int64_t row_pitch;
  const int32_t* slots;
  const int32_t* cu;
  int64_t n_seq, n_tokens;
  const int32_t* status;  // null, or nothing is written unless *status is 0
  int d;                  // head_dim
};

/// New rows of sequence b: [r0, r0 + n), positions [len - n, len).
__device__ __forceinline__ int wr_rows(const WrParams& p, int64_t b, int* slot, int64_t* r0,
                                       int* len) {
  *slot = kv_slot(p.c, p.slots, b);
  *len = kv_length(p.c, *slot);
  const int n = kv_rows(p.c, p.cu, b, p.n_tokens, r0);
  if (*slot < 0) return 0;
  if (n > *len) {
    atomicOr(p.c.err, kErrBadArgument);
    return 0;
  }
  return n;
}

/// Finds page `item` of the pages that the sequences' new rows touch, counted
/// sequence by sequence.  Returns the sequence, or -1; *nth = which of its pages.
__device__ int64_t wr_find(const WrParams& p, int64_t item, int* nth) {
  __shared__ int s_warp[kWrThreads / 32];
  __shared__ int64_t s_seq;
  __shared__ int s_nth;
  if (threadIdx.x == 0) s_seq = -1;
  __syncthreads();
  int64_t run = 0;
  for (int64_t base = 0; base < p.n_seq && run <= item; base += kWrThreads) {
    const int64_t b = base + threadIdx.x;
    int cnt = 0;
    if (b < p.n_seq) {
      int slot, len;
      int64_t r0;
      const int n = wr_rows(p, b, &slot, &r0, &len);
      if (n > 0) cnt = ((len - 1) >> p.c.shift) - ((len - n) >> p.c.shift) + 1;
    }
    int incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane_id() >= o) incl += v;
    }
    if (lane_id() == 31) s_warp[threadIdx.x >> 5] = incl;
    __syncthreads();
    int64_t before = run;
    for (int w = 0; w < kWrThreads / 32; ++w) {
      if (w < static_cast<int>(threadIdx.x >> 5)) before += s_warp[w];
      run += s_warp[w];
    }
    before += incl - cnt;
    if (item >= before && item < before + cnt) {
      s_seq = b;
      s_nth = static_cast<int>(item - before);
    }
    __syncthreads();
  }
  *nth = s_nth;
  return s_seq;
}

/// Whether a page with `users` users takes rows: one that others use too (or that is free) is left
/// as it is (error bit 2).  A write behind an extend that was refused comes to the slot's last
/// rows, which a fork may have shared.
__device__ __forceinline__ bool wr_own(const WrParams& p, int users) {
  if (users == 1) return true;
  if (threadIdx.x == 0) atomicOr(p.c.err, kErrBadArgument);
  return false;
}

/// Largest magnitude of 8 halves, as two packed bit patterns.
__device__ __forceinline__ uint32_t half8_max(const uint4& x) {
  return __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
}

/// Scale for new rows whose largest magnitude has the bit pattern mx, in a page of scale
/// `old` (0 for one without earlier rows); NaN where a row is not finite.
template <bool E4M3>
__device__ __forceinline__ float wr_scale(uint32_t mx, float old) {
  constexpr float kQ = E4M3 ? kQMaxE4M3 : kQMaxI8;
  const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(mx))) * (1.0f / kQ);
  return mx >= 0x7c00u || old != old ? __int_as_float(0x7fc00000) : fmaxf(s, old);
}

/// 16 codes times `ratio`, rounded again.
template <bool E4M3>
__device__ __forceinline__ uint4 wr_again(const uint4& in, float ratio) {
  const uint32_t q[4] = {in.x, in.y, in.z, in.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t lo, hi;
    codes_to_half4<E4M3>(q[j], lo, hi);
    const float2 f0 = __half22float2(*reinterpret_cast<__half2*>(&lo));
    const float2 f1 = __half22float2(*reinterpret_cast<__half2*>(&hi));
    o[j] = to_code<E4M3>(f0.x * ratio) | to_code<E4M3>(f0.y * ratio) << 8 | to_code<E4M3>(f1.x * ratio) << 16 |
           to_code<E4M3>(f1.y * ratio) << 24;
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

/// 8 halves as codes.  inv = 0 (a NaN scale, or all zeros) gives zeros.
template <bool E4M3>
__device__ __forceinline__ uint2 wr_codes(const uint4& x, float inv) {
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t o[2] = {0, 0};
  if (inv != 0.0f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&in[j]));
      o[j >> 1] |= (to_code<E4M3>(f.x * inv) | to_code<E4M3>(f.y * inv) << 8) << (16 * (j & 1));
    }
  }
  return make_uint2(o[0], o[1]);
}

// Several rows: a CTA takes kWrTiles (KV head, K | V) tiles of one page, one after the
// other with the next one's rows on their way, so that finding the page (three dependent
// lookups) is paid once for them.  (Tiles one by one 21 us, two 20.8, four 19.3, eight 18.9
// but fewer CTAs for short prompts.)
constexpr int kWrTiles = 4;

template <int PASSES, bool E4M3>
__global__ void __launch_bounds__(kWrThreads) kv_write_kernel(const WrParams p) {
  pdl_trigger();
  pdl_wait();
  if (p.status != nullptr && *p.status != 0) return;
  __shared__ uint32_t s_max[2][kWrThreads / 32];
  int nth = 0;
  const int64_t b = wr_find(p, blockIdx.x, &nth);
  if (b < 0) return;
  int slot, len;
  int64_t r0;
  const int n = wr_rows(p, b, &slot, &r0, &len);
  if (n == 0) return;
  const int page_size = 1 << p.c.shift;
  const int start = len - n;
  const int entry = (start >> p.c.shift) + nth;
  const int page = kv_page(p.c, slot, entry);
  if (page < 0) return;
  const int users = p.c.ref[page];
  const int first = max(start - entry * page_size, 0);  // first new row in the page
  const int rows = min(len - entry * page_size, page_size) - first;
  const int lpr = p.d >> 3;  // threads per row
  const int rpp = kWrThreads / lpr;
  const int tr = threadIdx.x / lpr, tc = (threadIdx.x % lpr) * 8;
  const int64_t src0 =
      (r0 + (static_cast<int64_t>(entry) * page_size + first - start)) * p.row_pitch + tc;
  const int end = min((static_cast<int>(blockIdx.y) + 1) * kWrTiles, 2 * p.c.heads);
  auto load = [&](int tile, uint4 (&x)[PASSES]) {
    const __half* src = ((tile & 1) ? p.v_new : p.k_new) + src0 + static_cast<int64_t>(tile >> 1) * p.d;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * rpp + tr;
      x[i] = r < rows ? __ldg(reinterpret_cast<const uint4*>(src + r * p.row_pitch)) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 next[PASSES];
  int tile = blockIdx.y * kWrTiles;
  load(tile, next);
  if (!wr_own(p, users)) return;  // (looked up beside the rows)
  for (; tile < end; ++tile) {
    const int h = tile >> 1;
    const bool is_v = tile & 1;
    uint4 x[PASSES];
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      x[i] = next[i];
      mx = __vmaxu2(mx, half8_max(x[i]));
    }
    if (tile + 1 < end) load(tile + 1, next);
    float* sp = (is_v ? p.c.vs : p.c.ks) + kv_scale_at(p.c, page, h);
    const float old = first > 0 ? *sp : 0.0f;
    mx = max(mx & 0xffffu, mx >> 16);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane_id() == 0) s_max[tile & 1][threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWrThreads / 32; ++w) mx = max(mx, s_max[tile & 1][w]);
    const float s = wr_scale<E4M3>(mx, old);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;  // 0 for NaN: its codes are 0
    uint8_t* dst = (is_v ? p.c.v : p.c.k) + ((static_cast<int64_t>(page) * p.c.heads + h) << p.c.shift) * p.d;
    if (first > 0 && s > old) {
      // The page's other rows, to the larger scale.
      const float ratio = old / s;
      uint4* w = reinterpret_cast<uint4*>(dst);
      const int lo = first * p.d / 16, hi = (first + rows) * p.d / 16;
      for (int i = threadIdx.x; i < page_size * p.d / 16; i += kWrThreads) {
        if (i < lo || i >= hi) w[i] = wr_again<E4M3>(w[i], ratio);
      }
    }
    dst += first * p.d + tc;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * rpp + tr;
      if (r < rows) *reinterpret_cast<uint2*>(dst + r * p.d) = wr_codes<E4M3>(x[i], inv);
    }
    if (threadIdx.x == 0 && (first == 0 || s != old)) *sp = s;
  }
}

// One row each: d / 8 threads to a (KV head, K | V) row.
template <bool E4M3>
__global__ void __launch_bounds__(kWrThreads) kv_append_kernel(const WrParams p) {
  pdl_trigger();
  pdl_wait();
  if (p.status != nullptr && *p.status != 0) return;
  const int lpr = p.d >> 3;
  const int tile = static_cast<int>(blockIdx.y) * (kWrThreads / lpr) + threadIdx.x / lpr;
  const int tc = threadIdx.x % lpr;
  int slot, len;
  int64_t r0;
  if (wr_rows(p, blockIdx.x, &slot, &r0, &len) == 0) return;
  const int page = kv_page(p.c, slot, (len - 1) >> p.c.shift);
  if (page < 0) return;
  const int users = p.c.ref[page];
  const int first = (len - 1) & ((1 << p.c.shift) - 1);
  const bool live = tile < 2 * p.c.heads, is_v = tile & 1;
  const int h = live ? tile >> 1 : 0;
  const __half* src = (is_v ? p.v_new : p.k_new) + r0 * p.row_pitch + static_cast<int64_t>(h) * p.d + tc * 8;
  const uint4 x = live ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
  float* sp = (is_v ? p.c.vs : p.c.ks) + kv_scale_at(p.c, page, h);
  const float old = live && first > 0 ? *sp : 0.0f;
  if (!wr_own(p, users)) return;
  uint32_t mx = half8_max(x);
  mx = max(mx & 0xffffu, mx >> 16);
  for (int o = 1; o < lpr; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  __syncwarp();
  if (!live) return;
  const float s = wr_scale<E4M3>(mx, old);
  const float inv = s > 0.0f ? 1.0f / s : 0.0f;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + ((static_cast<int64_t>(page) * p.c.heads + h) << p.c.shift) * p.d;
  if (first > 0 && s > old) {
    const float ratio = old / s;
    uint4* w = reinterpret_cast<uint4*>(dst);
    const int lo = first * p.d / 16, hi = (first + 1) * p.d / 16;
    for (int i = tc; i < (p.d << p.c.shift) / 16; i += lpr) {
      if (i < lo || i >= hi) w[i] = wr_again<E4M3>(w[i], ratio);
    }
  }
  *reinterpret_cast<uint2*>(dst + first * p.d + tc * 8) = wr_codes<E4M3>(x, inv);
  if (tc == 0 && (first == 0 || s != old)) *sp = s;
}

template <int PASSES>
int launch_write(const WrParams& p, dim3 grid, bool e4m3, cudaStream_t st) {
  if (e4m3) {
    B200_CUDA(launch_pdl(kv_write_kernel<PASSES, true>, grid, dim3(kWrThreads), 0, st, p));
  } else {
    B200_CUDA(launch_pdl(kv_write_kernel<PASSES, false>, grid, dim3(kWrThreads), 0, st, p));
  }
  return ENGINE_OK;
}

// ---------------------------------------------------------------- bookkeeping
//
// extend and fork hand out free pages (ref == 0), lowest id first.  One CTA does
// the whole call: it claims the slots (the top bit of their lengths, which also
// finds a slot named twice), adds up what they need, and counts the free pages
// before it changes anything, so a call that cannot be met leaves no trace.

constexpr int kBkThreads = 1024;

struct BkParams {
  int32_t* table;
  int32_t* length;
  int32_t* ref;
  int64_t n_pages;
  int64_t max_pages;
  int64_t n_slots;
  int shift;
  const int32_t* a;  // slots / parents
  const int32_t* b;  // n_new / children
  int32_t* status;
  int n;
  int2* pairs;       // fork: pages to copy (from, to)
  int32_t* n_pairs;
  unsigned int* err;
};

constexpr int32_t kClaim = static_cast<int32_t>(0x80000000u);

/// Inclusive sum over the CTA's threads; *total = the sum of all.
__device__ int block_scan(int v, int* total) {
  __shared__ int s_w[kBkThreads / 32];
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane_id() >= o) v += u;
  }
  __syncthreads();  // s_w may still be read from the last call
  if (lane_id() == 31) s_w[warp] = v;
  __syncthreads();
  int w = s_w[lane_id()];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane_id() >= o) w += u;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return v + (warp > 0 ? before : 0);
}

/// The free pages in ascending order: calls take(rank, id) for each with rank <
/// `want`; returns how many there are, counted up to at least `want`.
template <typename F>
__device__ int for_free_pages(const BkParams& p, int want, F take) {
  int run = 0;
  for (int64_t base = 0; base < p.n_pages && run < want; base += kBkThreads) {
    const int64_t id = base + threadIdx.x;
    const bool is_free = id < p.n_pages && p.ref[id] == 0;
    int total;
    const int rank = run + block_scan(is_free ? 1 : 0, &total) - 1;
    if (is_free && rank < want) take(rank, static_cast<int32_t>(id));
    run += total;
  }
  return run;
}

/// Slots' needs in s_start (exclusive sums); the page of rank r belongs to the
/// last i with s_start[i] <= r.
__device__ __forceinline__ int owner_of(const int* s_start, int n, int rank) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_start[mid] <= rank) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

/// Exclusive sums of need(i), i < n, into s_start; returns their total.
template <typename F>
__device__ int sum_needs(int n, int* s_start, F need) {
  int run = 0;
  for (int base = 0; base < n; base += kBkThreads) {
    const int i = base + threadIdx.x;
    const int v = i < n ? need(i) : 0;
    int total;
    const int incl = block_scan(v, &total);
    if (i < n) s_start[i] = run + incl - v;
    run += total;
  }
  __syncthreads();
  return run;
}

__global__ void __launch_bounds__(kBkThreads) kv_extend_kernel(const BkParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int s_start[ENGINE_KV_MAX_SLOTS];
  __shared__ int s_len[ENGINE_KV_MAX_SLOTS];  // length before; -1 where not claimed here
  __shared__ unsigned long long s_need;       // pages, which may be more than 32 bits hold
  if (threadIdx.x == 0) s_need = 0;
  const int64_t cap = p.max_pages << p.shift;
  const int page = 1 << p.shift;
  bool bad = false;
  for (int i = threadIdx.x; i < p.n; i += kBkThreads) {
    const int64_t slot = p.a != nullptr ? p.a[i] : i;
    const int add = p.b[i];
    s_len[i] = -1;
    if (slot < 0 || slot >= p.n_slots || add < 0) {
      bad = true;
      continue;
    }
    const int old = atomicOr(&p.length[slot], kClaim);
    if (old < 0) {
      bad = true;
      continue;
    }
    s_len[i] = old;
    if (static_cast<int64_t>(old) + add > cap) bad = true;
  }
  bad = __syncthreads_or(bad);
  int missing = 0;
  if (!bad) {
    auto need = [&](int i) {
      return ((s_len[i] + p.b[i] + page - 1) >> p.shift) - ((s_len[i] + page - 1) >> p.shift);
    };
    unsigned long long mine = 0;
    for (int i = threadIdx.x; i < p.n; i += kBkThreads) mine += need(i);
    if (mine != 0) atomicAdd(&s_need, mine);
    __syncthreads();
    const int64_t all = static_cast<int64_t>(s_need);
    const int want = static_cast<int>(min(all, p.n_pages + 1));  // enough to count them all
    const int have = for_free_pages(p, want, [](int, int32_t) {});
    if (all > have) missing = static_cast<int>(min(all - have, static_cast<int64_t>(0x7fffffff)));
    else sum_needs(p.n, s_start, need);
    if (missing == 0) {
      for_free_pages(p, want, [&](int rank, int32_t id) {
        const int i = owner_of(s_start, p.n, rank);
        const int64_t slot = p.a != nullptr ? p.a[i] : i;
        const int entry = ((s_len[i] + page - 1) >> p.shift) + rank - s_start[i];
        p.table[slot * p.max_pages + entry] = id;
        p.ref[id] = 1;
      });
    }
  }
  for (int i = threadIdx.x; i < p.n; i += kBkThreads) {
    if (s_len[i] < 0) continue;
    const int64_t slot = p.a != nullptr ? p.a[i] : i;
    p.length[slot] = s_len[i] + (!bad && missing == 0 ? p.b[i] : 0);
  }
  if (threadIdx.x == 0) {
    *p.status = bad ? -1 : missing;
    if (bad) atomicOr(p.err, kErrBadArgument);
  }
}

__global__ void __launch_bounds__(kBkThreads) kv_fork_kernel(const BkParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int s_start[ENGINE_KV_MAX_SLOTS];
  __shared__ int s_len[ENGINE_KV_MAX_SLOTS];  // length of the parent; -1: child not claimed here
  const int page = 1 << p.shift;
  bool bad = false;
  for (int i = threadIdx.x; i < p.n; i += kBkThreads) {
    const int64_t child = p.b[i], parent = p.a[i];
    s_len[i] = -1;
    if (child < 0 || child >= p.n_slots || parent < 0 || parent >= p.n_slots) {
      bad = true;
      continue;
    }
    const int old = atomicOr(&p.length[child], kClaim);
    if (old == 0) s_len[i] = 0;                       // claimed, to be given back
    else if (old > 0) p.length[child] = old;          // not empty (nobody else writes it: others see it claimed)
    if (old != 0) bad = true;
  }
  bad = __syncthreads_or(bad);
  if (!bad) {
    for (int i = threadIdx.x; i < p.n; i += kBkThreads) {
      const int len = __ldcg(&p.length[p.a[i]]);
      if (len < 0 || len > (p.max_pages << p.shift)) bad = true;  // a child, or no length
      else s_len[i] = len;
    }
    bad = __syncthreads_or(bad);
  }
  int missing = 0;
  if (!bad) {
    const int want = sum_needs(p.n, s_start, [&](int i) { return (s_len[i] & (page - 1)) != 0 ? 1 : 0; });
    const int have = for_free_pages(p, want, [](int, int32_t) {});
    missing = want > have ? want - have : 0;
    if (missing == 0) {
      for_free_pages(p, want, [&](int rank, int32_t id) {
        const int i = owner_of(s_start, p.n, rank);
        const int e = s_len[i] >> p.shift;
        const int from = p.table[p.a[i] * p.max_pages + e];
        const bool ok = from >= 0 && from < p.n_pages;
        if (!ok) atomicOr(p.err, kErrBadArgument);
        p.pairs[rank] = make_int2(ok ? from : id, id);
        p.table[p.b[i] * p.max_pages + e] = id;
        p.ref[id] = 1;
      });
      // The full pages, a warp per child.
      for (int i = threadIdx.x >> 5; i < p.n; i += kBkThreads / 32) {
        const int full = s_len[i] >> p.shift;
        for (int e = lane_id(); e < full; e += 32) {
          const int id = p.table[p.a[i] * p.max_pages + e];
          p.table[p.b[i] * p.max_pages + e] = id;
          if (id >= 0 && id < p.n_pages) atomicAdd(&p.ref[id], 1);
          else atomicOr(p.err, kErrBadArgument);
        }
      }
    }
    if (threadIdx.x == 0) *p.n_pairs = missing == 0 ? want : 0;
  } else if (threadIdx.x == 0) {
    *p.n_pairs = 0;
  }
  for (int i = threadIdx.x; i < p.n; i += kBkThreads) {
    if (s_len[i] < 0) continue;
    p.length[p.b[i]] = !bad && missing == 0 ? s_len[i] : 0;
  }
  if (threadIdx.x == 0) {
    *p.status = bad ? -1 : missing;
    if (bad) atomicOr(p.err, kErrBadArgument);
  }
}

/// A warp per slot; whoever takes the length empties the slot.
__global__ void __launch_bounds__(256) kv_free_kernel(const BkParams p) {
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= p.n) return;
  const int64_t slot = p.a != nullptr ? p.a[i] : i;
  if (slot < 0 || slot >= p.n_slots) {
    if (lane_id() == 0) atomicOr(p.err, kErrBadArgument);
    return;
  }
  int len = lane_id() == 0 ? atomicExch(&p.length[slot], 0) : 0;
  len = __shfl_sync(0xffffffffu, len, 0);
  int64_t used = len > 0 ? (static_cast<int64_t>(len) + (1 << p.shift) - 1) >> p.shift : 0;
  if (used > p.max_pages || len < 0) {
    used = used > p.max_pages ? p.max_pages : used;
    if (lane_id() == 0) atomicOr(p.err, kErrBadArgument);
  }
  int32_t* row = p.table + slot * p.max_pages;
  for (int64_t e = lane_id(); e < used; e += 32) {
    const int id = row[e];
    row[e] = -1;
    if (id >= 0 && id < p.n_pages) atomicSub(&p.ref[id], 1);
    else atomicOr(p.err, kErrBadArgument);
  }
}

/// Compaction, the plan (one CTA): the holes below the number of used pages, then
/// the used pages from there on, each moved to the hole of its rank.
__global__ void __launch_bounds__(kBkThreads) kv_compact_kernel(const BkParams p, int32_t* remap,
                                                                 int32_t* holes) {
  pdl_trigger();
  pdl_wait();
  int live = 0;
  for (int64_t id = threadIdx.x; id < p.n_pages; id += kBkThreads) live += p.ref[id] != 0 ? 1 : 0;
  int n_live;
  block_scan(live, &n_live);
  int run = 0;
  for (int64_t base = 0; base < n_live; base += kBkThreads) {
    const int64_t id = base + threadIdx.x;
    const bool hole = id < n_live && p.ref[id] == 0;
    int total;
    const int rank = run + block_scan(hole ? 1 : 0, &total) - 1;
    if (id < n_live) remap[id] = hole ? -1 : static_cast<int32_t>(id);
    if (hole) holes[rank] = static_cast<int32_t>(id);
    run += total;
  }
  __syncthreads();
  run = 0;
  for (int64_t base = n_live; base < p.n_pages; base += kBkThreads) {
    const int64_t id = base + threadIdx.x;
    const int users = id < p.n_pages ? p.ref[id] : 0;
    int total;
    const int rank = run + block_scan(users != 0 ? 1 : 0, &total) - 1;
    if (id < p.n_pages) remap[id] = -1;
    if (users != 0) {
      const int to = holes[rank];
      remap[id] = to;
      p.pairs[rank] = make_int2(static_cast<int>(id), to);
      p.ref[to] = users;
      p.ref[id] = 0;
    }
    run += total;
  }
  if (threadIdx.x == 0) *p.n_pairs = run;
}

// ---------------------------------------------------------------- page copies
//
// A page's codes are contiguous in each layer (all heads): a copy is a block of page_size *
// n_kv_heads * head_dim bytes for each pair, layer and K | V.  CTAs stride over chunks of
// 32 KB, every thread with eight 16-byte loads on their way before it stores.  640 pages in
// 32 layers (1.36 GB read and written): 244 us for the call, the plan and two small copies
// of the caller's in it; with four loads 248, with a ring of bulk copies in shared memory
// 234, but small calls 2 us slower (its 192 KB keep it from starting under its plan).
constexpr int kCpThreads = 256, kCpUnroll = 8;
constexpr int kCpChunk = kCpThreads * kCpUnroll;  // 16-byte words

struct CpParams {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  const int2* pairs;
  const int32_t* n_pairs;
  int64_t n_pages;
  int layers, heads;
  int64_t words;  // 16-byte words of one page in one layer
  // compact: rows to rewrite
  int32_t* table;
  const int32_t* remap;
  int64_t entries;
};

__global__ void __launch_bounds__(kCpThreads) kv_copy_kernel(const CpParams p) {
  pdl_trigger();
  pdl_wait();
  if (p.table != nullptr) {
    const int64_t nt = static_cast<int64_t>(gridDim.x) * kCpThreads;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kCpThreads) + threadIdx.x; i < p.entries; i += nt) {
      const int id = p.table[i];
      if (id >= 0 && id < p.n_pages) p.table[i] = p.remap[id];
    }
  }
  const int64_t chunks = (p.words + kCpChunk - 1) / kCpChunk;  // of a block
  const int64_t total = static_cast<int64_t>(*p.n_pairs) * p.layers * 2 * chunks;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int64_t block = u / chunks, part = u - block * chunks;
    const int64_t pl = block >> 1;
    const int64_t pair = pl / p.layers, layer = pl - pair * p.layers;
    const int2 m = p.pairs[pair];
    const uint4* src = reinterpret_cast<const uint4*>((block & 1) ? p.v : p.k) + (layer * p.n_pages + m.x) * p.words;
    uint4* dst = reinterpret_cast<uint4*>((block & 1) ? p.v : p.k) + (layer * p.n_pages + m.y) * p.words;
    const int64_t w0 = part * kCpChunk + threadIdx.x;
    uint4 x[kCpUnroll];
#pragma unroll
    for (int i = 0; i < kCpUnroll; ++i) {
      if (w0 + i * kCpThreads < p.words) x[i] = __ldcs(src + w0 + i * kCpThreads);
    }
    if (part == 0) {
      float* base = (block & 1) ? p.vs : p.ks;
      for (int h = threadIdx.x; h < p.heads; h += kCpThreads)
        base[(layer * p.n_pages + m.y) * p.heads + h] = base[(layer * p.n_pages + m.x) * p.heads + h];
    }
#pragma unroll
    for (int i = 0; i < kCpUnroll; ++i) {
      if (w0 + i * kCpThreads < p.words) __stcs(dst + w0 + i * kCpThreads, x[i]);
    }
  }
}

BkParams bk_params(const engine_kv_pages_t* kv, const int32_t* a, const int32_t* b, int64_t n) {
  BkParams p = {};
  p.table = kv->table;
  p.length = kv->length;
  p.ref = kv->ref;
  p.n_pages = kv->n_pages;
  p.max_pages = kv->max_pages;
  p.n_slots = kv->n_slots;
  p.shift = kv_view(kv, 0).shift;
  p.a = a;
  p.b = b;
  p.n = static_cast<int>(n);
  p.err = device_error_word();
  return p;
}

int launch_copy(const engine_kv_pages_t* kv, const int2* pairs, const int32_t* n_pairs,
                int64_t most, int32_t* table, const int32_t* remap, cudaStream_t st) {
  CpParams c = {};
  c.k = static_cast<uint8_t*>(kv->k);
  c.v = static_cast<uint8_t*>(kv->v);
  c.ks = kv->k_scale;
  c.vs = kv->v_scale;
  c.pairs = pairs;
  c.n_pairs = n_pairs;
  c.n_pages = kv->n_pages;
  c.layers = static_cast<int>(kv->n_layers);
  c.heads = static_cast<int>(kv->n_kv_heads);
  c.words = kv->n_kv_heads * kv->page_size * kv->head_dim / 16;
  c.table = table;
  c.remap = remap;
  c.entries = table != nullptr ? kv->n_slots * kv->max_pages : 0;
  int64_t blocks = most * kv->n_layers * 2 * ((c.words + kCpChunk - 1) / kCpChunk);
  blocks = std::max(blocks, (c.entries + kCpThreads - 1) / kCpThreads);
  blocks = std::min(blocks, static_cast<int64_t>(sm_count()) * 8);
  B200_CUDA(launch_pdl(kv_copy_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kCpThreads), 0, st, c));
  return ENGINE_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int engine_cuda_kv_pages_write(const engine_kv_pages_t* kv, int64_t layer,
                               const engine_half_t* k_new, const engine_half_t* v_new,
                               int64_t row_pitch, const int32_t* slots, const int32_t* cu_new,
                               int64_t n_seq, int64_t n_tokens, engine_stream_t stream) {
  return engine_cuda_kv_pages_write_if(kv, layer, k_new, v_new, row_pitch, slots, cu_new, n_seq, n_tokens,
                                       nullptr, stream);
}

int engine_cuda_kv_pages_write_if(const engine_kv_pages_t* kv, int64_t layer,
                                  const engine_half_t* k_new, const engine_half_t* v_new,
                                  int64_t row_pitch, const int32_t* slots, const int32_t* cu_new,
                                  int64_t n_seq, int64_t n_tokens, const int32_t* status,
                                  engine_stream_t stream) {
  B200_ENTRY_BEGIN
  if (const int rc = kv_pages_check(kv, layer, "kv_pages_write")) return rc;
  B200_REQUIRE(layer >= 0, "kv_pages_write: layer out of range");
  B200_REQUIRE(n_seq >= 0 && n_tokens >= 0, "kv_pages_write: n_seq and n_tokens must be non-negative");
  B200_REQUIRE(cu_new != nullptr || n_tokens == n_seq,
               "kv_pages_write: n_tokens must be n_seq where cu_new is null");
  B200_REQUIRE(slots != nullptr || n_seq <= kv->n_slots, "kv_pages_write: n_seq > n_slots");
  B200_REQUIRE(row_pitch >= kv->n_kv_heads * kv->head_dim,
               "kv_pages_write: row_pitch < n_kv_heads * head_dim");
  if (n_seq == 0 || n_tokens == 0) return ENGINE_OK;
  B200_REQUIRE(k_new != nullptr && v_new != nullptr, "kv_pages_write: k_new/v_new is null");
  const uintptr_t al = reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new);
  if (al % 16 != 0 || row_pitch % 8 != 0)
    return set_error(ENGINE_ERR_UNSUPPORTED,
                     "kv_pages_write: k_new/v_new must be 16-byte aligned, row_pitch a multiple of 8");
  // Pages that n_tokens rows of n_seq sequences can touch: a sequence's first row
  // and its second one a page each, then one page for every page_size rows.
  int64_t items = n_seq;
  if (cu_new != nullptr) {
    const int64_t most = 2 * n_seq + n_tokens / kv->page_size;
    items = n_tokens < most ? n_tokens : most;
  }
  if (items > 0x7fffffff || n_tokens > 0x7fffffff)
    return set_error(ENGINE_ERR_UNSUPPORTED, "kv_pages_write: n_tokens too large");
  WrParams p = {};
  p.c = kv_view(kv, layer);
  p.k_new = reinterpret_cast<const __half*>(k_new);
  p.v_new = reinterpret_cast<const __half*>(v_new);
  p.row_pitch = row_pitch;
  p.slots = slots;
  p.cu = cu_new;
  p.n_seq = n_seq;
  p.n_tokens = n_tokens;
  p.status = status;
  p.d = static_cast<int>(kv->head_dim);
  const bool e4m3 = kv->type == ENGINE_KV_E4M3;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = ENGINE_OK;
  const int64_t tiles = 2 * kv->n_kv_heads;
  if (cu_new == nullptr) {
    const int64_t per = kWrThreads / (kv->head_dim / 8);
    const dim3 grid(static_cast<unsigned>(items), static_cast<unsigned>((tiles + per - 1) / per));
    B200_CUDA(e4m3 ? launch_pdl(kv_append_kernel<true>, grid, dim3(kWrThreads), 0, st, p)
                   : launch_pdl(kv_append_kernel<false>, grid, dim3(kWrThreads), 0, st, p));
  } else {
    const dim3 grid(static_cast<unsigned>(items), static_cast<unsigned>((tiles + kWrTiles - 1) / kWrTiles));
    const int64_t passes = kv->page_size * kv->head_dim / 1024;  // 1024 elements each
    rc = passes <= 1   ? launch_write<1>(p, grid, e4m3, st)
         : passes <= 2 ? launch_write<2>(p, grid, e4m3, st)
         : passes <= 4 ? launch_write<4>(p, grid, e4m3, st)
         : passes <= 8 ? launch_write<8>(p, grid, e4m3, st)
                       : launch_write<16>(p, grid, e4m3, st);
  }
  if (rc != ENGINE_OK) return rc;
  return check_launch("kv_pages_write");
  B200_ENTRY_END
}

int engine_cuda_kv_pages_extend(const engine_kv_pages_t* kv, const int32_t* slots,
                                const int32_t* n_new, int32_t* status, int64_t n,
                                engine_stream_t stream) {
  B200_ENTRY_BEGIN
  if (const int rc = kv_pages_check(kv, -1, "kv_pages_extend")) return rc;
  B200_REQUIRE(n >= 0, "kv_pages_extend: n must be non-negative");
  B200_REQUIRE(n <= ENGINE_KV_MAX_SLOTS, "kv_pages_extend: n > ENGINE_KV_MAX_SLOTS");
  B200_REQUIRE(slots != nullptr || n <= kv->n_slots, "kv_pages_extend: n > n_slots");
  B200_REQUIRE(status != nullptr, "kv_pages_extend: status is null");
  B200_REQUIRE(n == 0 || n_new != nullptr, "kv_pages_extend: n_new is null");
  BkParams p = bk_params(kv, slots, n_new, n);
  p.status = status;
  B200_CUDA(launch_pdl(kv_extend_kernel, dim3(1), dim3(kBkThreads), 0,
                       static_cast<cudaStream_t>(stream), p));
  return check_launch("kv_pages_extend");
  B200_ENTRY_END
}

int engine_cuda_kv_pages_fork(const engine_kv_pages_t* kv, const int32_t* parents,
                              const int32_t* children, int32_t* status, int64_t n,
                              engine_stream_t stream) {
  B200_ENTRY_BEGIN
  if (const int rc = kv_pages_check(kv, -1, "kv_pages_fork")) return rc;
  B200_REQUIRE(n >= 0, "kv_pages_fork: n must be non-negative");
  B200_REQUIRE(n <= ENGINE_KV_MAX_SLOTS, "kv_pages_fork: n > ENGINE_KV_MAX_SLOTS");
  B200_REQUIRE(status != nullptr, "kv_pages_fork: status is null");
  B200_REQUIRE(n == 0 || (parents != nullptr && children != nullptr),
               "kv_pages_fork: parents/children is null");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(scratch_alloc(16 + n * sizeof(int2), st));
  if (ws == nullptr) return set_error(ENGINE_ERR_CUDA, "kv_pages_fork: workspace allocation failed");
  BkParams p = bk_params(kv, parents, children, n);
  p.status = status;
  p.n_pairs = reinterpret_cast<int32_t*>(ws);
  p.pairs = reinterpret_cast<int2*>(ws + 16);
  int rc = ENGINE_OK;
  const cudaError_t e = launch_pdl(kv_fork_kernel, dim3(1), dim3(kBkThreads), 0, st, p);
  if (e != cudaSuccess) rc = set_cuda_error(e, "kv_fork_kernel");
  if (rc == ENGINE_OK && n > 0) rc = launch_copy(kv, p.pairs, p.n_pairs, n, nullptr, nullptr, st);
  scratch_free(ws, st);
  if (rc != ENGINE_OK) return rc;
  return check_launch("kv_pages_fork");
  B200_ENTRY_END
}

int engine_cuda_kv_pages_free(const engine_kv_pages_t* kv, const int32_t* slots, int64_t n,
                              engine_stream_t stream) {
  B200_ENTRY_BEGIN
  if (const int rc = kv_pages_check(kv, -1, "kv_pages_free")) return rc;
  B200_REQUIRE(n >= 0, "kv_pages_free: n must be non-negative");
  B200_REQUIRE(slots != nullptr || n <= kv->n_slots, "kv_pages_free: n > n_slots");
  if (n == 0) return ENGINE_OK;
  if (n > 0x7fffffff / 32) return set_error(ENGINE_ERR_UNSUPPORTED, "kv_pages_free: n too large");
  const BkParams p = bk_params(kv, slots, nullptr, n);
  B200_CUDA(launch_pdl(kv_free_kernel, dim3(static_cast<unsigned>((n + 7) / 8)), dim3(256), 0,
                       static_cast<cudaStream_t>(stream), p));
  return check_launch("kv_pages_free");
  B200_ENTRY_END
}

int engine_cuda_kv_pages_compact(const engine_kv_pages_t* kv, int32_t* remap,
                                 engine_stream_t stream) {
  B200_ENTRY_BEGIN
  if (const int rc = kv_pages_check(kv, -1, "kv_pages_compact")) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t n = kv->n_pages, half = n / 2 + 1;  // at most half of the pages move
  const size_t bytes = 16 + half * sizeof(int2) + (half + n) * sizeof(int32_t);
  char* ws = static_cast<char*>(scratch_alloc(bytes, st));
  if (ws == nullptr)
    return set_error(ENGINE_ERR_CUDA, "kv_pages_compact: workspace allocation failed");
  BkParams p = bk_params(kv, nullptr, nullptr, 0);
  p.n_pairs = reinterpret_cast<int32_t*>(ws);
  p.pairs = reinterpret_cast<int2*>(ws + 16);
  int32_t* holes = reinterpret_cast<int32_t*>(p.pairs + half);
  if (remap == nullptr) remap = holes + half;
  int rc = ENGINE_OK;
  const cudaError_t e = launch_pdl(kv_compact_kernel, dim3(1), dim3(kBkThreads), 0, st, p, remap, holes);
  if (e != cudaSuccess) rc = set_cuda_error(e, "kv_compact_kernel");
  if (rc == ENGINE_OK) rc = launch_copy(kv, p.pairs, p.n_pairs, half, kv->table, remap, st);
  scratch_free(ws, st);
  if (rc != ENGINE_OK) return rc;
  return check_launch("kv_pages_compact");
  B200_ENTRY_END
}

}  // extern "C"
