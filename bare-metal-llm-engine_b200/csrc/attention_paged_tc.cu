// attention_paged_tc.cu -- attention over the paged 8-bit cache for many query rows
// per KV head (prompts, chunks of prompts) on the 5th-generation tensor cores.
//
// The computation is attention_paged.cu's: weights w_j = 2^(x_j + log2 vs_j - m) with
// the page's scale of V inside, products over the codes alone.  Its bound here is
// arithmetic: 4 d FLOP for each visible (row, key), on tcgen05 in FP16 (codes of both
// types are FP16 numbers), one exponential per (row, key), and the widening of the
// codes -- which is why one CTA takes 256 query rows, so that each code is widened
// once for 256 rows.
//
//   Rows: flat row = token * group + head within the group, so the query heads that
// share a KV head sit in one tile.  A CTA works on items of two tiles (sides A and B)
// of tq = 128 / group tokens each; keys come in tiles of 128.
//   Work split: the key tiles of all items, end to end, are dealt evenly to one CTA
// per SM, whatever the lengths are (they are on the device).  Items that are cut leave
// (m, l, O) in a workspace, and a second kernel joins the parts in order.
//   Warps: 0-3 widen codes (TMA'd bytes in, swizzled FP16 operand tiles out, two
// stages each of K and V); 4-7 and 8-11 are the softmax of side A and B, one thread
// per row; 12 looks up pages and scales and issues the TMA; 13 issues the MMAs; 14 and
// 15 only share their warpgroup's register split.
//   TMEM: S of A and B (128 columns each, overwritten by P as FP16 pairs) and O of A
// and B.  The MMA warp alternates the sides -- P V of the last tile, then S of the
// next -- so that one side's softmax runs under the other side's products.
//
// Every wait is bounded (ENGINE_WAIT_TIMEOUT_MS): on expiry the thread sets the device
// error word, its role ends, the others' waits run out too, and all meet at the
// teardown, where copies and MMAs in flight are waited for.
#include <algorithm>
#include <atomic>

#include "attention_paged.cuh"

namespace b200 {
namespace {

constexpr int kTcThreads = 512;
constexpr int kTcKeys = 128;
constexpr int kTcRows = 256;  // two sides
constexpr float kTcRescale = 8.0f;

template <int D>
struct TcCfg {
  static constexpr int kDH = D / 64;
  static constexpr int kSide = 128 * D * 2;   // one side's Q
  static constexpr int kWide = 128 * D * 2;   // a K or V tile as FP16
  static constexpr int kRaw = 128 * D;        // ... as codes
  static constexpr int kOffK = 2 * kSide;
  static constexpr int kOffV = kOffK + 2 * kWide;
  static constexpr int kOffRaw = kOffV + 2 * kWide;  // K, V
  static constexpr int kOffConst = kOffRaw + 2 * kRaw;
  static constexpr int kOffBar = kOffConst + 4 * 8 * 16;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  static constexpr int kColO = 256;           // S: 0, 128; O: 256, 256 + D
  static_assert(kSmem <= 232448, "shared memory budget");
  // The prefix sums of the prologue use the raw tiles' space.
  static_assert((kTcMaxSeq + 1) * 4 <= 2 * kRaw, "prefix sums");
};

struct TcParams {
  ApParams a;
  int tq;  // tokens per side
};

struct TcItem {
  int b, slot, len, n_tok;
  int64_t first;
  int head, qb;
  int t0, t1, tiles;
  int begin;  // the item's first tile, counted over all items
};

__device__ __forceinline__ int tc_tiles(const TcParams& p, int len, int n_tok, int qb) {
  const int last = min((qb + 1) * 2 * p.tq, n_tok);  // tokens before the item's end
  const int keys = p.a.causal ? len - n_tok + last : len;
  return max((keys + kTcKeys - 1) / kTcKeys, 1);
}

__device__ __forceinline__ void tc_sequence(const TcParams& p, int b, TcItem& it) {
  it.b = b;
  it.slot = kv_slot(p.a.c, p.a.slots, p.a.seq0 + b);
  it.len = kv_length(p.a.c, it.slot);
  it.n_tok = kv_rows(p.a.c, p.a.cu, p.a.seq0 + b, p.a.n_tokens, &it.first);
}

/// Moves on to the item after `it`, whose first tile is at `x` (< the total).
__device__ __forceinline__ void tc_next(const TcParams& p, TcItem& it, int x, int hi) {
  const int nb = (it.n_tok + 2 * p.tq - 1) / (2 * p.tq);
  if (++it.qb >= nb) {
    it.qb = 0;
    if (++it.head >= p.a.c.heads) {
      it.head = 0;
      do {
        tc_sequence(p, it.b + 1, it);
      } while (it.n_tok == 0 && it.b + 1 < p.a.n_seq);
    }
  }
  it.begin = x;
  it.tiles = tc_tiles(p, it.len, it.n_tok, it.qb);
  it.t0 = 0;
  it.t1 = min(it.tiles, hi - x);
}

/// The item at tile x, found by the whole warp.  pre: tiles before each sequence.
__device__ TcItem tc_find(const TcParams& p, const int32_t* pre, int x, int hi) {
  TcItem it;
  int lo = 0, up = p.a.n_seq - 1;
  while (lo < up) {
    const int mid = (lo + up + 1) >> 1;
    if (pre[mid] <= x) lo = mid;
    else up = mid - 1;
  }
  tc_sequence(p, lo, it);
  const int per_head = (pre[lo + 1] - pre[lo]) / p.a.c.heads;
  const int y = x - pre[lo];
  it.head = y / per_head;
  int z = y - it.head * per_head;  // tile among the head's
  const int nb = (it.n_tok + 2 * p.tq - 1) / (2 * p.tq);
  for (int base = 0; base < nb; base += 32) {
    const int qb = base + static_cast<int>(lane_id());
    const int v = qb < nb ? tc_tiles(p, it.len, it.n_tok, qb) : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane_id() >= o) incl += u;
    }
    const unsigned over = __ballot_sync(0xffffffffu, incl > z);
    if (over != 0) {
      const int src = __ffs(over) - 1;
      it.qb = base + src;
      it.tiles = __shfl_sync(0xffffffffu, v, src);
      it.t0 = z - __shfl_sync(0xffffffffu, incl - v, src);
      break;
    }
    z -= __shfl_sync(0xffffffffu, incl, 31);
  }
  it.t1 = min(it.tiles, it.t0 + hi - x);
  it.begin = x - it.t0;
  return it;
}

// Registers a thread: 128 at launch (65536 / 512); the softmax warps take from the rest
// (128 * 96 + 256 * 168 + 128 * 80 = 65536).
constexpr int kRegsWiden = 96, kRegsSoftmax = 168, kRegsOther = 80;
static_assert(128 * kRegsWiden + 256 * kRegsSoftmax + 128 * kRegsOther <= 65536, "register split");
template <int N>
__device__ __forceinline__ void set_max_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_max_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

/// Two FP32 lanes to an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct TcBars {
  uint64_t q_full, q_empty;
  uint64_t raw_full[2], raw_empty[2];  // K, V
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];  // stages
  uint64_t s_full[2], p_full[2], o_done[2], o_free[2];    // sides
  uint64_t drain;
  uint32_t tmem;
};

/// A row's maximum of x + log2 vs over a tile, S read from TMEM 32 columns at a time
/// (the next 32 on their way meanwhile).  MASK: keys from lim on and slices without a
/// page are left out.
template <bool MASK>
__device__ __forceinline__ float tc_row_max(uint32_t tS, const float4* con, int k0, int lim) {
  float mt = -INFINITY;
  uint32_t sv[2][32];
  tmem_ld_32x32b_x32(tS, sv[0]);
#pragma unroll
  for (int c4 = 0; c4 < 4; ++c4) {
    tmem_wait_ld();
    if (c4 < 3) tmem_ld_32x32b_x32(tS + (c4 + 1) * 32, sv[(c4 + 1) & 1]);
    const uint32_t(&v)[32] = sv[c4 & 1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 c = con[c4 * 2 + h];
      if (!MASK) {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          m0 = fmaxf(m0, __uint_as_float(v[h * 16 + e]));
          m1 = fmaxf(m1, __uint_as_float(v[h * 16 + e + 1]));
        }
        mt = fmaxf(mt, fmaf(fmaxf(m0, m1), c.x, c.y));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = fmaf(__uint_as_float(v[h * 16 + e]), c.x, c.y);
          if (k0 + (c4 * 2 + h) * 16 + e < lim && c.w != 0.0f) mt = fmaxf(mt, x);
        }
      }
    }
  }
  return mt;
}

/// The row's weights against the reference `base`, written over S as FP16 pairs (P's
/// columns trail those still to be read); returns the sum of w / vs.
template <bool MASK>
__device__ __forceinline__ float tc_row_weights(uint32_t tS, const float4* con, int k0, int lim, float base) {
  float l = 0.0f;
  uint32_t sv[2][32];
  tmem_ld_32x32b_x32(tS, sv[0]);
#pragma unroll
  for (int c4 = 0; c4 < 4; ++c4) {
    tmem_wait_ld();
    if (c4 < 3) tmem_ld_32x32b_x32(tS + (c4 + 1) * 32, sv[(c4 + 1) & 1]);
    const uint32_t(&v)[32] = sv[c4 & 1];
    uint32_t pk[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 c = con[c4 * 2 + h];
      const uint64_t kc = pack2(c.x, c.x), off = pack2(c.y - base, c.y - base);
      float2 w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e] = unpack2(fma2(pack2(__uint_as_float(v[h * 16 + 2 * e]), __uint_as_float(v[h * 16 + 2 * e + 1])), kc, off));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e].x = ex2_approx(w[e].x);
        w[e].y = ex2_approx(w[e].y);
        if (MASK) {
          const int k = k0 + (c4 * 2 + h) * 16 + 2 * e;
          if (k >= lim || c.w == 0.0f) w[e].x = 0.0f;
          if (k + 1 >= lim || c.w == 0.0f) w[e].y = 0.0f;
        }
      }
      uint64_t s0 = pack2(w[0].x, w[0].y), s1 = pack2(w[1].x, w[1].y);
#pragma unroll
      for (int e = 2; e < 8; e += 2) {
        s0 = add2(s0, pack2(w[e].x, w[e].y));
        s1 = add2(s1, pack2(w[e + 1].x, w[e + 1].y));
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const __half2 u = __floats2half2_rn(w[e].x, w[e].y);
        pk[h * 8 + e] = *reinterpret_cast<const uint32_t*>(&u);
      }
      const float2 t = unpack2(add2(s0, s1));
      const float sum = t.x + t.y;
      l = fmaf(sum, sum != 0.0f ? c.z : 0.0f, l);  // a NaN scale counts only where it is seen
    }
    tmem_st_32x32b_x16(tS + c4 * 16, pk);
  }
  return l;
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const TcParams p) {
  using Cfg = TcCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // [4 tiles][8 slices of 16 keys]: ks scale log2 e, log2 vs, 1 / vs, and whether the
  // slice has a page (0: no; 2: the tile's eight slices all have)
  float4* s_const = reinterpret_cast<float4*>(smem + Cfg::kOffConst);
  TcBars* bar = reinterpret_cast<TcBars*>(smem + Cfg::kOffBar);
  int32_t* s_pre = reinterpret_cast<int32_t*>(smem + Cfg::kOffRaw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvView& c = p.a.c;
  const unsigned long long limit = p.a.limit_ns;

  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    mbar_init(&bar->q_empty, 1);
    mbar_init(&bar->drain, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->raw_full[s], 1);
      mbar_init(&bar->raw_empty[s], 4);
      mbar_init(&bar->k_full[s], 128);
      mbar_init(&bar->k_empty[s], 1);
      mbar_init(&bar->v_full[s], 128);
      mbar_init(&bar->v_empty[s], 1);
      mbar_init(&bar->s_full[s], 1);
      mbar_init(&bar->p_full[s], 128);
      mbar_init(&bar->o_done[s], 1);
      mbar_init(&bar->o_free[s], 128);
    }
    fence_barrier_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 13) {
    tmem_alloc(&bar->tmem, 512);
    tmem_relinquish();
  }
  pdl_trigger();
  pdl_wait();
  // Tiles of each sequence (a warp each), then their sums.
  for (int b = warp; b < p.a.n_seq; b += kTcThreads / 32) {
    TcItem it;
    tc_sequence(p, b, it);
    const int nb = (it.n_tok + 2 * p.tq - 1) / (2 * p.tq);
    int sum = 0;
    for (int qb = lane; qb < nb; qb += 32) sum += tc_tiles(p, it.len, it.n_tok, qb);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) s_pre[b] = sum * c.heads;
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int base = 0; base < p.a.n_seq; base += 32) {
      const int v = base + lane < p.a.n_seq ? s_pre[base + lane] : 0;
      int incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (base + lane < p.a.n_seq) s_pre[base + lane] = run + incl - v;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_pre[p.a.n_seq] = run;
  }
  __syncthreads();
  const int total = s_pre[p.a.n_seq];
  const int per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int lo = min(static_cast<int64_t>(blockIdx.x) * per, static_cast<int64_t>(total));
  const int hi = min(lo + per, total);
  TcItem it = {};
  if (lo < hi) it = tc_find(p, s_pre, lo, hi);
  fence_proxy_async_smem();  // the sums' space becomes TMA's
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem;

  if (warp < 4) {
    // ------------------------------------------------------------- widening
    set_max_regs_dec<kRegsWiden>();
    int n = 0;
    bool ok = true;
    for (int x = lo; x < hi && ok;) {
      for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          const int st = n & 1;
          uint64_t* empty = kv ? &bar->v_empty[st] : &bar->k_empty[st];
          ok = mbar_wait_sleepy(&bar->raw_full[kv], n & 1, limit, c.err);
          ok = ok && mbar_wait_sleepy(empty, ((n >> 1) & 1u) ^ 1u, limit, c.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint8_t* raw = smem + Cfg::kOffRaw + kv * Cfg::kRaw;
          uint8_t* wide = smem + (kv ? Cfg::kOffV : Cfg::kOffK) + st * Cfg::kWide;
          constexpr int CH = D / 16;  // chunks per thread: its warp's 32 keys, 8 at a time
          uint4 w[CH];
          int key[CH], ch[CH];
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            // Eight lanes read and write all 32 banks: for d = 128 they take one half of a
            // row each of two keys, for d = 64 two whole rows.
            if constexpr (D == 128) {
              key[i] = warp * 32 + (i >> 1) * 8 + (lane >> 2);
              ch[i] = (lane & 3) + 4 * (((lane >> 2) ^ i) & 1);
              w[i] = *reinterpret_cast<const uint4*>(raw + key[i] * 128 + ((ch[i] ^ (key[i] & 7)) << 4));
            } else {
              key[i] = warp * 32 + i * 8 + (lane >> 2);
              ch[i] = lane & 3;
              const int line = key[i] >> 1;
              w[i] = *reinterpret_cast<const uint4*>(
                  raw + line * 128 + (((((key[i] & 1) << 2) | ch[i]) ^ (line & 7)) << 4));
            }
          }
          const float4* con = s_const + (n & 3) * 8;
          if (E4M3 && kv && ((t + 1) * kTcKeys > it.len || con[0].w != 2.0f)) {
            // Bytes that are no sequence's may be NaN, which a weight of 0 would not silence.
#pragma unroll
            for (int i = 0; i < CH; ++i) {
              if (t * kTcKeys + key[i] >= it.len || con[key[i] >> 4].w == 0.0f) w[i] = make_uint4(0, 0, 0, 0);
            }
          }
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            uint4 h0, h1;
            codes_to_half4<E4M3>(w[i].x, h0.x, h0.y);
            codes_to_half4<E4M3>(w[i].y, h0.z, h0.w);
            codes_to_half4<E4M3>(w[i].z, h1.x, h1.y);
            codes_to_half4<E4M3>(w[i].w, h1.z, h1.w);
            // K: [64 elements][128 keys]; V: [64 keys][64 elements][64 keys] blocks of 128-byte rows.
            uint8_t* row = wide + (kv ? (key[i] >> 6) * (Cfg::kDH * 8192) + (ch[i] >> 2) * 8192 + (key[i] & 63) * 128
                                      : (ch[i] >> 2) * 16384 + key[i] * 128);
            const int q = (ch[i] & 3) * 2;
            *reinterpret_cast<uint4*>(row + ((q ^ (key[i] & 7)) << 4)) = h0;
            *reinterpret_cast<uint4*>(row + (((q + 1) ^ (key[i] & 7)) << 4)) = h1;
          }
          fence_proxy_async_smem();
          mbar_arrive(kv ? &bar->v_full[st] : &bar->k_full[st]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->raw_empty[kv]);
        }
      }
      x += it.t1 - it.t0;
      if (x < hi) tc_next(p, it, x, hi);
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- softmax
    set_max_regs_inc<kRegsSoftmax>();
    const int side = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the side's tile, TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + side * 128;
    const uint32_t tO = tmem + lane_base + Cfg::kColO + side * D;
    int n = 0;
    bool ok = true;
    for (int x = lo; x < hi && ok;) {
      const int tok = (it.qb * 2 + side) * p.tq + r / p.a.group;
      const bool row = r < p.tq * p.a.group && tok < it.n_tok;
      const int lim = row && p.a.causal ? it.len - it.n_tok + tok + 1 : it.len;
      float m = -INFINITY, l = 0.0f;
      for (int t = it.t0; t < it.t1; ++t, ++n) {
        ok = __all_sync(0xffffffffu, mbar_wait_sleepy(&bar->s_full[side], n & 1, limit, c.err));
        if (!ok) break;
        tc_fence_after();
        const float4* con = s_const + (n & 3) * 8;
        const int k0 = t * kTcKeys;
        const bool clean = __all_sync(0xffffffffu, k0 + kTcKeys <= lim && con[0].w == 2.0f);
        const float mt = clean ? tc_row_max<false>(tS, con, k0, lim) : tc_row_max<true>(tS, con, k0, lim);
        // Lazy rescaling: the row keeps its reference until the maximum passes it by 2^8.
        const bool first = m == -INFINITY;
        const bool rescale = !first && mt > m + kTcRescale;
        const float m_new = first || rescale ? fmaxf(m, mt) : m;
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = first ? 1.0f : ex2_approx(m - base);
        if (__any_sync(0xffffffffu, rescale)) {
          // P V of the tile before is complete: s_full was committed behind it.
#pragma unroll 1
          for (int i = 0; i < D / 32; ++i) {
            uint32_t ov[32];
            tmem_ld_32x32b_x32(tO + i * 32, ov);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st_32x32b_x32(tO + i * 32, ov);
          }
        }
        m = m_new;
        const float ls = clean ? tc_row_weights<false>(tS, con, k0, lim, base)
                               : tc_row_weights<true>(tS, con, k0, lim, base);
        l = fmaf(l, alpha, ls);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar->p_full[side]);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait_sleepy(&bar->o_done[side], (n - 1) & 1, limit, c.err));
      if (!ok) break;
      tc_fence_after();
      const bool whole = it.t1 - it.t0 == it.tiles;
      const int64_t at = (it.first + tok) * p.a.n_heads + it.head * p.a.group + r % p.a.group;
      const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (it.t0 != 0 ? 0 : 1)) * kTcRows + side * 128 + r;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t ov[32];
        tmem_ld_32x32b_x32(tO + i * 32, ov);
        tmem_wait_ld();
        if (row && whole) {
          uint4* dst = reinterpret_cast<uint4*>(p.a.out + at * D + i * 32);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            __half2 h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              h[e] = __floats2half2_rn(__uint_as_float(ov[8 * q + 2 * e]) * inv,
                                       __uint_as_float(ov[8 * q + 2 * e + 1]) * inv);
            dst[q] = *reinterpret_cast<const uint4*>(h);
          }
        } else if (row) {
          uint4* dst = reinterpret_cast<uint4*>(p.a.ws_o + part * D + i * 32);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            dst[q] = make_uint4(ov[4 * q], ov[4 * q + 1], ov[4 * q + 2], ov[4 * q + 3]);
        }
      }
      if (row && whole && p.a.lse != nullptr)
        p.a.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
      if (row && !whole) p.a.ws_ml[part] = make_float2(m, l);
      tc_fence_before();
      mbar_arrive(&bar->o_free[side]);
      x += it.t1 - it.t0;
      if (x < hi) tc_next(p, it, x, hi);
    }
  } else {
    set_max_regs_dec<kRegsOther>();
    if (warp == 12) {
      // ----------------------------------------------------- lookups and TMA
      int n = 0, items = 0;
      bool ok = true;
      int4 cut = make_int4(-1, 0, 0, 0);
      const int per_box = min(4, 1 << (c.shift - 4));  // slices of 16 keys in a TMA box
      for (int x = lo; x < hi && ok; ++items) {
        if (it.t0 == 0 && it.t1 < it.tiles)
          cut = make_int4(it.b, it.qb, it.head, (it.begin + it.tiles - 1) / per);
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->q_empty, (items & 1) ^ 1u, limit, c.err));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bar->q_full, 2 * Cfg::kDH * p.tq * p.a.group * 128);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int dh = 0; dh < Cfg::kDH; ++dh)
              tma_load_3d(smem + s * Cfg::kSide + dh * 16384, &tmQ, &bar->q_full, dh * 64, it.head * p.a.group,
                          static_cast<int32_t>(it.first) + (it.qb * 2 + s) * p.tq);
          }
        }
        __syncwarp();
        // Slices of 16 keys: lane i of a batch has slice first + i; four tiles to a batch.
        const int end_slice = min(it.t1 * 8, (it.len + 15) >> 4);
        auto page_of = [&](int slice) {
          return slice < end_slice ? kv_page(c, it.slot, (slice << 4) >> c.shift) : -1;
        };
        int id = page_of(it.t0 * 8 + lane);
        for (int base = it.t0; base < it.t1 && ok; base += 4) {
          const int next = page_of((base + 4) * 8 + lane);
          float4 con = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
          if (id >= 0) {
            const float ks = c.ks[kv_scale_at(c, id, it.head)];
            float vs = c.vs[kv_scale_at(c, id, it.head)];
            if (vs == 0.0f) vs = 1.0f;
            con = make_float4(ks * p.a.scale_log2, log2f(vs), 1.0f / vs, 1.0f);
          }
          const unsigned valid = __ballot_sync(0xffffffffu, id >= 0);
          for (int i = 0; i < 4 && base + i < it.t1 && ok; ++i, ++n) {
            const int slice = lane & 7;
            const bool mine = (lane >> 3) == i && id >= 0 && slice % per_box == 0;
            const unsigned who = __ballot_sync(0xffffffffu, mine);
            float4 con_i = con;
            if (((valid >> (8 * i)) & 0xffu) == 0xffu) con_i.w = 2.0f;
            const int key = (base + i) * kTcKeys + slice * 16;
            const int row = mine ? ((id * c.heads + it.head) << c.shift) + (key & ((1 << c.shift) - 1)) : 0;
            for (int kv = 0; kv < 2; ++kv) {
              ok = __all_sync(0xffffffffu, mbar_wait(&bar->raw_empty[kv], (n & 1) ^ 1u, limit, c.err));
              if (!ok) break;
              if (kv == 0 && (lane >> 3) == i) s_const[(n & 3) * 8 + slice] = con_i;
              __syncwarp();
              if (lane == 0) mbar_arrive_expect_tx(&bar->raw_full[kv], __popc(who) * per_box * 16 * D);
              __syncwarp();
              if (mine)
                tma_load_2d(smem + Cfg::kOffRaw + kv * Cfg::kRaw + slice * 16 * D, kv ? &tmV : &tmK,
                            &bar->raw_full[kv], 0, D == 128 ? row : row >> 1);
            }
            if (!ok) break;
          }
          id = next;
        }
        x += it.t1 - it.t0;
        if (x < hi) tc_next(p, it, x, hi);
      }
      if (lane == 0) p.a.cut[blockIdx.x] = cut;
      // No copy may still be writing shared memory when the CTA leaves: what was issued last.
      if (items > 0) mbar_wait(&bar->q_full, (items - 1) & 1, limit, c.err);
      if (n > 0) {
        mbar_wait(&bar->raw_full[0], (n - 1) & 1, limit, c.err);
        mbar_wait(&bar->raw_full[1], (n - 1) & 1, limit, c.err);
      }
      __syncwarp();
    } else if (warp == 13 && lane == 0) {
      // ----------------------------------------------------------------- MMA
      constexpr uint32_t kIdescS = umma_idesc_f16(128, kTcKeys, false, false, false);
      constexpr uint32_t kIdescO = umma_idesc_f16(128, D, false, false, true);
      int n = 0, items = 0;
      bool ok = true;
      bool busy = false;  // something was issued
      auto s_mma = [&](int side) {
        const uint32_t qa = smem_u32(smem + side * Cfg::kSide);
        const uint32_t ka = smem_u32(smem + Cfg::kOffK + (n & 1) * Cfg::kWide);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t ad = umma_desc_sw128(qa + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024);
          const uint64_t bd = umma_desc_sw128(ka + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024);
          umma_f16(tmem + side * 128, ad, bd, kIdescS, kk > 0 ? 1u : 0u);
        }
        umma_commit(&bar->s_full[side]);
      };
      auto pv_mma = [&](int side, int i, bool start) {  // O += P V of tile i
        const uint32_t va = smem_u32(smem + Cfg::kOffV + (i & 1) * Cfg::kWide);
#pragma unroll
        for (int kk = 0; kk < kTcKeys / 16; ++kk) {
          const uint64_t bd =
              umma_desc_sw128(va + (kk >> 2) * (Cfg::kDH * 8192) + (kk & 3) * 2048, 8192, 1024);
          umma_f16_ts(tmem + Cfg::kColO + side * D, tmem + side * 128 + kk * 8, bd, kIdescO,
                      (start && kk == 0) ? 0u : 1u);
        }
        umma_commit(&bar->o_done[side]);
      };
      for (int x = lo; x < hi && ok; ++items) {
        ok = mbar_wait(&bar->q_full, items & 1, limit, c.err);
        for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
          ok = mbar_wait(&bar->k_full[n & 1], (n >> 1) & 1, limit, c.err);
          if (ok && t > it.t0) ok = mbar_wait(&bar->v_full[(n - 1) & 1], ((n - 1) >> 1) & 1, limit, c.err);
          for (int side = 0; side < 2 && ok; ++side) {
            if (t > it.t0) {
              ok = mbar_wait(&bar->p_full[side], (n - 1) & 1, limit, c.err);
              // The first product of an item overwrites O: the last item's rows have been read.
              if (ok && t == it.t0 + 1) ok = mbar_wait(&bar->o_free[side], (items & 1) ^ 1u, limit, c.err);
              if (!ok) break;
              tc_fence_after();
              pv_mma(side, n - 1, t == it.t0 + 1);
              busy = true;
              if (side == 1) umma_commit(&bar->v_empty[(n - 1) & 1]);
            }
            // S goes over P of the tile before: its product must have read it.
            if (n > 0) ok = mbar_wait(&bar->o_done[side], (n - 1) & 1, limit, c.err);
            if (!ok) break;
            tc_fence_after();
            s_mma(side);
            busy = true;
          }
          if (ok) umma_commit(&bar->k_empty[n & 1]);
        }
        if (!ok) break;
        umma_commit(&bar->q_empty);
        // The item's last tile.
        const bool start = it.t1 - it.t0 == 1;
        ok = mbar_wait(&bar->v_full[(n - 1) & 1], ((n - 1) >> 1) & 1, limit, c.err);
        for (int side = 0; side < 2 && ok; ++side) {
          ok = mbar_wait(&bar->p_full[side], (n - 1) & 1, limit, c.err);
          if (ok && start) ok = mbar_wait(&bar->o_free[side], (items & 1) ^ 1u, limit, c.err);
          if (!ok) break;
          tc_fence_after();
          pv_mma(side, n - 1, start);
          busy = true;
        }
        if (ok) umma_commit(&bar->v_empty[(n - 1) & 1]);
        x += it.t1 - it.t0;
        if (x < hi) tc_next(p, it, x, hi);
      }
      // No MMA may still use TMEM or shared memory when the CTA leaves.
      if (busy) {
        umma_commit(&bar->drain);
        mbar_wait(&bar->drain, 0, limit, c.err);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

/// Joins the parts of the item that CTA blockIdx.x began and did not finish (see
/// ApParams): 8 rows a block, D / 4 threads a row.
template <int D>
__global__ void __launch_bounds__(2 * D) attn_paged_tc_join_kernel(const TcParams p) {
  pdl_trigger();
  pdl_wait();
  const int4 cut = p.a.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int flat = blockIdx.y * 8 + threadIdx.x / (D / 4), col = threadIdx.x % (D / 4) * 4;
  const int side = flat >> 7, r = flat & 127;
  int64_t first;
  const int n_tok = kv_rows(p.a.c, p.a.cu, p.a.seq0 + cut.x, p.a.n_tokens, &first);
  const int tok = (cut.y * 2 + side) * p.tq + r / p.a.group;
  if (r >= p.tq * p.a.group || tok >= n_tok) return;
  const int parts = cut.w - static_cast<int>(blockIdx.x) + 1;
  auto part = [&](int i) {
    return (static_cast<int64_t>(blockIdx.x) * 2 + (i == 0 ? 1 : 2 * i)) * kTcRows + flat;
  };
  float m = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) m = fmaxf(m, p.a.ws_ml[part(i)].x);
  float l = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 2
  for (int i = 0; i < parts; ++i) {
    const float2 ml = p.a.ws_ml[part(i)];
    // A part without a visible key has m = -inf, l = 0 and o = 0 (or NaN in all: kept).
    const float a = ml.x == -INFINITY ? 1.0f : ex2_approx(ml.x - m);
    const float4 u = *reinterpret_cast<const float4*>(p.a.ws_o + part(i) * D + col);
    l = fmaf(ml.y, a, l);
    o = make_float4(fmaf(u.x, a, o.x), fmaf(u.y, a, o.y), fmaf(u.z, a, o.z), fmaf(u.w, a, o.w));
  }
  const int64_t at = (first + tok) * p.a.n_heads + cut.z * p.a.group + r % p.a.group;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const __half2 h[2] = {__floats2half2_rn(o.x * inv, o.y * inv), __floats2half2_rn(o.z * inv, o.w * inv)};
  *reinterpret_cast<uint2*>(p.a.out + at * D + col) = *reinterpret_cast<const uint2*>(h);
  if (p.a.lse != nullptr && col == 0)
    p.a.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <int D, bool E4M3>
int launch_tc(TcParams p, const engine_kv_pages_t* kv, int64_t most_tiles, cudaStream_t st) {
  using Cfg = TcCfg<D>;
  auto kern = attn_paged_tc_kernel<D, E4M3>;
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  B200_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if ((configured.load() & bit) == 0) {
    B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    configured.fetch_or(bit);
  }
  CUtensorMap tq, tk, tv;
  const uint64_t rows = static_cast<uint64_t>(kv->n_pages * kv->n_kv_heads * kv->page_size) * D / 128;
  const uint32_t box = static_cast<uint32_t>(kv->page_size < 64 ? kv->page_size : 64) * D / 128;
  if (!make_tmap_2d(&tk, p.a.c.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, 128, 128, box, 128) ||
      !make_tmap_2d(&tv, p.a.c.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, 128, 128, box, 128))
    return ENGINE_ERR_CUDA;
  const uint64_t dims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.n_heads),
                            static_cast<uint64_t>(p.a.n_tokens)};
  const uint64_t strides[2] = {static_cast<uint64_t>(D), static_cast<uint64_t>(p.a.q_pitch)};
  const uint32_t qbox[3] = {64, static_cast<uint32_t>(p.a.group), static_cast<uint32_t>(p.tq)};
  if (!make_tmap_3d(&tq, p.a.q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, dims, strides, qbox)) return ENGINE_ERR_CUDA;
  const int64_t ctas = std::min<int64_t>(sm_count(), most_tiles);
  const size_t o_bytes = 2 * ctas * kTcRows * D * sizeof(float), ml_bytes = 2 * ctas * kTcRows * sizeof(float2);
  char* ws = static_cast<char*>(scratch_alloc(o_bytes + ml_bytes + ctas * sizeof(int4), st));
  if (ws == nullptr)
    return set_error(ENGINE_ERR_CUDA, "attention_paged_prefill: workspace allocation failed");
  p.a.ws_o = reinterpret_cast<float*>(ws);
  p.a.ws_ml = reinterpret_cast<float2*>(ws + o_bytes);
  p.a.cut = reinterpret_cast<int4*>(ws + o_bytes + ml_bytes);
  int rc = ENGINE_OK;
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(ctas)), dim3(kTcThreads), Cfg::kSmem, st, tq, tk, tv, p);
  if (e == cudaSuccess)
    e = launch_pdl(attn_paged_tc_join_kernel<D>, dim3(static_cast<unsigned>(ctas), kTcRows / 8), dim3(2 * D), 0, st, p);
  if (e != cudaSuccess) rc = set_cuda_error(e, "attn_paged_tc_kernel");
  scratch_free(ws, st);
  return rc;
}

}  // namespace

int attention_paged_tc(const ApParams& a, const engine_kv_pages_t* kv, cudaStream_t st) {
  TcParams p;
  p.a = a;
  p.tq = 128 / a.group;
  // At most this many tiles (the kernel counts them in 32 bits).
  const int64_t tiles = std::max<int64_t>((kv->max_pages * kv->page_size + kTcKeys - 1) / kTcKeys, 1);
  const int64_t blocks = a.n_tokens / (2 * p.tq) + a.n_seq;
  if (blocks > 0x7fffffff / kv->n_kv_heads / tiles)
    return set_error(ENGINE_ERR_UNSUPPORTED, "attention_paged_prefill: too many query rows x positions");
  const int64_t most = blocks * kv->n_kv_heads * tiles;
  const bool e4m3 = kv->type == ENGINE_KV_E4M3;
  if (kv->head_dim == 64) return e4m3 ? launch_tc<64, true>(p, kv, most, st) : launch_tc<64, false>(p, kv, most, st);
  return e4m3 ? launch_tc<128, true>(p, kv, most, st) : launch_tc<128, false>(p, kv, most, st);
}

}  // namespace b200
