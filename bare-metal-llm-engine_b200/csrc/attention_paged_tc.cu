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
// stages each of K and V); 4-11 and 12-19 are the softmax of side A and B, four threads
// to a row; 20 looks up pages and scales and issues the TMA; 21 and 22 issue the MMAs of
// side A and B; 23 only shares its warpgroup's register split.
//   TMEM: S of A and B (128 columns each, overwritten by P as FP16 pairs) and O of A
// and B.  Within a side, S -> softmax -> P V is a chain; the two sides' chains interleave
// on the tensor cores and the exponential units.
//
//   Measured (B200, 32 / 8 heads of 128, calls back to back): 512 rows on 8704 keys 95 us (745
// TFLOP/s, 0.45 of the measured burst), a 4096-token prompt 180 us.  A side's chain bounds
// it: of about 4100 cycles a tile, 700 are the maxima, 1700 the weights (exponentials 512 of
// each half's 850), 1600 from the last weight to the next tile's S.  Steps: one thread a row
// with S in 128 registers 117 us; four threads a row 135; one MMA thread for both sides, whose
// issue was the bound, to a warp a side and descriptors that differ by constants 119; the
// sides' turns and the maxima before them 93; the first half's scores kept 92 to 94.  Without
// the turns 102; four prompts of 700-5000 tokens 405 without, 390 to 404 with them.  The 80
// registers at launch spill (460 to 596 bytes of stores, by -Xptxas -v): 1.4 % of the chunk's
// instructions.
//
// Every wait is bounded (ENGINE_WAIT_TIMEOUT_MS): on expiry the warp sets the device
// error word, its role ends, the others' waits run out too, and all meet at the
// teardown, where copies and MMAs in flight are waited for (by a limit of their own).
// Rows whose products are not complete are not stored, nor joined.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attention_paged.cuh"

namespace b200 {
namespace {

constexpr int kTcThreads = 768;
constexpr int kTcKeys = 128;
constexpr int kTcRows = 256;  // two sides
constexpr float kTcRescale = 14.0f;  // weights stay below 2^14 (FP16 ends at 2^16)

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

/// What an item costs beside its key tiles (its Q, the first tile's chain, O's way out;
/// about 7000 cycles against 4000 a tile), in tiles: the even shares count it, as steps in
/// front of the item's tiles in which nothing is done.
constexpr int kTcItemCost = 2;

struct TcItem {
  int b, slot, len, n_tok, nb;  // nb: the sequence's items per head
  int64_t first;
  int head, qb;
  int t0, t1, tiles;
  int begin;  // the item's first step, counted over all items
  bool two;   // side B has rows
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
  it.nb = (it.n_tok + 2 * p.tq - 1) / (2 * p.tq);
}

/// The tiles that the steps from x on, before hi, have of the item.
__device__ __forceinline__ void tc_range(const TcParams& p, TcItem& it, int x, int hi) {
  it.two = (it.qb * 2 + 1) * p.tq < it.n_tok;
  it.t0 = max(x - it.begin - kTcItemCost, 0);
  it.t1 = max(min(hi - it.begin - kTcItemCost, it.tiles), it.t0);
}
/// The step behind the item's part.
__device__ __forceinline__ int tc_end(const TcItem& it) { return it.begin + kTcItemCost + it.t1; }

/// Moves on to the item after `it`, whose first step is x (< the total).
__device__ __forceinline__ void tc_next(const TcParams& p, TcItem& it, int x, int hi) {
  if (++it.qb >= it.nb) {
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
  tc_range(p, it, x, hi);
}

/// The item at step x, found by the whole warp.  pre: steps before each sequence.
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
  int z = y - it.head * per_head;  // step among the head's
  for (int base = 0; base < it.nb; base += 32) {
    const int qb = base + static_cast<int>(lane_id());
    const int v = qb < it.nb ? kTcItemCost + tc_tiles(p, it.len, it.n_tok, qb) : 0;
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
      it.tiles = __shfl_sync(0xffffffffu, v, src) - kTcItemCost;
      it.begin = x - (z - __shfl_sync(0xffffffffu, incl - v, src));
      break;
    }
    z -= __shfl_sync(0xffffffffu, incl, 31);
  }
  tc_range(p, it, x, hi);
  return it;
}

// Registers a thread: 80 at launch (65536 / 768, in eights); the softmax warps take from
// the rest (128 * 72 + 512 * 88 + 128 * 56 = 768 * 80).
constexpr int kRegsWiden = 72, kRegsSoftmax = 88, kRegsOther = 56;
static_assert(128 * kRegsWiden + 512 * kRegsSoftmax + 128 * kRegsOther <= kTcThreads * 80, "register split");
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
  uint64_t s_full[2], p_full[2][2];                       // sides, halves of 64 keys
  uint64_t o_done[2], o_free[2], drain[2];                // sides
  uint64_t a_turn;                                        // A's weights, in items with a side B
  uint32_t tmem;
};
static_assert(sizeof(TcBars) <= 256, "space of the barriers");

/// A softmax warp has 16 rows of a side; a thread two of them (lane / 4 and + 8) and, of
/// every 8 columns, 2 (lane % 4) and the next: 32 values of a half tile of 64 keys, in
/// v[4 (column / 8) + 2 r + {0, 1}].  KG keys share their constants.
///
/// tc_half_load reads S.  In a tile that masks something (`clean` false) it makes x + log2 vs
/// of it, -inf from key lim[r] on; con_of then gives the constants that leave that alone.
template <int KG>
__device__ __forceinline__ void tc_half_load(uint32_t taddr, const float4* con, int key, const int (&lim)[2],
                                             bool clean, uint32_t (&v)[32]) {
  tmem_ld_16x256b_x8(taddr, v);
  tmem_wait_ld();
  if (!clean) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 c = con[j / 2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = fmaf(__uint_as_float(v[4 * j + 2 * r + e]), c.x, c.y);
          v[4 * j + 2 * r + e] = __float_as_uint(key + 8 * j + e < lim[r] ? x : -INFINITY);
        }
      }
    }
    __syncwarp();
  }
}
__device__ __forceinline__ float4 con_of(const float4& c, bool clean) {
  return clean ? c : make_float4(1.0f, 0.0f, c.z, c.w);
}

/// The rows' maxima of x + log2 vs.
template <int KG>
__device__ __forceinline__ void tc_half_max(const uint32_t (&v)[32], const float4* con, bool clean, float (&mt)[2]) {
#pragma unroll
  for (int gi = 0; gi < 64 / KG; ++gi) {
    const float4 c = con_of(con[gi * (KG / 16)], clean);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = gi * (KG / 8); j < (gi + 1) * (KG / 8); ++j)
        mx = fmaxf(mx, fmaxf(__uint_as_float(v[4 * j + 2 * r]), __uint_as_float(v[4 * j + 2 * r + 1])));
      mt[r] = fmaxf(mt[r], fmaf(mx, c.x, c.y));
    }
  }
}

/// The weights against the references m, as FP16 pairs (see attention_paged.cu) in the order of
/// tmem_st_16x128b_x8; adds the thread's w / vs to l, before that rounding.
template <int KG>
__device__ __forceinline__ void tc_half_weights(const uint32_t (&v)[32], const float4* con, bool clean,
                                                const float (&m)[2], float (&l)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (int gi = 0; gi < 64 / KG; ++gi) {
    const float4 c = con_of(con[gi * (KG / 16)], clean);
    const uint64_t kc = pack2(c.x, c.x);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float d = c.y - (m[r] == -INFINITY ? 0.0f : m[r]);
      const uint64_t off = pack2(d, d);
      uint64_t sum = 0;
#pragma unroll
      for (int j = gi * (KG / 8); j < (gi + 1) * (KG / 8); ++j) {
        float2 w = unpack2(fma2(pack2(__uint_as_float(v[4 * j + 2 * r]), __uint_as_float(v[4 * j + 2 * r + 1])), kc, off));
        w.x = ex2_approx(w.x);
        w.y = ex2_approx(w.y);
        sum = add2(sum, pack2(w.x, w.y));
        const __half2 u = __floats2half2_rn(w.x, w.y);
        pk[2 * j + r] = *reinterpret_cast<const uint32_t*>(&u);
      }
      const float2 s2 = unpack2(sum);
      const float s = s2.x + s2.y;
      l[r] = fmaf(s, s != 0.0f ? c.z : 0.0f, l[r]);  // a NaN scale counts only where it is seen
    }
  }
}

/// 4 x 4 transpose over the four lanes of a row: lane t's r[j] goes to lane j's r[t].
__device__ __forceinline__ void transpose4(uint32_t (&r)[4], int t) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {  // with lane t ^ 1
    const uint32_t u = __shfl_xor_sync(0xffffffffu, (t & 1) ? r[i] : r[i + 1], 1);
    if (t & 1) r[i] = u;
    else r[i + 1] = u;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // with lane t ^ 2
    const uint32_t u = __shfl_xor_sync(0xffffffffu, (t & 2) ? r[i] : r[i + 2], 2);
    if (t & 2) r[i] = u;
    else r[i + 2] = u;
  }
}

template <int D, bool E4M3, int KG>
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
    mbar_init(&bar->q_empty, 2);
    mbar_init(&bar->a_turn, 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar->raw_full[s], 1);
      mbar_init(&bar->raw_empty[s], 4);
      mbar_init(&bar->k_full[s], 128);
      mbar_init(&bar->k_empty[s], 2);
      mbar_init(&bar->v_full[s], 128);
      mbar_init(&bar->v_empty[s], 2);
      mbar_init(&bar->drain[s], 1);
      mbar_init(&bar->s_full[s], 1);
      mbar_init(&bar->p_full[s][0], 256);
      mbar_init(&bar->p_full[s][1], 256);
      mbar_init(&bar->o_done[s], 1);
      mbar_init(&bar->o_free[s], 256);
    }
    fence_barrier_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 21) {
    tmem_alloc(&bar->tmem, 512);
    tmem_relinquish();
  }
  pdl_trigger();
  pdl_wait();
  // Its two parts are not stored yet.
  if (threadIdx.x < 2 * kTcRows) p.a.ws_ml[blockIdx.x * (2 * kTcRows) + threadIdx.x] = make_float2(-INFINITY, kNoPart);
  static_assert(2 * kTcRows <= kTcThreads, "a mark a thread");
  // Steps of each sequence (a warp each), then their sums.  A CTA's share can end within an
  // item's leading steps: it then has no tile of it (t0 == t1), and nothing behind it either.
  for (int b = warp; b < p.a.n_seq; b += kTcThreads / 32) {
    TcItem it;
    tc_sequence(p, b, it);
    int sum = 0;
    for (int qb = lane; qb < it.nb; qb += 32) sum += kTcItemCost + tc_tiles(p, it.len, it.n_tok, qb);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) s_pre[b] = sum * c.heads;
  }
  __syncthreads();
  if (warp == 0) {
    unsigned run = 0;
    int64_t all = 0;
    for (int base = 0; base < p.a.n_seq; base += 32) {
      const int v = base + lane < p.a.n_seq ? s_pre[base + lane] : 0;
      unsigned incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (base + lane < p.a.n_seq) s_pre[base + lane] = static_cast<int>(run + incl - v);
      run += __shfl_sync(0xffffffffu, incl, 31);
      all += kv_wide_sum(v);
    }
    if (lane == 0) s_pre[p.a.n_seq] = kv_total(c, all);
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
    for (int x = lo; x < hi && ok && it.t0 < it.t1;) {
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
          if (E4M3 && ((t + 1) * kTcKeys > it.len || con[0].w != 2.0f)) {
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
      x = tc_end(it);
      if (x < hi) tc_next(p, it, x, hi);
    }
  } else if (warp < 20) {
    // -------------------------------------------------------------- softmax
    set_max_regs_inc<kRegsSoftmax>();
    const int side = (warp - 4) >> 3;
    const int r0 = (warp & 3) * 32 + ((warp - 4) >> 2 & 1) * 16;  // the warp's first row of the side's tile
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t tS = tmem + (static_cast<uint32_t>(r0) << 16) + side * 128;
    const uint32_t tO = tmem + (static_cast<uint32_t>(r0) << 16) + Cfg::kColO + side * D;
    int n = 0, own = 0, both = 0;  // tiles, those of this side, and those with a side B
    bool ok = true;
    // Token within the side's, or far past any, and head within the group of the thread's rows.
    int q_tok[2], q_head[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int q = r0 + g + 8 * r;
      q_tok[r] = q < p.tq * p.a.group ? q / p.a.group : 0x40000000;
      q_head[r] = q % p.a.group;
    }
    for (int x = lo; x < hi && ok && it.t0 < it.t1;) {
      if (side == 1 && !it.two) {
        n += it.t1 - it.t0;
        x = tc_end(it);
        if (x < hi) tc_next(p, it, x, hi);
        continue;
      }
      // Side B's first S of an item comes behind the tiles of those without rows for it (n - own so
      // far), each of which may take what a wait may.
      if (n != own) {
        ok = __all_sync(0xffffffffu, mbar_wait_sleepy(&bar->s_full[side], own & 1, limit * (min(n - own, 4095) + 1), c.err));
        if (!ok) break;
      }
      const int left = it.n_tok - (it.qb * 2 + side) * p.tq;  // tokens of the sequence from the side's first on
      int lim[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        lim[r] = p.a.causal && q_tok[r] < left ? it.len - left + q_tok[r] + 1 : it.len;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
      for (int t = it.t0; t < it.t1; ++t, ++n, ++own, both += it.two ? 1 : 0) {
        const float4* con = s_const + (n & 3) * 8;
        const int key = t * kTcKeys + 2 * t4;
        ok = __all_sync(0xffffffffu, mbar_wait_sleepy(&bar->s_full[side], own & 1, limit, c.err));
        if (!ok) break;
        tc_fence_after();
        const bool clean =
            __all_sync(0xffffffffu, (t + 1) * kTcKeys <= min(lim[0], lim[1]) && con[0].w == 2.0f);
        float mt[2] = {-INFINITY, -INFINITY};
        // The maxima of both halves; the first stays in registers for its weights (with the second
        // that would be 64, more than a thread has beside the rest).
        uint32_t v[32];
        tc_half_load<KG>(tS + 64, con + 4, key + 64, lim, clean, v);
        tc_half_max<KG>(v, con + 4, clean, mt);
        tc_half_load<KG>(tS, con, key, lim, clean, v);
        tc_half_max<KG>(v, con, clean, mt);
        // The rows keep their references until a maximum passes them by 2^14; only then do
        // the four threads of a row compare theirs, and O is rescaled.
        if (__any_sync(0xffffffffu, mt[0] > m[0] + kTcRescale || mt[1] > m[1] + kTcRescale)) {
          float alpha[2];
          bool rescale = false;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float u = fmaxf(mt[r], __shfl_xor_sync(0xffffffffu, mt[r], 1));
            u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 2));
            const bool grow = u > m[r] + kTcRescale;
            alpha[r] = grow && m[r] != -INFINITY ? ex2_approx(m[r] - u) : 1.0f;
            rescale |= alpha[r] != 1.0f;
            m[r] = grow ? u : m[r];
            l[r] *= alpha[r];
          }
          if (__any_sync(0xffffffffu, rescale)) {
            // P V of the tile before is complete: s_full was committed behind it.
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              uint32_t ov[16];
              tmem_ld_16x256b_x4(tO + i * 32, ov);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha[(e >> 1) & 1]);
              tmem_st_16x256b_x4(tO + i * 32, ov);
            }
          }
        }
        // The sides' exponentials take turns: A after B's last tile, B after A's this one.  In
        // step, both would want them at once and both would then want the tensor cores.  Both
        // count the tiles of items with a side B alone (a wait tells apart two phases only, and
        // A may be any number of other tiles ahead).
        if (side == 1 || (it.two && both > 0)) {
          ok = __all_sync(0xffffffffu, side ? mbar_wait_sleepy(&bar->a_turn, both & 1, limit, c.err)
                                            : mbar_wait_sleepy(&bar->p_full[1][1], (both - 1) & 1, limit, c.err));
          if (!ok) break;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[16];
          if (half == 1) tc_half_load<KG>(tS + 64, con + 4, key + 64, lim, clean, v);
          tc_half_weights<KG>(v, con + half * 4, clean, m, l, pk);
          __syncwarp();
          tmem_st_16x128b_x8(tS + half * 32, pk);  // over columns that have been read
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&bar->p_full[side][half]);
        }
        if (side == 0 && it.two) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->a_turn);
        }
      }
      if (!ok) break;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      ok = __all_sync(0xffffffffu, mbar_wait_sleepy(&bar->o_done[side], (own - 1) & 1, limit, c.err));
      if (!ok) break;
      tc_fence_after();
      const bool whole = it.t1 - it.t0 == it.tiles;
      // A lane stores 8 columns of each 32: its row's four lanes trade theirs.
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t ov[16];
        tmem_ld_16x256b_x4(tO + i * 32, ov);
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool row = q_tok[r] < left;
          const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
          if (whole) {
            uint32_t h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const __half2 u = __floats2half2_rn(__uint_as_float(ov[4 * j + 2 * r]) * inv,
                                                  __uint_as_float(ov[4 * j + 2 * r + 1]) * inv);
              h[j] = *reinterpret_cast<const uint32_t*>(&u);
            }
            transpose4(h, t4);
            const int64_t at = (it.first + it.n_tok - left + q_tok[r]) * p.a.n_heads + it.head * p.a.group + q_head[r];
            if (row)
              *reinterpret_cast<uint4*>(p.a.out + at * D + i * 32 + 8 * t4) = make_uint4(h[0], h[1], h[2], h[3]);
            if (row && i == 0 && t4 == 0 && p.a.lse != nullptr)
              p.a.lse[at] = l[r] == 0.0f ? -INFINITY : (m[r] + log2f(l[r])) * 0.69314718055994531f;
          } else {
            uint32_t f0[4], f1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f0[j] = ov[4 * j + 2 * r];
              f1[j] = ov[4 * j + 2 * r + 1];
            }
            transpose4(f0, t4);
            transpose4(f1, t4);
            const int64_t part = (static_cast<int64_t>(blockIdx.x) * 2 + (it.t0 != 0 ? 0 : 1)) * kTcRows +
                                 side * 128 + r0 + g + 8 * r;
            if (row) {
              uint4* dst = reinterpret_cast<uint4*>(p.a.ws_o + part * D + i * 32 + 8 * t4);
              dst[0] = make_uint4(f0[0], f1[0], f0[1], f1[1]);
              dst[1] = make_uint4(f0[2], f1[2], f0[3], f1[3]);
            }
            if (row && i == 0 && t4 == 0) p.a.ws_ml[part] = make_float2(m[r], l[r]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(&bar->o_free[side]);
      x = tc_end(it);
      if (x < hi) tc_next(p, it, x, hi);
    }
    __syncwarp();
    tmem_wait_st();  // behind a wait that ran out, a rescaled O may still be on its way
  } else {
    set_max_regs_dec<kRegsOther>();
    if (warp == 20) {
      // ----------------------------------------------------- lookups and TMA
      int n = 0, items = 0;  // tiles and items whose copies are on their way
      int n_k = 0;           // tiles whose K is
      bool ok = true;
      int4 cut = make_int4(-1, 0, 0, 0);
      const int per_box = min(4, 1 << (c.shift - 4));  // slices of 16 keys in a TMA box
      for (int x = lo; x < hi && ok && it.t0 < it.t1; ++items) {
        if (it.t0 == 0 && it.t1 < it.tiles)
          cut = make_int4(it.b, it.qb, it.head, (it.begin + kTcItemCost + it.tiles - 1) / per);
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
            if (vs == 0.0f) vs = kNoScale;
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
              n_k += kv == 0 ? 1 : 0;
              if (mine)
                tma_load_2d(smem + Cfg::kOffRaw + kv * Cfg::kRaw + slice * 16 * D, kv ? &tmV : &tmK,
                            &bar->raw_full[kv], 0, D == 128 ? row : row >> 1);
            }
            if (!ok) break;
          }
          id = next;
        }
        x = tc_end(it);
        if (x < hi) tc_next(p, it, x, hi);
      }
      if (lane == 0) p.a.cut[blockIdx.x] = cut;
      // No copy may still be writing shared memory when the CTA leaves: what was issued last.
      // (Behind a wait that ran out that may be a tile's K without its V.)
      const unsigned long long drain = drain_ns(limit);
      if (items > 0) mbar_wait(&bar->q_full, (items - 1) & 1, drain, c.err);
      if (n_k > 0) mbar_wait(&bar->raw_full[0], (n_k - 1) & 1, drain, c.err);
      if (n > 0) mbar_wait(&bar->raw_full[1], (n - 1) & 1, drain, c.err);
      __syncwarp();
    } else if (warp == 21 || warp == 22) {
      // ----------------------------------------------- MMA, a warp per side
      // The whole warp walks the tiles and one lane issues; the operands' descriptors differ
      // by constants only, so that an MMA costs an addition or two.
      constexpr uint32_t kIdescS = umma_idesc_f16(128, kTcKeys, false, false, false);
      constexpr uint32_t kIdescO = umma_idesc_f16(128, D, false, false, true);
      const int side = warp - 21;
      const bool leader = elect_one();
      const uint64_t dq = umma_desc_sw128(smem_u32(smem + side * Cfg::kSide), 16, 1024);
      const uint64_t dk = umma_desc_sw128(smem_u32(smem + Cfg::kOffK), 16, 1024);
      const uint64_t dv = umma_desc_sw128(smem_u32(smem + Cfg::kOffV), 8192, 1024);
      const uint32_t tS = tmem + side * 128, tO = tmem + Cfg::kColO + side * D;
      int n = 0;           // tiles
      int mine = 0;        // tiles of this side
      int items = 0, own = 0;  // items, and this side's
      bool ok = true;
      bool busy = false;  // something was issued
      // The warp goes on as one: a lane whose wait alone ran out would miss the others' votes.
      auto wait = [&](uint64_t* b, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(b, parity, limit, c.err));
      };
      auto pv = [&](int i, bool start) {  // O += P V of tile i, this side's last one; `start`: the item's first
        ok = wait(&bar->v_full[i & 1], (i >> 1) & 1);
        // It overwrites O: the last item's rows have been read.
        if (ok && start) ok = wait(&bar->o_free[side], (own & 1) ^ 1u);
        const uint64_t d = dv + static_cast<uint64_t>((i & 1) * (Cfg::kWide >> 4));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (ok) ok = wait(&bar->p_full[side][half], (mine - 1) & 1);
          if (!ok) return;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16_ts(tO, tS + half * 32 + kk * 8, d + ((half * (Cfg::kDH * 8192) + kk * 2048) >> 4), kIdescO,
                          (start && half == 0 && kk == 0) ? 0u : 1u);
            if (half == 1) {
              umma_commit(&bar->o_done[side]);
              umma_commit(&bar->v_empty[i & 1]);
            }
          }
          __syncwarp();
          busy = true;
        }
      };
      for (int x = lo; x < hi && ok && it.t0 < it.t1; ++items) {
        ok = wait(&bar->q_full, items & 1);
        if (side == 1 && !it.two) {
          // No rows here: the tiles are only given back.
          for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
            ok = wait(&bar->k_full[n & 1], (n >> 1) & 1);
            if (ok) ok = wait(&bar->v_full[n & 1], (n >> 1) & 1);
            if (ok && leader) {
              mbar_arrive(&bar->k_empty[n & 1]);
              mbar_arrive(&bar->v_empty[n & 1]);
            }
            __syncwarp();
          }
          if (ok && leader) mbar_arrive(&bar->q_empty);
          __syncwarp();
        } else {
          for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
            ok = wait(&bar->k_full[n & 1], (n >> 1) & 1);
            if (ok && t > it.t0) pv(n - 1, t == it.t0 + 1);
            // S goes over P of the tile before: its product must have read it.
            if (ok && mine > 0) ok = wait(&bar->o_done[side], (mine - 1) & 1);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint64_t d = dk + static_cast<uint64_t>((n & 1) * (Cfg::kWide >> 4));
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_f16(tS, dq + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                         d + (((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), kIdescS, kk > 0 ? 1u : 0u);
              umma_commit(&bar->s_full[side]);
              umma_commit(&bar->k_empty[n & 1]);
            }
            __syncwarp();
            busy = true;
            ++mine;
          }
          if (!ok) break;
          if (leader) umma_commit(&bar->q_empty);
          __syncwarp();
          pv(n - 1, it.t1 - it.t0 == 1);
          ++own;
        }
        x = tc_end(it);
        if (x < hi) tc_next(p, it, x, hi);
      }
      // No MMA may still use TMEM or shared memory when the CTA leaves.
      if (busy) {
        if (leader) umma_commit(&bar->drain[side]);
        __syncwarp();
        mbar_wait(&bar->drain[side], 0, drain_ns(limit), c.err);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 21) {
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
  float m = -INFINITY, least = 0.0f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float2 ml = p.a.ws_ml[part(i)];
    m = fmaxf(m, ml.x);
    least = fminf(least, ml.y);
  }
  if (least == kNoPart) return;
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

template <int D, bool E4M3, int KG>
int launch_tc(TcParams p, const engine_kv_pages_t* kv, int64_t most_steps, cudaStream_t st) {
  using Cfg = TcCfg<D>;
  auto kern = attn_paged_tc_kernel<D, E4M3, KG>;
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
  const int64_t ctas = std::min<int64_t>(sm_count(), most_steps);
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
  // At most this many steps (the kernel counts them in 32 bits).
  const int64_t tiles = std::max<int64_t>((kv->max_pages * kv->page_size + kTcKeys - 1) / kTcKeys, 1) + kTcItemCost;
  const int64_t blocks = a.n_tokens / (2 * p.tq) + a.n_seq;
  if (blocks > 0x7fffffff / kv->n_kv_heads / tiles)
    return set_error(ENGINE_ERR_UNSUPPORTED, "attention_paged_prefill: too many query rows x positions");
  const int64_t most = blocks * kv->n_kv_heads * tiles;
  // Keys that share constants within a half tile: the page's.
  auto run = [&](auto kg) {
    constexpr int KG = decltype(kg)::value;
    const bool e4m3 = kv->type == ENGINE_KV_E4M3;
    if (kv->head_dim == 64)
      return e4m3 ? launch_tc<64, true, KG>(p, kv, most, st) : launch_tc<64, false, KG>(p, kv, most, st);
    return e4m3 ? launch_tc<128, true, KG>(p, kv, most, st) : launch_tc<128, false, KG>(p, kv, most, st);
  };
  if (kv->page_size == 16) return run(std::integral_constant<int, 16>());
  if (kv->page_size == 32) return run(std::integral_constant<int, 32>());
  return run(std::integral_constant<int, 64>());
}

}  // namespace b200
