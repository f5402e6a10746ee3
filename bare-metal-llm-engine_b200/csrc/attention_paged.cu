// attention_paged.cu -- attention over the paged 8-bit KV cache.
//
// Both entry points are one computation: query row t of sequence b sees the
// positions [0, last] of its slot.  With x_j = scale log2(e) ks_j (q . ck_j), where
// ck, cv are codes and ks, vs the scales of their page,
//   w_j = 2^(x_j + log2 vs_j - m),  out = sum_j w_j cv_j / sum_j (w_j / vs_j),
// m the running maximum of x_j + log2 vs_j.  Keeping the page's scale of V inside
// the weight leaves the products to the codes alone, and the weight is scaled by
// what it contributes.  A page whose values are all zero has scale 0: it counts
// with vs = kNoScale = 2^-33 (its codes are zeros).  That is below every scale that a
// write gives, so its weights never set the m that the others' are rounded against
// (with 1, values of 1e-3 beside a dominant key in such a page lost 20 times the bound).
//
// w goes into the second product as FP16 (off by 2^-11 of itself at most, below 2^-14 by
// half a step of 2^-24): the tensor cores take 16 bits beside the codes, and the codes
// are exact there.  m, l and the sums of both products stay in FP32, l from the weights
// before that rounding.  Outputs are 2.3e-4 to 2.9e-4 (relative, RMS) from 64 bits, of which
// their own FP16 rounding is 2.0e-4.
//
// Few query rows per KV head (decode, and the verification of a few tokens): the
// keys and values are the traffic, 2 bytes for 4 * rows FLOP, so what counts is
// that the codes stream at HBM rate and cost few instructions each.
//   Work split: an item is (sequence, 16 query rows, KV head); its keys are tiles of
// 64.  All tiles of all items are laid end to end and every CTA takes an equal
// range of them, whatever the lengths are (they are on the device; the host knows
// none).  An item inside one range is written out at once; of one that is cut, each
// CTA leaves (m, l, O) in a workspace, and a second kernel joins them in order.
//   A CTA: one producer warp and four consumer warps.  The producer looks up pages
// and scales, 32 slices of 16 keys at a time and one batch ahead, and fetches each
// tile's K and V codes by TMA into a ring of kStages x 64 keys (rows of 128 bytes,
// 128-byte swizzle); each consumer warp owns 16 keys of every tile.
//   Products: mma.sync m16n8k16 with the keys (later the elements of the values) as
// A's 16 rows and the query rows as B's 8 columns: S^T = K q^T, O^T += V^T P^T, so
// eight rows cost one instruction where q as A would fill half of it.  tcgen05 would
// want its operands as FP16 in shared memory, and writing the widened codes there and
// back costs more than the products.  Here a lane turns the bytes that it has just
// loaded into A fragments in registers.  The order of the contraction is free, so they
// are consecutive bytes: D / 4 of two keys' rows for S^T, D / 8 of four keys' rows for
// O^T; P passes from one layout to the other by two 8 x 8 transpositions.
//   Measured (B200, 32 / 8 heads of 128, calls back to back): 131072 keys of one sequence
// 55 us (269 MB, 0.75 of the measured copy rate), 48 sequences of 200-16384 keys 74 us (372
// MB, 0.77), 64 x 4000 keys 94 us (0.85).  Within the kernel the tiles arrive at about 7 TB/s;
// the rest is the 5 us until the first tile is there (lengths, table, scales and codes, each
// looked up with the last), the spread of the shares' ends and the join (4 us).  With q as A
// and the int8 offset taken off every code the first was 66 us where it is 54 to 55.  Eight
// consumer warps a CTA, two CTAs: 96 registers, spills, 83.  Items of 16 rows with d = 128
// spill too (int8 124 bytes of stores, e4m3 32, by -Xptxas -v): 1.9 % of the instructions of 16
// x 4 rows on 4000 keys.
//
//   Every wait is bounded (ENGINE_WAIT_TIMEOUT_MS).  Behind one that ran out the CTA stores no
// more rows and marks its parts, so that the join leaves theirs alone; copies in flight are waited
// for before it ends.

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention_paged.cuh"

namespace b200 {
namespace {

constexpr int kPgKeys = 64;      // keys per tile
constexpr int kPgRows = 16;      // query rows per item, at most (PgCfg::kRows)
constexpr int kPgConsumers = 4;  // warps; each takes 16 keys of a tile
constexpr int kPgThreads = (kPgConsumers + 1) * 32;
constexpr int kPgMaxSeq = 1024;  // sequences per launch (their prefix sums sit in shared memory)
constexpr float kPgRescale = 8.0f;
/// What an item costs beside its key tiles (its q, the chain of its first tile, the join of
/// the warps: about 4 us against 1 a tile), in tiles: the even shares count it, as steps in
/// front of the item's tiles in which nothing is done.  48 sequences of 200-16384 keys: 75 us
/// with 2, 72 with 4, 74 with 8.
constexpr int kPgItemCost = 4;
/// Query rows of a sequence and KV head (the average: the host knows no more, and a call that
/// mixes prompts with single rows pays for it: 512 rows on 8704 keys with 63 or 200 single rows on
/// 4000 keys take 368 and 765 us, in two calls 198 and 392) from which
/// attention_paged_tc takes the call: what needs a third group of 16 here.  One sequence of
/// 4000 keys: 32 rows 23 us either way, 48 rows 23 us there and 24 here, 64 rows 23 and 25;
/// sixteen of them: 16 rows 83 and 52, 32 rows 81 and 77, 48 rows 82 and 103.
constexpr int64_t kManyRows = 33;
/// Slots of at most so many tiles (by the table's width: the host knows no lengths) have a CTA to an
/// item: no workspace, no join.  1000 keys: one
/// sequence 13 us and 16 split, 8 sequences 14 and 16, 256 sequences 102 and 103; at 2000 keys
/// (32 tiles) it would be 21 and 16, 26 and 20, 176 and 179.
constexpr int64_t kWholeTiles = 16;
static_assert(kPgMaxSeq <= kTcMaxSeq, "both kernels take a launch's sequences");

/// NQ: groups of 8 query rows of an item.  Three CTAs an SM with 128 registers a thread
/// either way: of sixteen rows the fragments of q stay in shared memory.
template <int D, int NQ>
struct PgCfg {
  static constexpr int kRows = 8 * NQ;
  static constexpr int kCtas = 3;
  static constexpr int kTile = kPgKeys * D;  // bytes of K (or V) of a tile
  static constexpr int kStages = D == 128 ? 3 : 5;
  static constexpr int kOW = D + 4;          // pitch of a row of O in shared memory
  static constexpr int kBufs = 4 / NQ;       // copies of it: warps to a copy one after the other
  static constexpr int kOffO = kStages * 2 * kTile;
  static constexpr int kOffQ = kOffO + kBufs * kRows * kOW * 4;  // [D / 16][32 lanes], 16 bytes each
  static constexpr int kOffConst = kOffQ + (NQ == 1 ? 0 : D / 16 * 512);
  static constexpr int kOffBar = kOffConst + kStages * 4 * 16;
  static constexpr int kOffFail = kOffBar + 2 * kStages * 8;
  static constexpr int kOffMl = kOffFail + 16;
  static constexpr int kOffSeq = kOffMl + kPgConsumers * kRows * 8;
  static size_t smem(int n_seq) { return kOffSeq + 12 * (static_cast<size_t>(n_seq) + 1) + 1024; }
};

/// d += a b, m16n8k16.  The whole warp has to come here together: callers put
/// __syncwarp() behind code that the lanes' rows may branch in.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

/// The 8 x 8 transpose of a matrix of 16-bit elements, two of row lane / 4 in each lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

/// Four codes of a key as the two fragment registers of a contraction step.  e4m3:
/// bytes (0, 1) and (2, 3), exactly.  int8: bytes (0, 2) and (1, 3) as the FP16
/// subnormals (q + 128) 2^-24 -- the byte itself, its sign bit flipped, in a 16-bit
/// lane: 3 instructions for 4 codes, 5 where the 128 is taken off here.  It is taken
/// off the sums instead, which start at -128 2^-24 sum(q) (below full scale of the
/// codes, so it costs the FP32 sums no more than their largest values do).  P V cannot
/// do so: there the sum over thousands of keys can be far below the offset's.
template <bool E4M3>
__device__ __forceinline__ void k_fragment(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    codes_to_half4<true>(w, lo, hi);
  } else {
    lo = (w & 0x00ff00ffu) ^ 0x00800080u;
    hi = __byte_perm(w, 0, 0x4341) ^ 0x00800080u;
  }
}
constexpr float kKeyUnit = 5.9604644775390625e-8f;  // 2^-24

/// Shared-memory offset, within a tile, of the 16 bytes `c` of key `key`'s row.
template <int D>
__device__ __forceinline__ uint32_t pg_at(int key, int c) {
  if constexpr (D == 128) {
    return key * 128 + ((c ^ (key & 7)) << 4);
  } else {  // two keys to a 128-byte row
    const int line = key >> 1;
    return line * 128 + (((((key & 1) << 2) | c) ^ (line & 7)) << 4);
  }
}

/// Barrier of the consumer warps.  bar.sync wants whole warps: lanes that parted
/// before it (a row's own branch, a loop's early exit) are brought together first.
__device__ __forceinline__ void consumer_sync() {
  __syncwarp();
  named_barrier_sync(1, kPgConsumers * 32);
}

/// An item and the part of it that a CTA takes.
struct PgItem {
  int b;         // sequence, within the launch
  int slot, len;
  int head;      // KV head
  int row0;      // first flat query row (token * group + head within the group)
  int n_rows;    // flat rows of the sequence
  int n_tok;     // its tokens
  int64_t first; // its first token
  int t0, t1;    // tiles; none where the share ends within the item's leading steps
  int begin;     // the item's first step, counted over all items
  int end;       // the step behind this part
  int tiles;     // of the whole item
};

struct PgLists {
  const int32_t* pre;   // steps before each sequence
  const int32_t* slot;
  const int32_t* len;
};

/// The item at step `x` (`whole`: the item of that number), up to step `hi`.
template <int ROWS>
__device__ __forceinline__ PgItem pg_item(const ApParams& p, const PgLists& s, int x, int hi) {
  int lo = 0, up = p.n_seq - 1;
  while (lo < up) {  // the last sequence that starts at or before x
    const int mid = (lo + up + 1) >> 1;
    if (s.pre[mid] <= x) lo = mid;
    else up = mid - 1;
  }
  PgItem it;
  it.b = lo;
  it.slot = s.slot[lo];
  it.len = s.len[lo];
  it.tiles = max((it.len + kPgKeys - 1) / kPgKeys, 1);
  const int y = x - s.pre[lo];
  const int steps = p.whole ? 1 : kPgItemCost + it.tiles;
  const int j = y / steps;
  it.begin = s.pre[lo] + j * steps;
  it.t0 = p.whole ? 0 : max(x - it.begin - kPgItemCost, 0);
  it.t1 = p.whole ? it.tiles : max(min(hi - it.begin - kPgItemCost, it.tiles), it.t0);
  it.end = it.begin + (p.whole ? 1 : kPgItemCost + it.t1);
  it.head = j % p.c.heads;
  it.row0 = j / p.c.heads * ROWS;
  it.n_tok = kv_rows(p.c, p.cu, p.seq0 + lo, p.n_tokens, &it.first);
  it.n_rows = it.n_tok * p.group;
  return it;
}

/// Row of out / lse of a flat query row of a sequence.
__device__ __forceinline__ int64_t pg_row(const ApParams& p, int64_t first, int head, int flat) {
  const int tok = flat / p.group;
  return (first + tok) * p.n_heads + head * p.group + (flat - tok * p.group);
}

template <int D, bool E4M3, int NQ>
__global__ void __launch_bounds__(kPgThreads, PgCfg<D, NQ>::kCtas)
    attn_paged_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const ApParams p) {
  using Cfg = PgCfg<D, NQ>;
  constexpr int ST = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* s_o = reinterpret_cast<float*>(smem + Cfg::kOffO);
  uint4* s_q = reinterpret_cast<uint4*>(smem + Cfg::kOffQ);
  float4* s_const = reinterpret_cast<float4*>(smem + Cfg::kOffConst);  // [ST][4]: of 16 keys each
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* empty = full + ST;
  volatile int* s_fail = reinterpret_cast<int*>(smem + Cfg::kOffFail);  // a consumer's wait ran out
  float2* s_ml = reinterpret_cast<float2*>(smem + Cfg::kOffMl);        // [warps][rows]
  int32_t* s_pre = reinterpret_cast<int32_t*>(smem + Cfg::kOffSeq);    // [n_seq + 1]
  int32_t* s_slot = s_pre + p.n_seq + 1;
  int32_t* s_len = s_slot + p.n_seq + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kPgConsumers);
    }
    *s_fail = 0;
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  pdl_trigger();
  pdl_wait();
  // Steps of each sequence, then their sums.
  for (int b = threadIdx.x; b < p.n_seq; b += kPgThreads) {
    const int slot = kv_slot(p.c, p.slots, p.seq0 + b);
    const int len = kv_length(p.c, slot);
    int64_t first;
    const int rows = kv_rows(p.c, p.cu, p.seq0 + b, p.n_tokens, &first) * p.group;
    s_slot[b] = slot;
    s_len[b] = len;
    s_pre[b] = (rows + Cfg::kRows - 1) / Cfg::kRows * p.c.heads * (p.whole ? 1 : kPgItemCost + max((len + kPgKeys - 1) / kPgKeys, 1));
  }
  __syncthreads();
  if (warp == 0) {
    unsigned run = 0;
    int64_t all = 0;
    for (int base = 0; base < p.n_seq; base += 32) {
      const int v = base + lane < p.n_seq ? s_pre[base + lane] : 0;
      unsigned incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (base + lane < p.n_seq) s_pre[base + lane] = static_cast<int>(run + incl - v);
      run += __shfl_sync(0xffffffffu, incl, 31);
      all += kv_wide_sum(v);
    }
    if (lane == 0) s_pre[p.n_seq] = kv_total(p.c, all);
  }
  __syncthreads();
  const PgLists lists{s_pre, s_slot, s_len};
  const int total = s_pre[p.n_seq];
  // Steps (items, where `whole`) to a CTA.
  const int per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const int lo = min(static_cast<int64_t>(blockIdx.x) * per, static_cast<int64_t>(total));
  const int hi = min(lo + per, total);

  if (warp == kPgConsumers) {
    // ------------------------------------------------------------ producer
    const float kc_unit = p.scale_log2 * (E4M3 ? 1.0f : 1.0f / kKeyUnit);
    int n = 0, issued = 0;  // tiles handed over, and fetched
    int page_base = 0;
    bool ok = true;
    for (int x = lo; x < hi && ok;) {
      const PgItem it = pg_item<Cfg::kRows>(p, lists, x, hi);
      x = it.end;
      if (it.t0 == it.t1) break;
      const int n_keys = it.len;
      const int first_slice = it.t0 * 4, end_slice = min(it.t1 * 4, (n_keys + 15) >> 4);
      // Lane i of batch k looks after slice first_slice + 32 k + i.  Entries and scales are read
      // a batch ahead, and checked only when they are wanted.
      auto entry_of = [&](int slice) {
        return slice < end_slice
                   ? p.c.table[static_cast<int64_t>(it.slot) * p.c.max_pages + ((slice << 4) >> p.c.shift)]
                   : -1;
      };
      auto checked = [&](int id, int slice) {
        if (id >= 0 && id < p.c.n_pages) return id;
        if (slice < end_slice) atomicOr(p.c.err, kErrBadArgument);
        return -1;
      };
      int id = entry_of(first_slice + lane), id1 = entry_of(first_slice + 32 + lane);
      id = checked(id, first_slice + lane);
      float ks = 0.0f, vs = 0.0f, ks1 = 0.0f, vs1 = 0.0f;
      if (id >= 0) {
        ks = p.c.ks[kv_scale_at(p.c, id, it.head)];
        vs = p.c.vs[kv_scale_at(p.c, id, it.head)];
      }
      // One load per page of a tile, by the lane of the page's first slice.
      const int per_box = p.c.shift >= 6 ? 4 : 1 << (p.c.shift - 4);
      auto fetch = [&](int at, int i) {  // tile number `at`, the batch's i-th
        const int s = at % ST;
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((at / ST) & 1u) ^ 1u, p.limit_ns, p.c.err));
        if (!ok) return;
        const int slice = lane & 3;
        const bool mine = (lane >> 2) == i && id >= 0 && slice % per_box == 0;
        const unsigned who = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) mbar_expect_tx(&full[s], __popc(who) * per_box * 16 * D * 2);
        __syncwarp();
        if (mine) {
          uint8_t* sk = smem + s * 2 * Cfg::kTile + slice * 16 * D;
          const int key = (first_slice + lane) * 16 + page_base;
          const int off = key & ((1 << p.c.shift) - 1);  // row within the page
          const int row = ((id * p.c.heads + it.head) << p.c.shift) + off;
          const int y = D == 128 ? row : row >> 1;
          tma_load_2d(sk, &tmK, &full[s], 0, y);
          tma_load_2d(sk + Cfg::kTile, &tmV, &full[s], 0, y);
        }
      };
      for (int base = it.t0; base < it.t1 && ok; base += 8) {
        page_base = (base - it.t0) * kPgKeys;
        const int count = min(8, it.t1 - base);
        // At the CTA's start the first tiles are on their way before the scales are here.
        int ahead = 0;
        if (n == 0) {
          while (ahead < min(count, ST) && ok) {
            fetch(ahead, ahead);
            if (ok) ++ahead;
          }
        }
        const float v1 = vs == 0.0f ? kNoScale : vs;
        const float4 con = id >= 0 ? make_float4(ks * kc_unit, log2f(v1), 1.0f / v1, 1.0f)
                                   : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
        int id2 = -1;
        for (int i = 0; i < count && ok; ++i, ++n) {
          if (i >= ahead) fetch(n, i);
          if (!ok) break;
          const int s = n % ST;
          if (lane >> 2 == i) s_const[s * 4 + (lane & 3)] = con;
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
          if (i == min(ahead, count - 1)) {  // the next batch's scales, and the entries behind it
            id2 = entry_of((base + 16) * 4 + lane);
            id1 = checked(id1, (base + 8) * 4 + lane);
            if (id1 >= 0) {
              ks1 = p.c.ks[kv_scale_at(p.c, id1, it.head)];
              vs1 = p.c.vs[kv_scale_at(p.c, id1, it.head)];
            }
          }
        }
        issued = max(n, ahead);
        id = id1;
        ks = ks1;
        vs = vs1;
        id1 = id2;
      }
    }
    // No copy may still be writing shared memory when the CTA leaves.
    // (Behind a wait that ran out, tiles that were fetched ahead have not been arrived for.)
    if (n < issued) {
      for (; n < issued; ++n) {
        if (lane == 0) mbar_arrive(&full[n % ST]);
        __syncwarp();
      }
    }
    for (int j = max(n - ST, 0); j < n; ++j) mbar_wait(&full[j % ST], (j / ST) & 1u, drain_ns(p.limit_ns), p.c.err);
  } else {
    // ----------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    constexpr int NK = D / 16;  // contraction steps of S^T, and 16-row tiles of O^T
    int n = 0;
    bool ok = true;
    if (threadIdx.x == 0 && !p.whole && !p.by_item) p.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    for (int x = lo; x < hi;) {
      const PgItem it = pg_item<Cfg::kRows>(p, lists, x, hi);
      x = it.end;
      if (it.t0 == it.t1) break;
      // q^T as B fragments: the lane's D / 4 elements of query row g (and g + 8), from
      // t * D / 4.  In the sums' columns a lane has rows 2t and 2t + 1 (and + 8).
      uint32_t bq[NQ == 1 ? NK : 1][2];
      float init[NQ][2];
      int lim[NQ][2];
      int least = it.len;
      uint4 qw[NQ][NK / 2];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        const int flat = it.row0 + 8 * nq + g;
        const bool row = flat < it.n_rows;
        const uint4* src = reinterpret_cast<const uint4*>(
            p.q + (it.first + (row ? flat / p.group : 0)) * p.q_pitch +
            static_cast<int64_t>(it.head * p.group + (row ? flat % p.group : 0)) * D + t * (D / 4));
#pragma unroll
        for (int i = 0; i < NK / 2; ++i) qw[nq][i] = row ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NK / 2; ++i) {
          const uint32_t q[4] = {qw[nq][i].x, qw[nq][i].y, qw[nq][i].z, qw[nq][i].w};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t u0 = q[2 * e], u1 = q[2 * e + 1];
            if constexpr (!E4M3) {  // elements (0, 2) and (1, 3), as k_fragment pairs the codes
              const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&u0));
              const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&u1));
              sum += (f0.x + f0.y) + (f1.x + f1.y);
              const uint32_t v0 = u0;
              u0 = __byte_perm(v0, u1, 0x5410);
              u1 = __byte_perm(v0, u1, 0x7632);
            }
            if constexpr (NQ == 1) {
              bq[2 * i + e][0] = u0;
              bq[2 * i + e][1] = u1;
            } else if (warp == 0) {
              reinterpret_cast<uint2*>(s_q + (2 * i + e) * 32 + lane)[nq] = make_uint2(u0, u1);
            }
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          init[nq][e] = -128.0f * kKeyUnit * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
          const int f = it.row0 + 8 * nq + 2 * t + e;
          lim[nq][e] = it.len;
          if (p.causal && f < it.n_rows) lim[nq][e] = it.len - it.n_tok + f / p.group + 1;
          least = min(least, lim[nq][e]);
        }
      }
      least = __reduce_min_sync(0xffffffffu, least);
      if (NQ > 1) consumer_sync();  // s_q
      float o[NQ][NK][4];
      float m[NQ][2], l[NQ][2];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
        for (int j = 0; j < NK; ++j) o[nq][j][0] = o[nq][j][1] = o[nq][j][2] = o[nq][j][3] = 0.0f;
        m[nq][0] = m[nq][1] = -INFINITY;
        l[nq][0] = l[nq][1] = 0.0f;
      }

      for (int tile = it.t0; tile < it.t1; ++tile, ++n) {
        const int s = n % ST;
        if (ok) ok = mbar_wait(&full[s], (n / ST) & 1u, p.limit_ns, p.c.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) continue;
        const uint8_t* sk = smem + s * 2 * Cfg::kTile;
        const uint8_t* sv = sk + Cfg::kTile;
        const int k0 = warp * 16;  // this warp's first key of the tile
        const float4 con = s_const[s * 4 + warp];
        // S^T: keys g and g + 8 in rows, element [nq][0..3] = (g, 2t) (g, 2t+1) (g+8, 2t) (g+8, 2t+1).
        uint32_t kw[2][NK];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            *reinterpret_cast<uint4*>(&kw[r][4 * c]) =
                *reinterpret_cast<const uint4*>(sk + pg_at<D>(k0 + 8 * r + g, t * (D / 64) + c));
        }
        float sc[NQ][4];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nq][e] = E4M3 ? 0.0f : init[nq][e & 1];
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          uint32_t a[4];
          k_fragment<E4M3>(kw[0][i], a[0], a[2]);
          k_fragment<E4M3>(kw[1][i], a[1], a[3]);
          if constexpr (NQ == 1) {
            mma16816(sc[0], a, bq[i][0], bq[i][1]);
          } else {
            const uint4 b = s_q[i * 32 + lane];
            mma16816(sc[0], a, b.x, b.y);
            mma16816(sc[NQ - 1], a, b.z, b.w);
          }
        }
        // The lane's D / 8 elements, from g * D / 8, of keys 2t, 2t+1, 2t+8, 2t+9: on their way
        // while the weights are formed.
        const int pos = tile * kPgKeys + k0;
        uint32_t v[4][D / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (D == 128) {
            *reinterpret_cast<uint4*>(v[i]) = *reinterpret_cast<const uint4*>(sv + pg_at<D>(key, g));
          } else {
            *reinterpret_cast<uint2*>(v[i]) =
                *reinterpret_cast<const uint2*>(sv + pg_at<D>(key, g >> 1) + (g & 1) * 8);
          }
        }
        // x = S kc + lv; masked keys -inf.
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nq][e] = fmaf(sc[nq][e], con.x, con.y);
        }
        if (pos + 16 > least || con.w == 0.0f) {
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pos + g + 8 * (e >> 1) >= lim[nq][e & 1] || con.w == 0.0f) sc[nq][e] = -INFINITY;
          }
          if (E4M3) {  // bytes that are no sequence's may be NaN, which a weight of 0 would not silence
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool none = pos + 2 * t + (i & 1) + 8 * (i >> 1) >= it.len || con.w == 0.0f;
#pragma unroll
              for (int j = 0; j < D / 32; ++j) v[i][j] = none ? 0u : v[i][j];
            }
          }
        }
        bool grow = false;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
          for (int e = 0; e < 2; ++e) grow |= fmaxf(sc[nq][e], sc[nq][e + 2]) > m[nq][e] + kPgRescale;
        }
        // The reference m follows the running maximum only where that passed it by 2^8
        // (weights stay below 2^8); the result does not depend on it.
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float u = fmaxf(sc[nq][e], sc[nq][e + 2]);
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, w));
              u = fmaxf(u, m[nq][e]);
              const float a = u == -INFINITY ? 1.0f : ex2_approx(m[nq][e] - u);
              m[nq][e] = u;
              l[nq][e] *= a;
#pragma unroll
              for (int j = 0; j < NK; ++j) {
                o[nq][j][e] *= a;
                o[nq][j][e + 2] *= a;
              }
            }
          }
        }
        uint32_t bp[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float base = m[nq][e & 1] == -INFINITY ? 0.0f : m[nq][e & 1];
            w[e] = ex2_approx(sc[nq][e] - base);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float sum = w[e] + w[e + 2];
            // a NaN scale counts only where it is seen
            l[nq][e] = fmaf(sum, sum != 0.0f ? con.z : 0.0f, l[nq][e]);
          }
          const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
          bp[nq][0] = *reinterpret_cast<const uint32_t*>(&h0);
          bp[nq][1] = *reinterpret_cast<const uint32_t*>(&h1);
        }
        __syncwarp();
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
          bp[nq][0] = transpose8x8(bp[nq][0]);
          bp[nq][1] = transpose8x8(bp[nq][1]);
        }
        // O^T: 16-row tile i has elements g * D / 8 + 2i (row g) and + 2i + 1 (row g + 8).
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          uint32_t lo[4], hi[4];  // of the four bytes: keys 2t, 2t+1 and keys 2t+8, 2t+9
          codes_to_half4<E4M3>(__byte_perm(v[0][j], v[1][j], 0x5140), lo[0], lo[1]);
          codes_to_half4<E4M3>(__byte_perm(v[0][j], v[1][j], 0x7362), lo[2], lo[3]);
          codes_to_half4<E4M3>(__byte_perm(v[2][j], v[3][j], 0x5140), hi[0], hi[1]);
          codes_to_half4<E4M3>(__byte_perm(v[2][j], v[3][j], 0x7362), hi[2], hi[3]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t a[4] = {lo[2 * e], lo[2 * e + 1], hi[2 * e], hi[2 * e + 1]};
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) mma16816(o[nq][2 * j + e], a, bp[nq][0], bp[nq][1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }

      // Join the four warps: (m, l) of each row, then O in warp order.
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], w);
          if (g == 0) s_ml[warp * Cfg::kRows + 8 * nq + 2 * t + e] = make_float2(m[nq][e], l[nq][e]);
        }
      }
      if (!ok) *s_fail = 1;  // rows without this warp's keys: none go out from here on
      consumer_sync();
      float a[NQ][2];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mm = -INFINITY;
#pragma unroll
          for (int w = 0; w < kPgConsumers; ++w) mm = fmaxf(mm, s_ml[w * Cfg::kRows + 8 * nq + 2 * t + e].x);
          a[nq][e] = m[nq][e] == -INFINITY ? (l[nq][e] != l[nq][e] ? l[nq][e] : 0.0f) : ex2_approx(m[nq][e] - mm);
        }
      }
#pragma unroll
      for (int w = 0; w < kPgConsumers / Cfg::kBufs; ++w) {
        if (warp / Cfg::kBufs == w) {
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float* row = s_o + ((warp % Cfg::kBufs) * Cfg::kRows + 8 * nq + 2 * t + e) * Cfg::kOW + g * (D / 8);
#pragma unroll
              for (int j = 0; j < NK; j += 2) {
                float4* dst = reinterpret_cast<float4*>(row + 2 * j);
                float4 u = w == 0 ? make_float4(0, 0, 0, 0) : *dst;
                u.x = fmaf(o[nq][j][e], a[nq][e], u.x);
                u.y = fmaf(o[nq][j][e + 2], a[nq][e], u.y);
                u.z = fmaf(o[nq][j + 1][e], a[nq][e], u.z);
                u.w = fmaf(o[nq][j + 1][e + 2], a[nq][e], u.w);
                *dst = u;
              }
            }
          }
        }
        consumer_sync();
      }
      // The rows go out, 4 elements a thread and pass.
      const bool whole = it.t1 - it.t0 == it.tiles;
      const int wslot = blockIdx.x * 2 + (it.t0 != 0 ? 0 : 1);
      for (int i = threadIdx.x; i < Cfg::kRows * (D / 4); i += kPgConsumers * 32) {
        const int row = i / (D / 4), col = (i % (D / 4)) * 4;
        if (it.row0 + row >= it.n_rows) continue;
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kPgConsumers; ++w) mm = fmaxf(mm, s_ml[w * Cfg::kRows + row].x);
#pragma unroll
        for (int w = 0; w < kPgConsumers; ++w) {
          const float2 e = s_ml[w * Cfg::kRows + row];
          if (e.x != -INFINITY) ll = fmaf(e.y, ex2_approx(e.x - mm), ll);
          else if (e.y != e.y) ll = e.y;  // a NaN weight
        }
        float4 u = *reinterpret_cast<const float4*>(s_o + row * Cfg::kOW + col);
#pragma unroll
        for (int w = 1; w < Cfg::kBufs; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_o + (w * Cfg::kRows + row) * Cfg::kOW + col);
          u = make_float4(u.x + y.x, u.y + y.y, u.z + y.z, u.w + y.w);
        }
        const bool complete = *s_fail == 0;
        if (whole) {
          if (!complete) continue;
          const int64_t at = pg_row(p, it.first, it.head, it.row0 + row);
          const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
          const __half2 h[2] = {__floats2half2_rn(u.x * inv, u.y * inv), __floats2half2_rn(u.z * inv, u.w * inv)};
          *reinterpret_cast<uint2*>(p.out + at * D + col) = *reinterpret_cast<const uint2*>(h);
          if (p.lse != nullptr && col == 0)
            p.lse[at] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
        } else {
          *reinterpret_cast<float4*>(p.ws_o + (static_cast<int64_t>(wslot) * kPgRows + row) * D + col) = u;
          if (col == 0) p.ws_ml[wslot * kPgRows + row] = make_float2(mm, complete ? ll : kNoPart);
        }
      }
      if (threadIdx.x == 0 && it.t0 == 0 && !p.whole && (p.by_item || !whole)) {
        const int parts = (it.begin + kPgItemCost + it.tiles - 1) / per - static_cast<int>(blockIdx.x) + 1;
        const int at = p.by_item ? (it.b * ((p.group + Cfg::kRows - 1) / Cfg::kRows) + it.row0 / Cfg::kRows) * p.c.heads + it.head
                                 : static_cast<int>(blockIdx.x);
        p.cut[at] = make_int4(whole ? -1 : it.b, it.row0, it.head | parts << 16, static_cast<int>(blockIdx.x));
      }
      consumer_sync();  // s_o, s_ml and s_q are free again
    }
  }
}

/// The k-th (from 0) of the entries that hold a cut item; its x is -1 where there is none.
/// The whole warp comes with one k.
__device__ __forceinline__ int4 nth_cut(const int4* cuts, int n, int k) {
  constexpr int J = 8;
  for (int base = 0; base < n; base += 32 * J) {
    int x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = base + 32 * j + static_cast<int>(lane_id());
      x[j] = i < n ? cuts[i].x : -1;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      unsigned some = __ballot_sync(0xffffffffu, x[j] >= 0);
      const int count = __popc(some);
      if (k < count) {
        for (; k > 0; --k) some &= some - 1;
        return cuts[base + 32 * j + __ffs(some) - 1];
      }
      k -= count;
    }
  }
  return make_int4(-1, 0, 0, 0);
}

/// Joins the parts of a cut item (part 1 of the CTA that began it, and part 0 of each one
/// up to that which finished it); blockIdx.x is the item (the entry of p.cut, or, where a
/// few are spread over many entries, the number among those that hold one), blockIdx.y the
/// row.  One sequence of 131072 keys has 55 parts of a row: eight warps take every eighth,
/// so that all of them are on their way at once.
constexpr int kJoinWarps = 8;
/// RPB: rows of a block.  One where an item has many parts; eight, a warp each, where it
/// has a few.
template <int D, int RPB>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_paged_join_kernel(const ApParams p) {
  pdl_trigger();
  pdl_wait();
  const int4 cut = RPB == 1 && !p.by_item ? nth_cut(p.cut, p.n_cut, blockIdx.x) : p.cut[blockIdx.x];
  if (cut.x < 0) return;
  constexpr int E = D / 32;            // columns of a lane
  constexpr int W = kJoinWarps / RPB;  // warps of a row
  __shared__ float s_o[RPB == 1 ? kJoinWarps : 1][D];
  __shared__ float s_l[RPB == 1 ? kJoinWarps : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y * RPB + warp / W;
  int64_t first;
  const int n_rows = kv_rows(p.c, p.cu, p.seq0 + cut.x, p.n_tokens, &first) * p.group;
  if (cut.y + row >= n_rows) return;  // (whole blocks where RPB is 1)
  const int parts = static_cast<int>(static_cast<unsigned>(cut.z) >> 16);
  const int part0 = 2 * cut.w;
  auto slot = [&](int i) { return static_cast<int64_t>(part0 + (i == 0 ? 1 : 2 * i)) * kPgRows + row; };
  float m = -INFINITY, least = 0.0f;
  for (int i = lane; i < parts; i += 32) {
    const float2 ml = p.ws_ml[slot(i)];
    m = fmaxf(m, ml.x);
    least = fminf(least, ml.y);
  }
  if (__any_sync(0xffffffffu, least == kNoPart)) return;  // (every warp of a row looks at all parts)
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  float l = 0.0f, o[E] = {};
#pragma unroll 4
  for (int i = warp % W; i < parts; i += W) {
    const float2 ml = p.ws_ml[slot(i)];
    float v[E];
    if constexpr (E == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p.ws_o + slot(i) * D + lane * E);
    else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p.ws_o + slot(i) * D + lane * E);
    // A part without a visible key has m = -inf, l = 0 and o = 0 (or NaN in all: kept).
    const float a = ml.x == -INFINITY ? 1.0f : ex2_approx(ml.x - m);
    l = fmaf(ml.y, a, l);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], a, o[e]);
  }
  if constexpr (RPB == 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    if (warp != 0) return;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      l += s_l[w];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += s_o[w][lane * E + e];
    }
  }
  const int64_t at = pg_row(p, first, cut.z & 0xffff, cut.y + row);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  __half2 h[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) h[e] = __floats2half2_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
  if constexpr (E == 4) *reinterpret_cast<uint2*>(p.out + at * D + lane * E) = *reinterpret_cast<const uint2*>(h);
  else *reinterpret_cast<__half2*>(p.out + at * D + lane * E) = h[0];
  if (p.lse != nullptr && lane == 0)
    p.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

/// `most`: steps (items, where p.whole) that there can be; `items`: as it says.
template <int D, bool E4M3, int NQ>
int launch_paged(ApParams p, const engine_kv_pages_t* kv, int64_t most, int64_t items, cudaStream_t st) {
  using Cfg = PgCfg<D, NQ>;
  auto kern = attn_paged_kernel<D, E4M3, NQ>;
  const size_t smem = Cfg::smem(p.n_seq);
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  B200_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if ((configured.load() & bit) == 0) {
    B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(Cfg::smem(kPgMaxSeq))));
    B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    configured.fetch_or(bit);
  }
  CUtensorMap tk, tv;
  const uint64_t rows = static_cast<uint64_t>(kv->n_pages * kv->n_kv_heads * kv->page_size) * D / 128;
  const uint32_t box = static_cast<uint32_t>(kv->page_size < kPgKeys ? kv->page_size : kPgKeys) * D / 128;
  if (!make_tmap_2d(&tk, p.c.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, 128, 128, box, 128) ||
      !make_tmap_2d(&tv, p.c.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, 128, 128, box, 128))
    return ENGINE_ERR_CUDA;
  // kCtas an SM while their shared memory fits (three: up to about 300 sequences).
  const int64_t per_sm = std::min<int64_t>(Cfg::kCtas, (max_smem_optin() + 1024) / static_cast<int64_t>(smem + 1024));
  if (p.whole) {
    const cudaError_t e =
        launch_pdl(kern, dim3(static_cast<unsigned>(most)), dim3(kPgThreads), smem, st, tk, tv, p);
    return e == cudaSuccess ? ENGINE_OK : set_cuda_error(e, "attn_paged_kernel");
  }
  const int64_t ctas = std::min<int64_t>(sm_count() * std::max<int64_t>(per_sm, 1), most);
  // One row per sequence: the items are numbered, and the join has a block column for each.
  // Else they are known by the CTA that began them.
  p.by_item = p.cu == nullptr && items <= ctas ? 1 : 0;
  const int64_t cuts = p.by_item ? items : ctas;
  p.n_cut = static_cast<int>(cuts);
  const size_t o_bytes = 2 * ctas * kPgRows * D * sizeof(float), ml_bytes = 2 * ctas * kPgRows * sizeof(float2);
  char* ws = static_cast<char*>(scratch_alloc(o_bytes + ml_bytes + cuts * sizeof(int4), st));
  if (ws == nullptr) return set_error(ENGINE_ERR_CUDA, "attention_paged: workspace allocation failed");
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(ws + o_bytes);
  p.cut = reinterpret_cast<int4*>(ws + o_bytes + ml_bytes);
  int rc = ENGINE_OK;
  // A plain launch: an SM that still runs blocks of the kernel before keeps their split of its
  // storage, and begun under it takes two of these CTAs where it should take three; the shares
  // left over then begin when the others are done (85 us against 71 for the call).
  kern<<<static_cast<unsigned>(ctas), kPgThreads, smem, st>>>(tk, tv, p);
  cudaError_t e = cudaGetLastError();
  const unsigned c = static_cast<unsigned>(cuts);
  if (e == cudaSuccess) {
    // With few items a block looks for its entry: of the 444 x 16 that one block an entry and
    // row would be nearly all had nothing to do (16 rows on 4000 keys 25 us then, 21 so).
    if (ctas >= 8 * items)
      e = launch_pdl(attn_paged_join_kernel<D, 1>, dim3(static_cast<unsigned>(items), Cfg::kRows), dim3(kJoinWarps * 32), 0, st, p);
    else
      e = launch_pdl(attn_paged_join_kernel<D, 8>, dim3(c, Cfg::kRows / 8), dim3(kJoinWarps * 32), 0, st, p);
  }
  if (e != cudaSuccess) rc = set_cuda_error(e, "attn_paged_kernel");
  scratch_free(ws, st);
  return rc;
}

/// The sequences, in launches of at most kPgMaxSeq.
int run_paged(ApParams p, const engine_kv_pages_t* kv, int64_t n_seq, cudaStream_t st, const char* what) {
  const bool e4m3 = kv->type == ENGINE_KV_E4M3;
  const int64_t tiles = std::max<int64_t>((kv->max_pages * kv->page_size + kPgKeys - 1) / kPgKeys, 1);
  const int64_t steps = tiles + kPgItemCost;
  // Rows per sequence and KV head, on the average (the host knows no more).  Where that is at
  // most 8 an item has 8 rows (8 of 16 sequences of 4000 keys 37 us, 50 with items of 16; of
  // one sequence 16 and 19), else 16, so that the keys are read half as often.
  const int64_t all = p.cu == nullptr ? p.group * n_seq : p.n_tokens * p.group;
  const bool r8 = all <= 8 * n_seq;
  const bool many = p.cu != nullptr && p.group <= 128 && all >= kManyRows * n_seq;
  const int64_t rows = r8 ? 8 : 16;  // of an item
  for (int64_t at = 0; at < n_seq; at += kPgMaxSeq) {
    const int64_t n = std::min<int64_t>(kPgMaxSeq, n_seq - at);
    p.seq0 = static_cast<int>(at);
    p.n_seq = static_cast<int>(n);
    if (many) {
      if (const int rc = attention_paged_tc(p, kv, st)) return rc;
      continue;
    }
    // At most this many steps (the kernel counts them in 32 bits).
    const int64_t groups = p.cu == nullptr ? n * ((p.group + rows - 1) / rows)
                                           : p.n_tokens * p.group / rows + n;
    if (groups > 0x7fffffff / kv->n_kv_heads / steps)
      return set_error(ENGINE_ERR_UNSUPPORTED, std::string(what) + ": too many query rows x positions");
    p.whole = tiles <= kWholeTiles ? 1 : 0;
    const int64_t most = groups * kv->n_kv_heads * (p.whole ? 1 : steps);
    int rc;
    if (kv->head_dim == 64) {
      rc = e4m3 ? (r8 ? launch_paged<64, true, 1>(p, kv, most, groups * kv->n_kv_heads, st) : launch_paged<64, true, 2>(p, kv, most, groups * kv->n_kv_heads, st))
                : (r8 ? launch_paged<64, false, 1>(p, kv, most, groups * kv->n_kv_heads, st) : launch_paged<64, false, 2>(p, kv, most, groups * kv->n_kv_heads, st));
    } else {
      rc = e4m3 ? (r8 ? launch_paged<128, true, 1>(p, kv, most, groups * kv->n_kv_heads, st) : launch_paged<128, true, 2>(p, kv, most, groups * kv->n_kv_heads, st))
                : (r8 ? launch_paged<128, false, 1>(p, kv, most, groups * kv->n_kv_heads, st) : launch_paged<128, false, 2>(p, kv, most, groups * kv->n_kv_heads, st));
    }
    if (rc != ENGINE_OK) return rc;
  }
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

ApParams paged_params(const engine_kv_pages_t* kv, int64_t layer, const engine_half_t* q,
                      int64_t q_pitch, const int32_t* slots, const int32_t* cu, engine_half_t* out,
                      float* lse, int64_t n_tokens, int64_t n_heads, float scale, bool causal) {
  ApParams p = {};
  p.c = kv_view(kv, layer);
  p.q = reinterpret_cast<const __half*>(q);
  p.q_pitch = q_pitch;
  p.slots = slots;
  p.cu = cu;
  p.out = reinterpret_cast<__half*>(out);
  p.lse = lse;
  p.n_tokens = n_tokens;
  p.n_heads = static_cast<int>(n_heads);
  p.group = static_cast<int>(n_heads / kv->n_kv_heads);
  p.causal = causal ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.limit_ns = wait_limit_ns();
  return p;
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
  const ApParams p = paged_params(kv, layer, q, q_pitch, slots, nullptr, out, out_lse, n_seq, n_heads,
                                  scale, false);
  return run_paged(p, kv, n_seq, static_cast<cudaStream_t>(stream), what);
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
  const ApParams p = paged_params(kv, layer, q, q_pitch, slots, cu_q, out, out_lse, n_tokens, n_heads,
                                  scale, is_causal != 0);
  return run_paged(p, kv, n_seq, static_cast<cudaStream_t>(stream), what);
  B200_ENTRY_END
}

}  // extern "C"
