// attention_paged.cuh -- what the two kernels of attention over the paged cache
// share (attention_paged.cu: few query rows per KV head; attention_paged_tc.cu: many).
#pragma once

#include "kernels.cuh"
#include "kv_pages.cuh"

namespace b200 {

struct ApParams {
  KvView c;
  const __half* q;
  int64_t q_pitch;
  const int32_t* slots;
  const int32_t* cu;  // null: one row per sequence
  __half* out;
  float* lse;
  int seq0, n_seq;    // sequences [seq0, seq0 + n_seq) of the call
  int64_t n_tokens;
  int n_heads, group;
  int causal;
  float scale_log2;
  float* ws_o;        // [2 * CTAs][rows][D]: unfinished items, part 1 of the CTA that began one,
  float2* ws_ml;      // [2 * CTAs][rows]     part 0 of those that went on with it
  int4* cut;          // items that are cut: sequence (-1: none), first row, KV head (16-row
                      // kernel: and parts << 16), last CTA (16-row kernel: the first)
  int by_item;        // 16-row kernel: cut[item], one row per sequence; else cut[CTA that began it]
  int n_cut;          // 16-row kernel: entries of cut
  int whole;          // a CTA to an item: none is cut, no workspace
  unsigned long long limit_ns;
};

/// Many query rows per KV head, on tcgen05 (attention_paged_tc.cu): the sequences
/// [p.seq0, p.seq0 + p.n_seq), at most kTcMaxSeq.  p.group must be at most 128.
constexpr int kTcMaxSeq = 1024;
int attention_paged_tc(const ApParams& p, const engine_kv_pages_t* kv, cudaStream_t st);

/// l of a part that was not stored (a wait ran out), which no sum of weights is: the join then
/// leaves the row as it was, as the kernels leave the rows of items that are not cut.
constexpr float kNoPart = -1.0f;

/// The limit of a wait for a CTA's own copies and products in flight.  They end by themselves, and
/// the CTA must not leave before them, however short the limit of its roles' waits for each other is.
__device__ __forceinline__ unsigned long long drain_ns(unsigned long long limit_ns) {
  return limit_ns > 2000000000ull ? limit_ns : 2000000000ull;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace b200
