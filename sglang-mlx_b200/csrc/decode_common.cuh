// decode_common.cuh — what the attention kernels' translation units share: the
// parameter block of a decode launch, the sticky status word, programmatic
// dependent launch, and the partition, zero-row and merge helpers.
#pragma once

#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "kvc_common.cuh"

namespace kvc {


// (one word for each translation unit that includes this; kvc_get_status ORs them)
static __device__ unsigned int g_decode_status = 0;

struct DecodeParams {
  void* out;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const uint32_t* block_tables;
  const uint32_t* context_lens;
  const float* alibi;
  float* part_max;
  float* part_sum;
  float* part_out;
  int num_seqs, num_heads, num_kv_heads, block_size;
  int max_seq_len, partition_size, num_partitions;
  int heads_per_cta;  // q heads of one KV group handled by one CTA
  int64_t num_blocks;
  int64_t q_seq_stride, q_head_stride, out_seq_stride, out_head_stride;
  int64_t k_block_stride, k_head_stride, v_block_stride, v_head_stride;
  int64_t k_tok_stride, v_tok_stride;  // token-major caches: elements between a block's tokens
  // shared-prefix decode: partitions [0, prefix_parts) are chunks of prefix_part_size tokens of the shared
  // prefix (the cascade kernel writes them); partition prefix_parts + i covers tokens
  // prefix_len + i * partition_size onwards.  part_offset is added to blockIdx.z by the partition kernels.
  int prefix_len, prefix_parts, prefix_part_size, part_offset;
  float k_scale, v_scale;  // one-byte caches: dequantisation scales (value = code * scale)
  int wait_prior_at_end;   // partition kernel: griddepcontrol.wait before exiting (shared-prefix launch order)
  int wait_prior_at_start; // partition kernel launched as a programmatic dependent of the kernel before it
                           // (an append): griddepcontrol.wait before its first global read
  int64_t table_stride;
  int64_t part_seq_stride, part_head_stride;
  int64_t part_out_seq_stride, part_out_head_stride, part_out_part_stride;
  float scale;
  // Planned split-K: CTA i of a 1-D grid runs work item i / num_kv_heads of the
  // plan (kvc_decode_plan) for KV head i % num_kv_heads; a sequence split in
  // several partitions has its partials merged by the CTA that finishes last
  // (plan_counters) when fused_merge is set, else by the reduce kernel.
  const uint32_t* plan_header;
  const uint32_t* plan_items;
  uint32_t* plan_counters;
  int fused_merge;
  // The step's append, folded into the decode (kvc_paged_attention_planned_append):
  // the CTA holding a sequence's last token writes that token's K row and V
  // column to slot slots[seq] before its first cache copy.
  const void* new_k;
  const void* new_v;
  const void* slots;
  int slots_i64;
  int64_t nk_tok_stride, nk_head_stride, nv_tok_stride, nv_head_stride;
};

// What the queries at positions first .. last of a sequence see under a sliding
// window of `window` tokens with `sinks` first tokens that stay visible, as a
// run of whole blocks: the blocks of the sinks, then those from the first
// query's window start on, numbered without the gap between them ("virtual"
// positions; a virtual position differs from the real one by `jump` tokens from
// virtual block `sink_blocks` on).  Every kernel of the window form works in
// virtual positions and looks blocks up with real_block.  A query at real
// position i sees the virtual positions v < i + 1 - jump with v < sinks or
// v >= i + 1 - window - jump: where jump > 0 the sinks end before the gap.
struct Seen {
  int sink_blocks, skip;  // blocks before the gap, blocks in it
  int jump;               // tokens in the gap
  int beg, end;           // virtual: the first query's window start, one past the last query
  __device__ __forceinline__ int real_block(int vb) const { return vb + (vb >= sink_blocks ? skip : 0); }
};
__device__ __forceinline__ Seen seen_range(int first, int last, int window, int sinks, int bs) {
  Seen s;
  const int start = first + 1 > window ? first + 1 - window : 0;
  const int sink_end = sinks < start ? sinks : start;
  s.sink_blocks = (sink_end + bs - 1) / bs;
  const int wb = start / bs;
  s.skip = wb > s.sink_blocks ? wb - s.sink_blocks : 0;
  s.jump = s.skip * bs;
  s.beg = start - s.jump;
  s.end = last + 1 - s.jump;
  return s;
}

// Programmatic dependent launch: the partition kernels let the split-K reduce be
// scheduled early; the reduce waits for their completion before reading.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Token range [begin, end) of this CTA's partition; returns false when the
// CTA has nothing to do.  `zero_out` is set when the sequence must produce
// zeros (reference edge rule) and this CTA owns writing them.
__device__ __forceinline__ bool partition_range(const DecodeParams& p, int seq, int part, uint32_t ctx, int* begin,
                                                int* end, bool* zero_out) {
  *zero_out = false;
  if (ctx == 0 || ctx > (uint32_t)p.max_seq_len) {
    // Single pass: this CTA writes the zeros.  Split: the reduce does.
    *zero_out = (p.num_partitions == 1);
    return false;
  }
  if (p.prefix_len > 0) {
    // shared-prefix decode: this kernel only runs the partitions after the prefix
    const int64_t b = (int64_t)p.prefix_len + (int64_t)(part - p.prefix_parts) * p.partition_size;
    if (part < p.prefix_parts || b >= (int64_t)ctx) return false;
    *begin = (int)b;
    const int64_t e = b + p.partition_size;
    *end = (int)((int64_t)ctx < e ? (int64_t)ctx : e);
    return true;
  }
  if (p.num_partitions == 1) {
    *begin = 0;
    *end = (int)ctx;
    return true;
  }
  const int64_t b = (int64_t)part * p.partition_size;
  if (b >= (int64_t)ctx) return false;  // the reduce never reads this partition
  *begin = (int)b;
  const int64_t e = b + p.partition_size;
  *end = (int)((int64_t)ctx < e ? (int64_t)ctx : e);
  return true;
}

template <typename T>
__device__ __forceinline__ void write_zero_heads(const DecodeParams& p, int seq, int h0, int nh, int D) {
  T* out = reinterpret_cast<T*>(p.out);
  for (int i = threadIdx.x; i < nh * D; i += blockDim.x) {
    const int g = i / D, d = i - g * D;
    out[(int64_t)seq * p.out_seq_stride + (int64_t)(h0 + g) * p.out_head_stride + d] = from_float<T>(0.f);
  }
}

// ---------------------------------------------------------------------------
// Planned split-K (kvc_decode_plan + kvc_paged_attention_planned).
// ---------------------------------------------------------------------------

// The work item of this CTA: false when the CTA has none (past the plan's item
// count, or a plan written for other launch parameters, which is flagged).
__device__ __forceinline__ bool planned_item(const DecodeParams& p, int* kvh, int* seq, int* part) {
  const uint32_t* h = p.plan_header;
  if (h[0] != kPlanMagic || h[1] != (uint32_t)p.num_seqs || h[2] != (uint32_t)p.num_kv_heads ||
      h[3] != (uint32_t)p.max_seq_len || h[4] != (uint32_t)p.partition_size) {
    if (blockIdx.x == 0 && threadIdx.x == 0) set_status(&g_decode_status, KVC_STATUS_PLAN_MISMATCH);
    return false;
  }
  const uint32_t item_idx = blockIdx.x / (uint32_t)p.num_kv_heads;
  if (item_idx >= h[5]) return false;
  const uint32_t item = p.plan_items[item_idx];
  *kvh = (int)(blockIdx.x - item_idx * (uint32_t)p.num_kv_heads);
  *seq = (int)(item & 0xFFFFu);
  *part = (int)(item >> 16);
  return true;
}

// Partitions of a sequence of `ctx` tokens (valid ctx only).
__device__ __forceinline__ int planned_parts(const DecodeParams& p, uint32_t ctx) {
  return (int)((ctx + (uint32_t)p.partition_size - 1) / (uint32_t)p.partition_size);
}

// Merges the `nparts` (<= 32) partials of heads h0 .. h0 + G - 1 of `seq` into
// the output.  Every thread of the CTA calls it; the partials must be visible to
// the CTA, and `scratch` (at least G * 32 + G floats of shared memory) free.
template <typename T>
__device__ __forceinline__ void merge_head_partials(const DecodeParams& p, int seq, int h0, int G, int D, int nparts,
                                                    float* scratch) {
  // weights e^{m_k - M} of every partition, and 1 / (L + 1e-6), per head
  float* w = scratch;                 // [G][32]
  float* inv = scratch + G * 32;      // [G]
  for (int g = threadIdx.x; g < G; g += blockDim.x) {
    const int64_t o = (int64_t)seq * p.part_seq_stride + (int64_t)(h0 + g) * p.part_head_stride;
    float M = -INFINITY;
    for (int k = 0; k < nparts; ++k) M = fmaxf(M, __ldcg(p.part_max + o + k));
    float L = 0.f;
    for (int k = 0; k < nparts; ++k) {
      const float mk = __ldcg(p.part_max + o + k);
      const float wt = (M == -INFINITY || mk == -INFINITY) ? 0.f : expf(mk - M);
      w[g * 32 + k] = wt;
      L += wt * __ldcg(p.part_sum + o + k);
    }
    inv[g] = 1.f / (L + 1e-6f);  // paged_attention_kernels.metal:144
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(p.out);
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    const int g = i / D, d = i - g * D;
    const float* po = p.part_out + (int64_t)seq * p.part_out_seq_stride + (int64_t)(h0 + g) * p.part_out_head_stride + d;
    float a = 0.f;
    for (int k = 0; k < nparts; ++k) a += w[g * 32 + k] * __ldcg(po + (int64_t)k * p.part_out_part_stride);
    out[(int64_t)seq * p.out_seq_stride + (int64_t)(h0 + g) * p.out_head_stride + d] = from_float<T>(a * inv[g]);
  }
}

// Called by every thread of the CTA after it wrote its partition's partials:
// counts the arrival, and the CTA that completes the sequence's set merges
// the `nparts` (<= 32) partials into the output and resets the counter.
template <typename T>
__device__ __forceinline__ void planned_arrive_and_merge(const DecodeParams& p, int seq, int kvh, int h0, int G,
                                                         int D, int nparts, float* scratch) {
  __shared__ uint32_t s_last;
  __threadfence();  // this thread's partials are visible before the arrival below
  __syncthreads();
  uint32_t* counter = p.plan_counters + (int64_t)seq * p.num_kv_heads + kvh;
  if (threadIdx.x == 0) s_last = atomicAdd(counter, 1u) == (uint32_t)(nparts - 1) ? 1u : 0u;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  merge_head_partials<T>(p, seq, h0, G, D, nparts, scratch);
  if (threadIdx.x == 0) *counter = 0u;  // ready for the next call with this plan
}

// Writes one merged (max, sum, acc) triple: the final output in single-pass
// mode, the partition's partials in split mode.
template <typename T>
__device__ __forceinline__ void emit(const DecodeParams& p, int seq, int head, int part, int d, float m, float l,
                                     float acc, bool first_d, bool direct) {
  if (direct) {
    T* out = reinterpret_cast<T*>(p.out);
    // paged_attention_kernels.metal:144 — inv_sum = 1 / (sum + 1e-6)
    const float inv = 1.f / (l + 1e-6f);
    out[(int64_t)seq * p.out_seq_stride + (int64_t)head * p.out_head_stride + d] = from_float<T>(acc * inv);
  } else {
    p.part_out[(int64_t)seq * p.part_out_seq_stride + (int64_t)head * p.part_out_head_stride +
               (int64_t)part * p.part_out_part_stride + d] = acc;
    if (first_d) {
      const int64_t o = (int64_t)seq * p.part_seq_stride + (int64_t)head * p.part_head_stride + part;
      p.part_max[o] = m;
      p.part_sum[o] = l;
    }
  }
}

}  // namespace kvc
