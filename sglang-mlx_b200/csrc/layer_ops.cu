// layer_ops.cu — what surrounds the attention of a step, for sm_100a: the block
// tables, positions and slot maps of a batch built from its lengths, and the
// per-head RMS norm with the rotary position of queries and keys, on its own or
// fused with the append of keys and values into the cache.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kvc_common.cuh"

namespace kvc {

__device__ unsigned int g_layer_ops_status = 0;

// SMs of the current device (cached per device; any racing writer stores the same value).
static int sm_count() {
  static std::atomic<int> sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  int n = dev >= 0 && dev < 64 ? sms[dev].load() : 0;
  if (n <= 0) {
    if (dev < 0 || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    if (dev >= 0 && dev < 64) sms[dev] = n;
  }
  return n;
}

// ---------------------------------------------------------------------------
// Step tables.  Request b holds prefix[b] cached tokens and brings fresh[b] new
// ones.  With bs tokens per block, F_b = ceil(prefix[b] / bs) its blocks so far
// and N_b = ceil((prefix[b] + fresh[b]) / bs) - F_b the ones it needs, the new
// blocks come off the free list in request order:
//   tables[b][F_b + j] = free[sum_{c < b} N_c + j],   j < N_b
// and new token i of request b (row sum_{c < b} fresh[c] + i) has
//   position  prefix[b] + i
//   slot      tables[b][position / bs] * bs + position % bs.
// One launch.  A chunk is 1024 requests; CTA (s, c) sums the requests before
// chunk c, scans the chunk's own (each CTA of a chunk does so for itself: a few
// KB out of L2, cheaper than a second launch or a wait between CTAs) and then
// does slice s of the chunk's new blocks and new tokens, found by binary search
// in the scanned offsets.  A token in a new block reads the free list, not the
// table, so no CTA needs what another one writes.
// ---------------------------------------------------------------------------
constexpr int kTablesThreads = 512;
constexpr int kTablesChunk = 2 * kTablesThreads;

__device__ __forceinline__ uint64_t warp_inclusive(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// last i with off[i] <= x, for off[0 .. n] ascending and off[0] <= x < off[n]
__device__ __forceinline__ int find_request(const uint32_t* off, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kTablesThreads) step_tables_kernel(StepTablesArgs p) {
  __shared__ uint32_t tok_off[kTablesChunk + 1], blk_off[kTablesChunk + 1];
  __shared__ int32_t first_tok[kTablesChunk];
  __shared__ uint64_t warp_tok[kTablesThreads / 32], warp_blk[kTablesThreads / 32];
  __shared__ uint64_t base_tok_s, base_blk_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b0 = blockIdx.y * kTablesChunk;
  const int nb = p.num_seqs - b0 < kTablesChunk ? p.num_seqs - b0 : kTablesChunk;
  const bool last_chunk = blockIdx.y == gridDim.y - 1;
  const uint32_t bs = (uint32_t)p.block_size;
  bool bad = false;
  // request b's cached tokens, new tokens and new blocks (lengths below zero, or
  // past 2^31 - 1 together, are input errors: flagged, read as zero)
  auto request = [&](int b, uint32_t* pre, uint32_t* fresh, uint32_t* blocks) {
    const int32_t x = p.prefix_lens[b], y = p.new_lens[b];
    const bool ok = x >= 0 && y >= 0 && (int64_t)x + y <= 0x7fffffffll;
    bad |= !ok;
    *pre = ok ? (uint32_t)x : 0u;
    *fresh = ok ? (uint32_t)y : 0u;
    *blocks = (*pre + *fresh + bs - 1) / bs - (*pre + bs - 1) / bs;
  };

  // the requests before this chunk
  uint64_t tok = 0, blk = 0;
  for (int b = tid; b < b0; b += kTablesThreads) {
    uint32_t pre, fresh, blocks;
    request(b, &pre, &fresh, &blocks);
    tok += fresh;
    blk += blocks;
  }
  if (b0 > 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      tok += __shfl_xor_sync(0xffffffffu, tok, o);
      blk += __shfl_xor_sync(0xffffffffu, blk, o);
    }
    if (lane == 0) {
      warp_tok[warp] = tok;
      warp_blk[warp] = blk;
    }
    __syncthreads();
    if (tid == 0) {
      uint64_t a = 0, c = 0;
      for (int w = 0; w < kTablesThreads / 32; ++w) {
        a += warp_tok[w];
        c += warp_blk[w];
      }
      base_tok_s = a;
      base_blk_s = c;
    }
  } else if (tid == 0) {
    base_tok_s = base_blk_s = 0;
  }
  __syncthreads();
  const uint64_t base_tok = base_tok_s, base_blk = base_blk_s;

  // this chunk's two requests of the thread, and the scan over the chunk
  uint32_t pre[2] = {0u, 0u}, fresh[2] = {0u, 0u}, blocks[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (2 * tid + e < nb) request(b0 + 2 * tid + e, &pre[e], &fresh[e], &blocks[e]);
  const uint64_t st = warp_inclusive((uint64_t)fresh[0] + fresh[1], lane);
  const uint64_t sb = warp_inclusive((uint64_t)blocks[0] + blocks[1], lane);
  if (lane == 31) {
    warp_tok[warp] = st;
    warp_blk[warp] = sb;
  }
  __syncthreads();
  uint64_t at = st - fresh[0] - fresh[1], ab = sb - blocks[0] - blocks[1];
  for (int w = 0; w < warp; ++w) {
    at += warp_tok[w];
    ab += warp_blk[w];
  }
  const uint64_t limit = 0x7fffffffull;  // (offsets past int32 are past every output too: saturated)
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * tid + e;
    const uint64_t t = at + (e ? fresh[0] : 0u), k = ab + (e ? blocks[0] : 0u);
    if (i < nb) {
      tok_off[i] = (uint32_t)(t < limit ? t : limit);
      blk_off[i] = (uint32_t)(k < limit ? k : limit);
      first_tok[i] = (int32_t)pre[e];
      if (blockIdx.x == 0) {
        p.kv_lens[b0 + i] = (int32_t)(pre[e] + fresh[e]);
        const uint64_t row = base_tok + t;
        p.qo_indptr[b0 + i] = (int32_t)(row < limit ? row : limit);
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    uint64_t a = 0, c = 0;
    for (int w = 0; w < kTablesThreads / 32; ++w) {
      a += warp_tok[w];
      c += warp_blk[w];
    }
    tok_off[nb > 0 ? nb : 0] = (uint32_t)(a < limit ? a : limit);
    blk_off[nb > 0 ? nb : 0] = (uint32_t)(c < limit ? c : limit);
    if (last_chunk && blockIdx.x == 0) {
      const uint64_t total = base_tok + a, used = base_blk + c;
      p.qo_indptr[p.num_seqs] = (int32_t)(total < limit ? total : limit);
      *p.blocks_used = (int32_t)(used < limit ? used : limit);
      bad |= total > (uint64_t)p.num_tokens;
    }
  }
  __syncthreads();
  const int n = nb > 0 ? nb : 0;
  const uint32_t ntok = tok_off[n], nblk = blk_off[n];
  const uint64_t threads = (uint64_t)gridDim.x * kTablesThreads;
  const uint64_t me = (uint64_t)blockIdx.x * kTablesThreads + tid;

  // new blocks: free list -> table rows
  for (uint64_t k = me; k < nblk; k += threads) {
    const int i = find_request(blk_off, n, (uint32_t)k);
    const uint64_t f = base_blk + k;
    const int64_t col = ((int64_t)first_tok[i] + bs - 1) / bs + (int64_t)((uint32_t)k - blk_off[i]);
    const bool have = f < (uint64_t)p.num_free;
    bad |= !have || col >= p.table_len;
    if (col < p.table_len) p.tables[(int64_t)(b0 + i) * p.table_stride + col] = have ? p.free_blocks[f] : -1;
  }

  // new tokens, four consecutive rows to a thread; the last chunk also fills the
  // rows past the batch (capacity of a captured step) with -1
  const int64_t row0 = (int64_t)(base_tok < (uint64_t)p.num_tokens ? base_tok : (uint64_t)p.num_tokens);
  int64_t row1 = last_chunk ? p.num_tokens : row0 + (int64_t)ntok;
  if (row1 > p.num_tokens) row1 = p.num_tokens;
  const bool vec = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15u) == 0;
  for (int64_t g = row0 / 4 + (int64_t)me; g * 4 < row1; g += (int64_t)threads) {
    int32_t pos[4];
    int64_t slot[4];
    int i = -1;
    int64_t id = -1;      // block of the token before, to be carried on inside it
    uint32_t in_blk = 0;  // its place in that block
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t r = g * 4 + e;
      pos[e] = -1;
      slot[e] = -1;
      if (r < row0 || r - row0 >= (int64_t)ntok) continue;
      const uint32_t x = (uint32_t)(r - row0);
      const bool same = i >= 0 && x < tok_off[i + 1];
      if (!same) i = find_request(tok_off, n, x);
      const int32_t t = first_tok[i] + (int32_t)(x - tok_off[i]);
      pos[e] = t;
      if (same && in_blk + 1 < bs) {
        ++in_blk;
      } else {
        const uint32_t col = (uint32_t)t / bs, had = ((uint32_t)first_tok[i] + bs - 1) / bs;
        in_blk = (uint32_t)t - col * bs;
        const uint64_t f = base_blk + blk_off[i] + (col - had);
        id = -1;
        if ((int64_t)col < p.table_len) {
          if (col < had) id = p.tables[(int64_t)(b0 + i) * p.table_stride + col];
          else if (f < (uint64_t)p.num_free) id = p.free_blocks[f];
        }
      }
      if (id >= 0) slot[e] = id * (int64_t)bs + in_blk;
      bad |= id < 0;
    }
    if (!p.slots_i64) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (slot[e] > 0x7fffffffll) {
          slot[e] = -1;
          bad = true;
        }
    }
    if (vec && g * 4 >= row0 && g * 4 + 4 <= row1) {
      reinterpret_cast<int4*>(p.positions)[g] = make_int4(pos[0], pos[1], pos[2], pos[3]);
      if (p.slots_i64) {
        reinterpret_cast<longlong2*>(p.slots)[2 * g] = make_longlong2(slot[0], slot[1]);
        reinterpret_cast<longlong2*>(p.slots)[2 * g + 1] = make_longlong2(slot[2], slot[3]);
      } else {
        reinterpret_cast<int4*>(p.slots)[g] = make_int4((int)slot[0], (int)slot[1], (int)slot[2], (int)slot[3]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t r = g * 4 + e;
        if (r < row0 || r >= row1) continue;
        p.positions[r] = pos[e];
        if (p.slots_i64) reinterpret_cast<int64_t*>(p.slots)[r] = slot[e];
        else reinterpret_cast<int32_t*>(p.slots)[r] = (int32_t)slot[e];
      }
    }
  }
  if (bad) set_status(&g_layer_ops_status, KVC_STATUS_INDEX_OOB);
}

cudaError_t launch_step_tables(const StepTablesArgs& a, cudaStream_t stream) {
  const int64_t chunks = a.num_seqs > 0 ? ((int64_t)a.num_seqs + kTablesChunk - 1) / kTablesChunk : 1;
  if (chunks > 65535) return cudaErrorInvalidValue;
  // a thread's four rows at a time, up to two CTAs to an SM
  int64_t slices = (a.num_tokens + 4 * kTablesThreads - 1) / (4 * kTablesThreads);
  const int64_t most = 2 * (int64_t)sm_count() / chunks;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  step_tables_kernel<<<dim3((unsigned)slices, (unsigned)chunks), kTablesThreads, 0, stream>>>(a);
  count_launch();
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Rotary table: row p is [cos(p f_i)] then [sin(p f_i)], i < R / 2, times the
// attention factor of the scaling rule.  The angle is formed and reduced in 64
// bits (at position 10^6 a 32-bit angle is off by 0.03 rad) and rounded once.
// Written once per model; the division of work is of no weight.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) rotary_table_kernel(RotaryTableArgs p) {
  const int64_t total = p.rows * p.half;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / p.half;
    const int f = (int)(i - row * p.half);
    double s, c;
    sincos((double)row * p.inv_freq[f], &s, &c);
    p.table[row * p.stride + f] = (float)(c * p.factor);
    p.table[row * p.stride + p.half + f] = (float)(s * p.factor);
  }
}

cudaError_t launch_rotary_table(const RotaryTableArgs& a, cudaStream_t stream) {
  const int64_t total = a.rows * a.half;
  if (total <= 0) return cudaSuccess;
  int64_t ctas = (total + 255) / 256;
  const int64_t most = 8 * (int64_t)sm_count();
  if (ctas > most) ctas = most;
  rotary_table_kernel<<<(unsigned)ctas, 256, 0, stream>>>(a);
  count_launch();
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Per-head RMS norm and rotary position.  For a head's row x of D elements,
// its weight w and its token's cosines c and sines s (R = 2 * half rotated
// dims, the rest pass):
//   y_d = x_d w_d / sqrt(sum_e x_e^2 / D + eps)          (or y = x)
//   half layout         (y_i, y_{i + half}),   interleaved   (y_2i, y_2i+1):
//   (a, b) -> (a c_i - b s_i, b c_i + a s_i)
// in 32 bits, rounded once to the output's type.
// ---------------------------------------------------------------------------
template <typename T, int VEC>
struct Vec {  // VEC consecutive elements as the widest loads and stores up to 16 bytes
  static constexpr int BYTES = VEC * (int)sizeof(T);
  static_assert(BYTES % 8 == 0, "whole 8-byte words");
  T e[VEC];
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(src);
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(src)[i];
    }
  }
  __device__ __forceinline__ void store(T* dst) const {
    if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(e)[i];
    }
  }
};

// The token's table row and cache place; false: its rows are skipped (a negative
// position or slot is padding, one past the table or the cache is flagged).
__device__ __forceinline__ int64_t load_index(const void* a, bool i64, int64_t i) {
  return i64 ? reinterpret_cast<const int64_t*>(a)[i] : (int64_t)reinterpret_cast<const int32_t*>(a)[i];
}

__device__ __forceinline__ bool token_place(const RopeArgs& p, int64_t slot, bool flag, int64_t* blk, int* off) {
  if (slot < 0) return false;
  *blk = slot / p.block_size;
  *off = (int)(slot - *blk * p.block_size);
  if (*blk >= p.num_blocks) {
    if (flag) set_status(&g_layer_ops_status, KVC_STATUS_SLOT_OOB);
    return false;
  }
  return true;
}

// How a launch divides a token's rows: chunks of U passes of the warp, each over
// 32 >> lpr_shift rows; first the q heads, then the k heads, then (append) the v
// heads.  CTAs from `row_ctas` on move V through shared-memory tiles instead.
struct RopePlan {
  int lpr_shift, q_chunks, k_chunks, v_chunks;
  unsigned row_ctas;
};
constexpr int kRopeWarps = 8;
constexpr int kVTile = 32;  // tokens of a V tile

// V of kVTile tokens and one head into [block][head][dim][offset]: rows in, then
// lane = token, so tokens at consecutive offsets of a block make one run.
template <typename T, int VEC>
__device__ __forceinline__ void store_v_tile(const RopeArgs& p, int64_t tile, unsigned char* smem) {
  constexpr int PAD = sizeof(T) == 2 ? 2 : 1;  // an odd number of words to a row
  __shared__ int64_t s_dst[kVTile];
  const int64_t t0 = tile / p.num_kv_heads * kVTile;
  const int h = (int)(tile % p.num_kv_heads), D = p.head_size, stride = D + PAD;
  T* rows = reinterpret_cast<T*>(smem);
  const int ntok = (int)(p.num_tokens - t0 < kVTile ? p.num_tokens - t0 : kVTile);
  if (threadIdx.x < kVTile) {
    int64_t blk = 0;
    int off = 0;
    const bool on = (int)threadIdx.x < ntok &&
                    token_place(p, load_index(p.slots, p.slots_i64, t0 + threadIdx.x), h == 0, &blk, &off);
    s_dst[threadIdx.x] = on ? blk * p.vc_block + (int64_t)h * p.vc_head + off : -1;
  }
  const T* v = reinterpret_cast<const T*>(p.v) + (int64_t)h * p.v_head;
  const int nvec = D / VEC;
  for (int i = threadIdx.x; i < ntok * nvec; i += kRopeWarps * 32) {
    const int t = i / nvec, d = (i - t * nvec) * VEC;
    Vec<T, VEC> x;
    x.load(v + (t0 + t) * p.v_tok + d);
    constexpr int W = VEC * (int)sizeof(T) / 4;
#pragma unroll
    for (int e = 0; e < W; ++e)
      reinterpret_cast<uint32_t*>(rows + t * stride + d)[e] = reinterpret_cast<const uint32_t*>(x.e)[e];
  }
  __syncthreads();
  T* vc = reinterpret_cast<T*>(p.v_cache);
  for (int i = threadIdx.x; i < kVTile * D; i += kRopeWarps * 32) {
    const int t = i % kVTile, d = i / kVTile;
    const int64_t dst = s_dst[t];
    if (dst >= 0) vc[dst + (int64_t)d * p.block_size] = rows[t * stride + d];
  }
}

template <typename T, int VEC, bool INTER, int U>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(const RopeArgs p, const RopePlan pl) {
  extern __shared__ __align__(16) unsigned char smem_rope[];
  if (blockIdx.x >= pl.row_ctas) {
    store_v_tile<T, VEC>(p, blockIdx.x - pl.row_ctas, smem_rope);
    return;
  }
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  const unsigned per = (unsigned)(pl.q_chunks + pl.k_chunks + pl.v_chunks);
  const unsigned tok = w / per;
  if (tok >= p.num_tokens) return;
  int chunk = (int)(w - tok * per);
  const int kind = chunk < pl.q_chunks ? 0 : (chunk < pl.q_chunks + pl.k_chunks ? 1 : 2);
  if (kind > 0) chunk -= pl.q_chunks;
  if (kind > 1) chunk -= pl.k_chunks;
  const bool to_cache = kind > 0 && p.k_cache != nullptr;
  const int64_t pos = load_index(p.positions, p.pos_i64, tok);
  const int64_t slot = to_cache ? load_index(p.slots, p.slots_i64, tok) : 0;

  const int lpr = 1 << pl.lpr_shift, rpw = 32 >> pl.lpr_shift;
  const int sub = lane >> pl.lpr_shift, li = lane & (lpr - 1);
  const int D = p.head_size, d0 = li * VEC, half = p.rot >> 1;
  const int heads = kind ? p.num_kv_heads : p.num_heads;
  const int h0 = chunk * rpw * U + sub;
  const bool on = d0 < D;
  const T* src = reinterpret_cast<const T*>(kind == 0 ? p.q : (kind == 1 ? p.k : p.v));
  const int64_t s_tok = kind == 0 ? p.q_tok : (kind == 1 ? p.k_tok : p.v_tok);
  const int64_t s_head = kind == 0 ? p.q_head : (kind == 1 ? p.k_head : p.v_head);
  src += (int64_t)tok * s_tok + d0;

  // every load of the warp's rows before any is used
  Vec<T, VEC> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * rpw;
    if (on && h < heads) x[u].load(src + (int64_t)h * s_head);
    else
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[u].e[e] = from_float<T>(0.f);
  }
  int64_t blk = 0;
  int off = 0;
  if (to_cache && !token_place(p, slot, chunk == 0 && kind == 1 && lane == 0, &blk, &off)) return;

  if (kind == 2) {
    T* vc = reinterpret_cast<T*>(p.v_cache) + blk * p.vc_block;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * rpw;
      if (!on || h >= heads) continue;
      T* dst = vc + (int64_t)h * p.vc_head;
      if (p.paged) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dst[(int64_t)(d0 + e) * p.block_size + off] = x[u].e[e];
      } else {
        x[u].store(dst + (int64_t)off * p.vc_tok + d0);
      }
    }
    return;
  }
  if (pos < 0 || pos >= p.table_rows) {  // (the whole warp: one token)
    if (pos >= 0 && lane == 0) set_status(&g_layer_ops_status, KVC_STATUS_INDEX_OOB);
    return;
  }

  // this lane's cosines and sines (in the half layout an element's own, so that
  // the pair is formed by one exchange with the lane that holds the other half)
  constexpr int NC = INTER ? VEC / 2 : VEC;
  float c[NC], s[NC];
  const bool rotated = on && d0 < p.rot;
  const bool upper = !INTER && d0 >= half;
  const float* cs = p.table + pos * p.table_stride + (INTER ? d0 / 2 : (upper ? d0 - half : d0));
#pragma unroll
  for (int i = 0; i < NC; i += 2) {
    const float2 a = rotated ? __ldg(reinterpret_cast<const float2*>(cs + i)) : make_float2(1.f, 1.f);
    const float2 b = rotated ? __ldg(reinterpret_cast<const float2*>(cs + half + i)) : make_float2(0.f, 0.f);
    c[i] = a.x;
    c[i + 1] = a.y;
    s[i] = upper ? b.x : (INTER ? b.x : -b.x);
    s[i + 1] = upper ? b.y : (INTER ? b.y : -b.y);
  }
  const void* wp = kind ? p.k_weight : p.q_weight;
  float wt[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) wt[e] = 1.f;
  if (wp && on) {
    if (p.weight_type == ElemType::F32) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) wt[e] = __ldg(reinterpret_cast<const float*>(wp) + d0 + e);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) wt[e] = to_float(reinterpret_cast<const T*>(wp)[d0 + e]);
    }
  }
  // the lane that holds the other element of each pair (half layout)
  const int mate = rotated ? (upper ? lane - half / VEC : lane + half / VEC) : lane;
  T* dst = reinterpret_cast<T*>(kind == 0 ? p.q_out : p.k_out);
  const int64_t o_head = kind == 0 ? p.qo_head : p.ko_head;
  if (to_cache) dst = reinterpret_cast<T*>(p.k_cache) + blk * p.kc_block;
  else dst += (int64_t)tok * (kind == 0 ? p.qo_tok : p.ko_tok) + d0;
  constexpr int X = 16 / (int)sizeof(T);

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * rpw;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] = to_float(x[u].e[e]);
    if (wp) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss = fmaf(y[e], y[e], ss);
      for (int o = 1; o < lpr; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] *= inv * wt[e];
    }
    Vec<T, VEC> out;
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float a = y[2 * i], b = y[2 * i + 1];
        out.e[2 * i] = from_float<T>(rotated ? a * c[i] - b * s[i] : a);
        out.e[2 * i + 1] = from_float<T>(rotated ? fmaf(b, c[i], a * s[i]) : b);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float m = __shfl_sync(0xffffffffu, y[e], mate);
        out.e[e] = from_float<T>(rotated ? fmaf(m, s[e], y[e] * c[e]) : y[e]);
      }
    }
    if (!on || h >= heads) continue;
    if (!to_cache) {
      out.store(dst + (int64_t)h * o_head);
    } else if (p.paged) {  // 16-byte places [d / X][offset] of the page
      T* page = dst + (int64_t)h * p.kc_head;
      if constexpr (VEC >= X) {
#pragma unroll
        for (int i = 0; i < VEC / X; ++i)
          *reinterpret_cast<uint4*>(page + ((int64_t)(d0 / X + i) * p.block_size + off) * X) =
              reinterpret_cast<const uint4*>(out.e)[i];
      } else {
        out.store(page + ((int64_t)(d0 / X) * p.block_size + off) * X + d0 % X);
      }
    } else {
      out.store(dst + (int64_t)off * p.kc_tok + (int64_t)h * p.kc_head + d0);
    }
  }
}

// The same for every other case: odd head sizes, halves that no vector divides,
// unaligned rows, 32-bit rows into a 16-bit cache.  A warp per row, element by
// element, the normed row in shared memory between norm and rotation.
constexpr int kRopeMaxHead = 512;

template <typename T, typename C>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_any_kernel(const RopeArgs p) {
  __shared__ float row_s[kRopeWarps][kRopeMaxHead];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned per = (unsigned)(p.num_heads + p.num_kv_heads * (p.k_cache ? 2 : 1));
  const unsigned w = blockIdx.x * kRopeWarps + warp, tok = w / per;
  if (tok >= p.num_tokens) return;
  int h = (int)(w - tok * per);
  const int kind = h < p.num_heads ? 0 : (h < p.num_heads + p.num_kv_heads ? 1 : 2);
  if (kind > 0) h -= p.num_heads;
  if (kind > 1) h -= p.num_kv_heads;
  const bool to_cache = kind > 0 && p.k_cache != nullptr;
  const int D = p.head_size, half = p.rot >> 1;
  int64_t blk = 0;
  int off = 0;
  if (to_cache && !token_place(p, load_index(p.slots, p.slots_i64, tok), h == 0 && kind == 1 && lane == 0, &blk, &off))
    return;
  const T* src = kind == 0   ? reinterpret_cast<const T*>(p.q) + (int64_t)tok * p.q_tok + (int64_t)h * p.q_head
                 : kind == 1 ? reinterpret_cast<const T*>(p.k) + (int64_t)tok * p.k_tok + (int64_t)h * p.k_head
                             : reinterpret_cast<const T*>(p.v) + (int64_t)tok * p.v_tok + (int64_t)h * p.v_head;
  C* kc = reinterpret_cast<C*>(p.k_cache);
  C* vc = reinterpret_cast<C*>(p.v_cache);
  if (kind == 2) {
    for (int d = lane; d < D; d += 32)
      vc[blk * p.vc_block + (int64_t)h * p.vc_head +
         (p.paged ? (int64_t)d * p.block_size + off : (int64_t)off * p.vc_tok + d)] = Convert<T, C>::apply(src[d]);
    return;
  }
  const int64_t pos = load_index(p.positions, p.pos_i64, tok);
  if (pos < 0 || pos >= p.table_rows) {
    if (pos >= 0 && lane == 0) set_status(&g_layer_ops_status, KVC_STATUS_INDEX_OOB);
    return;
  }
  float* row = row_s[warp];
  float ss = 0.f;
  for (int d = lane; d < D; d += 32) {
    const float x = to_float(src[d]);
    row[d] = x;
    ss = fmaf(x, x, ss);
  }
  const void* wp = kind ? p.k_weight : p.q_weight;
  if (wp) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / (float)D + p.eps);
    for (int d = lane; d < D; d += 32)
      row[d] *= inv * (p.weight_type == ElemType::F32 ? reinterpret_cast<const float*>(wp)[d]
                                                      : to_float(reinterpret_cast<const T*>(wp)[d]));
  }
  __syncwarp();
  const float* cs = p.table + pos * p.table_stride;
  constexpr int X = 16 / (int)sizeof(C);
  for (int d = lane; d < D; d += 32) {
    float y = row[d];
    if (d < p.rot) {
      const int i = p.interleaved ? d >> 1 : (d < half ? d : d - half);
      const bool second = p.interleaved ? d & 1 : d >= half;
      const float m = row[p.interleaved ? d ^ 1 : (second ? d - half : d + half)];
      const float s = cs[half + i];
      y = fmaf(m, second ? s : -s, y * cs[i]);
    }
    if (!to_cache) {
      T* dst = kind == 0 ? reinterpret_cast<T*>(p.q_out) + (int64_t)tok * p.qo_tok + (int64_t)h * p.qo_head
                         : reinterpret_cast<T*>(p.k_out) + (int64_t)tok * p.ko_tok + (int64_t)h * p.ko_head;
      dst[d] = from_float<T>(y);
    } else {
      kc[blk * p.kc_block + (int64_t)h * p.kc_head +
         (p.paged ? ((int64_t)(d / X) * p.block_size + off) * X + d % X : (int64_t)off * p.kc_tok + d)] =
          from_float<C>(y);
    }
  }
}

template <typename T, typename C>
static cudaError_t launch_rope_any(const RopeArgs& a, cudaStream_t stream) {
  const int64_t rows = a.num_tokens * (a.num_heads + (int64_t)a.num_kv_heads * (a.k_cache ? 2 : 1));
  if (a.head_size > kRopeMaxHead || rows > 0x7fffffffll) return cudaErrorInvalidValue;
  qk_norm_rope_any_kernel<T, C><<<(unsigned)((rows + kRopeWarps - 1) / kRopeWarps), kRopeWarps * 32, 0, stream>>>(a);
  count_launch();
  return cudaGetLastError();
}

template <typename T, int VEC, bool INTER, int U>
static cudaError_t launch_rope_u(const RopeArgs& a, RopePlan pl, bool v_tiles, cudaStream_t stream) {
  const int rpw = 32 >> pl.lpr_shift;
  pl.q_chunks = (a.num_heads + rpw * U - 1) / (rpw * U);
  pl.k_chunks = (a.num_kv_heads + rpw * U - 1) / (rpw * U);
  pl.v_chunks = a.k_cache && !v_tiles ? pl.k_chunks : 0;
  const int64_t warps = a.num_tokens * (pl.q_chunks + pl.k_chunks + pl.v_chunks);
  const int64_t tiles = v_tiles ? (a.num_tokens + kVTile - 1) / kVTile * a.num_kv_heads : 0;
  const int64_t ctas = (warps + kRopeWarps - 1) / kRopeWarps;
  if (ctas + tiles > 0x7fffffffll / kRopeWarps) return cudaErrorInvalidValue;
  pl.row_ctas = (unsigned)ctas;
  const size_t smem = v_tiles ? (size_t)kVTile * (a.head_size + (sizeof(T) == 2 ? 2 : 1)) * sizeof(T) : 0;
  qk_norm_rope_kernel<T, VEC, INTER, U><<<(unsigned)(ctas + tiles), kRopeWarps * 32, smem, stream>>>(a, pl);
  count_launch();
  return cudaGetLastError();
}

template <typename T, int VEC>
static cudaError_t launch_rope_vec(const RopeArgs& a, cudaStream_t stream) {
  RopePlan pl = {};
  while ((VEC << pl.lpr_shift) < a.head_size) ++pl.lpr_shift;
  const int rpw = 32 >> pl.lpr_shift;
  const int64_t rows = a.num_tokens * (a.num_heads + (int64_t)a.num_kv_heads * (a.k_cache ? 2 : 1));
  // four passes to a warp once that still fills the GPU (16 warps to an SM)
  const bool four = rows >= (int64_t)sm_count() * 16 * 4 * rpw;
  const bool v_tiles = a.k_cache && a.paged && a.num_tokens >= 1024;
  if (a.interleaved)
    return four ? launch_rope_u<T, VEC, true, 4>(a, pl, v_tiles, stream)
                : launch_rope_u<T, VEC, true, 1>(a, pl, v_tiles, stream);
  return four ? launch_rope_u<T, VEC, false, 4>(a, pl, v_tiles, stream)
              : launch_rope_u<T, VEC, false, 1>(a, pl, v_tiles, stream);
}

// Whether every row the launch touches can be moved VEC elements at a time.
static bool rope_vec_ok(const RopeArgs& a, int vec, int es) {
  const int D = a.head_size;
  const int64_t align = vec * es < 16 ? vec * es : 16;
  // the rotated part is whole vectors, and so is each half of it in the half layout
  if (D % vec || D > 32 * vec || a.rot % (a.interleaved ? vec : 2 * vec) || a.type != a.cache_type) return false;
  auto rows = [&](const void* base, int64_t s1, int64_t s2, int64_t s3) {
    return reinterpret_cast<uintptr_t>(base) % align == 0 && (s1 * es) % align == 0 && (s2 * es) % align == 0 &&
           (s3 * es) % align == 0;
  };
  if (!rows(a.q, a.q_tok, a.q_head, 0) || !rows(a.k, a.k_tok, a.k_head, 0) || !rows(a.q_out, a.qo_tok, a.qo_head, 0))
    return false;
  if ((reinterpret_cast<uintptr_t>(a.table) & 7u) || (a.table_stride & 1)) return false;  // (float2 loads)
  if ((a.rot >> 1) & 1) return false;
  if (!a.k_cache) return rows(a.k_out, a.ko_tok, a.ko_head, 0);
  return rows(a.v, a.v_tok, a.v_head, 0) && rows(a.k_cache, a.kc_block, a.kc_head, a.kc_tok) &&
         (a.paged || rows(a.v_cache, a.vc_block, a.vc_head, a.vc_tok));
}

template <typename T>
static cudaError_t launch_rope_t(const RopeArgs& a, cudaStream_t stream) {
  if (rope_vec_ok(a, 8, sizeof(T))) return launch_rope_vec<T, 8>(a, stream);
  if (rope_vec_ok(a, 4, sizeof(T))) return launch_rope_vec<T, 4>(a, stream);
  return launch_rope_any<T, T>(a, stream);
}

cudaError_t launch_qk_norm_rope(const RopeArgs& a, cudaStream_t stream) {
  if (a.type == ElemType::F16) return launch_rope_t<__half>(a, stream);
  if (a.type == ElemType::BF16) return launch_rope_t<__nv_bfloat16>(a, stream);
  if (a.cache_type == ElemType::F16) return launch_rope_any<float, __half>(a, stream);
  if (a.cache_type == ElemType::BF16) return launch_rope_any<float, __nv_bfloat16>(a, stream);
  return launch_rope_t<float>(a, stream);
}

}  // namespace kvc

unsigned int kvc_layer_ops_status(int clear, cudaError_t* err) {
  unsigned int v = 0;
  *err = cudaMemcpyFromSymbol(&v, kvc::g_layer_ops_status, sizeof(v));
  if (*err == cudaSuccess && clear) {
    const unsigned int zero = 0;
    *err = cudaMemcpyToSymbol(kvc::g_layer_ops_status, &zero, sizeof(zero));
  }
  return v;
}
