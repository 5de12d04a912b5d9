// layer_ops.cu — what surrounds the attention of a step, for sm_100a: the block
// tables, positions and slot maps of a batch built from its lengths, and the
// per-head RMS norm with the rotary position of queries and keys, on its own or
// fused with the append of keys and values into the cache.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "kvc_common.cuh"

namespace kvc {

__device__ unsigned int g_layer_ops_status = 0;

// Every kernel here is a programmatic dependent of the kernel before it on the
// stream: its launch overlaps that kernel's end, and it waits for it before it
// reads or writes anything (with coherent loads: the non-coherent ones want data
// that nothing writes while the kernel runs).  None lets its own dependents start
// early: the whole-context decode kernels read queries, tables and lengths, which
// are written here, before they wait.
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
static cudaError_t launch_dependent(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                    A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

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
// table, so no CTA needs what another one writes, and none may write what another
// one still reads: lengths that are updated in place (kv_lens is prefix_lens or
// new_lens) are left to a second kernel (0.85 us more).  A few KB move: what counts is the
// chain of launch, loads, scan, search and stores (64 requests with one token each
// 4.9 us back to back, 528 of a mixed step 6.8; 256 prompts of up to 4096 tokens, 7.2
// MB of positions and slots, 6.6; an empty kernel launched the same way takes about
// 2.1).
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

// A request's lengths: below zero, or past 2^31 - 1 together, is an input error, read
// as zero (false).
__device__ __forceinline__ bool request_lens(const StepTablesArgs& p, int b, uint32_t* pre, uint32_t* fresh) {
  const int32_t x = p.prefix_lens[b], y = p.new_lens[b];
  const bool ok = x >= 0 && y >= 0 && (int64_t)x + y <= 0x7fffffffll;
  *pre = ok ? (uint32_t)x : 0u;
  *fresh = ok ? (uint32_t)y : 0u;
  return ok;
}

// The lengths in place: each thread reads a request's own before it writes them.
__global__ void __launch_bounds__(256) step_lens_kernel(StepTablesArgs p) {
  wait_for_prior();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= p.num_seqs) return;
  uint32_t pre, fresh;
  request_lens(p, b, &pre, &fresh);
  p.kv_lens[b] = (int32_t)(pre + fresh);
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
  wait_for_prior();
  // request b's cached tokens, new tokens and new blocks (input errors are flagged)
  auto request = [&](int b, uint32_t* pre, uint32_t* fresh, uint32_t* blocks) {
    bad |= !request_lens(p, b, pre, fresh);
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
        if (!p.lens_in_place) p.kv_lens[b0 + i] = (int32_t)(pre[e] + fresh[e]);
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

  // new blocks: free list -> table rows (the first one's id is on its way while
  // the tokens are done)
  auto free_id = [&](uint64_t k) {
    const uint64_t f = base_blk + k;
    return f < (uint64_t)p.num_free ? p.free_blocks[f] : -1;
  };
  int32_t next_id = me < nblk ? free_id(me) : -1;

  // new tokens, four consecutive rows to a thread, the block ids of all four read
  // before one is used; the last chunk also fills the rows past the batch (capacity
  // of a captured step) with -1
  const int64_t row0 = (int64_t)(base_tok < (uint64_t)p.num_tokens ? base_tok : (uint64_t)p.num_tokens);
  int64_t row1 = last_chunk ? p.num_tokens : row0 + (int64_t)ntok;
  if (row1 > p.num_tokens) row1 = p.num_tokens;
  const bool vec = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15u) == 0;
  for (int64_t g = row0 / 4 + (int64_t)me; g * 4 < row1; g += (int64_t)threads) {
    int32_t pos[4];
    int64_t slot[4];
    uint32_t in_blk[4];
    const int32_t* id_at[4];  // (nullptr: no block)
    int i = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t r = g * 4 + e;
      pos[e] = -1;
      slot[e] = -1;
      in_blk[e] = 0u;
      id_at[e] = nullptr;
      if (r < row0 || r - row0 >= (int64_t)ntok) continue;
      const uint32_t x = (uint32_t)(r - row0);
      if (i < 0 || x >= tok_off[i + 1]) i = find_request(tok_off, n, x);
      const int32_t t = first_tok[i] + (int32_t)(x - tok_off[i]);
      const uint32_t col = (uint32_t)t / bs, had = ((uint32_t)first_tok[i] + bs - 1) / bs;
      pos[e] = t;
      in_blk[e] = (uint32_t)t - col * bs;
      const uint64_t f = base_blk + blk_off[i] + (col - had);
      if ((int64_t)col < p.table_len) {
        if (col < had) id_at[e] = p.tables + (int64_t)(b0 + i) * p.table_stride + col;
        else if (f < (uint64_t)p.num_free) id_at[e] = p.free_blocks + f;
      }
    }
    int32_t id[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) id[e] = id_at[e] ? *id_at[e] : -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (id[e] >= 0) slot[e] = (int64_t)id[e] * (int64_t)bs + in_blk[e];
      bad |= pos[e] >= 0 && id[e] < 0;
      if (!p.slots_i64 && slot[e] > 0x7fffffffll) {
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

  for (uint64_t k = me; k < nblk; k += threads) {
    const int i = find_request(blk_off, n, (uint32_t)k);
    const int64_t col = ((int64_t)first_tok[i] + bs - 1) / bs + (int64_t)((uint32_t)k - blk_off[i]);
    bad |= base_blk + k >= (uint64_t)p.num_free || col >= p.table_len;
    if (col < p.table_len) p.tables[(int64_t)(b0 + i) * p.table_stride + col] = next_id;
    if (k + threads < nblk) next_id = free_id(k + threads);
  }
  if (bad) set_status(&g_layer_ops_status, KVC_STATUS_INDEX_OOB);
}

cudaError_t launch_step_tables(const StepTablesArgs& a, cudaStream_t stream) {
  const int64_t chunks = a.num_seqs > 0 ? ((int64_t)a.num_seqs + kTablesChunk - 1) / kTablesChunk : 1;
  if (chunks > 65535) return cudaErrorInvalidValue;
  // four rows to every fourth thread (the latency of a CTA's scan hides better
  // behind more CTAs than behind fuller ones), up to two CTAs to an SM
  int64_t slices = (a.num_tokens + kTablesThreads - 1) / kTablesThreads;
  const int64_t most = 2 * (int64_t)sm_count() / chunks;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  const cudaError_t e =
      launch_dependent(step_tables_kernel, dim3((unsigned)slices, (unsigned)chunks), kTablesThreads, 0, stream, a);
  if (e != cudaSuccess || !a.lens_in_place || a.num_seqs == 0) return e;
  return launch_dependent(step_lens_kernel, dim3((unsigned)((a.num_seqs + 255) / 256)), 256, 0, stream, a);
}

// ---------------------------------------------------------------------------
// Rotary table: row p is [cos(p f_i)] then [sin(p f_i)], i < R / 2, times the
// attention factor of the scaling rule.  The angle is formed and reduced in 64
// bits (at position 10^6 a 32-bit angle is off by 0.03 rad) and rounded once.
// Written once per model; the division of work is of no weight.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) rotary_table_kernel(RotaryTableArgs p) {
  wait_for_prior();
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
  return launch_dependent(rotary_table_kernel, dim3((unsigned)ctas), 256, 0, stream, a);
}

// ---------------------------------------------------------------------------
// Per-head RMS norm and rotary position.  For a head's row x of D elements,
// its weight w and its token's cosines c and sines s (R = 2 * half rotated
// dims, the rest pass):
//   y_d = x_d w_d / sqrt(sum_e x_e^2 / D + eps)          (or y = x)
//   half layout         (y_i, y_{i + half}),   interleaved   (y_2i, y_2i+1):
//   (a, b) -> (a c_i - b s_i, b c_i + a s_i)
// in 32 bits, rounded once to the output's type.  Memory sets the pace for many tokens
// (8192 tokens of 28 + 4 heads of 128, fp16, 136 MB: 25.6 us, 5.3 TB/s; with norm and
// append to 32-token pages 34.4 us, 4.5 TB/s; 28 + 4 heads in fp32 with norm 46.0 us, 5.9
// TB/s, and with the append 51.1, 6.0 TB/s), latency for few (256 tokens of 32 + 8
// heads: 4.0 us; with the append 7.5, half of it V's elements, each a sector of its
// own).
// ---------------------------------------------------------------------------
// Two fp32 lanes per instruction (the f32x2 arithmetic of sm_100), rounded as two
// scalar operations are.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmul.rn.f32x2 rd, ra, rb;\n"
      "mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 ra, rb, rc, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmov.b64 rc, {%6, %7};\n"
      "fma.rn.f32x2 rd, ra, rb, rc;\nmov.b64 {%0, %1}, rd;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 pair_to_float(uint32_t w, __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pair_from_float(float2 x, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair_from_float(float2 x, __half*) {
  const __half2 v = __floats2half2_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
struct Quad {  // four consecutive elements, one load or store (8 or 16 bytes)
  using Word = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
  Word w;
  __device__ __forceinline__ void load(const T* src) { w = *reinterpret_cast<const Word*>(src); }
  __device__ __forceinline__ void store(T* dst) const { *reinterpret_cast<Word*>(dst) = w; }
  __device__ __forceinline__ void get(float2& x, float2& y) const {
    if constexpr (sizeof(T) == 2) {
      x = pair_to_float(w.x, (T*)nullptr);
      y = pair_to_float(w.y, (T*)nullptr);
    } else {
      x = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
      y = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    }
  }
  __device__ __forceinline__ void put(float2 x, float2 y) {
    if constexpr (sizeof(T) == 2) {
      w.x = pair_from_float(x, (T*)nullptr);
      w.y = pair_from_float(y, (T*)nullptr);
    } else {
      w = make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
    }
  }
};

__device__ __forceinline__ int64_t load_index(const void* a, bool i64, int64_t i) {
  return i64 ? reinterpret_cast<const int64_t*>(a)[i] : (int64_t)reinterpret_cast<const int32_t*>(a)[i];
}

// The cache place of a slot; false: the token's rows are skipped (a negative
// slot is padding, one past the cache is flagged).
__device__ __forceinline__ bool token_place(const RopeArgs& p, int64_t slot, bool flag, int64_t* blk, int* off) {
  if (slot < 0) return false;
  if (slot <= 0xffffffffll) {  // (a 64-bit division costs a hundred instructions)
    const uint32_t s = (uint32_t)slot, b = s / (uint32_t)p.block_size;
    *blk = b;
    *off = (int)(s - b * (uint32_t)p.block_size);
  } else {
    *blk = slot / p.block_size;
    *off = (int)(slot - *blk * p.block_size);
  }
  if (*blk >= p.num_blocks) {
    if (flag) set_status(&g_layer_ops_status, KVC_STATUS_SLOT_OOB);
    return false;
  }
  return true;
}

// How a launch divides a token's rows.  A group is the 32 >> lpr_shift rows that a
// warp holds at a time; a token's groups are its q heads', then its k heads', then
// (append) its v heads', and a warp takes `span` of one token's groups.  CTAs from
// `row_ctas` on move V through shared-memory tiles instead.
struct RopePlan {
  int lpr_shift, q_groups, k_groups, v_groups, span;
  unsigned warps_per_token, row_ctas;
  float inv_d;
};
constexpr int kRopeWarps = 8;
constexpr int kVTile = 32;  // tokens of a V tile

// V of kVTile tokens and one head into [block][head][dim][offset].  The rows are
// staged in shared memory (16 bytes of padding: 8 rows cover all banks).  16-bit
// elements: a transposed matrix load whose matrix i takes tokens 8q + 2i, 8q + 2i
// + 1 for q = 0..3 leaves lane (dim, q) the tokens 8q .. 8q + 7 of its dim in
// order, so 8 tokens that lie in one block at consecutive offsets from a multiple
// of 8 on are one 16-byte store.  Tokens that do not, and 32-bit elements, go
// one by one, lane = token.
template <typename T>
__device__ __forceinline__ void store_v_tile(const RopeArgs& p, unsigned tile, unsigned char* smem) {
  __shared__ int64_t s_dst[kVTile];
  __shared__ uint32_t s_runs;  // bit q: tokens 8q .. 8q + 7 make such a run
  const unsigned tt = tile / (unsigned)p.num_kv_heads;
  const int64_t t0 = (int64_t)tt * kVTile;
  const int h = (int)(tile - tt * (unsigned)p.num_kv_heads), D = p.head_size;
  const int stride = D + 16 / (int)sizeof(T);
  T* rows = reinterpret_cast<T*>(smem);
  const int ntok = (int)(p.num_tokens - t0 < kVTile ? p.num_tokens - t0 : kVTile);
  if (threadIdx.x < kVTile) {
    const int lane = threadIdx.x;
    int64_t blk = 0;
    int off = 0;
    const bool on = lane < ntok && token_place(p, load_index(p.slots, p.slots_i64, t0 + lane), h == 0, &blk, &off);
    const int64_t dst = on ? blk * p.vc_block + (int64_t)h * p.vc_head + off : -1;
    s_dst[lane] = dst;
    const int64_t lead = __shfl_sync(0xffffffffu, dst, lane & ~7);
    const int lead_off = __shfl_sync(0xffffffffu, off, lane & ~7);
    const bool run = on && lead >= 0 && lead_off % 8 == 0 && off == lead_off + (lane & 7) && dst == lead + (lane & 7);
    const uint32_t m = __ballot_sync(0xffffffffu, run);
    uint32_t runs = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) runs |= ((m >> (8 * q)) & 0xffu) == 0xffu ? 1u << q : 0u;
    if (lane == 0) s_runs = runs;
  }
  const T* v = reinterpret_cast<const T*>(p.v) + (int64_t)h * p.v_head + t0 * p.v_tok;
  const int nq = D / 4;
  for (int i = threadIdx.x; i < kVTile * nq; i += kRopeWarps * 32) {
    const int t = i / nq, d = (i - t * nq) * 4;
    Quad<T> x;
    x.w = typename Quad<T>::Word{};
    if (t < ntok) x.load(v + t * p.v_tok + d);
    x.store(rows + t * stride + d);
  }
  __syncthreads();
  T* vc = reinterpret_cast<T*>(p.v_cache);
  // (16-byte stores need 16-byte pages: block sizes of 8, 16 and 32 tokens in aligned caches)
  const bool wide = sizeof(T) == 2 && p.v_wide;
  const uint32_t runs = wide ? s_runs : 0u;
  if constexpr (sizeof(T) == 2) {
    if (runs) {
      const int lane = threadIdx.x & 31, q = lane & 3;
      // lane l gives row l % 8 of matrix l / 8: token 8 (row / 2) + 2 matrix + row % 2
      const int row = lane & 7, tok = 8 * (row >> 1) + 2 * (lane >> 3) + (row & 1);
      const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(rows + tok * stride));
      const int64_t dst = s_dst[8 * q];
      for (int d = (threadIdx.x >> 5) * 8; d < D; d += kRopeWarps * 8) {
        uint4 x;
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                     : "r"(base + (uint32_t)d * 2u));
        if ((runs >> q) & 1u) *reinterpret_cast<uint4*>(vc + dst + (int64_t)(d + (lane >> 2)) * p.block_size) = x;
      }
    }
  }
  if (runs == 0xfu) return;
  const int t = threadIdx.x % kVTile;
  const int64_t dst = s_dst[t];
  if (dst < 0 || ((runs >> (t >> 3)) & 1u)) return;
  for (int d = threadIdx.x / kVTile; d < D; d += kRopeWarps * 32 / kVTile)
    vc[dst + (int64_t)d * p.block_size] = rows[t * stride + d];
}

// A lane holds 8 elements of a row as two quads: in the half layout quads a and
// a + half of the rotated part, so that its pairs are its own and share four
// cosines and sines; otherwise 8 neighbours.  The elements past the rotated part
// are 8 neighbours to a lane in both layouts.
struct RopeLane {
  int sub, lpr, rpw;  // row of the warp's group, lanes to a row, rows to a group
  int da, db;         // first elements of the two quads
  bool on, rotated;
};

// A lane's ring of quad pairs in shared memory, filled by its own asynchronous
// copies and read by itself alone: no barrier, and what is in flight costs no
// registers (with 16 bytes to a lane and group, 32 warps to an SM and 5 groups
// ahead, 80 KB to an SM; loads into registers reached 4.1 TB/s at 8192 tokens,
// the ring 4.9).  Quad e of place i of lane l lies at (i * 2 + e) * 32 + l.
// 32-bit elements take twice the place: 4 stages are 32 KB to a CTA, while 6 would
// be the whole 48 KB that a kernel has without asking for more, with none left for
// the V tiles' static words.
template <typename T>
constexpr int kRopeStages = sizeof(T) == 4 ? 4 : 6;

template <typename T>
__device__ __forceinline__ void quad_async(Quad<T>* dst, const T* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (sizeof(T) == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void quads_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void quads_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rows of groups [g0, g1) of one tensor (heads of one token); STAGES > 1: through
// the ring, STAGES 1: loads into registers.  `oa`, `ob`: where the two quads of a
// row go.  Arithmetic in pairs: what bounds the kernel next to memory is issue
// slots (about 60 instructions to a lane's 8 elements; 160 with scalar arithmetic
// and 64-bit index arithmetic, which ran at 3.2 TB/s).
template <typename T, bool INTER, int STAGES>
__device__ __forceinline__ void rope_rows(const RopeLane& ln, Quad<T>* ring, const T* src, int s_head, T* dst, int d_head,
                                          int oa, int ob, int heads, int g0, int g1, const void* weight, bool w_f32,
                                          float eps, float inv_d, float4 c, float4 s) {
  const float2 cc[4] = {INTER ? make_float2(c.x, c.x) : make_float2(c.x, c.y),
                        INTER ? make_float2(c.y, c.y) : make_float2(c.z, c.w), make_float2(c.z, c.z),
                        make_float2(c.w, c.w)};
  const float2 sn[4] = {INTER ? make_float2(-s.x, s.x) : make_float2(s.x, s.y),
                        INTER ? make_float2(-s.y, s.y) : make_float2(s.z, s.w), make_float2(-s.z, s.z),
                        make_float2(-s.w, s.w)};
  float2 wt[4];
  if (weight && ln.on) {
    if (w_f32) {
      const float* w = reinterpret_cast<const float*>(weight);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        wt[i] = make_float2(w[ln.da + 2 * i], w[ln.da + 2 * i + 1]);
        wt[2 + i] = make_float2(w[ln.db + 2 * i], w[ln.db + 2 * i + 1]);
      }
    } else {
      const T* w = reinterpret_cast<const T*>(weight);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        wt[i] = make_float2(to_float(w[ln.da + 2 * i]), to_float(w[ln.da + 2 * i + 1]));
        wt[2 + i] = make_float2(to_float(w[ln.db + 2 * i]), to_float(w[ln.db + 2 * i + 1]));
      }
    }
  }
  int h = g0 * ln.rpw + ln.sub;
  const int h_end = ln.on ? (g1 * ln.rpw < heads ? g1 * ln.rpw : heads) : 0;
  const T* row = src + (int64_t)h * s_head;
  T* out = dst + (int64_t)h * d_head;
  const int64_t s_step = (int64_t)ln.rpw * s_head, d_step = (int64_t)ln.rpw * d_head;
  int h_in = h, stage_in = 0, stage = 0;  // (ring) the next row to be asked for, and where it goes
  auto ask = [&]() {
    if (h_in < h_end) {
      quad_async(ring + stage_in * 64, row + ln.da);
      quad_async(ring + stage_in * 64 + 32, row + ln.db);
    }
    quads_commit();
    row += s_step;
    h_in += ln.rpw;
    stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
  };
  if constexpr (STAGES > 1) {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) ask();
  }
  for (int g = g0; g < g1; ++g) {
    Quad<T> a, b;
    a.w = b.w = typename Quad<T>::Word{};
    if constexpr (STAGES > 1) {
      ask();
      quads_wait<STAGES - 1>();
      if (h < h_end) {
        a = ring[stage * 64];
        b = ring[stage * 64 + 32];
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    } else {
      if (h < h_end) {
        a.load(row + ln.da);
        b.load(row + ln.db);
      }
      row += s_step;
    }
    float2 y[4];
    a.get(y[0], y[1]);
    b.get(y[2], y[3]);
    if (weight) {
      float2 q = mul2(y[0], y[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) q = fma2(y[i], y[i], q);
      float ss = q.x + q.y;
      for (int o = 1; o < ln.lpr; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(fmaf(ss, inv_d, eps));
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = mul2(y[i], mul2(make_float2(inv, inv), wt[i]));
    }
    if (ln.rotated) {
      if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = fma2(make_float2(y[i].y, y[i].x), sn[i], mul2(y[i], cc[i]));
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 va = y[i], vb = y[2 + i];
          y[i] = fma2(vb, make_float2(-sn[i].x, -sn[i].y), mul2(va, cc[i]));
          y[2 + i] = fma2(va, sn[i], mul2(vb, cc[i]));
        }
      }
    }
    if (h < h_end) {
      a.put(y[0], y[1]);
      b.put(y[2], y[3]);
      a.store(out + oa);
      b.store(out + ob);
    }
    out += d_step;
    h += ln.rpw;
  }
}

template <typename T, bool INTER, int STAGES>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(const RopeArgs p, const RopePlan pl) {
  extern __shared__ __align__(16) unsigned char smem_rope[];
  wait_for_prior();
  if (blockIdx.x >= pl.row_ctas) {
    store_v_tile<T>(p, blockIdx.x - pl.row_ctas, smem_rope);
    return;
  }
  const int lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  const unsigned tok = w / pl.warps_per_token;
  if (tok >= p.num_tokens) return;
  const int all = pl.q_groups + pl.k_groups + pl.v_groups;
  const int g0 = (int)(w - tok * pl.warps_per_token) * pl.span, g1 = g0 + pl.span < all ? g0 + pl.span : all;

  const int half = p.rot >> 1;
  RopeLane ln;
  ln.lpr = 1 << pl.lpr_shift;
  ln.rpw = 32 >> pl.lpr_shift;
  ln.sub = lane >> pl.lpr_shift;
  const int li = lane & (ln.lpr - 1);
  ln.on = li * 8 < p.head_size;
  ln.rotated = li * 8 < p.rot;
  ln.da = !INTER && ln.rotated ? 4 * li : 8 * li;
  ln.db = !INTER && ln.rotated ? ln.da + half : ln.da + 4;
  const int64_t pos = load_index(p.positions, p.pos_i64, tok);
  int64_t blk = 0;
  int off = 0;
  bool place = false;  // the token has a cache place
  if (p.k_cache != nullptr && g1 > pl.q_groups)
    place = token_place(p, load_index(p.slots, p.slots_i64, tok), lane == 0, &blk, &off);
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  if (pos >= p.table_rows && lane == 0) set_status(&g_layer_ops_status, KVC_STATUS_INDEX_OOB);
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (ln.rotated && pos_ok) {
    const float* cs = p.table + pos * p.table_stride + 4 * li;
    c = *reinterpret_cast<const float4*>(cs);
    s = *reinterpret_cast<const float4*>(cs + half);
  }
  const bool w_f32 = p.weight_type == ElemType::F32;
  Quad<T>* ring = reinterpret_cast<Quad<T>*>(smem_rope) + (threadIdx.x >> 5) * (STAGES * 64) + lane;

  if (g0 < pl.q_groups && pos_ok)
    rope_rows<T, INTER, STAGES>(ln, ring, reinterpret_cast<const T*>(p.q) + (int64_t)tok * p.q_tok, (int)p.q_head,
                           reinterpret_cast<T*>(p.q_out) + (int64_t)tok * p.qo_tok, (int)p.qo_head, ln.da, ln.db,
                           p.num_heads, g0, g1 < pl.q_groups ? g1 : pl.q_groups, p.q_weight, w_f32, p.eps, pl.inv_d, c,
                           s);
  const int k0 = g0 > pl.q_groups ? g0 - pl.q_groups : 0;
  int k1 = g1 - pl.q_groups;
  k1 = k1 < pl.k_groups ? k1 : pl.k_groups;
  if (k0 < k1 && pos_ok && (place || p.k_cache == nullptr)) {
    T* dst;
    int d_head, oa = ln.da, ob = ln.db;
    if (p.k_cache == nullptr) {
      dst = reinterpret_cast<T*>(p.k_out) + (int64_t)tok * p.ko_tok;
      d_head = (int)p.ko_head;
    } else {
      dst = reinterpret_cast<T*>(p.k_cache) + blk * p.kc_block;
      d_head = (int)p.kc_head;
      if (p.paged) {  // 16-byte places [d / X][offset] of the page
        constexpr int X = 16 / (int)sizeof(T);
        oa = (oa / X * p.block_size + off) * X + oa % X;
        ob = (ob / X * p.block_size + off) * X + ob % X;
      } else {
        dst += (int64_t)off * p.kc_tok;
      }
    }
    rope_rows<T, INTER, STAGES>(ln, ring, reinterpret_cast<const T*>(p.k) + (int64_t)tok * p.k_tok, (int)p.k_head, dst, d_head, oa,
                           ob, p.num_kv_heads, k0, k1, p.k_weight, w_f32, p.eps, pl.inv_d, c, s);
  }
  const int vg = pl.q_groups + pl.k_groups;
  if (g1 > vg && place) {  // values: as they are
    const T* src = reinterpret_cast<const T*>(p.v) + (int64_t)tok * p.v_tok;
    T* dst = reinterpret_cast<T*>(p.v_cache) + blk * p.vc_block + (p.paged ? (int64_t)off : (int64_t)off * p.vc_tok);
    const int d = 8 * li;
    for (int g = g0 > vg ? g0 - vg : 0; g < g1 - vg; ++g) {
      const int h = g * ln.rpw + ln.sub;
      if (!ln.on || h >= p.num_kv_heads) continue;
      Quad<T> a, b;
      a.load(src + h * p.v_head + d);
      b.load(src + h * p.v_head + d + 4);
      T* o = dst + h * p.vc_head;
      if (p.paged) {
        const T* ea = reinterpret_cast<const T*>(&a.w);
        const T* eb = reinterpret_cast<const T*>(&b.w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[(d + e) * p.block_size] = ea[e];
          o[(d + 4 + e) * p.block_size] = eb[e];
        }
      } else {
        a.store(o + d);
        b.store(o + d + 4);
      }
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
  wait_for_prior();
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
  return launch_dependent(qk_norm_rope_any_kernel<T, C>, dim3((unsigned)((rows + kRopeWarps - 1) / kRopeWarps)),
                          kRopeWarps * 32, 0, stream, a);
}

template <typename T, bool INTER, int STAGES>
static cudaError_t launch_rope_u(const RopeArgs& a, RopePlan pl, bool v_tiles, int span, cudaStream_t stream) {
  const int rpw = 32 >> pl.lpr_shift;
  pl.q_groups = (a.num_heads + rpw - 1) / rpw;
  pl.k_groups = (a.num_kv_heads + rpw - 1) / rpw;
  pl.v_groups = a.k_cache && !v_tiles ? pl.k_groups : 0;
  const int all = pl.q_groups + pl.k_groups + pl.v_groups;
  pl.span = span;
  pl.warps_per_token = (unsigned)((all + pl.span - 1) / pl.span);
  const int64_t warps = a.num_tokens * pl.warps_per_token;
  const int64_t tiles = v_tiles ? (a.num_tokens + kVTile - 1) / kVTile * a.num_kv_heads : 0;
  const int64_t ctas = (warps + kRopeWarps - 1) / kRopeWarps;
  if (ctas + tiles > 0x7fffffffll / kRopeWarps) return cudaErrorInvalidValue;
  pl.row_ctas = (unsigned)ctas;
  size_t smem = STAGES > 1 ? (size_t)kRopeWarps * STAGES * 64 * sizeof(Quad<T>) : 0;
  static_assert(STAGES == 1 || kRopeWarps * STAGES * 64 * sizeof(Quad<T>) <= 40 * 1024,
                "dynamic shared memory beside the static words, within 48 KB");
  const size_t tile = v_tiles ? (size_t)kVTile * (a.head_size * sizeof(T) + 16) : 0;
  if (tile > smem) smem = tile;
  return launch_dependent(qk_norm_rope_kernel<T, INTER, STAGES>, dim3((unsigned)(ctas + tiles)), kRopeWarps * 32, smem,
                          stream, a, pl);
}

template <typename T>
static cudaError_t launch_rope_vec(RopeArgs a, cudaStream_t stream) {
  RopePlan pl = {};
  while ((8 << pl.lpr_shift) < a.head_size) ++pl.lpr_shift;
  pl.inv_d = 1.f / (float)a.head_size;
  // Many tokens: a token's rows to one warp, kRopeStages<T> of its groups in flight
  // through the lanes' rings; else one group to a warp.  bf16, 32 + 8 heads of
  // 128 (20 groups to a token), one group / rings: 512 tokens 8.3 / 12.4 us, 1024
  // 12.4 / 12.4, 2048 24.5 / 16.4, 6000 61.5 / 32.8.  Without enough tokens the
  // rings leave SMs with too few warps, with few groups a ring hardly fills.
  const int rpw = 32 >> pl.lpr_shift;
  const int64_t groups = a.num_tokens * ((a.num_heads + rpw - 1) / rpw + (a.num_kv_heads + rpw - 1) / rpw);
  const bool whole = a.num_tokens >= 7 * (int64_t)sm_count() && groups >= 128 * (int64_t)sm_count();
  // V by tiles of 32 tokens: 16-byte stores where slots run on, but a poor scatter
  // where they do not.  bf16, heads of 128, 64 / 256 / 1024 tokens, one by one and by
  // tiles: a prompt's slots (28 + 4 heads) 3.3 / 4.9 / 13.1 us and 2.7 / 3.4 / 9.4
  // (8192: 65 and 35), one slot of each request (32 + 8 heads) 4.9 / 7.6 / 25.7 and
  // 7.0 / 12.8 / 39.5.  The host does not see the slots: fewer than 1024 new tokens
  // are taken for a decode step's.
  const bool v_tiles = a.k_cache && a.paged && a.num_tokens >= 1024;
  a.v_wide = a.block_size % 8 == 0 && reinterpret_cast<uintptr_t>(a.v_cache) % 16 == 0 && a.vc_block % 8 == 0 &&
             a.vc_head % 8 == 0;
  if (a.interleaved)
    return whole ? launch_rope_u<T, true, kRopeStages<T>>(a, pl, v_tiles, 1 << 20, stream)
                 : launch_rope_u<T, true, 1>(a, pl, v_tiles, 1, stream);
  return whole ? launch_rope_u<T, false, kRopeStages<T>>(a, pl, v_tiles, 1 << 20, stream)
               : launch_rope_u<T, false, 1>(a, pl, v_tiles, 1, stream);
}

// Whether every row the launch touches is whole quads of 8 (16-bit) or 16 bytes.
static bool rope_vec_ok(const RopeArgs& a, int es) {
  const int64_t align = 4 * es;
  if (a.head_size % 8 || a.head_size > 256 || a.rot % 8 || a.type != a.cache_type) return false;
  // (head strides are 32-bit in the kernel)
  for (int64_t s : {a.q_head, a.k_head, a.v_head, a.qo_head, a.ko_head, a.kc_head, a.vc_head})
    if (s > 0x7fffffffll || s < -0x7fffffffll) return false;
  auto rows = [&](const void* base, int64_t s1, int64_t s2, int64_t s3) {
    return reinterpret_cast<uintptr_t>(base) % align == 0 && (s1 * es) % align == 0 && (s2 * es) % align == 0 &&
           (s3 * es) % align == 0;
  };
  if (!rows(a.q, a.q_tok, a.q_head, 0) || !rows(a.k, a.k_tok, a.k_head, 0) || !rows(a.q_out, a.qo_tok, a.qo_head, 0))
    return false;
  // the table's rows as four floats at a time (half a multiple of 4)
  if ((reinterpret_cast<uintptr_t>(a.table) & 15u) || (a.table_stride & 3)) return false;
  if (!a.k_cache) return rows(a.k_out, a.ko_tok, a.ko_head, 0);
  // (places within a head's page are 32-bit in the kernel)
  if (a.paged && (int64_t)a.head_size * a.block_size > 0x7fffffffll) return false;
  return rows(a.v, a.v_tok, a.v_head, 0) && rows(a.k_cache, a.kc_block, a.kc_head, a.kc_tok) &&
         (a.paged || rows(a.v_cache, a.vc_block, a.vc_head, a.vc_tok));
}

template <typename T>
static cudaError_t launch_rope_t(const RopeArgs& a, cudaStream_t stream) {
  return rope_vec_ok(a, sizeof(T)) ? launch_rope_vec<T>(a, stream) : launch_rope_any<T, T>(a, stream);
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
