// window.cu — attention over a sliding window with a few first tokens that stay
// visible (sinks), on the paged and token-major caches, for sm_100a: one new
// token per sequence (decode, below) and the new tokens of a ragged batch
// (extend).
//
// The query at position i of a sequence sees position j <= i when j < sinks or
// j > i - window:
//   out = sum_j e^{s_j - m} v_j / (sum_j e^{s_j - m} + 1e-6),  s_j = scale q.k_j
// with m the largest s_j; a sequence of length 0 or past max_seq_len gives zeros.
#include "decode_common.cuh"
#include "decode_mma.cuh"
#include "prefill.cuh"
#include "prefill_umma.cuh"
#include "window_umma.cuh"

namespace kvc {

// ---------------------------------------------------------------------------
// Decode.  What a sequence sees is at most window + sinks tokens (and the rest
// of their blocks), whatever its length, so instead of partitions of the
// context with partials in device memory and a second kernel, the seen blocks of
// one (sequence, KV head) go to the CTAs of one thread-block cluster in equal
// runs, and the cluster joins its softmax states through distributed shared
// memory: CTA r owns a slice of the output elements, every CTA stores its
// (max, sum) and its unnormalised values of that slice into r's shared memory,
// and after one cluster barrier each CTA finishes its own slice.  One launch, no
// workspace, a fixed order of summation.
// ---------------------------------------------------------------------------
constexpr int kMaxCluster = 16;

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// This CTA's shared address `p` in CTA `rank` of the cluster, and stores to it.
__device__ __forceinline__ uint32_t remote_address(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return a;
}
__device__ __forceinline__ void store_remote(const float2* dst, uint32_t rank, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote_address(dst, rank)), "f"(v.x), "f"(v.y)
               : "memory");
}
__device__ __forceinline__ void store_remote(const float4* dst, uint32_t rank, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote_address(dst, rank)), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}

__device__ __forceinline__ void add_scaled(float4& a, float w, float4 b) {
  a.x += w * b.x;
  a.y += w * b.y;
  a.z += w * b.z;
  a.w += w * b.w;
}

// a / L as four elements of an output row, of any alignment; 0 where L is 0 (a NaN
// sum, from a score that is NaN or +inf, gives NaN).
template <typename T>
__device__ __forceinline__ void store_quotient(T* dst, float4 a, float L, float eps) {
  const float n = L + eps;
  const bool any = L != 0.f;
  struct alignas(4 * sizeof(T)) Four {
    T e[4];
  } v = {{from_float<T>(any ? a.x / n : 0.f), from_float<T>(any ? a.y / n : 0.f), from_float<T>(any ? a.z / n : 0.f),
          from_float<T>(any ? a.w / n : 0.f)}};
  if ((reinterpret_cast<uintptr_t>(dst) & (sizeof(Four) - 1)) == 0) {
    *reinterpret_cast<Four*>(dst) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = v.e[i];
  }
}

// The exchange area of one CTA: [C][nh] (max, sum) pairs, then [C][S] values of
// its slice of the nh * D elements, four to a value, S = ceil(nh * D / 4 / C).
__host__ __device__ constexpr int exchange_floats(int nh, int D) {
  return kMaxCluster * nh * 2 + nh * D + 4 * kMaxCluster;
}

// Joins the CTA states of a cluster.  part(g, d, &M, &L): the CTA's unnormalised
// elements d .. d + 3 of row g, and the row's max (natural log units) and sum;
// dest(g): the output row.  `eps` is added to a row's sum (a row that sees nothing
// has sum 0 and gives 0).  Every thread of every CTA of the cluster calls it; each
// CTA has arrived once on the cluster barrier before (its shared memory is live).
template <typename T, typename FPart, typename FDest>
__device__ __forceinline__ void cluster_join(int nh, int D, int C, int rank, float* xch, float eps, FPart part, FDest dest) {
  const int n4 = nh * D / 4;
  if (C == 1) {
    for (int i = threadIdx.x; i < n4; i += blockDim.x) {
      const int g = 4 * i / D, d = 4 * i - g * D;
      float M, L;
      const float4 a = part(g, d, &M, &L);
      store_quotient(dest(g) + d, a, L, eps);
    }
    return;
  }
  const int S = (n4 + C - 1) / C;
  float2* ml = reinterpret_cast<float2*>(xch);                          // [C][nh]
  float4* val = reinterpret_cast<float4*>(xch + kMaxCluster * nh * 2);  // [C][S]
  cluster_wait();  // every CTA of the cluster runs: its exchange area may be written
  for (int i = threadIdx.x; i < n4; i += blockDim.x) {
    const int g = 4 * i / D, d = 4 * i - g * D, r = i / S;
    float M, L;
    const float4 a = part(g, d, &M, &L);
    store_remote(val + rank * S + (i - r * S), (uint32_t)r, a);
    // the row's state goes to every CTA, one by each of the row's threads
    for (int c = d / 4; c < C; c += D / 4) store_remote(ml + rank * nh + g, (uint32_t)c, make_float2(M, L));
  }
  cluster_arrive();
  cluster_wait();
  for (int j = threadIdx.x; j < S && rank * S + j < n4; j += blockDim.x) {
    const int i = rank * S + j, g = 4 * i / D, d = 4 * i - g * D;
    float M = -INFINITY;
    for (int c = 0; c < C; ++c) M = fmaxf(M, ml[c * nh + g].x);
    float L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < C; ++c) {
      const float2 s = ml[c * nh + g];
      const float w = s.x == -INFINITY ? 0.f : expf(s.x - M);
      L += w * s.y;
      add_scaled(a, w, val[c * S + j]);
    }
    store_quotient(dest(g) + d, a, L, eps);
  }
}

// Tensor-core form: 16 (new token, query head of the group) rows of one KV head
// are the rows of the decode's m16n8k16 tile (mma_group, decode_mma.cuh); each warp
// streams every NW-th group of GT tokens of the CTA's run through its own ring of
// STAGES stages, as paged_decode_mma_kernel does.  MODE: kBulk (whole pages),
// kSwizzledV (32-token pages), kFlashTma (token rows in blocks of 16k), kFlash
// (token rows).  EXT: several such tiles to a sequence and KV head: the
// extend's few new tokens (indptr), or, without indptr, more than 16 heads of one.
template <int D, int BS, int NW, int STAGES, int GT, int MODE>
struct WindowGeom {
  using Geo = MmaGeom<D, BS, NW, STAGES, GT, MODE>;
  static constexpr int XCH_OFF = (Geo::SMEM + 15) / 16 * 16;
  static constexpr int SMEM = XCH_OFF + exchange_floats(16, D) * 4;
};

template <typename T, int D, int BS, int NW, int STAGES, int GTOK, int MODE, bool EXT>
__global__ void __launch_bounds__(NW * 32)
    window_decode_kernel(const DecodeParams p, const WindowArgs wa, const __grid_constant__ TmaMaps tm) {
  using namespace mma_detail;
  using WG = WindowGeom<D, BS, NW, STAGES, GTOK, MODE>;
  using Geo = typename WG::Geo;
  constexpr int GT = Geo::GT, NBOX = Geo::NBOX, BOX = Geo::BOX, VBS = Geo::VBS;
  constexpr int KS = D / 16, NT = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];

  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int unit = blockIdx.x / C, seq = blockIdx.y;
  const int tile = EXT ? unit / p.num_kv_heads : 0, kvh = unit - tile * p.num_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, q4 = lane & 3;
  const int G = p.num_heads / p.num_kv_heads, h0 = kvh * G;
  grid_dependents_launch();
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Geo::BAR_OFF) + warp * STAGES;
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem + Geo::MASK_OFF) + warp * STAGES;
  constexpr int IDC = Geo::IDC, IDV = IDC * GT / 32;
  uint32_t* ids = reinterpret_cast<uint32_t*>(smem + Geo::IDS_OFF) + warp * 2 * IDC * GT;
  uint8_t* ring_base = smem;
  if constexpr (Geo::ALIGN > 0) {
    constexpr uint32_t A = (uint32_t)Geo::ALIGN;
    ring_base += (A - (smem_u32(smem) & (A - 1u))) & (A - 1u);
  }
  uint8_t* ring = ring_base + (size_t)warp * STAGES * Geo::STAGE;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&bars[s], Geo::CP_ASYNC ? 32 : 1);
    mbar_fence_init();
  }
  __syncwarp();

  // The kernel before this one may have written anything that is read from here on,
  // lengths, tables and queries (an attention output as the next query) included.
  grid_dependency_wait();
  const int rbs = Geo::TROWS || Geo::FLASH ? p.block_size : BS;
  // rows R0 .. R0 + nh - 1 of the sequence's new tokens, whose first is row q0 of
  // q / out and position `prefix`
  const int R0 = tile * 16;
  const uint32_t ctx = p.context_lens[seq];
  int64_t q0 = seq;
  int rows = G, prefix = (int)ctx - 1;
  bool zero = ctx == 0 || ctx > (uint32_t)p.max_seq_len;
  if (EXT && wa.indptr) {
    const int64_t a = wa.indptr[seq], b = wa.indptr[seq + 1];
    const int64_t ql = b - a;
    q0 = a;
    if (ql <= 0 || R0 >= ql * G) return;  // (the same for the whole cluster, as every early end here)
    // rows past q may not be written; other index errors give zeros
    zero = ql > wa.max_q_len || (int64_t)ctx < ql || (int64_t)ctx > wa.table_len * (int64_t)rbs || ctx > 0x7fffff00u;
    const bool past = b > wa.num_tokens;
    if ((zero || past) && threadIdx.x == 0 && blockIdx.x == 0) set_status(&g_decode_status, KVC_STATUS_INDEX_OOB);
    if (past) return;
    rows = (int)(ql * G < 0x7fffffff ? ql * G : 0x7fffffff);
    prefix = (int)((int64_t)ctx - ql);
  }
  const int nh = EXT ? (rows - R0 < 16 ? rows - R0 : 16) : G;
  // row R0 + g: new token t, head of the group
  auto token_of = [&](int g) { return EXT ? (R0 + g) / G : 0; };
  auto dest = [&](int g) -> T* {
    if constexpr (!EXT)  // (fewer registers live across the loop: 256 sequences, window 1024: 170 -> 165 us)
      return reinterpret_cast<T*>(p.out) + (int64_t)seq * p.out_seq_stride + (int64_t)(h0 + g) * p.out_head_stride;
    const int t = token_of(g);
    return reinterpret_cast<T*>(p.out) + (q0 + t) * p.out_seq_stride + (int64_t)(h0 + R0 + g - t * G) * p.out_head_stride;
  };
  if (zero) {
    if (rank == 0)
      for (int i = threadIdx.x; i < nh * D; i += NW * 32) dest(i / D)[i % D] = from_float<T>(0.f);
    return;
  }
  if (C > 1) cluster_arrive();
  const Seen seen = seen_range(prefix + token_of(0), prefix + token_of(nh - 1), wa.window, wa.sinks, rbs);
  // this CTA's run of groups
  const int all = (seen.end + GT - 1) / GT, per = (all + C - 1) / C;
  const int begin = rank * per * GT;
  const int end = begin + per * GT < seen.end ? begin + per * GT : seen.end;
  const int ngroups = end > begin ? (end - begin + GT - 1) / GT : 0;
  const int n_mine = warp < ngroups ? (ngroups - warp + NW - 1) / NW : 0;

  const T* kbase = reinterpret_cast<const T*>(p.k_cache) + (int64_t)kvh * p.k_head_stride;
  const T* vbase = reinterpret_cast<const T*>(p.v_cache) + (int64_t)kvh * p.v_head_stride;
  const uint32_t* table = p.block_tables + (int64_t)seq * p.table_stride;
  const int tbs = p.block_size;
  const bool tok_blocks = tbs == 1, group_blocks = (tbs & 15) == 0;

  // block ids: lane i holds box i's of group k (paged, tensor rows); token rows
  // keep chunks of IDC groups, an id per token, loaded a chunk ahead
  auto load_block = [&](int k) -> uint32_t {
    uint32_t b = 0xffffffffu;
    if constexpr (!Geo::TOKIDS) {
      const int tok = begin + (warp + k * NW) * GT + lane * VBS;
      if (lane < NBOX && k < n_mine && tok < end) b = table[seen.real_block(tok / rbs)];
    }
    return b;
  };
  auto load_ids = [&](int c, uint32_t (&v)[IDV]) {
#pragma unroll
    for (int i = 0; i < IDV; ++i) {
      const int j = lane + 32 * i, kg = c * IDC + j / GT;
      const int tt = begin + (warp + kg * NW) * GT + j % GT;
      v[i] = kg < n_mine && tt < end ? table[seen.real_block(tok_blocks ? tt : tt / tbs)] : 0xffffffffu;
    }
  };
  auto store_ids = [&](int c, const uint32_t (&v)[IDV]) {
#pragma unroll
    for (int i = 0; i < IDV; ++i) ids[(c & 1) * IDC * GT + lane + 32 * i] = v[i];
    __syncwarp();
  };
  auto issue = [&](int k, int s, uint32_t blk) {
    const int t0 = begin + (warp + k * NW) * GT;
    uint8_t* st = ring + (size_t)s * Geo::STAGE;
    if constexpr (Geo::FLASH) {
      constexpr int CPR = Geo::ROWB / 16, RPP = 32 / CPR, RPL = GT / RPP;
      const uint32_t* cid = ids + ((k / IDC) & 1) * IDC * GT + (k % IDC) * GT;
      const bool in_ctx = lane < GT && t0 + lane < end;
      const bool ok = in_ctx && (int64_t)cid[lane < GT ? lane : 0] < p.num_blocks;
      if (in_ctx && !ok) set_status(&g_decode_status, KVC_STATUS_BLOCK_OOB);
      const uint32_t mask = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) masks[s] = mask;
      if (mask) {  // (a set bit means num_blocks > 0: block 0 is mapped for the masked rows)
        const int in0 = tok_blocks ? 0 : (group_blocks ? t0 % tbs : 0);
        const int col = lane % CPR, r0 = (lane / CPR) * RPL;
        uint32_t rid[RPL];
#pragma unroll
        for (int i = 0; i < RPL; i += 4) {
          const uint4 v4 = *reinterpret_cast<const uint4*>(cid + r0 + i);
          rid[i] = v4.x;
          rid[i + 1] = v4.y;
          rid[i + 2] = v4.z;
          rid[i + 3] = v4.w;
        }
#pragma unroll
        for (int i = 0; i < RPL; ++i) {
          const int row = r0 + i;
          const bool on = (mask >> row) & 1u;
          const int64_t b = on ? rid[i] : 0;
          const int64_t in_blk = tok_blocks ? 0 : (group_blocks ? in0 + row : (t0 + row) % tbs);
          cp_async16_zfill(st + row * BOX + col * 16, kbase + col * 8 + b * p.k_block_stride + in_blk * p.k_tok_stride,
                           on ? 16u : 0u);
          cp_async16_zfill(st + (NBOX + row) * BOX + col * 16,
                           vbase + col * 8 + b * p.v_block_stride + in_blk * p.v_tok_stride, on ? 16u : 0u);
        }
      }
      cp_async_arrive(&bars[s]);
    } else {
      uint32_t bid[NBOX];
#pragma unroll
      for (int i = 0; i < NBOX; ++i) bid[i] = __shfl_sync(0xffffffffu, blk, i);
      if (lane == 0) {
        uint32_t mask = 0, bytes = 0;
#pragma unroll
        for (int i = 0; i < NBOX; ++i) {
          if (t0 + i * VBS < end) {
            if ((int64_t)bid[i] < p.num_blocks) {
              mask |= 1u << i;
              bytes += 2 * BOX;
            } else {
              set_status(&g_decode_status, KVC_STATUS_BLOCK_OOB);
            }
          }
        }
        masks[s] = mask;
        if (bytes) mbar_arrive_expect_tx(&bars[s], bytes);
        else mbar_arrive(&bars[s]);
#pragma unroll
        for (int i = 0; i < NBOX; ++i) {
          if (!(mask & (1u << i))) continue;
          if constexpr (Geo::TROWS) {
            const int row = (int)bid[i] * rbs + t0 % rbs;  // (rows are below 2^31: the host checked)
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              tma_load_3d(st + i * BOX + h * GT * 128, &tm.k, 64 * h, kvh, row, &bars[s]);
              tma_load_3d(st + (NBOX + i) * BOX + h * GT * 128, &tm.v, 64 * h, kvh, row, &bars[s]);
            }
          } else {
            bulk_g2s(st + i * BOX, kbase + (int64_t)bid[i] * p.k_block_stride, BOX, &bars[s]);
            if constexpr (MODE == kSwizzledV)
              tma_load_4d(st + (NBOX + i) * BOX, &tm.v, 0, 0, kvh, (int)bid[i], &bars[s]);
            else
              bulk_g2s(st + (NBOX + i) * BOX, vbase + (int64_t)bid[i] * p.v_block_stride, BOX, &bars[s]);
          }
        }
      }
    }
  };

  // the first groups' ids and the query rows are on their way together
  uint32_t first_blk[STAGES], ids_next[IDV];
#pragma unroll
  for (int s = 0; s < STAGES; ++s) first_blk[s] = load_block(s);
  if constexpr (Geo::TOKIDS) {
    uint32_t first[IDV];
    load_ids(0, first);
    load_ids(1, ids_next);
    store_ids(0, first);
  }
  uint32_t qa[KS][4];
  const int t_lo = token_of(r), t_hi = token_of(r + 8);
  const T* q_lo = reinterpret_cast<const T*>(p.q) + (q0 + t_lo) * p.q_seq_stride +
                  (int64_t)(h0 + R0 + r - t_lo * G) * p.q_head_stride;
  const T* q_hi = reinterpret_cast<const T*>(p.q) + (q0 + t_hi) * p.q_seq_stride +
                  (int64_t)(h0 + R0 + r + 8 - t_hi * G) * p.q_head_stride;
  // what this lane's two rows see (rows past the last: nothing)
  int end_lo = 2147483647, end_hi = 2147483647, beg_lo = seen.beg, beg_hi = seen.beg;
  if constexpr (EXT) {
    end_lo = r < nh ? prefix + t_lo + 1 - seen.jump : 0;
    end_hi = r + 8 < nh ? prefix + t_hi + 1 - seen.jump : 0;
    beg_lo = end_lo > wa.window ? end_lo - wa.window : 0;
    beg_hi = end_hi > wa.window ? end_hi - wa.window : 0;
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d0 = ks * 16 + 2 * q4;
    qa[ks][0] = qa[ks][1] = qa[ks][2] = qa[ks][3] = 0u;
    if (r < nh) {
      const T* row = q_lo;
      qa[ks][0] = *reinterpret_cast<const uint32_t*>(row + d0);
      qa[ks][2] = *reinterpret_cast<const uint32_t*>(row + d0 + 8);
    }
    if (r + 8 < nh) {
      const T* row = q_hi;
      qa[ks][1] = *reinterpret_cast<const uint32_t*>(row + d0);
      qa[ks][3] = *reinterpret_cast<const uint32_t*>(row + d0 + 8);
    }
  }
  const float qk_scale = p.scale * kLog2e;
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < n_mine) issue(s, s, first_blk[s]);

  GroupState<D> gs;
  gs.reset();
  int k_fail = -1;
  for (int k = 0; k < n_mine; ++k) {
    const int s = k % STAGES;
    if constexpr (Geo::TOKIDS) {
      if (k % IDC == 0 && k + STAGES < n_mine) {
        store_ids(k / IDC + 1, ids_next);
        load_ids(k / IDC + 2, ids_next);
      }
    }
    const uint32_t next_blk = load_block(k + STAGES);
    if (!mbar_wait_bounded(&bars[s], (uint32_t)((k / STAGES) & 1))) {
      k_fail = k;
      break;
    }
    const uint8_t* st = ring + (size_t)s * Geo::STAGE;
    mma_group<T, Geo, D, true, true>(gs, qa, smem_u32(st), smem_u32(st + NBOX * BOX), begin + (warp + k * NW) * GT, end,
                                     masks[s], 0, qk_scale, false, 0.f, 0.f, lane, end_lo, end_hi, beg_lo, beg_hi,
                                     wa.sinks, seen.beg);
    __syncwarp();
    if (k + STAGES < n_mine) {
      fence_proxy_async();
      issue(k + STAGES, s, next_blk);
    }
  }
  if (k_fail >= 0) {  // the copies in flight land (or time out) before the ring is reused
    if (lane == 0) set_status(&g_decode_status, KVC_STATUS_WAIT_TIMEOUT);
    for (int kk = k_fail; kk < n_mine && kk < k_fail + STAGES; ++kk)
      mbar_wait_bounded(&bars[kk % STAGES], (uint32_t)((kk / STAGES) & 1));
  }

  // ---- the warps' states, then the cluster's
  const float l_lo = gs.quad_sum_lo(), l_hi = gs.quad_sum_hi();
  __syncthreads();  // every warp is done with its ring
  float* red_o = reinterpret_cast<float*>(smem);  // [NW][16][D]
  float* red_ml = red_o + NW * 16 * D;            // [NW][16][2]
  {
    // (16-byte pieces of a row in an order of its own, so that the rows' stores meet
    // in no bank; rows past the last stay unwritten)
    float* ow = red_o + (size_t)warp * 16 * D;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int d = ((2 * nt + (q4 >> 1)) ^ r) * 4 + 2 * (q4 & 1);
      if (r < nh) *reinterpret_cast<float2*>(ow + r * D + d) = make_float2(gs.o[nt][0], gs.o[nt][1]);
      if (r + 8 < nh) *reinterpret_cast<float2*>(ow + (r + 8) * D + d) = make_float2(gs.o[nt][2], gs.o[nt][3]);
    }
    if (q4 == 0) {
      red_ml[(warp * 16 + r) * 2] = gs.m_lo;
      red_ml[(warp * 16 + r) * 2 + 1] = l_lo;
      red_ml[(warp * 16 + r + 8) * 2] = gs.m_hi;
      red_ml[(warp * 16 + r + 8) * 2 + 1] = l_hi;
    }
  }
  __syncthreads();
  auto part = [&](int g, int d, float* M, float* L) -> float4 {
    float m = -INFINITY, l = 0.f;  // log2 units
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, red_ml[(w * 16 + g) * 2]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 s = *reinterpret_cast<const float2*>(red_ml + (w * 16 + g) * 2);
      const float e = s.x == -INFINITY ? 0.f : fast_exp2(s.x - m);
      l += e * s.y;
      add_scaled(a, e, *reinterpret_cast<const float4*>(red_o + (size_t)w * 16 * D + g * D + (d ^ ((g & 7) * 4))));
    }
    *M = m * kLn2;
    *L = l;
    return a;
  };
  cluster_join<T>(nh, D, C, rank, reinterpret_cast<float*>(smem + WG::XCH_OFF), EXT && wa.indptr ? 0.f : 1e-6f, part, dest);
}

// CUDA-core form, for every other pair of types, head size and group: the
// generic decode's page walk (4 warps, fp32 math, up to 8 heads of a KV group to
// a CTA) over the cluster's share of the seen blocks.
constexpr int kWinWarps = 4, kWinGC = 8;

template <typename Q_T, typename CACHE_T, int D>
__global__ void __launch_bounds__(kWinWarps * 32) window_decode_any_kernel(const DecodeParams p, const WindowArgs wa) {
  constexpr int X = 16 / sizeof(CACHE_T), NCHUNK = D / X, DPL = (D + 31) / 32, GC = kWinGC;
  __shared__ float qs[GC][D];
  __shared__ float ps[kWinWarps][GC][32];
  __shared__ float red_ml[kWinWarps][GC][2];
  __shared__ __align__(16) float red_o[kWinWarps][GC * D];
  extern __shared__ __align__(16) float xch[];
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int G = p.num_heads / p.num_kv_heads, per_kv = (G + GC - 1) / GC;
  const int cx = blockIdx.x / C, kvh = cx / per_kv, hc = cx - kvh * per_kv;
  const int h0 = kvh * G + hc * GC, nh = min(GC, G - hc * GC), seq = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bs = p.block_size;
  grid_dependents_launch();
  grid_dependency_wait();
  const uint32_t ctx = p.context_lens[seq];
  if (ctx == 0 || ctx > (uint32_t)p.max_seq_len) {
    if (rank == 0) write_zero_heads<Q_T>(p, seq, h0, nh, D);
    return;
  }
  if (C > 1) cluster_arrive();
  const Seen seen = seen_range((int)ctx - 1, (int)ctx - 1, wa.window, wa.sinks, bs);
  const int pages = (seen.end + bs - 1) / bs, per = (pages + C - 1) / C;
  const int page0 = rank * per, page1 = min(pages, page0 + per);

  const Q_T* q = reinterpret_cast<const Q_T*>(p.q);
  for (int i = threadIdx.x; i < GC * D; i += blockDim.x) {
    const int g = i / D, d = i - g * D;
    qs[g][d] = g < nh ? to_float(q[(int64_t)seq * p.q_seq_stride + (int64_t)(h0 + g) * p.q_head_stride + d]) : 0.f;
  }
  __syncthreads();
  float m[GC], l[GC], o[GC][DPL];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[g][i] = 0.f;
  }
  const CACHE_T* kcache = reinterpret_cast<const CACHE_T*>(p.k_cache);
  const CACHE_T* vcache = reinterpret_cast<const CACHE_T*>(p.v_cache);
  const uint32_t* table = p.block_tables + (int64_t)seq * p.table_stride;
  const int tpl = 32 / bs, t = lane % bs, sub = lane / bs;
  auto visible = [&](int v) { return v < seen.end && (v >= seen.beg || v < wa.sinks); };

  for (int pg = page0 + warp; pg < page1; pg += kWinWarps) {
    const int64_t blk = (int64_t)table[seen.real_block(pg)];
    if (blk >= p.num_blocks) {
      if (lane == 0) set_status(&g_decode_status, KVC_STATUS_BLOCK_OOB);
      continue;
    }
    const CACHE_T* kp = kcache + blk * p.k_block_stride + (int64_t)kvh * p.k_head_stride;
    float acc[GC];
#pragma unroll
    for (int g = 0; g < GC; ++g) acc[g] = 0.f;
    for (int c = sub; c < NCHUNK; c += tpl) {
      const uint4 raw = *reinterpret_cast<const uint4*>(kp + ((int64_t)c * bs + t) * X);
      const CACHE_T* kv = reinterpret_cast<const CACHE_T*>(&raw);
#pragma unroll
      for (int e = 0; e < X; ++e) {
        const float kf = to_float(kv[e]);
#pragma unroll
        for (int g = 0; g < GC; ++g) acc[g] += qs[g][c * X + e] * kf;
      }
    }
    for (int off = bs; off < 32; off <<= 1) {
#pragma unroll
      for (int g = 0; g < GC; ++g) acc[g] += __shfl_xor_sync(0xffffffffu, acc[g], off);
    }
    const bool on = visible(pg * bs + t);
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      const float s = on ? acc[g] * p.scale : -INFINITY;
      float pm = s;
      for (int off = 1; off < bs; off <<= 1) pm = fmaxf(pm, __shfl_xor_sync(0xffffffffu, pm, off));
      const float mn = fmaxf(m[g], pm);
      const float ref = mn == -INFINITY ? 0.f : mn;  // (a page none of whose tokens is seen)
      const float alpha = m[g] == -INFINITY ? 0.f : expf(m[g] - ref);
      const float e = on ? expf(s - ref) : 0.f;
      float es = e;
      for (int off = 1; off < bs; off <<= 1) es += __shfl_xor_sync(0xffffffffu, es, off);
      l[g] = l[g] * alpha + es;
      m[g] = mn;
#pragma unroll
      for (int i = 0; i < DPL; ++i) o[g][i] *= alpha;
      if (sub == 0) ps[warp][g][t] = e;
    }
    __syncwarp();
    // tokens nobody sees are skipped: their slots may hold anything, and 0 * NaN would poison the sum
    const CACHE_T* vp = vcache + blk * p.v_block_stride + (int64_t)kvh * p.v_head_stride;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
      const int d = lane + 32 * i;
      if (d < D) {
        const CACHE_T* row = vp + (int64_t)d * bs;
        for (int t0 = 0; t0 < bs; t0 += X) {
          const uint4 raw = *reinterpret_cast<const uint4*>(row + t0);
          const CACHE_T* vv = reinterpret_cast<const CACHE_T*>(&raw);
#pragma unroll
          for (int e = 0; e < X; ++e) {
            const float vf = visible(pg * bs + t0 + e) ? to_float(vv[e]) : 0.f;
#pragma unroll
            for (int g = 0; g < GC; ++g) o[g][i] += ps[warp][g][t0 + e] * vf;
          }
        }
      }
    }
    __syncwarp();
  }

  if (lane == 0) {
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      red_ml[warp][g][0] = m[g];
      red_ml[warp][g][1] = l[g];
    }
  }
#pragma unroll
  for (int g = 0; g < GC; ++g)
#pragma unroll
    for (int i = 0; i < DPL; ++i)
      if (lane + 32 * i < D) red_o[warp][g * D + lane + 32 * i] = o[g][i];
  __syncthreads();
  auto part = [&](int g, int d, float* M, float* L) -> float4 {
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) top = fmaxf(top, red_ml[w][g][0]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWinWarps; ++w) {
      const float e = red_ml[w][g][0] == -INFINITY ? 0.f : expf(red_ml[w][g][0] - top);
      l += e * red_ml[w][g][1];
      add_scaled(a, e, *reinterpret_cast<const float4*>(&red_o[w][g * D + d]));
    }
    *M = top;
    *L = l;
    return a;
  };
  auto dest = [&](int g) -> Q_T* {
    return reinterpret_cast<Q_T*>(p.out) + (int64_t)seq * p.out_seq_stride + (int64_t)(h0 + g) * p.out_head_stride;
  };
  cluster_join<Q_T>(nh, D, C, rank, xch, 1e-6f, part, dest);
}

// ---- launches -------------------------------------------------------------------
// How a CTA of the tensor-core form is cut: kNarrow (two or three to an SM), kWide
// (one, with the SM's shared memory: more warps, each with fewer groups one after
// another), kSmall (four).
enum Form { kNarrow, kWide, kSmall };

// The longest run that a query can see, in whole blocks.
static int64_t longest_seen(const DecodeParams& p, const WindowArgs& w) {
  const int64_t sinks = (w.sinks + (int64_t)p.block_size - 1) / p.block_size * p.block_size;
  const int64_t seen = sinks + w.window + p.block_size;
  return seen < p.max_seq_len ? seen : p.max_seq_len;
}

// CTAs to a cluster of the CUDA-core form, whose CTAs share SMs: the smallest power
// of two (at most 16) that brings the launch to one CTA per SM, while a CTA keeps at
// least `least` tokens of the longest run.
static int window_cluster(const DecodeParams& p, const WindowArgs& w, int64_t units, int least) {
  const int64_t seen = longest_seen(p, w), n = units * p.num_seqs, sms = decode_sm_count();
  int c = 1;
  while (c < kMaxCluster && n * c < sms && seen >= (int64_t)least * 2 * c) c *= 2;
  return c;
}

// Shared memory and cluster sizes of a kernel, once per device (twice is harmless).
template <typename K>
static cudaError_t configure_clustered(K kern, int smem, std::atomic<bool>* configured) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && configured[dev]) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev] = true;
  return e;
}

// Clusters of c CTAs that run at once on the current device, asked once per size.
template <typename K>
static int active_clusters(K kern, int smem, int threads, int c, int dev, std::atomic<int> (*known)[kMaxCluster + 1]) {
  const bool keep = dev >= 0 && dev < 64;
  int n = keep ? known[dev][c].load() : 0;
  if (n > 0) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (keep) known[dev][c] = n + 1;
  return n;
}

template <typename K, typename... Args>
static cudaError_t launch_clustered(K kern, int smem, int cluster, int64_t units, unsigned seqs, int threads,
                                    std::atomic<bool>* configured, cudaStream_t stream, Args... args) {
  if (units * cluster > 0x7fffffffll) return cudaErrorInvalidValue;
  if (const cudaError_t e = configure_clustered(kern, smem, configured); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)units * (unsigned)cluster, seqs);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int D, int BS, int NW, int STAGES, int GT, int MODE, bool EXT, Form FORM>
static cudaError_t launch_window_nw(const DecodeParams& p, const WindowArgs& w, cudaStream_t stream) {
  using WG = WindowGeom<D, BS, NW, STAGES, GT, MODE>;
  TmaMaps maps;
  memset(&maps, 0, sizeof(maps));
  if (MODE == kSwizzledV || MODE == kFlashTma) {
    const ElemType et = std::is_same<T, __nv_bfloat16>::value ? ElemType::BF16 : ElemType::F16;
    if (!make_tensor_maps(p, et, D, BS, WG::Geo::VBS, WG::Geo::VSWZ, MODE, &maps)) return cudaErrorNotSupported;
  }
  static std::atomic<bool> configured[64];
  // 16-row tiles of a sequence
  const int64_t rows = (EXT ? (int64_t)w.max_q_len : 1) * (p.num_heads / p.num_kv_heads), tiles = (rows + 15) / 16;
  const int64_t units = p.num_kv_heads * tiles;
  auto kern = window_decode_kernel<T, D, BS, NW, STAGES, GT, MODE, EXT>;
  int cluster = 1;
  if constexpr (FORM == kWide) {
    // the largest cluster (at most 16 CTAs) of which all run at once, one CTA to an
    // SM, while a CTA keeps half of its warps' groups.  What fits a GPC is the
    // device's own affair, hence the question (two sequences of 8 KV heads, window
    // 4096 / 16384: powers of two up to 8 18.3 / 44.0 us, any size up to all SMs, where
    // the last clusters wait, 18.3 / 42.5, so 12.1 / 28.7).
    static std::atomic<int> known[64][kMaxCluster + 1];
    int dev = 0;
    cudaGetDevice(&dev);
    if (const cudaError_t e = configure_clustered(kern, WG::SMEM, configured); e != cudaSuccess) return e;
    const int64_t n = units * p.num_seqs, sms = decode_sm_count(), most = longest_seen(p, w) / (NW * GT / 2);
    for (int c = (int)(most < kMaxCluster ? most : kMaxCluster); c > 1 && cluster == 1; --c)
      if (n * c <= sms && active_clusters(kern, WG::SMEM, NW * 32, c, dev, known) >= n) cluster = c;
  }
  return launch_clustered(kern, WG::SMEM, cluster, units, (unsigned)p.num_seqs, NW * 32, configured, stream, p, w, maps);
}

// Token-major blocks whose rows a tensor map can address: 16k rows one after another.
static bool token_row_map(const DecodeParams& p) {
  return p.block_size % 16 == 0 && p.k_block_stride == (int64_t)p.block_size * p.k_tok_stride &&
         p.v_block_stride == (int64_t)p.block_size * p.v_tok_stride &&
         p.num_blocks * (int64_t)p.block_size < (int64_t)1 << 31;
}

template <typename T, int D, bool EXT, Form FORM>
static cudaError_t launch_window_layout(const DecodeParams& p, bool flash, const WindowArgs& w, cudaStream_t stream) {
  // 16-token groups: as the decode (decode_mma.cuh), or 12 warps, or half the
  // decode's; 32-token pages: 2 warps (three CTAs to an SM), or 6 (12 at D = 64)
  constexpr int NW = FORM == kWide ? 12 : (D == 128 ? 6 : 4) / (FORM == kSmall ? 2 : 1), ST = D == 128 ? 2 : 3;
  constexpr int NP = FORM == kWide ? (D == 128 ? 6 : 12) : 2;
  if (flash) {
    if (token_row_map(p)) {
      const cudaError_t e = launch_window_nw<T, D, 16, NW, ST, 16, kFlashTma, EXT, FORM>(p, w, stream);
      if (e != cudaErrorNotSupported) return e;
    }
    return launch_window_nw<T, D, 16, NW, ST, 16, kFlash, EXT, FORM>(p, w, stream);
  }
  if (p.block_size == 8) return launch_window_nw<T, D, 8, NW, ST, 16, kBulk, EXT, FORM>(p, w, stream);
  if (p.block_size == 16) return launch_window_nw<T, D, 16, NW, ST, 16, kBulk, EXT, FORM>(p, w, stream);
  constexpr Form FP = FORM == kSmall ? kNarrow : FORM;  // (kNarrow is as small)
  const cudaError_t e = launch_window_nw<T, D, 32, NP, 2, 32, kSwizzledV, EXT, FP>(p, w, stream);
  if (e != cudaErrorNotSupported) return e;
  return launch_window_nw<T, D, 32, NP, 2, 32, kBulk, EXT, FP>(p, w, stream);
}

// 16-row tiles of a call: (tiles of a sequence) x sequences x KV heads.
static int64_t window_units(const DecodeParams& p, int64_t new_tokens) {
  return (new_tokens * (p.num_heads / p.num_kv_heads) + 15) / 16 * p.num_seqs * p.num_kv_heads;
}

// kWide where every tile gets an SM or more (decode, 8 KV heads, 1 / 2 / 4 / 8 / 16
// sequences: window 1024, 32-token pages 27.6 / 27.5 / 27.6 / 28.9 / 29.8 us narrow, 6.5 /
// 7.0 / 8.4 / 12.4 / 17.4 wide; slot lists 22.3 / 22.3 / 22.3 / 22.9 / 23.5 and 7.6 / 8.1 /
// 10.1 / 13.0 / 19.0; window 4096, 16-token pages 52.9 / 53.8 / 57.5 / 60.8 / 62.7 and 9.5 /
// 12.0 / 18.0 / 28.5 / 48.0).
// kSmall where every SM gets four tiles or more, so that it pays to have more CTAs in
// their start and end, and the groups are short (D = 64, single token rows) or few
// (decode, 8 KV heads, 128 sequences, window 64 / 128 / 256 / 1024: D = 128, 16-token
// pages 19.4 / 24.5 / 33.9 / 89.8 us narrow, 17.3 / 23.0 / 34.7 / 101.4 small, and with
// 256 sequences 34.1 / 42.9 / 58.2 / 166.2 and 29.2 / 38.1 / 57.8 / 171.9; D = 64 9.5 /
// 13.4 / 20.2 / 49.9 and 7.3 / 11.6 / 17.3 / 51.7; slot lists 32.6 / 41.9 / 57.7 / 154.0 and
// 20.0 / 27.3 / 43.1 / 138.2; 64 sequences of D = 64, under four tiles to an SM: 5.3 / 6.7 /
// 11.0 / 28.1 and 6.1 / 8.7 / 13.3 / 39.9).
template <typename T, int D, bool EXT>
static cudaError_t launch_window_mma(const DecodeParams& p, bool flash, const WindowArgs& w, cudaStream_t stream) {
  const int64_t units = window_units(p, EXT ? w.max_q_len : 1), sms = decode_sm_count();
  if (units <= sms) return launch_window_layout<T, D, EXT, kWide>(p, flash, w, stream);
  if constexpr (!EXT) {
    const bool slots = flash && !token_row_map(p), pages32 = !flash && p.block_size == 32;
    if (units >= 4 * sms && !pages32 && (D == 64 || slots || longest_seen(p, w) <= 160))
      return launch_window_layout<T, D, EXT, kSmall>(p, flash, w, stream);
  }
  return launch_window_layout<T, D, EXT, kNarrow>(p, flash, w, stream);
}

template <typename Q_T, typename CACHE_T, int D>
static cudaError_t launch_window_any(const DecodeParams& p, const WindowArgs& w, cudaStream_t stream) {
  const int G = p.num_heads / p.num_kv_heads;
  const int units = p.num_kv_heads * ((G + kWinGC - 1) / kWinGC);
  static std::atomic<bool> configured[64];
  return launch_clustered(window_decode_any_kernel<Q_T, CACHE_T, D>, exchange_floats(kWinGC, D) * 4,
                          window_cluster(p, w, units, kWinWarps * p.block_size), units, (unsigned)p.num_seqs,
                          kWinWarps * 32, configured, stream, p, w);
}

template <typename Q_T, typename CACHE_T>
static cudaError_t launch_window_any_d(const DecodeParams& p, const WindowArgs& w, int D, cudaStream_t stream) {
  switch (D) {
    case 32: return launch_window_any<Q_T, CACHE_T, 32>(p, w, stream);
    case 64: return launch_window_any<Q_T, CACHE_T, 64>(p, w, stream);
    case 80: return launch_window_any<Q_T, CACHE_T, 80>(p, w, stream);
    case 96: return launch_window_any<Q_T, CACHE_T, 96>(p, w, stream);
    case 112: return launch_window_any<Q_T, CACHE_T, 112>(p, w, stream);
    case 120: return launch_window_any<Q_T, CACHE_T, 120>(p, w, stream);
    case 128: return launch_window_any<Q_T, CACHE_T, 128>(p, w, stream);
    case 192: return launch_window_any<Q_T, CACHE_T, 192>(p, w, stream);
    case 256: return launch_window_any<Q_T, CACHE_T, 256>(p, w, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_window_decode(const DecodeArgs& a, const WindowArgs& w, cudaStream_t stream) {
  if (a.num_seqs > 65535) return cudaErrorInvalidValue;
  const int cs = elem_size(a.cache_type);
  auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; };
  if (!al(a.k_cache) || !al(a.v_cache) || (a.k_block_stride * cs) % 16 || (a.k_head_stride * cs) % 16 ||
      (a.v_block_stride * cs) % 16 || (a.v_head_stride * cs) % 16 || (a.k_tok_stride * cs) % 16 ||
      (a.v_tok_stride * cs) % 16)
    return cudaErrorMisalignedAddress;
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.out = a.out;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.block_tables = a.block_tables;
  p.context_lens = a.context_lens;
  p.num_seqs = a.num_seqs;
  p.num_heads = a.num_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.block_size = a.block_size;
  p.max_seq_len = a.max_seq_len;
  p.num_partitions = 1;
  p.num_blocks = a.num_blocks;
  p.q_seq_stride = a.q_seq_stride;
  p.q_head_stride = a.q_head_stride;
  p.out_seq_stride = a.out_seq_stride;
  p.out_head_stride = a.out_head_stride;
  p.k_block_stride = a.k_block_stride;
  p.k_head_stride = a.k_head_stride;
  p.v_block_stride = a.v_block_stride;
  p.v_head_stride = a.v_head_stride;
  p.k_tok_stride = a.k_tok_stride;
  p.v_tok_stride = a.v_tok_stride;
  p.table_stride = a.table_stride;
  p.scale = a.scale;
  // tensor cores: 16-bit query and cache of one type, head size 64 / 128, query
  // rows read as pairs of elements
  const bool mma = a.q_type == a.cache_type && a.q_type != ElemType::F32 && (a.head_size == 64 || a.head_size == 128) &&
                   (reinterpret_cast<uintptr_t>(a.q) & 3u) == 0 &&
                   ((a.q_seq_stride | a.q_head_stride) & 1) == 0;
  if (mma && a.num_heads / a.num_kv_heads > 16) {
    const WindowArgs one = {w.window, w.sinks, nullptr, 1, a.num_seqs, 0};
    if (a.q_type == ElemType::BF16)
      return a.head_size == 128 ? launch_window_mma<__nv_bfloat16, 128, true>(p, a.flash, one, stream)
                                : launch_window_mma<__nv_bfloat16, 64, true>(p, a.flash, one, stream);
    return a.head_size == 128 ? launch_window_mma<__half, 128, true>(p, a.flash, one, stream)
                              : launch_window_mma<__half, 64, true>(p, a.flash, one, stream);
  }
  if (mma) {
    if (a.q_type == ElemType::BF16)
      return a.head_size == 128 ? launch_window_mma<__nv_bfloat16, 128, false>(p, a.flash, w, stream)
                                : launch_window_mma<__nv_bfloat16, 64, false>(p, a.flash, w, stream);
    return a.head_size == 128 ? launch_window_mma<__half, 128, false>(p, a.flash, w, stream)
                              : launch_window_mma<__half, 64, false>(p, a.flash, w, stream);
  }
  if (a.flash) return cudaErrorNotSupported;  // no CUDA-core kernel for token-major caches
  const int D = a.head_size;
  if (a.q_type == ElemType::F32) {
    if (a.cache_type == ElemType::F32) return launch_window_any_d<float, float>(p, w, D, stream);
    if (a.cache_type == ElemType::F16) return launch_window_any_d<float, __half>(p, w, D, stream);
    return launch_window_any_d<float, __nv_bfloat16>(p, w, D, stream);
  }
  if (a.q_type == ElemType::F16) return launch_window_any_d<__half, __half>(p, w, D, stream);
  return launch_window_any_d<__nv_bfloat16, __nv_bfloat16>(p, w, D, stream);
}

// ---------------------------------------------------------------------------
// Extend.  The tcgen05 kernel (window_umma.cuh) serves every paged and token-major
// cache that tensor maps describe (pages a whole number of K chunk rows apart, token
// rows that hold all heads a fixed distance apart, fewer than 2^31 of either); the
// decode's kernel serves few new tokens, and any number from the other caches.
// ---------------------------------------------------------------------------
// K as rows of one 8-dim chunk of one page, [rows][BS * 8], over whatever lies
// between the pages of a strided cache.
static bool make_k_chunk_map(const PrefillArgs& a, int D, int BS, CUtensorMap* map) {
  auto enc = tensor_map_encoder();
  const int64_t row = (int64_t)BS * 8;
  if (!enc || a.k_block_stride % row || a.k_head_stride % row || a.k_block_stride < 0 || a.k_head_stride < 0) return false;
  const int64_t rows = ((a.num_blocks - 1) * a.k_block_stride + (a.num_kv_heads - 1) * a.k_head_stride) / row + D / 8;
  if (rows <= 0 || rows > 0x7fffffffll) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)row, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row * 2};
  const cuuint32_t box[2] = {(cuuint32_t)row, 1};
  const cuuint32_t ones[2] = {1, 1};
  return enc(map, a.q_type == ElemType::BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(a.k_cache), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// Token rows of a token-major cache, [rows][all heads of a row]: row `token` of block
// b is row b * (block stride / token stride) + token.
static bool make_token_row_map(const PrefillArgs& a, const void* base, int D, int64_t block, int64_t tok, int64_t head,
                               CUtensorMap* map) {
  auto enc = tensor_map_encoder();
  if (!enc || tok <= 0 || block <= 0 || head < 0 || block % tok) return false;
  const int64_t width = (a.num_kv_heads - 1) * head + D;
  const int64_t rows = (a.num_blocks - 1) * (block / tok) + a.block_size;
  if (width > tok || rows <= 0 || rows > 0x7fffffffll || width > 0x7fffffffll) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)tok * 2};
  const cuuint32_t box[2] = {64, 1};
  const cuuint32_t ones[2] = {1, 1};
  return enc(map, a.q_type == ElemType::BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int BS, int LOAD, bool OUT16>
static cudaError_t launch_window_umma_out(const PrefillArgs& a, cudaStream_t stream) {
  using WG = WinUmmaGeom<D, BS, LOAD>;
  DecodeParams dp;
  memset(&dp, 0, sizeof(dp));
  dp.k_cache = a.k_cache;
  dp.v_cache = a.v_cache;
  dp.num_blocks = a.num_blocks;
  dp.num_kv_heads = a.num_kv_heads;
  dp.block_size = a.block_size;
  dp.k_head_stride = a.k_head_stride;
  dp.k_block_stride = a.k_block_stride;
  dp.v_head_stride = a.v_head_stride;
  dp.v_block_stride = a.v_block_stride;
  dp.k_tok_stride = a.k_tok_stride;
  dp.v_tok_stride = a.v_tok_stride;
  TmaMaps maps;
  memset(&maps, 0, sizeof(maps));
  const ElemType et = std::is_same<T, __nv_bfloat16>::value ? ElemType::BF16 : ElemType::F16;
  if (LOAD == kPages) {
    if ((BS > 8 && !make_tensor_maps(dp, et, D, BS, BS, BS * 2, kTiles, &maps)) || !make_k_chunk_map(a, D, BS, &maps.k))
      return cudaErrorNotSupported;
  } else if (LOAD == kRows) {
    if (!make_tensor_maps(dp, et, D, 16, 16, 128, kFlashTma, &maps)) return cudaErrorNotSupported;
  } else {
    // (block size 1, the pool's [slots, H, D]: a block is one row and carries no token stride)
    const bool one = a.block_size == 1;
    if (!make_token_row_map(a, a.k_cache, D, a.k_block_stride, one ? a.k_block_stride : a.k_tok_stride, a.k_head_stride,
                            &maps.k) ||
        !make_token_row_map(a, a.v_cache, D, a.v_block_stride, one ? a.v_block_stride : a.v_tok_stride, a.v_head_stride,
                            &maps.v))
      return cudaErrorNotSupported;
  }
  auto kern = window_umma_kernel<T, D, BS, LOAD, OUT16>;
  static std::atomic<bool> configured[64];  // per device; setting the attribute twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WG::SMEM);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int G = a.num_heads / a.num_kv_heads;
  const int64_t tiles = ((int64_t)a.max_q_len * G + kUmmaRows - 1) / kUmmaRows;
  const int64_t items = tiles * a.num_seqs * a.num_kv_heads;
  if (items > 0x7fffffffll - 1024) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)umma_persistent_ctas(dev, items));
  cfg.blockDim = dim3(kWinThreads);
  cfg.dynamicSmemBytes = WG::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, kern, a, maps, (int)tiles, (int)a.num_seqs, umma_sched_slot(stream));
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int D, int BS, int LOAD>
static cudaError_t launch_window_umma(const PrefillArgs& a, cudaStream_t stream) {
  return (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && ((a.out_tok_stride | a.out_head_stride) & 7) == 0
             ? launch_window_umma_out<T, D, BS, LOAD, true>(a, stream)
             : launch_window_umma_out<T, D, BS, LOAD, false>(a, stream);
}

// The decode's kernel over 16-row tiles, split over clusters.
template <typename T, int D>
static cudaError_t launch_window_few(const PrefillArgs& a, cudaStream_t stream) {
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.out = a.out;
  p.q = a.q;
  p.k_cache = a.k_cache;
  p.v_cache = a.v_cache;
  p.block_tables = a.block_tables;
  p.context_lens = a.kv_lens;
  p.num_seqs = a.num_seqs;
  p.num_heads = a.num_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.block_size = a.block_size;
  p.max_seq_len = (int)(a.table_len * a.block_size < 0x7fffffffll ? a.table_len * a.block_size : 0x7fffffffll);
  p.num_partitions = 1;
  p.num_blocks = a.num_blocks;
  p.q_seq_stride = a.q_tok_stride;
  p.q_head_stride = a.q_head_stride;
  p.out_seq_stride = a.out_tok_stride;
  p.out_head_stride = a.out_head_stride;
  p.k_block_stride = a.k_block_stride;
  p.k_head_stride = a.k_head_stride;
  p.v_block_stride = a.v_block_stride;
  p.v_head_stride = a.v_head_stride;
  p.k_tok_stride = a.k_tok_stride;
  p.v_tok_stride = a.v_tok_stride;
  p.table_stride = a.table_stride;
  p.scale = a.scale;
  WindowArgs w = {a.window, a.sinks, a.qo_indptr, a.max_q_len, a.num_tokens, a.table_len};
  return launch_window_mma<T, D, true>(p, a.token_major, w, stream);
}

template <typename T, int D>
static cudaError_t launch_window_prefill_t(const PrefillArgs& a, cudaStream_t stream) {
  // A 16-row tile for every SM or fewer: the decode's kernel, which splits the keys
  // too (4 sequences, 4 KV heads, 7 heads each, window 1024; 16 / 64 / 112 / 224
  // tiles: 8.6 / 13.3 / 17.4 / 30.5 us against 20 of 128-row items one after
  // another).
  const int64_t units = ((int64_t)a.max_q_len * (a.num_heads / a.num_kv_heads) + 15) / 16 * a.num_seqs * a.num_kv_heads;
  const int64_t sms = decode_sm_count();
  if (units <= sms) return launch_window_few<T, D>(a, stream);
  cudaError_t e = cudaErrorNotSupported;
  if (!a.token_major) {
    if (a.block_size == 32) e = launch_window_umma<T, D, 32, kPages>(a, stream);
    else if (a.block_size == 16) e = launch_window_umma<T, D, 16, kPages>(a, stream);
    else if (a.block_size == 8) e = launch_window_umma<T, D, 8, kPages>(a, stream);
  } else {
    const int64_t bs = a.block_size;
    if (bs % 16 == 0 && a.k_block_stride == bs * a.k_tok_stride && a.v_block_stride == bs * a.v_tok_stride &&
        a.num_blocks * bs < (int64_t)1 << 31)
      e = launch_window_umma<T, D, 16, kRows>(a, stream);
    if (e == cudaErrorNotSupported) e = launch_window_umma<T, D, 16, kSlots>(a, stream);
  }
  // (a cache that no tensor map describes: per-lane or bulk copies)
  return e != cudaErrorNotSupported ? e : launch_window_few<T, D>(a, stream);
}

cudaError_t launch_window_prefill(const PrefillArgs& a, cudaStream_t stream) {
  if (a.num_seqs <= 0 || a.max_q_len <= 0) return cudaSuccess;
  if (a.num_seqs > 65535 || a.num_kv_heads > 65535) return cudaErrorInvalidValue;
  if (a.q_type == ElemType::BF16)
    return a.head_size == 128 ? launch_window_prefill_t<__nv_bfloat16, 128>(a, stream)
                              : launch_window_prefill_t<__nv_bfloat16, 64>(a, stream);
  return a.head_size == 128 ? launch_window_prefill_t<__half, 128>(a, stream)
                            : launch_window_prefill_t<__half, 64>(a, stream);
}

}  // namespace kvc

unsigned int kvc_window_status(int clear, cudaError_t* err) {
  unsigned int v = 0;
  *err = cudaMemcpyFromSymbol(&v, kvc::g_decode_status, sizeof(v));
  if (*err == cudaSuccess && clear) {
    const unsigned int zero = 0;
    *err = cudaMemcpyToSymbol(kvc::g_decode_status, &zero, sizeof(zero));
  }
  return v;
}
