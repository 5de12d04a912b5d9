// window_umma.cuh — tcgen05 extend attention over a sliding window with sinks
// (sm_100a), for the paged layout and for token-major caches.
//
// Included by window.cu after prefill_umma.cuh, whose work items (umma_item: 128
// (new token, query head) rows of one sequence and KV head), persistent grid and
// descriptors it shares.  An item's keys are its sink blocks and its window's
// blocks without the gap between them (struct Seen), in tiles of 128 tokens that
// are filled block by block, so the few sink tokens share a tile with the window's
// first blocks and no tile is spent on alignment.
//
// What sets it apart from the causal kernel: that one's two halves of softmax warps
// (each thread one row and 64 of a tile's 128 tokens) share one O and so must agree
// on a row maximum before every exponential, an exchange of about 630 of a tile's
// 3260 cycles.  Here each half accumulates into an O of its own with its own lazy
// maximum and sum, and the two meet once per item:
//   out = (w_0 O_0 + w_1 O_1) / (w_0 l_0 + w_1 l_1),  w_h = 2^(m_h - max(m_0, m_1)).
// The second O takes the tensor memory that Q had, so Q goes to shared memory
// (S = Q K^T from two descriptors, N = 128), and K and V have rings of their own: K
// is free after S, V after P V.
//   TMEM (512 columns): S 2 x 128 (P over it: per half 32 columns of hi pairs and
//   32 of lo pairs, zeros where the rows have none), O 2 x D.
//   Warps 0-7 softmax (warp w and w + 4: the two halves of rows 32 (w & 3) ..),
//   warp 8 K, warp 9 (one lane) products, warp 10 V, warp 11 items and Q.
// K and V have a warp each because V waits for a product that comes a softmax
// later than K's: behind V's wait in one warp, K came 800 cycles late for S.  Warp
// 11 claims and decodes an item while the one before it runs and copies its Q
// rows: done by the softmax warps between two items, that cost 12000 cycles an
// item, against 3300 a tile.  The products run over the tiles of all items in one
// sequence, S of the next tile (or item) ahead of P V of this one.
//
// LOAD: how a tile reaches shared memory.
//   kPages  paged layout: K by 4-row gathers of 8-dim chunk rows ([D/8][128][8],
//           no swizzle), V a page at a time ([D][bs], K-major for P V: rows swizzled
//           over their bs * 2 bytes, or as they are for 8 tokens).
//   kRows   token-major, blocks of 16k dense rows: 16 rows x 64 dims to a copy,
//           128-byte swizzle; K is K-major as it lies, V is MN-major (its
//           dims, the N of P V, run along the row).
//   kSlots  token-major, any block size (the pool's slot lists) and row distance: the
//           same tile from 4-row gathers, each token's row where its own slot is.
// Every wait is bounded; a timeout sets KVC_STATUS_WAIT_TIMEOUT and an abort flag
// that ends every loop; TMEM is freed after a final commit.
#pragma once

namespace kvc {

constexpr int kPages = 0, kRows = 1, kSlots = 2;
constexpr uint32_t kLayoutSw128 = 2;

constexpr int kWinThreads = 384;
constexpr int kKWarp = 8, kVWarp = 10, kItemWarp = 11;
constexpr int kWinItems = 4;  // item slots
// bf16 P is rounded once (8 bits) where no weight of a warp's 32 rows in a half tile is
// more than 1 / kSharp of its row's sum so far (and so of its whole sum), and carried as
// hi + lo (16 bits, a second product per 16 tokens) elsewhere: a few large weights on
// nearly cancelling V rows show the rounding, many small ones average it out.  16 x 512
// tokens, window 1024, N(0, 1) keys and values, queries N(0, f^2); elements of 2.2e7 past
// 2e-3 + 1e-2 |value| at f = 2 / 6 (the worst by), and the time at f = 1:
//   once wherever a row sees 64 keys   16 / 1746 (5e-3)      134.6 us
//   kSharp 2                            1 / 4    (6e-4)      141.6
//   kSharp 4                            0 / 0    (7e-4 to go) 144.7
//   kSharp 8                            0 / 0    (1.4e-3)    150.3
//   always hi + lo                      0 / 0    (2.0e-3)    164.2
constexpr float kSharp = 4.f;

// 16 bytes of an output row: one store, or, where the rows do not start on 16-byte
// boundaries, four (a row's pairs are 4-byte aligned: the host checked).
template <bool OUT16>
__device__ __forceinline__ void store_row16(void* dst, uint4 v) {
  if constexpr (OUT16) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
    uint32_t* d = reinterpret_cast<uint32_t*>(dst);
    d[0] = v.x;
    d[1] = v.y;
    d[2] = v.z;
    d[3] = v.w;
  }
}

// Products whose accumulation is known as the code is written, with the second
// operand's descriptor as its low word (the address, which is all that changes:
// shared addresses stay below 256 KB, no carry) and its constant high word.  The
// one lane that issues them competes with eight softmax warps for issue slots: at
// 160 cycles a product (64-bit descriptor arithmetic, a predicate and a branch
// each) they, not the tensor cores, set the pace.
template <bool ADD>
__device__ __forceinline__ void mma_ts_lo(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 b;\nmov.b64 b, {%2, %3};\nsetp.ne.b32 p, %5, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(ADD ? 1 : 0));
}
template <bool ADD>
__device__ __forceinline__ void mma_ss_lo(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                          uint32_t idesc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %2};\nmov.b64 b, {%3, %4};\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(ADD ? 1 : 0));
}

// A decoded work item, handed by warp 11 to the others.
struct WinItem {
  int64_t q0;         // row of q / out of the sequence's first new token
  Seen seen;
  int t0, g0, nrows;  // (new token, head of the group) of the item's first row; rows
  int y, kvh, prefix; // prefix less the gap: row's end = prefix + token + 1, virtual
  int kv_end, ntiles;
  int state;          // 0 work, 1 rows to be zeroed (bad indices), 2 no further item
};

template <int D, int BS, int LOAD>
struct WinUmmaGeom {
  static constexpr int TILE = kUmmaTile * D * 2;  // bytes of one K (or V) tile
  static constexpr int KS = D == 128 ? 3 : 4, VS = D == 128 ? 2 : 4;  // ring stages
  static constexpr int Q_OFF = (KS + VS) * TILE;
  static constexpr int XBUF_OFF = Q_OFF + 2 * TILE;          // [2 halves][128 rows] (max, sum)
  static constexpr int BAR_OFF = XBUF_OFF + 2 * 128 * 8;
  static constexpr int NBARS = 2 * KS + 3 * VS + 2 + 4 + 1 + 1 + 4 + 1 + 1 + 2 * kWinItems;
  static constexpr int MASK_OFF = BAR_OFF + NBARS * 8;       // [8 tiles][4] loaded blocks (kSlots: tokens)
  static constexpr int ITEM_OFF = (MASK_OFF + 8 * 16 + 15) / 16 * 16;
  static constexpr int MISC_OFF = ITEM_OFF + kWinItems * (int)sizeof(WinItem);  // abort, tmem address, lo parts
  static constexpr int SMEM = MISC_OFF + 8 + 16;
  static constexpr int UNIT = LOAD == kPages ? BS : (LOAD == kRows ? 16 : 1);  // tokens to a mask bit
  static constexpr int UNITS = LOAD == kSlots ? 128 : kUmmaTile / UNIT;
  static constexpr uint32_t SCOL = 0, OCOL = 256;
  static_assert(OCOL + 2 * D <= 512, "TMEM columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// OUT16: output rows start on 16-byte boundaries (a run-time choice costs the softmax
// warps registers: 16 x 512 tokens 5 us).
template <typename T, int D, int BS, int LOAD, bool OUT16>
__global__ void __launch_bounds__(kWinThreads, 1)
    window_umma_kernel(const PrefillArgs p, const __grid_constant__ TmaMaps maps, int tiles_x, int ny, int slot) {
  using namespace mma_detail;
  using WG = WinUmmaGeom<D, BS, LOAD>;
  constexpr int KT = kUmmaTile, TILE = WG::TILE, KS = WG::KS, VS = WG::VS, UNIT = WG::UNIT;
  constexpr int PAGES = KT / BS, PAGE = D * BS * 2;  // kPages
  constexpr int HALF = KT * 128;                     // token-major: bytes of 64 dims of a tile
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  // (no static shared memory: the dynamic window then starts on a 1024-byte
  // boundary, as the 128-byte swizzle needs; checked below)
  extern __shared__ __align__(1024) uint8_t smem_wu[];
  uint8_t* kring = smem_wu;
  uint8_t* vring = smem_wu + KS * TILE;
  uint8_t* qsm = smem_wu + WG::Q_OFF;
  float2* xbuf = reinterpret_cast<float2*>(smem_wu + WG::XBUF_OFF);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_wu + WG::BAR_OFF);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* v_ready = v_empty + VS;  // what nobody sees is cleared
  uint64_t* s_full = v_ready + VS;   // [2 buffers]
  uint64_t* p_full = s_full + 2;    // [2 buffers][2 halves]
  uint64_t* pv_done = p_full + 4;
  uint64_t* o_done = pv_done + 1;
  uint64_t* q_full = o_done + 1;    // [2 buffers]
  uint64_t* q_empty = q_full + 2;
  uint64_t* all_done = q_empty + 2;
  uint64_t* xchg = all_done + 1;
  uint64_t* item_full = xchg + 1;   // [kWinItems]
  uint64_t* item_empty = item_full + kWinItems;
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem_wu + WG::MASK_OFF);
  WinItem* items = reinterpret_cast<WinItem*>(smem_wu + WG::ITEM_OFF);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem_wu + WG::MISC_OFF);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem_wu + WG::MISC_OFF + 4);
  // [2 buffers][2 halves][4 warps]: the warp's rows of P have lo parts (else those are 0)
  volatile uint8_t* s_lo = reinterpret_cast<volatile uint8_t*>(smem_wu + WG::MISC_OFF + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.num_heads / p.num_kv_heads;
  const int n_items = tiles_x * ny * p.num_kv_heads;
  const bool dynamic = n_items > (int)gridDim.x;
  grid_dependents_launch();
  if ((smem_u32(smem_wu) & 1023u) != 0) {  // (the same for every thread)
    grid_dependency_wait();
    if (threadIdx.x == 0) set_status(&g_decode_status, KVC_STATUS_WAIT_TIMEOUT);
    return;
  }
  if (threadIdx.x == 0) {
    *s_abort = 0;
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&v_ready[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s_full[b], 2);
      mbar_init(&q_full[b], 1);
      mbar_init(&q_empty[b], 8);
    }
    for (int b = 0; b < 4; ++b) mbar_init(&p_full[b], 4);
    for (int b = 0; b < kWinItems; ++b) {
      mbar_init(&item_full[b], 1);
      mbar_init(&item_empty[b], 11);
    }
    mbar_init(pv_done, 1);
    mbar_init(o_done, 1);
    mbar_init(all_done, 1);
    mbar_init(xchg, 8);
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == kKWarp && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.v)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.k)) : "memory");
  }
  umma::fence_before();
  __syncthreads();
  umma::fence_after();
  const uint32_t tmem = *s_tmem;
  // (a programmatic dependent: the set-up above overlaps the kernel before this one)
  grid_dependency_wait();
  auto abort_now = [&]() -> bool { return *s_abort != 0; };
  auto give_up = [&]() {
    *s_abort = 1;
    set_status(&g_decode_status, KVC_STATUS_WAIT_TIMEOUT);
  };

  // Item k of this CTA, for a whole warp: false on a failed wait.
  auto take_item = [&](int k, WinItem& it) -> bool {
    const int sl = k % kWinItems;
    if (!__all_sync(0xffffffffu, umma::wait(&item_full[sl], (uint32_t)((k / kWinItems) & 1)))) return false;
    it = items[sl];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[sl]);
    return true;
  };

  if (warp == kItemWarp) {
    // ---- items and their Q
    UmmaSched* sched = &g_umma_sched[slot];
    int npub = 0, nq = 0;  // items handed over, of them with keys
    bool ok = true;
    auto publish = [&](const WinItem& it) -> bool {
      const int sl = npub % kWinItems;
      bool fine = true;
      if (lane == 0) {
        if (npub >= kWinItems) fine = umma::wait(&item_empty[sl], (uint32_t)((npub / kWinItems - 1) & 1));
        if (fine) {
          items[sl] = it;
          mbar_arrive(&item_full[sl]);  // (release)
        }
      }
      ++npub;
      return __shfl_sync(0xffffffffu, fine, 0) && !__shfl_sync(0xffffffffu, abort_now() ? 1 : 0, 0);
    };
    for (int idx = blockIdx.x; idx < n_items && ok;) {
      const UmmaItem u = umma_item<false, true>(p, idx, tiles_x, ny);
      if (u.bad && u.first_tile && u.kvh == 0 && lane == 0) set_status(&g_decode_status, KVC_STATUS_INDEX_OOB);
      if (!u.skip) {
        WinItem it;
        it.q0 = u.q0;
        it.seen = u.seen;
        it.t0 = (int)(u.R0 / G);
        it.g0 = (int)(u.R0 - (int64_t)it.t0 * G);
        it.nrows = (int)(u.rows - u.R0 < kUmmaRows ? u.rows - u.R0 : kUmmaRows);
        it.y = u.y;
        it.kvh = u.kvh;
        it.prefix = u.prefix;
        it.kv_end = u.kv_end;
        it.ntiles = u.ntiles;
        it.state = u.bad ? 1 : 0;
        ok = publish(it);
        if (ok && it.ntiles > 0) {
          // Q rows into buffer nq & 1 ([D/8 chunks][128 rows][8 dims]; rows past the
          // last are zero), free once the item two back has left its output rows in it
          const int buf = nq & 1;
          bool free = true;
          if (nq >= 2 && lane == 0) free = umma::wait(&q_empty[buf], (uint32_t)(((nq >> 1) - 1) & 1));
          ok = __shfl_sync(0xffffffffu, free, 0);
          if (ok) {
            const T* qbase = reinterpret_cast<const T*>(p.q);
            const T* row[4];
            bool on[4], wide = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 32 + lane, x = it.g0 + r, dt = x / G;
              on[i] = r < it.nrows;
              row[i] = on[i] ? qbase + (it.q0 + it.t0 + dt) * p.q_tok_stride +
                                   (int64_t)(it.kvh * G + (x - dt * G)) * p.q_head_stride
                             : qbase;
              wide = wide && (!on[i] || (reinterpret_cast<uintptr_t>(row[i]) & 15u) == 0);
            }
            // (a row past the last reads nothing, but its address must be aligned too)
            wide = __all_sync(0xffffffffu, wide) && (reinterpret_cast<uintptr_t>(qbase) & 15u) == 0;
            uint8_t* qb = qsm + buf * TILE + lane * 16;
            if (wide) {
#pragma unroll 4
              for (int c = 0; c < D / 8; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  cp_async16_zfill(qb + c * (kUmmaRows * 16) + i * 512, row[i] + c * 8, on[i] ? 16u : 0u);
              asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
              for (int c = 0; c < D / 8; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t* q32 = reinterpret_cast<const uint32_t*>(row[i] + c * 8);
                  *reinterpret_cast<uint4*>(qb + c * (kUmmaRows * 16) + i * 512) =
                      on[i] ? make_uint4(q32[0], q32[1], q32[2], q32[3])
                            : make_uint4(0u, 0u, 0u, 0u);
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[buf]);
            ++nq;
          }
        }
      }
      // the next item, once Q of this one is in (so at most one item is claimed ahead)
      unsigned nx = (unsigned)n_items;
      if (dynamic && lane == 0) nx = gridDim.x + atomicAdd(&sched->next, 1u);
      nx = __shfl_sync(0xffffffffu, nx, 0);
      idx = nx < (unsigned)n_items ? (int)nx : n_items;
    }
    if (ok) {
      WinItem it;
      memset(&it, 0, sizeof(it));
      it.state = 2;
      ok = publish(it);
    }
    if (!ok && lane == 0) give_up();
    __syncwarp();
  } else if (warp == kKWarp || warp == kVWarp) {
    // ---- one ring's tiles, K or V
    const bool is_k = warp == kKWarp;
    const int stages = is_k ? KS : VS;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    uint8_t* ring = is_k ? kring : vring;
    const CUtensorMap* map = is_k ? &maps.k : &maps.v;
    // kSlots: rows of the map from one block to the next (all rows are below 2^31: the host checked)
    const int64_t rows_per_block = LOAD != kSlots || p.block_size == 1 ? 1
                                   : is_k                              ? p.k_block_stride / p.k_tok_stride
                                                                       : p.v_block_stride / p.v_tok_stride;
    int g = 0, st = 0, round = 0;  // tiles asked for, the next one's stage and turn of the ring
    bool ok = true;
    for (int k = 0; ok; ++k) {
      WinItem it;
      if (!take_item(k, it)) {
        ok = false;
        break;
      }
      if (it.state == 2) break;
      const int kvh = it.kvh, kv_end = it.kv_end, ntiles = it.ntiles;
      const uint32_t* table = p.block_tables + (int64_t)it.y * p.table_stride;
      const int tbs = p.block_size;
      const int col = (int)(kvh * (is_k ? p.k_head_stride : p.v_head_stride));  // kSlots: the head's first column
      // ids of tile j: lane i holds unit i's (kSlots: tokens 4i .. 4i + 3)
      auto load_ids = [&](int j, uint32_t (&id)[4]) {
        if constexpr (LOAD == kSlots) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = j * KT + 4 * lane + e;
            id[e] = j < ntiles && tok < kv_end ? table[it.seen.real_block(tbs == 1 ? tok : tok / tbs)] : 0xffffffffu;
          }
        } else {
          const int tok = j * KT + lane * UNIT;
          id[0] = lane < WG::UNITS && j < ntiles && tok < kv_end
                      ? table[it.seen.real_block(LOAD == kPages ? tok / BS : tok / tbs)]
                      : 0xffffffffu;
        }
      };
      uint32_t id[4];
      load_ids(0, id);
      for (int j = 0; j < ntiles; ++j) {
        const int t0 = j * KT;
        bool free = true;
        if (round > 0 && lane == 0) free = umma::wait(&empty[st], (uint32_t)((round - 1) & 1));
        free = __shfl_sync(0xffffffffu, free, 0);
        if (!free || __shfl_sync(0xffffffffu, abort_now() ? 1 : 0, 0)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + (size_t)st * TILE;
        uint32_t* tm = masks + (g & 7) * 4;
        uint32_t next[4];
        uint32_t loaded = 0, bad4 = 0;  // units that are loaded; kSlots: which of my four tokens have no block
        if constexpr (LOAD == kSlots) {
          // a token without a block gathers a loaded token's row (and is masked)
          uint32_t good4 = 0, oob = 0;
          int row[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = t0 + 4 * lane + e;
            const bool in = tok < kv_end, good = in && (int64_t)id[e] < p.num_blocks;
            good4 |= good ? 1u << e : 0u;
            oob |= in && !good ? 1u << e : 0u;
            row[e] = good ? (int)(id[e] * rows_per_block) + (tbs == 1 ? 0 : tok % tbs) : -1;
          }
          if (oob) set_status(&g_decode_status, KVC_STATUS_BLOCK_OOB);
          bad4 = oob;
          const uint32_t any = __ballot_sync(0xffffffffu, good4 != 0u);
          int spare = good4 ? row[__ffs(good4) - 1] : 0;
          spare = __shfl_sync(0xffffffffu, spare, any ? __ffs(any) - 1 : 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) row[e] = row[e] >= 0 ? row[e] : spare;
          if (is_k) {  // lanes 8w .. 8w + 7 hold the 32 tokens of word w
            uint32_t word = good4 << (4 * (lane & 7));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
            if ((lane & 7) == 0) tm[lane >> 3] = word;
          }
          load_ids(j + 1, next);
          __syncwarp();
          if (lane == 0) {
            if (any) mbar_arrive_expect_tx(&full[st], (uint32_t)TILE);
            else mbar_arrive(&full[st]);
          }
          __syncwarp();
          if (any) {
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              tma_gather4(dst + h * HALF + lane * 512, map, col + 64 * h, row[0], row[1], row[2], row[3], &full[st]);
          }
        } else {
          const int tok = t0 + lane * UNIT;
          const bool in = lane < WG::UNITS && tok < kv_end, good = in && (int64_t)id[0] < p.num_blocks;
          if (in && !good) set_status(&g_decode_status, KVC_STATUS_BLOCK_OOB);
          const uint32_t mask = __ballot_sync(0xffffffffu, good);
          const uint32_t mine = id[0];
          loaded = mask;
          load_ids(j + 1, next);
          if (lane == 0) {
            if (is_k) tm[0] = mask;
            if (!mask) mbar_arrive(&full[st]);
            else
              mbar_arrive_expect_tx(&full[st], LOAD == kPages && is_k ? (uint32_t)TILE
                                                                      : (uint32_t)__popc(mask) * (uint32_t)(UNIT * D * 2));
          }
          __syncwarp();
          if (mask) {
            if constexpr (LOAD == kPages) {
              if (is_k) {
                // chunk row c of a page: row base + c; pages without keys gather a loaded page's rows
                const int base = (int)(((int64_t)mine * p.k_block_stride + (int64_t)kvh * p.k_head_stride) / (BS * 8));
                const int any = __shfl_sync(0xffffffffu, base, __ffs(mask) - 1);
                int rb[PAGES];
#pragma unroll
                for (int i = 0; i < PAGES; ++i) {
                  const int b = __shfl_sync(0xffffffffu, base, i);
                  rb[i] = (mask >> i) & 1u ? b : any;
                }
                if (lane < D / 8) {
#pragma unroll
                  for (int q = 0; q < PAGES; q += 4)
                    tma_gather4(dst + lane * KT * 16 + q * BS * 16, map, 0, rb[q] + lane, rb[q + 1] + lane,
                                rb[q + 2] + lane, rb[q + 3] + lane, &full[st]);
                }
              } else if (good) {
                if constexpr (BS == 8)
                  bulk_g2s(dst + lane * PAGE, reinterpret_cast<const T*>(p.v_cache) + (int64_t)mine * p.v_block_stride +
                                                  (int64_t)kvh * p.v_head_stride, PAGE, &full[st]);
                else
                  tma_load_4d(dst + lane * PAGE, map, 0, 0, kvh, (int)mine, &full[st]);
              }
            } else if (good) {
              const int row = (int)mine * tbs + tok % tbs;  // (rows are below 2^31: the host checked)
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_load_3d(dst + h * HALF + lane * 16 * 128, map, 64 * h, kvh, row, &full[st]);
            }
          }
        }
        if (!is_k) {
          // V of tokens nobody sees, in blocks that are loaded for others, becomes 0
          // (their slots may hold anything, and 0 * NaN = NaN): between the sinks and
          // the first row's window, and past the last row's end up to the 16 tokens
          // of a product.  So does V of blocks past the cache, in whose place the
          // stage holds another tile's tokens or another token's row.  This warp runs
          // ahead of the products.
          const int a0 = p.sinks > t0 ? p.sinks : t0, a1 = it.seen.beg < t0 + KT ? it.seen.beg : t0 + KT;
          const int e0 = kv_end > t0 ? kv_end : t0, e1r = (kv_end + 15) / 16 * 16, e1 = e1r < t0 + KT ? e1r : t0 + KT;
          uint32_t holes;  // units (kSlots: of my four tokens) below kv_end without a block
          bool any_hole;
          if constexpr (LOAD == kSlots) {
            holes = bad4;
            any_hole = __any_sync(0xffffffffu, bad4 != 0u);
          } else {
            const int n = (kv_end - t0 + UNIT - 1) / UNIT;
            holes = (n >= WG::UNITS ? (1u << WG::UNITS) - 1u : (1u << n) - 1u) & ~loaded;
            any_hole = holes != 0u;
          }
          if (a0 < a1 || e0 < e1 || any_hole) {
            if (!__all_sync(0xffffffffu, umma::wait(&full[st], (uint32_t)(round & 1)))) {
              ok = false;
              break;
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int c0 = (w ? e0 : a0) - t0, c1 = (w ? e1 : a1) - t0;
              if constexpr (LOAD == kPages) {
                // 8 tokens (16 bytes) of one dim's row of a page at a time
                for (int tk = c0 & ~7; tk < c1; tk += 8) {
                  const int ch = (tk % BS) / 8, lo = c0 - tk, hi = c1 - tk;
                  uint32_t keep[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    keep[i] = (2 * i < lo || 2 * i >= hi ? 0x0000ffffu : 0u) |
                              (2 * i + 1 < lo || 2 * i + 1 >= hi ? 0xffff0000u : 0u);
                  const bool whole = lo <= 0 && hi >= 8;
                  for (int d = lane; d < D; d += 32) {
                    const int phys = BS == 32 ? (ch ^ ((d >> 1) & 3)) : (BS == 16 ? (ch ^ ((d >> 2) & 1)) : 0);
                    uint4* w16 = reinterpret_cast<uint4*>(dst + (tk / BS) * PAGE + d * BS * 2 + phys * 16);
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (!whole) {
                      v = *w16;
                      v.x &= keep[0];
                      v.y &= keep[1];
                      v.z &= keep[2];
                      v.w &= keep[3];
                    }
                    *w16 = v;
                  }
                }
              } else {
                for (int i = lane; i < (c1 - c0) * (D / 8); i += 32) {
                  const int tk = c0 + i / (D / 8), ch = i % (D / 8);
                  *reinterpret_cast<uint4*>(dst + (ch >> 3) * HALF + tk * 128 + (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
              }
            }
            if constexpr (LOAD == kSlots) {
              for (; holes; holes &= holes - 1u) {
                uint8_t* row = dst + (4 * lane + __ffs(holes) - 1) * 128;
                for (int ch = 0; ch < D / 8; ++ch)
                  *reinterpret_cast<uint4*>(row + (ch >> 3) * HALF + (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
              }
            } else {
              for (; holes; holes &= holes - 1u) {
                const int u = __ffs(holes) - 1;
                if constexpr (LOAD == kPages) {
                  for (int i = lane; i < PAGE / 16; i += 32)
                    reinterpret_cast<uint4*>(dst + u * PAGE)[i] = make_uint4(0u, 0u, 0u, 0u);
                } else {
                  for (int i = lane; i < UNIT * (D / 8); i += 32)
                    reinterpret_cast<uint4*>(dst + (i / (UNIT * 8)) * HALF + u * UNIT * 128)[i % (UNIT * 8)] =
                        make_uint4(0u, 0u, 0u, 0u);
                }
              }
            }
            fence_proxy_async();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&v_ready[st]);
        }
        ++g;
        if (++st == stages) {
          st = 0;
          ++round;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) id[e] = next[e];
      }
    }
    if (!ok && lane == 0) give_up();
    // shared memory outlives every copy, after an abort too: bounded waits on the
    // last copy asked for in each stage
    if (lane == 0)
      for (int i = g > stages ? g - stages : 0; i < g; ++i) umma::wait(&full[i % stages], (uint32_t)((i / stages) & 1));
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---- products (one lane)
    if (lane == 0) {
      const uint32_t idS = umma::instr_desc(BF16, 128, KT);
      const uint32_t idO = umma::instr_desc(BF16, 128, D) | (LOAD == kPages ? 0u : 1u << 16);  // (B is MN-major)
      const uint64_t q_desc0 = umma::smem_desc(smem_u32(qsm), kUmmaRows * 16, 128, umma::kLayoutNone);
      const uint64_t k_desc0 = LOAD == kPages ? umma::smem_desc(smem_u32(kring), KT * 16, 128, umma::kLayoutNone)
                                              : umma::smem_desc(smem_u32(kring), 16, 1024, kLayoutSw128);
      const uint64_t v_desc0 =
          LOAD != kPages ? umma::smem_desc(smem_u32(vring), HALF, 1024, kLayoutSw128)
                         : (BS == 32   ? umma::smem_desc(smem_u32(vring), 16, 512, umma::kLayoutSw64)
                            : BS == 16 ? umma::smem_desc(smem_u32(vring), 16, 256, umma::kLayoutSw32)
                                       : umma::smem_desc(smem_u32(vring), PAGE, 128, umma::kLayoutNone));
      // S of tile g, then P V of tile g - 1, over the tiles of all items
      int g = 0, nq = 0;                        // tiles, items with keys so far
      int pv_left = 0, pv_j = -1;               // the tile whose P V is due: keys from its first token on, its place
      bool pv_last = false;                     // .. whether its item ends with it
      bool ok = true;
      auto issue_pv = [&]() -> bool {
        const int t = g - 1, b = t & 1, vs = t % VS;
        if (!umma::wait(&v_ready[vs], (uint32_t)((t / VS) & 1)) || !umma::wait(&v_full[vs], (uint32_t)((t / VS) & 1)))
          return false;
        const uint64_t vd = v_desc0 + (uint64_t)((vs * TILE) >> 4);
        // an item's first product overwrites both O, which every softmax warp has
        // read by the time it hands over its part of the first tile
        if (pv_j == 0 && !umma::wait(&p_full[2 * b + 1], (uint32_t)((t >> 1) & 1))) return false;
        const uint32_t vd_lo = (uint32_t)vd, vd_hi = (uint32_t)(vd >> 32);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!umma::wait(&p_full[2 * b + h], (uint32_t)((t >> 1) & 1))) return false;
          umma::fence_after();
          const int left = pv_left - h * 64;
          const bool two = BF16 && *reinterpret_cast<volatile uint32_t*>(smem_wu + WG::MISC_OFF + 8 + (2 * b + h) * 4) != 0u;
          const uint32_t pcol = tmem + WG::SCOL + b * 128 + h * 64, ocol = tmem + WG::OCOL + h * D;
          // 16 tokens of V: k-step ks of this half
          auto vlo = [&](int ks) -> uint32_t {
            const int tk = h * 64 + 16 * ks;
            return vd_lo + (uint32_t)((LOAD == kPages ? (tk / BS) * PAGE + (tk % BS) * 2 : tk * 128) >> 4);
          };
          if (left > 0) {
            if (pv_j > 0) mma_ts_lo<true>(ocol, pcol, vlo(0), vd_hi, idO);
            else mma_ts_lo<false>(ocol, pcol, vlo(0), vd_hi, idO);
          }
          if (left > 48 && !two) {
#pragma unroll
            for (int ks = 1; ks < 4; ++ks) mma_ts_lo<true>(ocol, pcol + 8 * ks, vlo(ks), vd_hi, idO);
          } else if (left > 0) {
            const int steps = left > 48 ? 4 : (left + 15) / 16;
            if (two) mma_ts_lo<true>(ocol, pcol + 32, vlo(0), vd_hi, idO);
#pragma unroll
            for (int ks = 1; ks < 4; ++ks) {
              if (ks < steps) {
                mma_ts_lo<true>(ocol, pcol + 8 * ks, vlo(ks), vd_hi, idO);
                if (two) mma_ts_lo<true>(ocol, pcol + 32 + 8 * ks, vlo(ks), vd_hi, idO);
              }
            }
          }
        }
        umma::commit(pv_done);
        umma::commit(&v_empty[vs]);
        if (pv_last) umma::commit(o_done);
        return true;
      };
      for (int k = 0; ok; ++k) {
        const int sl = k % kWinItems;
        if (abort_now() || !umma::wait(&item_full[sl], (uint32_t)((k / kWinItems) & 1))) {
          ok = false;
          break;
        }
        const int kv_end = items[sl].kv_end, ntiles = items[sl].ntiles, state = items[sl].state;
        mbar_arrive(&item_empty[sl]);
        if (state == 2) break;
        if (ntiles == 0) continue;
        const int buf = nq & 1;
        if (abort_now() || !umma::wait(&q_full[buf], (uint32_t)((nq >> 1) & 1))) {
          ok = false;
          break;
        }
        ++nq;
        const uint64_t qd = q_desc0 + (uint64_t)((buf * TILE) >> 4);
        for (int j = 0; j < ntiles; ++j) {
          const int ks0 = g % KS, b = g & 1;
          if (!umma::wait(&k_full[ks0], (uint32_t)((g / KS) & 1))) {
            ok = false;
            break;
          }
          umma::fence_after();
          const uint64_t kd = k_desc0 + (uint64_t)((ks0 * TILE) >> 4);
          const uint32_t qlo = (uint32_t)qd, qhi = (uint32_t)(qd >> 32), klo = (uint32_t)kd, khi = (uint32_t)(kd >> 32);
          mma_ss_lo<false>(tmem + WG::SCOL + b * 128, qlo, qhi, klo, khi, idS);
#pragma unroll
          for (int ks = 1; ks < D / 16; ++ks)
            mma_ss_lo<true>(tmem + WG::SCOL + b * 128, qlo + (uint32_t)((ks * 2 * kUmmaRows * 16) >> 4), qhi,
                            klo + (uint32_t)((LOAD == kPages ? ks * 2 * KT * 16 : (ks / 4) * HALF + (ks % 4) * 32) >> 4),
                            khi, idS);
          umma::commit(&s_full[b]);
          mbar_arrive(&s_full[b]);  // (release: the tile's masks, seen through k_full, are seen by whoever waits)
          umma::commit(&k_empty[ks0]);
          if (pv_j >= 0 && !issue_pv()) {
            ok = false;
            break;
          }
          ++g;
          pv_j = j;
          pv_left = kv_end - j * KT;
          pv_last = j == ntiles - 1;
        }
      }
      if (ok && pv_j >= 0) ok = issue_pv();
      if (!ok) give_up();
      umma::commit(all_done);
      umma::wait(all_done, 0);
    }
    __syncwarp();
  } else {
    // ---- softmax / epilogue.  Decisions ahead of warp-collective TMEM accesses
    // are made for the whole warp.
    auto uwait = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, umma::wait(bar, parity));
    };
    auto uabort = [&]() -> bool { return __any_sync(0xffffffffu, abort_now()); };
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    constexpr int HK = 64;      // tokens of a tile per half
    constexpr int HD = D / 2;   // output columns per half
    // (a zero scale would make 0 * inf of a hidden score: the least normal number
    // instead, whose scores round to the same exponentials)
    const float qk_scale = p.scale == 0.f ? 1.1754944e-38f : p.scale * kLog2e;
    bool ok = true;
    int gt = 0, nx = 0;  // tiles and items with keys so far
    for (int k = 0; ok; ++k) {
      WinItem it;
      if (uabort() || !take_item(k, it)) {
        ok = false;
        break;
      }
      if (it.state == 2) break;
      const int ntiles = it.ntiles;
      const bool in_tile = r < it.nrows;
      const int x0 = it.g0 + r, dt = x0 / G, row_t = it.t0 + dt, row_g = x0 - dt * G;
      const int64_t o_off = (it.q0 + row_t) * p.out_tok_stride + (int64_t)(it.kvh * G + row_g) * p.out_head_stride;
      const int end_r = in_tile && it.state == 0 ? it.prefix + row_t + 1 : 0;
      const int beg_r = end_r > p.window ? end_r - p.window : 0;
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < ntiles; ++j) {
        const int gg = gt + j, b = gg & 1;
        if (uabort() || !uwait(&s_full[b], (uint32_t)((gg >> 1) & 1))) {
          ok = false;
          break;
        }
        umma::fence_after();
        const int tile0 = j * KT, t0 = tile0 + half * HK;  // first token of my half
        const uint32_t* tm = masks + (gg & 7) * 4;
        float x[HK];
#pragma unroll
        for (int c = 0; c < HK; c += 32) {
          uint32_t v[32];
          umma::ld32(lane_base + WG::SCOL + b * 128 + half * HK + c, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c + i] = __uint_as_float(v[i]);
        }
        // bit c / UNIT of m0 (c < 32) and m1: the block of token t0 + c is loaded
        uint32_t m0, m1;
        bool all_in;
        if constexpr (LOAD == kSlots) {
          m0 = tm[2 * half];
          m1 = tm[2 * half + 1];
          all_in = (m0 & m1) == 0xffffffffu;
        } else {
          constexpr int UH = HK / UNIT;
          const uint32_t mine = (tm[0] >> (half * UH)) & ((1u << UH) - 1u);
          m0 = mine & ((1u << (UH / 2)) - 1u);
          m1 = mine >> (UH / 2);
          all_in = mine == (1u << UH) - 1u;
        }
        umma::wait_ld();
        // a half tile every row of the warp sees whole needs no per-token mask
        const bool whole = __all_sync(0xffffffffu, all_in && t0 >= beg_r && t0 + HK <= end_r);
        if (!whole) {
          // seen: tokens [beg, end) and [0, sinks) of this half, as bits
          auto below = [](int n) -> uint64_t { return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1ull); };
          uint64_t vis = below(end_r - t0) & (~below(beg_r - t0) | below(p.sinks - t0));
          if (!all_in) {
            uint64_t in = 0;
            if constexpr (LOAD == kSlots) {
              in = (uint64_t)m1 << 32 | m0;
            } else {
              constexpr int UH = HK / UNIT;
              const uint32_t mine = m0 | m1 << (UH / 2);
#pragma unroll
              for (int u = 0; u < UH; ++u) in |= (mine >> u) & 1u ? below(UNIT) << (u * UNIT % 64) : 0ull;
            }
            vis &= in;
          }
          const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
          // (a hidden score is whatever the scale takes to -inf)
          const float hidden = qk_scale >= 0.f ? -INFINITY : INFINITY;
#pragma unroll
          for (int c = 0; c < HK; ++c) x[c] = ((c < 32 ? v0 : v1) >> (c & 31)) & 1u ? x[c] : hidden;
        }
        // row max of my scaled scores (log2 units): the largest raw score, or the
        // smallest for a negative scale; four chains
        float mx;
        {
          float h[4] = {x[0], x[1], x[2], x[3]};
          if (qk_scale >= 0.f) {
#pragma unroll
            for (int c = 4; c < HK; c += 4)
#pragma unroll
              for (int e = 0; e < 4; ++e) h[e] = fmaxf(h[e], x[c + e]);
            mx = fmaxf(fmaxf(h[0], h[1]), fmaxf(h[2], h[3])) * qk_scale;
          } else {
#pragma unroll
            for (int c = 4; c < HK; c += 4)
#pragma unroll
              for (int e = 0; e < 4; ++e) h[e] = fminf(h[e], x[c + e]);
            mx = fminf(fminf(h[0], h[1]), fminf(h[2], h[3])) * qk_scale;
          }
        }
        // lazy max: rescale only when it rises by more than 2^8
        float alpha = 1.f;
        if (mx > m_ref + 8.f) {
          alpha = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - mx);
          m_ref = mx;
        }
        const float neg_ref = m_ref == -INFINITY ? 0.f : -m_ref;
        float2 ps = make_float2(0.f, 0.f);
        // P over this tile's own S, the sum before the first store (what is carried
        // depends on it: a sum of the tiles before alone, with the stores among the
        // exponentials, carries lo parts oftener, 147.6 us against 144.7 at 16 x 512
        // tokens): one rounding, or hi = the upper 16 bits of each fp32 (a bf16,
        // truncated) and lo = the exact remainder rounded to bf16.  (No wait: S's last
        // reader, P V two tiles back, completed before this S did.)
        const float2 sc = make_float2(qk_scale, qk_scale), nr = make_float2(neg_ref, neg_ref);
#pragma unroll
        for (int i = 0; i < HK / 2; ++i) {
          const float2 e = fma_x2(make_float2(x[2 * i], x[2 * i + 1]), sc, nr);  // (hidden: exp2(-inf) = 0)
          x[2 * i] = fast_exp2(e.x);
          x[2 * i + 1] = fast_exp2(e.y);
          ps = add_x2(ps, make_float2(x[2 * i], x[2 * i + 1]));
        }
        l = l * alpha + (ps.x + ps.y);
        const bool two = BF16 && __any_sync(0xffffffffu, fast_exp2(mx + neg_ref) * kSharp > l);
        const uint32_t pcol = lane_base + WG::SCOL + b * 128 + half * 64;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t hi[16], lo[16];
          if (two) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float p0 = x[32 * q + 2 * i], p1 = x[32 * q + 2 * i + 1];
              const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
              hi[i] = __byte_perm(u0, u1, 0x7632);
              const float2 rem = sub_x2(make_float2(p0, p1),
                                        make_float2(__uint_as_float(u0 & 0xFFFF0000u), __uint_as_float(u1 & 0xFFFF0000u)));
              lo[i] = MmaOp<T>::pack(rem.x, rem.y);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              hi[i] = MmaOp<T>::pack(x[32 * q + 2 * i], x[32 * q + 2 * i + 1]);
              lo[i] = 0u;
            }
          }
          umma::st16(pcol + 16 * q, hi);
          if constexpr (BF16) umma::st16(pcol + 32 + 16 * q, lo);
        }
        if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
          if (!uwait(pv_done, (uint32_t)((gg - 1) & 1))) {
            ok = false;
            break;
          }
          umma::fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t v[16];
            umma::ld16(lane_base + WG::OCOL + half * D + c, v);
            umma::wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            umma::st16(lane_base + WG::OCOL + half * D + c, v);
          }
        }
        umma::wait_st();
        umma::fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (BF16) s_lo[(2 * b + half) * 4 + (warp & 3)] = two;
          mbar_arrive(&p_full[2 * b + half]);
        }
      }
      bool have = ok && ntiles > 0;
      if (have) {
        // (a barrier of its own, once per item: the other half may be a tile behind,
        // and the parity of pv_done cannot tell the last P V from the one two back)
        have = uwait(o_done, (uint32_t)(nx & 1));
        if (!have) ok = false;
        umma::fence_after();
      }
      // the halves' (max, sum) of this row: one exchange per item (the buffer is
      // free again before any warp can be at its next item's: that item's products
      // need every warp)
      float m_o = -INFINITY, l_o = 0.f;
      if (ntiles > 0) {
        xbuf[half * 128 + r] = make_float2(m_ref, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(xchg);
        if (!uwait(xchg, (uint32_t)(nx & 1))) ok = false;
        ++nx;
        const float2 o = xbuf[(half ^ 1) * 128 + r];
        m_o = o.x;
        l_o = o.y;
      }
      have = have && ok;
      const float M = fmaxf(m_ref, m_o);
      const float w_me = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - M);
      const float w_o = m_o == -INFINITY ? 0.f : fast_exp2(m_o - M);
      const float total = w_me * l + w_o * l_o;
      // a row with no visible key (or after an abort) is 0; a half without any has
      // an O that nothing has written, and takes no part (unless the total is NaN,
      // from a score that is NaN or +inf, which makes the row NaN)
      const bool nonzero = have && total != 0.f;
      const float inv = nonzero ? 1.f / total : 0.f;
      const float f0 = (half == 0 ? w_me : w_o) * inv, f1 = (half == 0 ? w_o : w_me) * inv;
      const bool u0 = nonzero && f0 != 0.f, u1 = nonzero && f1 != 0.f;
      if (ntiles > 0) {
        // through the item's Q buffer (S is done with it) to whole 128- or 64-byte
        // pieces of rows: 16-byte chunk c of row r at c ^ (r & 7), this warp's rows
        // and half of the columns only
        constexpr int RB = D * 2, CPR = HD / 8;  // bytes of a row, chunks of my half of it
        uint8_t* ob = qsm + ((nx - 1) & 1) * TILE;
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t v[32], w[32];
          umma::ld32(lane_base + WG::OCOL + half * HD + c, v);
          umma::ld32(lane_base + WG::OCOL + D + half * HD + c, w);
          umma::wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t packed[4];
#pragma unroll
            for (int k2 = 0; k2 < 4; ++k2) {
              float y[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float o0 = u0 ? __uint_as_float(v[i + 2 * k2 + e]) * f0 : 0.f;
                y[e] = u1 ? fmaf(__uint_as_float(w[i + 2 * k2 + e]), f1, o0) : o0;
              }
              packed[k2] = pack_out<T>(y[0], y[1]);
            }
            const int ch = half * CPR + (c + i) / 8;
            *reinterpret_cast<uint4*>(ob + r * RB + ((ch & ~7) | ((ch ^ r) & 7)) * 16) =
                make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
        }
        umma::fence_before();
        __syncwarp();
        // lane -> chunk lane % CPR of row (lane / CPR) + 32 / CPR * i of my warp's 32
        const int ch = half * CPR + lane % CPR;
#pragma unroll
        for (int i = 0; i < CPR; ++i) {
          const int from = lane / CPR + (32 / CPR) * i, rr = (warp & 3) * 32 + from;
          const int64_t off = __shfl_sync(0xffffffffu, o_off, from);  // (that row's own thread knows where it goes)
          if (rr < it.nrows)
            store_row16<OUT16>(reinterpret_cast<T*>(p.out) + off + ch * 8,
                               *reinterpret_cast<const uint4*>(ob + rr * RB + ((ch & ~7) | ((ch ^ rr) & 7)) * 16));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_empty[(nx - 1) & 1]);
      } else if (in_tile) {  // (bad indices: zeros)
        T* orow = reinterpret_cast<T*>(p.out) + o_off + half * HD;
#pragma unroll
        for (int c = 0; c < HD; c += 8) store_row16<OUT16>(orow + c, make_uint4(0u, 0u, 0u, 0u));
      }
      gt += ntiles;
    }
    if (!ok && lane == 0) give_up();
  }

  umma::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    umma::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (dynamic && threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(&g_umma_sched[slot].done, 1u) == gridDim.x - 1) {
      atomicExch(&g_umma_sched[slot].next, 0u);
      atomicExch(&g_umma_sched[slot].done, 0u);
    }
  }
}

}  // namespace kvc
