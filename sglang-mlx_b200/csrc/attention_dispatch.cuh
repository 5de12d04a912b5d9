// attention_dispatch.cuh — which tensor-core kernel serves a decode, prefill or
// shared-prefix call (included by decode.cu after the kernels).
#pragma once

namespace kvc {

static bool mma_disabled_by_env() {
  const char* v = getenv("KVC_DECODE_KERNEL");
  return v && (v[0] == 'g' || v[0] == 'G');  // "generic"
}

static bool mma_supported(const DecodeArgs& a) {
  if (a.cache_type == ElemType::U8) {  // one-byte caches have no other kernel
    const int G = a.num_heads / a.num_kv_heads;
    return (a.q_type == ElemType::F16 || a.q_type == ElemType::BF16) && (a.head_size == 64 || a.head_size == 128) &&
           (a.block_size == 8 || a.block_size == 16 || a.block_size == 32) && G >= 1 && G <= 16 && !a.flash &&
           (a.num_partitions == 1 || a.partition_size % 32 == 0) && (reinterpret_cast<uintptr_t>(a.q) & 3u) == 0 &&
           (a.q_seq_stride & 1) == 0 && (a.q_head_stride & 1) == 0;
  }
  if (mma_disabled_by_env()) return false;
  if (a.q_type != a.cache_type) return false;
  if (a.q_type != ElemType::F16 && a.q_type != ElemType::BF16) return false;
  if (!(a.head_size == 64 || a.head_size == 128)) return false;
  if (!a.flash && a.block_size != 8 && a.block_size != 16 && a.block_size != 32) return false;
  const int G = a.num_heads / a.num_kv_heads;
  if (G < 1 || G > 16) return false;
  if (a.num_partitions > 1 && a.partition_size % 32 != 0) return false;
  if (a.flash) return (reinterpret_cast<uintptr_t>(a.q) & 3u) == 0 && (a.q_seq_stride & 1) == 0 &&
                      (a.q_head_stride & 1) == 0;
  // q rows are read as 4-byte pairs
  if ((reinterpret_cast<uintptr_t>(a.q) & 3u) || (a.q_seq_stride & 1) || (a.q_head_stride & 1)) return false;
  return true;
}

// Variant id = warps * 1000 + stages * 100 + group tokens, + 100000 for tiled
// tensor copies ("<warps>x<stages>x<group>t"), + 200000 for bulk K with the
// swizzled whole-page V ("<warps>x<stages>x<group>s").
static int mma_variant() {
  const char* v = getenv("KVC_MMA_CONFIG");
  if (!v) return 0;
  int w = 0, s = 0, g = 32;
  char t = 0;
  const int n = sscanf(v, "%dx%dx%d%c", &w, &s, &g, &t);
  if (n < 2) return 0;
  return (t == 't' ? 100000 : (t == 's' ? 200000 : 0)) + w * 1000 + s * 100 + g;
}

template <typename T, int D, int BS>
static cudaError_t launch_mma_typed(const DecodeParams& p, cudaStream_t stream) {
  const int v = mma_variant();
  const int g = v % 100;
  const bool part_ok = p.num_partitions == 1 || (g > 0 && p.partition_size % g == 0);
  if (D == 128 && v && part_ok) {
    cudaError_t e = cudaErrorNotSupported;
    switch (v) {
      case 2332: e = launch_mma_nw<T, D, BS, 2, 3, 32>(p, stream); break;
      case 2232: e = launch_mma_nw<T, D, BS, 2, 2, 32>(p, stream); break;
      case 4316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 4, 3, 16>(p, stream); break;
      case 1316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 1, 3, 16>(p, stream); break;
      case 1416: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 1, 4, 16>(p, stream); break;
      case 2316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 2, 3, 16>(p, stream); break;
      case 6216: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 6, 2, 16>(p, stream); break;
      case 8216: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 8, 2, 16>(p, stream); break;
      case 6316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 6, 3, 16>(p, stream); break;
      case 8316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 8, 3, 16>(p, stream); break;
      case 10216: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 10, 2, 16>(p, stream); break;
      case 12216: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 12, 2, 16>(p, stream); break;
      case 104316: e = launch_mma_nw<T, D, BS, 4, 3, 16, kTiles>(p, stream); break;
      case 102232: e = launch_mma_nw<T, D, BS, 2, 2, 32, kTiles>(p, stream); break;
      case 204316: if constexpr (BS <= 16) e = launch_mma_nw<T, D, BS, 4, 3, 16, kSwizzledV>(p, stream); break;
      case 202232: e = launch_mma_nw<T, D, BS, 2, 2, 32, kSwizzledV>(p, stream); break;
      case 203232: e = launch_mma_nw<T, D, BS, 3, 2, 32, kSwizzledV>(p, stream); break;
      case 202332: e = launch_mma_nw<T, D, BS, 2, 3, 32, kSwizzledV>(p, stream); break;
      default: break;
    }
    if (e != cudaErrorNotSupported) return e;
  }
  // The tail partitions of a shared-prefix decode (short, at most 256 tokens):
  // 2 warps x 3 stages, so each warp streams more of its partition before the
  // CTA's merge (config 4: 57.8 us against 62.2 us with 4 warps).
  if constexpr (BS <= 16) {
    if (p.part_offset > 0 && p.partition_size <= 256 && p.partition_size % 16 == 0)
      return launch_mma_nw<T, D, BS, 2, 3, 16>(p, stream);
  }
  // Defaults from sweeps on B200: 16-token groups, 4 warps x 3 stages (96 KB,
  // two CTAs and 8 warps per SM; 6 x 2 at D = 128, below) with whole-page 1-D bulk copies where the
  // block size allows (98% of copy bandwidth on config 2, against 81% for
  // 32-token groups).  32-token blocks: 32-token groups, 2 warps x 2 stages
  // (64 KB, three CTAs per SM), K by bulk copy and V through the 128-byte
  // swizzled tensor map (config 3: 77.7% against 73.9% with the 4-way bank
  // conflicts of unswizzled 64-byte V rows; config 5: 91% against 89%).
  // Tiled 16-token boxes of 32-token pages measured slower: such a box is
  // hundreds of 16-32 byte rows.  If no tensor map can be encoded for the
  // cache, plain bulk copies are used.
  if constexpr (BS <= 16) {
    // One rank's share of a head-sharded batch: a planned decode with at most
    // two (sequence, KV head) pairs per SM whose partitions hold whole
    // sequences runs on 10 warps x 2 stages (160 KB, one CTA per SM), so the
    // longest sequences, which end the launch, stream on more warps (256
    // sequences of U[512, 4096] tokens, one KV head: 1.71 ms per 32-layer step
    // against 1.89 with 4 warps and 2048-token partitions; 8 warps 1.74, 12
    // warps 1.71; with more pairs per SM the 4-warp CTAs are faster).
    if (D == 128 && p.plan_items && p.part_offset == 0 && p.partition_size >= 4096 && p.partition_size % 16 == 0 &&
        p.max_seq_len <= p.partition_size + 2 * BS &&
        (int64_t)p.num_seqs * p.num_kv_heads <= 2 * (int64_t)decode_sm_count())
      return launch_mma_nw<T, D, BS, 10, 2, 16>(p, stream);
    // Otherwise, at D = 128, 6 warps x 2 stages (96 KB, two CTAs and 12 warps
    // per SM).  Config 2 per 32-layer step against 4 warps x 3 stages: planned
    // at 2 / 4 / 8 KV heads per GPU 3.02 / 6.15 / 12.06 ms against 3.12 / 6.33 /
    // 12.62; single pass (v1) 12.22 against 13.11; split-K (v2) 15.29 against
    // 15.61.
    if (p.num_partitions == 1 || p.partition_size % 16 == 0) {
      if constexpr (D == 128) return launch_mma_nw<T, D, BS, 6, 2, 16>(p, stream);
      return launch_mma_nw<T, D, BS, 4, 3, 16>(p, stream);
    }
  } else {
    cudaError_t e = launch_mma_nw<T, D, BS, 2, 2, 32, kSwizzledV>(p, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  return launch_mma_nw<T, D, BS, 2, 2, 32>(p, stream);
}

// One-byte caches: 16-token groups, 4 warps x 4 stages of 4 KB (three CTAs per
// SM) for blocks of up to 16 tokens; 32-token groups, 4 warps x 3 stages of
// 8 KB for 32-token blocks.
template <typename T, int D, int MODE>
static cudaError_t launch_mma_fp8(const DecodeParams& p, int block_size, cudaStream_t stream) {
  if (block_size == 8) return launch_mma_nw<T, D, 8, 4, 4, 16, MODE>(p, stream);
  if (block_size == 16) return launch_mma_nw<T, D, 16, 4, 4, 16, MODE>(p, stream);
  return launch_mma_nw<T, D, 32, 4, 3, 32, MODE>(p, stream);
}

template <typename T>
static cudaError_t launch_mma_t(const DecodeParams& p, const DecodeArgs& a, cudaStream_t stream) {
  if (a.cache_type == ElemType::U8) {
    const bool e5m2 = a.fp8_format == 1 || a.fp8_format == 3;  // the -sat formats decode alike
    if (a.head_size == 128)
      return e5m2 ? launch_mma_fp8<T, 128, kFp8E5M2>(p, a.block_size, stream)
                  : launch_mma_fp8<T, 128, kFp8E4M3>(p, a.block_size, stream);
    return e5m2 ? launch_mma_fp8<T, 64, kFp8E5M2>(p, a.block_size, stream)
                : launch_mma_fp8<T, 64, kFp8E4M3>(p, a.block_size, stream);
  }
  if (a.flash) {
    // token-major caches: 16-token groups, 6 warps x 2 stages for D = 128 and
    // 4 warps x 3 stages for D = 64 (two CTAs per SM); the block size is read
    // at run time.
    // KVC_FLASH_COPY=bulk selects per-row bulk copies (tuning runs).
    // KVC_FLASH_COPY=cpasync keeps the per-lane row copies where tensor copies apply (tuning runs).
    // KVC_FLASH_COPY=gather reads dense rows in any order by tensor gathers (below).
    const char* fc = getenv("KVC_FLASH_COPY");
    if (fc && fc[0] == 'b') {
      if (a.head_size == 128) return launch_mma_nw<T, 128, 16, 4, 3, 16, kFlashBulk>(p, stream);
      return launch_mma_nw<T, 64, 16, 4, 3, 16, kFlashBulk>(p, stream);
    }
    // blocks of 16k consecutive token rows: a tensor copy per (16-token group, head, 64 dims)
    const bool rows_ok = a.block_size % 16 == 0 && a.k_block_stride == (int64_t)a.block_size * a.k_tok_stride &&
                         a.v_block_stride == (int64_t)a.block_size * a.v_tok_stride &&
                         a.num_blocks * (int64_t)a.block_size < (int64_t)1 << 31 && !(fc && fc[0] == 'c');
    // D = 128: 6 warps x 2 stages (two CTAs and 12 warps per SM; config 2 on
    // the pool: page tables 12.67 against 13.54 ms per step with 4 x 3, slot
    // lists 15.67 against 16.66)
    const bool six = a.head_size == 128;
    if (rows_ok) {
      cudaError_t e = six ? launch_mma_nw<T, 128, 16, 6, 2, 16, kFlashTma>(p, stream)
                    : a.head_size == 128 ? launch_mma_nw<T, 128, 16, 4, 3, 16, kFlashTma>(p, stream)
                                         : launch_mma_nw<T, 64, 16, 4, 3, 16, kFlashTma>(p, stream);
      if (e != cudaErrorNotSupported) return e;
    }
    // KVC_FLASH_COPY=gather: dense token rows in any order (the pool's slot
    // lists) by 4-row tensor gathers.  Not the default: on config 2's slot-list
    // pool they measured 0.661 of the copy peak against 0.708 for the per-lane
    // row copies (16 gather requests per 16-token group and head, against 4
    // tensor copies for blocks of consecutive rows).
    // (block size 1, the pool's [slots, H, D]: a block is one row and carries no token stride)
    const int64_t D = a.head_size, H = a.num_kv_heads, rbs = a.block_size;
    const int64_t ktok = rbs == 1 ? H * D : a.k_tok_stride, vtok = rbs == 1 ? H * D : a.v_tok_stride;
    const bool dense = a.k_head_stride == D && ktok == H * D && a.k_block_stride == rbs * H * D &&
                       a.v_head_stride == D && vtok == H * D && a.v_block_stride == rbs * H * D &&
                       a.num_blocks * rbs * H < (int64_t)1 << 31 && fc && fc[0] == 'g';
    if (dense) {
      cudaError_t e = a.head_size == 128 ? launch_mma_nw<T, 128, 16, 4, 3, 16, kFlashGather>(p, stream)
                                         : launch_mma_nw<T, 64, 16, 4, 3, 16, kFlashGather>(p, stream);
      if (e != cudaErrorNotSupported) return e;
    }
    if (six) return launch_mma_nw<T, 128, 16, 6, 2, 16, kFlash>(p, stream);
    if (a.head_size == 128) return launch_mma_nw<T, 128, 16, 4, 3, 16, kFlash>(p, stream);
    return launch_mma_nw<T, 64, 16, 4, 3, 16, kFlash>(p, stream);
  }
  if (a.head_size == 128) {
    if (a.block_size == 8) return launch_mma_typed<T, 128, 8>(p, stream);
    if (a.block_size == 16) return launch_mma_typed<T, 128, 16>(p, stream);
    return launch_mma_typed<T, 128, 32>(p, stream);
  }
  if (a.block_size == 8) return launch_mma_typed<T, 64, 8>(p, stream);
  if (a.block_size == 16) return launch_mma_typed<T, 64, 16>(p, stream);
  return launch_mma_typed<T, 64, 32>(p, stream);
}

static cudaError_t launch_mma(const DecodeParams& p, const DecodeArgs& a, cudaStream_t stream) {
  if (a.q_type == ElemType::BF16) return launch_mma_t<__nv_bfloat16>(p, a, stream);
  return launch_mma_t<__half>(p, a, stream);
}

// The mma.sync kernel: every layout, head size 64 / 128.
static cudaError_t launch_prefill_mma_any(const PrefillArgs& a, cudaStream_t stream) {
  if (a.head_size == 128)
    return a.q_type == ElemType::BF16 ? launch_prefill_layout<__nv_bfloat16, 128>(a, a.token_major, stream)
                                      : launch_prefill_layout<__half, 128>(a, a.token_major, stream);
  if (a.head_size == 64)
    return a.q_type == ElemType::BF16 ? launch_prefill_layout<__nv_bfloat16, 64>(a, a.token_major, stream)
                                      : launch_prefill_layout<__half, 64>(a, a.token_major, stream);
  return cudaErrorNotSupported;
}

// K viewed as rows of one 8-dim chunk of one page of one head: [nb * H * D/8][BS * 8]
// (needs the dense paged layout).
static bool make_k_gather_map(const PrefillArgs& a, int D, int BS, CUtensorMap* map) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)BS * 8, (cuuint64_t)a.num_blocks * a.num_kv_heads * (D / 8)};
  const cuuint64_t strides[1] = {(cuuint64_t)BS * 16};
  const cuuint32_t box[2] = {(cuuint32_t)BS * 8, 1};
  const cuuint32_t ones[2] = {1, 1};
  return enc(map, a.q_type == ElemType::BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(a.k_cache), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// KVC_PREFILL_ISSUE=single: the producer's lane 0 issues every copy (tuning runs).
static int umma_single_issue() {
  const char* v = getenv("KVC_PREFILL_ISSUE");
  return v && v[0] == 's' ? 1 : 0;
}

template <typename T, int D, int BS, bool GK>
static cudaError_t launch_prefill_umma(const PrefillArgs& a, cudaStream_t stream) {
  using UG = UmmaGeom<D, BS>;
  DecodeParams dp;
  memset(&dp, 0, sizeof(dp));
  dp.k_cache = a.k_cache;
  dp.v_cache = a.v_cache;
  dp.num_blocks = a.num_blocks;
  dp.num_kv_heads = a.num_kv_heads;
  dp.k_head_stride = a.k_head_stride;
  dp.k_block_stride = a.k_block_stride;
  dp.v_head_stride = a.v_head_stride;
  dp.v_block_stride = a.v_block_stride;
  TmaMaps maps;
  memset(&maps, 0, sizeof(maps));
  // the kTiles maps: V as [nb][H][D][BS] pages, one whole page per box, bs*2-byte swizzle
  if (!make_tensor_maps(dp, std::is_same<T, __nv_bfloat16>::value ? ElemType::BF16 : ElemType::F16, D, BS, BS, BS * 2,
                        kTiles, &maps))
    return cudaErrorNotSupported;
  if (GK && !make_k_gather_map(a, D, BS, &maps.k)) return cudaErrorNotSupported;
  if constexpr (GK) {
    if (pair_enabled()) {
      const int G2 = a.num_heads / a.num_kv_heads;
      const int64_t tiles2 = ((int64_t)a.max_q_len * G2 + kUmmaRows - 1) / kUmmaRows;
      if (tiles2 <= 0 || a.num_seqs <= 0) return cudaSuccess;
      const cudaError_t e = launch_pair<T, D, BS, false>(a, maps, tiles2, (int)a.num_seqs, stream);
      if (e != cudaErrorNotSupported) return e;
    }
  }
  auto kern = prefill_umma_kernel<T, D, BS, GK>;
  static std::atomic<bool> configured[64];  // per device; setting the attribute twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, UG::SMEM);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int G = a.num_heads / a.num_kv_heads;
  const int64_t tiles = ((int64_t)a.max_q_len * G + kUmmaRows - 1) / kUmmaRows;
  if (tiles <= 0 || a.num_seqs <= 0) return cudaSuccess;
  const int64_t items = tiles * a.num_seqs * a.num_kv_heads;
  if (items > 0x7fffffffll - 1024) return cudaErrorInvalidValue;
  const int ctas = umma_persistent_ctas(dev, items);
  const int slot = umma_sched_slot(stream);  // (runtime queries stay outside the launch statement)
  PrefillArgs aa = a;
  aa.single_issue = umma_single_issue();
  kern<<<ctas, kUmmaThreads, UG::SMEM, stream>>>(aa, maps, (int)tiles, (int)a.num_seqs, slot);
  count_launch();
  return cudaGetLastError();
}

// The tcgen05 kernel serves the paged layout with block size 16 or 32 (pages
// tile a 128-token S tile; V rows of 32 or 64 bytes match a swizzle mode).
static bool prefill_umma_supported(const PrefillArgs& a) {
  if (a.token_major || !(a.block_size == 16 || a.block_size == 32) || !(a.head_size == 64 || a.head_size == 128))
    return false;
  // rows are stored as 16-byte vectors
  if ((reinterpret_cast<uintptr_t>(a.out) & 15u) || (a.out_tok_stride & 7) || (a.out_head_stride & 7)) return false;
  const char* v = getenv("KVC_PREFILL_KERNEL");
  return !(v && (v[0] == 'm' || v[0] == 'M'));  // "mma": the mma.sync kernel
}

static cudaError_t launch_prefill_umma_any(const PrefillArgs& a, cudaStream_t stream) {
  const bool bf = a.q_type == ElemType::BF16;
  const int64_t D = a.head_size, BS = a.block_size;
  // the 4-row gathers need K rows uniformly strided: the dense paged layout
  const bool dense = a.k_head_stride == D * BS && a.k_block_stride == (int64_t)a.num_kv_heads * D * BS &&
                     a.num_blocks * a.num_kv_heads * (D / 8) < 0x7fffffffll;  // (row indices are 32-bit)
  if (a.head_size == 128) {
    if (a.block_size == 32) {
      if (dense)
        return bf ? launch_prefill_umma<__nv_bfloat16, 128, 32, true>(a, stream)
                  : launch_prefill_umma<__half, 128, 32, true>(a, stream);
      return bf ? launch_prefill_umma<__nv_bfloat16, 128, 32, false>(a, stream)
                : launch_prefill_umma<__half, 128, 32, false>(a, stream);
    }
    if (dense)
      return bf ? launch_prefill_umma<__nv_bfloat16, 128, 16, true>(a, stream)
                : launch_prefill_umma<__half, 128, 16, true>(a, stream);
    return bf ? launch_prefill_umma<__nv_bfloat16, 128, 16, false>(a, stream)
              : launch_prefill_umma<__half, 128, 16, false>(a, stream);
  }
  if (a.block_size == 32) {
    if (dense)
      return bf ? launch_prefill_umma<__nv_bfloat16, 64, 32, true>(a, stream)
                : launch_prefill_umma<__half, 64, 32, true>(a, stream);
    return bf ? launch_prefill_umma<__nv_bfloat16, 64, 32, false>(a, stream)
              : launch_prefill_umma<__half, 64, 32, false>(a, stream);
  }
  if (dense)
    return bf ? launch_prefill_umma<__nv_bfloat16, 64, 16, true>(a, stream)
              : launch_prefill_umma<__half, 64, 16, true>(a, stream);
  return bf ? launch_prefill_umma<__nv_bfloat16, 64, 16, false>(a, stream)
            : launch_prefill_umma<__half, 64, 16, false>(a, stream);
}

// ---- shared-prefix (cascade) decode through the tcgen05 kernel ----
template <typename T, int D, int BS, bool GK>
static cudaError_t launch_cascade_umma(const PrefillArgs& a, int prefix_parts, cudaStream_t stream) {
  using UG = UmmaGeom<D, BS>;
  DecodeParams dp;
  memset(&dp, 0, sizeof(dp));
  dp.k_cache = a.k_cache;
  dp.v_cache = a.v_cache;
  dp.num_blocks = a.num_blocks;
  dp.num_kv_heads = a.num_kv_heads;
  dp.k_head_stride = a.k_head_stride;
  dp.k_block_stride = a.k_block_stride;
  dp.v_head_stride = a.v_head_stride;
  dp.v_block_stride = a.v_block_stride;
  TmaMaps maps;
  memset(&maps, 0, sizeof(maps));
  if (!make_tensor_maps(dp, std::is_same<T, __nv_bfloat16>::value ? ElemType::BF16 : ElemType::F16, D, BS, BS, BS * 2,
                        kTiles, &maps))
    return cudaErrorNotSupported;
  if (GK && !make_k_gather_map(a, D, BS, &maps.k)) return cudaErrorNotSupported;
  if constexpr (GK) {
    if (pair_enabled()) {
      const int G2 = a.num_heads / a.num_kv_heads;
      const cudaError_t e = launch_pair<T, D, BS, true>(
          a, maps, ((int64_t)a.num_seqs * G2 + kUmmaRows - 1) / kUmmaRows, prefix_parts, stream);
      if (e != cudaErrorNotSupported) return e;
    }
  }
  auto kern = prefill_umma_kernel<T, D, BS, GK, true>;
  static std::atomic<bool> configured[64];  // per device; setting the attribute twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, UG::SMEM);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  const int G = a.num_heads / a.num_kv_heads;
  const int64_t tiles = ((int64_t)a.num_seqs * G + kUmmaRows - 1) / kUmmaRows;
  const int64_t items = tiles * prefix_parts * a.num_kv_heads;
  if (items <= 0) return cudaSuccess;
  if (items > 0x7fffffffll - 1024) return cudaErrorInvalidValue;
  const int ctas = umma_persistent_ctas(dev, items);
  const int slot = umma_sched_slot(stream);
  PrefillArgs aa = a;
  aa.single_issue = umma_single_issue();
  // a programmatic dependent of the kernel before it (see the kernel's start)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kUmmaThreads);
  cfg.dynamicSmemBytes = UG::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, aa, maps, (int)tiles, prefix_parts, slot);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

// The prefix of a shared-prefix decode on the tensor cores' own pipeline when
// the cache suits the gathered-K tcgen05 kernel (dense paged layout, block size
// 16 or 32, head size 64 / 128, prefix and chunks in whole blocks, partial
// buffers of 16-byte rows);
// cudaErrorNotSupported otherwise (the caller then runs the mma.sync prefix
// kernel).
static cudaError_t launch_cascade_prefix_umma(const DecodeParams& p, const DecodeArgs& da, cudaStream_t stream) {
  const int D = da.head_size, BS = da.block_size;
  // Only the gathered-K form (dense K): with per-page S chains (N = 16 for
  // block size 16, 64 products per tile) the single-lane product issue set the
  // pace and config 4 measured 69.0 us against 65.9 us for the mma.sync prefix
  // kernel.
  if (!(BS == 16 || BS == 32) || !(D == 64 || D == 128)) return cudaErrorNotSupported;
  if (!(p.k_head_stride == (int64_t)D * BS && p.k_block_stride == (int64_t)p.num_kv_heads * D * BS))
    return cudaErrorNotSupported;
  if ((reinterpret_cast<uintptr_t>(p.part_out) & 15u) || (p.part_out_seq_stride & 3) || (p.part_out_head_stride & 3) ||
      (p.part_out_part_stride & 3) || (p.prefix_len % BS) || (p.prefix_part_size % BS))
    return cudaErrorNotSupported;
  const char* v = getenv("KVC_PREFILL_KERNEL");
  if (v && (v[0] == 'm' || v[0] == 'M')) return cudaErrorNotSupported;
  PrefillArgs a;
  memset(&a, 0, sizeof(a));
  a.q = p.q;
  a.k_cache = p.k_cache;
  a.v_cache = p.v_cache;
  a.block_tables = p.block_tables;
  a.num_seqs = p.num_seqs;
  a.num_heads = p.num_heads;
  a.num_kv_heads = p.num_kv_heads;
  a.block_size = BS;
  a.num_blocks = p.num_blocks;
  a.table_stride = p.table_stride;
  a.q_tok_stride = p.q_seq_stride;
  a.q_head_stride = p.q_head_stride;
  a.k_block_stride = p.k_block_stride;
  a.k_head_stride = p.k_head_stride;
  a.v_block_stride = p.v_block_stride;
  a.v_head_stride = p.v_head_stride;
  a.scale = p.scale;
  a.q_type = da.q_type;
  a.head_size = D;
  a.context_lens = p.context_lens;
  a.max_seq_len = p.max_seq_len;
  a.prefix_len = p.prefix_len;
  a.prefix_part_size = p.prefix_part_size;
  a.part_max = p.part_max;
  a.part_sum = p.part_sum;
  a.part_out = p.part_out;
  a.part_seq_stride = p.part_seq_stride;
  a.part_head_stride = p.part_head_stride;
  a.part_out_seq_stride = p.part_out_seq_stride;
  a.part_out_head_stride = p.part_out_head_stride;
  a.part_out_part_stride = p.part_out_part_stride;
  const bool bf = a.q_type == ElemType::BF16;
  const bool dense = a.k_head_stride == (int64_t)D * BS && a.k_block_stride == (int64_t)a.num_kv_heads * D * BS &&
                     a.num_blocks * a.num_kv_heads * (D / 8) < 0x7fffffffll;
  const int parts = p.prefix_parts;
  if (!dense) return cudaErrorNotSupported;
  if (D == 128)
    return BS == 32 ? (bf ? launch_cascade_umma<__nv_bfloat16, 128, 32, true>(a, parts, stream)
                          : launch_cascade_umma<__half, 128, 32, true>(a, parts, stream))
                    : (bf ? launch_cascade_umma<__nv_bfloat16, 128, 16, true>(a, parts, stream)
                          : launch_cascade_umma<__half, 128, 16, true>(a, parts, stream));
  return BS == 32 ? (bf ? launch_cascade_umma<__nv_bfloat16, 64, 32, true>(a, parts, stream)
                        : launch_cascade_umma<__half, 64, 32, true>(a, parts, stream))
                  : (bf ? launch_cascade_umma<__nv_bfloat16, 64, 16, true>(a, parts, stream)
                        : launch_cascade_umma<__half, 64, 16, true>(a, parts, stream));
}

cudaError_t launch_paged_prefill(const PrefillArgs& a, cudaStream_t stream) {
  if (a.num_seqs <= 0 || a.max_q_len <= 0) return cudaSuccess;
  if (a.num_seqs > 65535 || a.num_kv_heads > 65535) return cudaErrorInvalidValue;
  if (prefill_umma_supported(a)) return launch_prefill_umma_any(a, stream);
  return launch_prefill_mma_any(a, stream);
}

}  // namespace kvc
