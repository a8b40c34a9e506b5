// Grouped GEMM by expert on MXFP4 operands: block-scaled tcgen05 MMAs
// (kind::mxf4, K = 64, one e8m0 scale per 32), fp32 accumulation in TMEM.
//   plain:   out[rows of g] = x[rows of g] @ w[g]^T               -> bf16
//   SwiGLU:  h = silu(x @ gate^T) * (x @ up^T), in fp32           -> bf16 or
//            MXFP4 records (the next product's input; h never exists in bf16)
//
// One persistent CTA per SM, 128-row tiles.  A k-block is 256 elements: a
// 128-byte swizzled row of codes per operand row.  Warp 0 loads A (row
// records through a tensor map whose row stride is the record), B and B's
// scale atoms; warps 2-3 bring A's scales (row-major in the records, 8 bytes
// per row and k-block) into the atom layout; warp 1 copies the atoms to TMEM
// and issues the MMAs; eight warps run the epilogue.  Each stage has its own
// TMEM scale columns, so a stage's empty barrier covers its scales as well.
#include "gemm_mxfp4.cuh"

namespace hmoe {
namespace mx {
namespace {

constexpr int kThreads = 384;  // 4 control warps, 8 epilogue warps
constexpr int kAccs = 2;

template <int BN>
struct Tile {
  static constexpr int kStages = 5;
  static constexpr int kNB = (BN + 127) / 128;  // scale chunks of B
  static constexpr int kABytes = MM * kRowB;
  static constexpr int kBBytes = BN * kRowB;
  static constexpr int kSfA = 2 * kAtom;
  static constexpr int kSfB = 2 * kAtom * kNB;
  static constexpr int kStageBytes = kABytes + kBBytes + kSfA + kSfB;
  static constexpr int kSfCols = 8 + 8 * kNB;  // TMEM scale columns of a stage
  static constexpr int kSfBase = kAccs * BN;
  static_assert(kSfBase + kStages * kSfCols <= kTmemCols, "TMEM columns");
};

template <int STAGES>
struct Ctl {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t acc_full[kAccs];
  uint64_t acc_empty[kAccs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  GroupTables tab;
};

template <int BN>
constexpr size_t smem_bytes() {
  return 1024 + static_cast<size_t>(Tile<BN>::kStages) * Tile<BN>::kStageBytes +
         8 * kEpiBox + sizeof(Ctl<Tile<BN>::kStages>);
}
static_assert(smem_bytes<128>() <= 232448, "shared memory budget of one sm_100 CTA");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
struct TilePos : RowBlock {
  int n;
};
__device__ __forceinline__ TilePos decode_tile(const GroupTables& tab, int G, int n_tiles, int tile) {
  const int mt = tile / n_tiles;
  TilePos t;
  static_cast<RowBlock&>(t) = find_block(tab, G, mt, MM);
  t.n = tile - mt * n_tiles;
  return t;
}

template <int BN, bool SWIGLU, bool QOUT>
__global__ void __launch_bounds__(kThreads, 1)
grouped_gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA,
                          const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const Params p) {
  using T = Tile<BN>;
  constexpr int ST = T::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  auto& ctl = *reinterpret_cast<Ctl<ST>*>(smem + ST * T::kStageBytes + 8 * kEpiBox);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.G;

  // ---------------------------------------------------------------- setup
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < ST; ++s) {
        mbar_init(smem_u32(&ctl.full[s]), 3);   // the producer's arm, two scale warps
        mbar_init(smem_u32(&ctl.empty[s]), 1);  // one commit per stage use
      }
      for (int a = 0; a < kAccs; ++a) {
        mbar_init(smem_u32(&ctl.acc_full[a]), 1);
        mbar_init(smem_u32(&ctl.acc_empty[a]), 8);  // the epilogue warps
      }
      mbar_init(smem_u32(&ctl.drain), 1);
      ctl.abort = 0;
      fence_mbar_init();
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmC);
    }
    __syncwarp();
    grid_dependency_wait();  // launched early (launch_pdl): the counts are written before this
    build_tables(ctl.tab, p.counts, G, p.M, MM);
  } else if (warp == 1) {
    tmem_alloc(smem_u32(&ctl.tmem_base), kTmemCols);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();

  const uint32_t tmem_base = ctl.tmem_base;
  const int num_tiles = ctl.tab.num_m_tiles * p.n_tiles;
  const int kp = mx_padded_k(p.K);
  const int nkb = cdiv(kp, kMxKBlock);
  volatile int* abort = &ctl.abort;
  int never = 0;
  const unsigned long long lim = p.wait_limit_ns;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const TilePos t = decode_tile(ctl.tab, G, p.n_tiles, tile);
        const int boxes = cdiv(min(MM, t.row_end - t.row0), p.a_box_rows);
        const int brow = t.g * p.b_rows + t.n * BN;
        const int nchunks = min(T::kNB, p.b_chunks - t.n * BN / 128);
        const uint8_t* bs = p.b_scales +
                            (static_cast<int64_t>(t.g) * p.b_chunks + t.n * BN / 128) * nkb * 1024;
        const uint32_t bytes = boxes * p.a_box_rows * kRowB + T::kBBytes + nchunks * 1024;
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait_bounded(smem_u32(&ctl.empty[stage]), phase ^ 1u, abort, p.err, lim)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&ctl.full[stage]);
          const uint32_t sa = sbase + stage * T::kStageBytes;
          mbar_arrive_expect_tx(fb, bytes);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(sa + b * p.a_box_rows * kRowB, &tmA, kb * kRowB,
                        t.row0 + b * p.a_box_rows, fb);
          tma_load_2d(sa + T::kABytes, &tmB, kb * kRowB, brow, fb);
          for (int c = 0; c < nchunks; ++c)
            bulk_load(sa + T::kABytes + T::kBBytes + T::kSfA + c * 1024,
                      bs + (static_cast<int64_t>(c) * nkb + kb) * 1024, 1024, fb);
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
      }
      // wait until every stage filled has been released by the MMAs
      for (int i = 0; i < ST; ++i) {
        if (!mbar_wait_bounded(smem_u32(&ctl.empty[stage]), phase ^ 1u, &never, p.err, lim)) break;
        if (++stage == ST) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        if (!mbar_wait_bounded(smem_u32(&ctl.acc_empty[acc]), acc_phase ^ 1u, abort, p.err, lim))
          break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait_bounded(smem_u32(&ctl.full[stage]), phase, abort, p.err, lim)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = sbase + stage * T::kStageBytes;
          const uint32_t sb = sa + T::kABytes;
          const uint32_t ssfa = sb + T::kBBytes, ssfb = ssfa + T::kSfA;
          const uint32_t tsfa = tmem_base + T::kSfBase + stage * T::kSfCols, tsfb = tsfa + 8;
          // the scales of 128 elements: four columns per 128 rows
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tmem_cp_atom(tsfa + 4 * j, smem_desc_atom(ssfa + j * kAtom));
#pragma unroll
            for (int c = 0; c < T::kNB; ++c)
              tmem_cp_atom(tsfb + 4 * T::kNB * j + 4 * c,
                           smem_desc_atom(ssfb + c * 1024 + j * kAtom));
          }
          const int mmas = min(4, cdiv(kp - kb * kMxKBlock, 64));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk >= mmas) break;
            mma_mxf4(d_tmem, smem_desc_sw128(sa + kk * 32), smem_desc_sw128(sb + kk * 32),
                     idesc_mxf4(MM, BN, (kk & 1) * 2), tsfa + 4 * (kk >> 1),
                     tsfb + 4 * T::kNB * (kk >> 1), (kb | kk) != 0 ? 1u : 0u);
          }
          tc_commit(smem_u32(&ctl.empty[stage]));
          if (++stage == ST) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        tc_commit(smem_u32(&ctl.acc_full[acc]));
        if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
      }
      // every MMA issued has completed before TMEM is freed
      tc_commit(smem_u32(&ctl.drain));
      mbar_wait_bounded(smem_u32(&ctl.drain), 0, &never, p.err, lim);
    }
  } else if (warp < 4) {
    // ------------------------------------------------------ scales of A
    // Thread i brings rows i and i + 64: batches of four k-blocks, the next
    // batch's loads in flight while this one is stored.
    const int r0 = (warp - 2) * 32 + lane;
    const int soff = mx_code_bytes(p.K);
    int stage = 0;
    uint32_t phase = 0;
    uint2 cur[2][4], nxt[2][4];
    auto load = [&](int tile, int kb0, uint2 (&v)[2][4]) {
      const TilePos t = decode_tile(ctl.tab, G, p.n_tiles, tile);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = t.row0 + r0 + 64 * h;
        const uint8_t* src = p.a_rows + static_cast<int64_t>(row) * p.a_row_bytes + soff;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[h][i] = row < t.row_end && kb0 + i < nkb
                        ? *reinterpret_cast<const uint2*>(src + (kb0 + i) * 8)
                        : make_uint2(0, 0);
      }
    };
    int tile = blockIdx.x, kb0 = 0;
    bool ok = true;
    if (tile < num_tiles) load(tile, 0, cur);
    while (ok && tile < num_tiles) {
      int ntile = tile, nkb0 = kb0 + 4;
      if (nkb0 >= nkb) { nkb0 = 0; ntile += gridDim.x; }
      if (ntile < num_tiles) load(ntile, nkb0, nxt);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (kb0 + i >= nkb) break;
        if (!mbar_wait_bounded(smem_u32(&ctl.empty[stage]), phase ^ 1u, abort, p.err, lim)) {
          ok = false;
          break;
        }
        const uint32_t dst = sbase + stage * T::kStageBytes + T::kABytes + T::kBBytes + lane * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t d = dst + ((warp - 2) + 2 * h) * 4;
          st_shared_u32(d, cur[h][i].x);
          st_shared_u32(d + kAtom, cur[h][i].y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.full[stage]));
        if (++stage == ST) { stage = 0; phase ^= 1u; }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) cur[h][i] = nxt[h][i];
      tile = ntile;
      kb0 = nkb0;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    const int half = (warp - 4) >> 2;
    const int r_in_tile = quad * 32 + lane;
    const uint32_t stg = sbase + ST * T::kStageBytes + (warp - 4) * kEpiBox;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const TilePos t = decode_tile(ctl.tab, G, p.n_tiles, tile);
      const int nrows = min(MM, t.row_end - t.row0);
      if (!mbar_wait_bounded(smem_u32(&ctl.acc_full[acc]), acc_phase, abort, p.err, lim)) break;
      tc_fence_after();
      const uint32_t trow = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                            static_cast<uint32_t>(acc * BN);
      const int64_t grow = static_cast<int64_t>(t.row0) + r_in_tile;
      const bool row_ok = r_in_tile < nrows;
      const bool quad_full = (quad + 1) * 32 <= nrows;
      constexpr int kChunks = SWIGLU ? BN / 64 : BN / 32;  // of 32 output columns
      if (quad * 32 < nrows) {
#pragma unroll 1
        for (int c = half; c < kChunks; c += 2) {
          const int col0 = (t.n * kChunks + c) * 32;
          if (col0 >= p.N) break;
          float v[32];
          load_chunk<SWIGLU>(trow + (SWIGLU ? 64 : 32) * c, v);
          store_chunk<QOUT>(v, p, &tmC, col0, grow, t.row0 + quad * 32, row_ok, quad_full, stg);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.acc_empty[acc]));
      if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
    }
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  // --------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------ host side ----
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

template <int BN, bool SWIGLU, bool QOUT>
cudaError_t launch_variant(unsigned grid, const CUtensorMap& ma, const CUtensorMap& mb,
                           const CUtensorMap& mc, const Params& p, cudaStream_t st) {
  static int done[64] = {0};
  static std::mutex mu;
  const cudaError_t e =
      allow_smem(grouped_gemm_mxfp4_kernel<BN, SWIGLU, QOUT>, smem_bytes<BN>(), done, mu);
  if (e != cudaSuccess) return e;
  return launch_pdl(kPdlGemm, grouped_gemm_mxfp4_kernel<BN, SWIGLU, QOUT>, dim3(grid),
                    dim3(kThreads), smem_bytes<BN>(), st, ma, mb, mc, p);
}

}  // namespace

bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t rows,
              uint64_t cols, uint64_t stride, uint32_t box_rows, uint32_t box_cols,
              CUtensorMapSwizzle swizzle) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {stride};
  const cuuint32_t box[2] = {box_cols, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_scale_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t nkb) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[3] = {256, nkb, rows};
  const cuuint64_t strides[2] = {1024, 1024 * nkb};
  const cuuint32_t box[3] = {256, 1, 2};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mx

cudaError_t launch_grouped_gemm_mxfp4(const MxGemmArgs& a, cudaStream_t st) {
  using namespace mx;
  if (a.M == 0 || a.G == 0) return cudaSuccess;
  if (a.G > kMaxGroups || a.K % 8 != 0 || a.N % 8 != 0) return cudaErrorInvalidValue;
  const int forced = forced_gemm_kernel();
  if (forced >= 0 ? forced == 1 : a.M > 192 * static_cast<int64_t>(a.G))
    return launch_grouped_gemm_mxfp4_pair(a, st);
  constexpr int BN = 128;
  Params p = make_params(a);
  p.a_box_rows = a.M > 64 * static_cast<int64_t>(a.G) ? 128 : 32;
  p.n_tiles = cdiv(p.b_rows, BN);
  const uint64_t cb = static_cast<uint64_t>(mx_code_bytes(a.K));
  CUtensorMap ma, mb, mc;
  if (!make_code_map(&ma, a.rows, static_cast<uint64_t>(a.M), cb, p.a_row_bytes, p.a_box_rows) ||
      !make_code_map(&mb, a.weight, static_cast<uint64_t>(a.G) * p.b_rows, cb, cb, BN))
    return cudaErrorInvalidValue;
  if (a.quantized_out)
    mc = ma;  // not used
  else if (!make_out_map(&mc, a.out, static_cast<uint64_t>(a.M), static_cast<uint64_t>(a.N)))
    return cudaErrorInvalidValue;
  const int sms = num_sms_for_current_device();
  const int64_t max_tiles = (cdiv64(a.M, MM) + a.G) * p.n_tiles;
  const unsigned grid = static_cast<unsigned>(max_tiles < sms ? max_tiles : sms);
  if (!a.swiglu) return launch_variant<BN, false, false>(grid, ma, mb, mc, p, st);
  if (a.quantized_out) return launch_variant<BN, true, true>(grid, ma, mb, mc, p, st);
  return launch_variant<BN, true, false>(grid, ma, mb, mc, p, st);
}

}  // namespace hmoe
