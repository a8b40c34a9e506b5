// Grouped GEMM by expert on MXFP4 operands: block-scaled tcgen05 MMAs
// (kind::mxf4, K = 64, one e8m0 scale per 32), fp32 accumulation in TMEM.
//   plain:   out[rows of g] = x[rows of g] @ w[g]^T               -> bf16 or fp32
//   SwiGLU:  h = silu(x @ gate^T) * (x @ up^T), in fp32           -> bf16 or
//            MXFP4 records (the next product's input; h never exists in bf16)
//
// This file: one persistent CTA per SM, tiles of 128 rows x (up to) 192
// columns.  (CTA pairs, for much work in groups of many rows:
// gemm_mxfp4_pair.cu; the rule is use_pairs.)  A k-block is 256 elements: a 128-byte swizzled row of
// codes per operand row.  Warp 0 loads A (row records through a tensor map
// whose row stride is the record; only the 32-row boxes that the group
// reaches), A's scales as the records hold them, B and B's scale atoms; warp 2
// brings A's scales into the atom layout; warp 3 copies the atoms to TMEM;
// warp 1 issues the MMAs; twelve warps run the epilogue.  Each stage has its
// own TMEM scale columns, so a stage's empty barrier covers its scales as well.
//
// Such calls read each expert's weights once: XL 64x8 at T=64 53.5 MB for
// gate_up, 15.7 us, and 26.7 MB for down, 9.8 us alone, two sets of weights in
// turn (a large part is the launch, the group tables and the first tile's way
// through the pipeline, 8 us for a single gate_up tile).
#include "gemm_mxfp4.cuh"

namespace hmoe {
namespace mx {
namespace {

constexpr int ST = 4;          // stages
constexpr int kRaw = 3;        // pairs of k-blocks of A's scales as they come
constexpr int kABytes = MM * kRowB;
constexpr int kBBytes = kAccCols * kRowB;
constexpr int kOffSfa = kABytes + kBBytes;  // in a stage
constexpr int kOffSfb = kOffSfa + 2 * kAtom;
constexpr int kStageBytes = (kOffSfb + kSfbBytes + 1023) / 1024 * 1024;
constexpr int kSfCol = kAccs * kAccCols;
constexpr int kSfCols = kSfaCols + kSfbCols;  // of a stage
static_assert(kSfCol + ST * kSfCols <= kTmemCols, "TMEM columns");

struct Ctl {
  uint64_t full[ST];
  uint64_t empty[ST];
  uint64_t sf_full[ST];  // the stage's scales are in TMEM
  uint64_t raw_full[kRaw], raw_empty[kRaw];
  uint64_t acc_full[kAccs];
  uint64_t acc_empty[kAccs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  GroupTables tab;
};
constexpr int kOffRaw = ST * kStageBytes;  // [128 rows][16 scales]
constexpr int kOffEpi = kOffRaw + kRaw * 2048;
template <int OUT>
constexpr int kOffCtl = kOffEpi + epi_bytes<OUT>();
template <int OUT>
constexpr size_t kSmemBytes = 1024 + kOffCtl<OUT> + sizeof(Ctl);
static_assert(kSmemBytes<kBf16> <= 232448 && kSmemBytes<kRecords> <= 232448,
              "shared memory budget of one sm_100 CTA");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
struct Tile : RowBlock {
  int c0, nc;  // 64-column chunks
};
__device__ __forceinline__ Tile decode_tile(const GroupTables& tab, const Params& p, int tile) {
  const int mt = tile / p.ct.tiles;
  const int n = tile - mt * p.ct.tiles;
  Tile t;
  static_cast<RowBlock&>(t) = find_block(tab, p.G, mt, MM);
  t.c0 = p.ct.first(n);
  t.nc = p.ct.count(n);
  return t;
}

template <bool SWIGLU, int OUT>
__global__ void __launch_bounds__(kThreads, 1)
grouped_gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA,
                          const __grid_constant__ CUtensorMap tmA1,
                          const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmB1,
                          const __grid_constant__ CUtensorMap tmR,
                          const __grid_constant__ CUtensorMap tmR1,
                          const __grid_constant__ CUtensorMap tmC, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Ctl& ctl = *reinterpret_cast<Ctl*>(smem + kOffCtl<OUT>);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // ---------------------------------------------------------------- setup
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < ST; ++s) {
        mbar_init(smem_u32(&ctl.full[s]), 2);   // the producer's arm, the scale warp
        mbar_init(smem_u32(&ctl.empty[s]), 1);  // one commit per stage use
        mbar_init(smem_u32(&ctl.sf_full[s]), 1);
      }
      for (int s = 0; s < kRaw; ++s) {
        mbar_init(smem_u32(&ctl.raw_full[s]), 1);
        mbar_init(smem_u32(&ctl.raw_empty[s]), 1);
      }
      for (int a = 0; a < kAccs; ++a) {
        mbar_init(smem_u32(&ctl.acc_full[a]), 1);
        mbar_init(smem_u32(&ctl.acc_empty[a]), kEpiWarps);
      }
      mbar_init(smem_u32(&ctl.drain), 1);
      ctl.abort = 0;
      fence_mbar_init();
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmB1);
      tma_prefetch_desc(&tmR);
      tma_prefetch_desc(&tmC);
    }
    __syncwarp();
    grid_dependency_wait();  // launched early (launch_pdl): the counts are written before this
    build_tables(ctl.tab, p.counts, p.G, p.M, MM);
  } else if (warp == 1) {
    tmem_alloc(smem_u32(&ctl.tmem_base), kTmemCols);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();

  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl.tmem_base, 0);
  const int num_tiles = ctl.tab.num_m_tiles * p.ct.tiles;
  const int kp = mx_padded_k(p.K);
  const int nkb = mx_num_kblocks(p.K);
  volatile int* abort = &ctl.abort;
  int never = 0;
  const unsigned long long lim = p.wait_limit_ns;
  const auto wait = [&](uint64_t& bar, uint32_t parity) {
    return mbar_wait_bounded(smem_u32(&bar), parity, abort, p.err, lim);
  };
  const auto wait_warp = [&](uint64_t& bar, uint32_t parity) {
    return mbar_wait_warp(smem_u32(&bar), parity, abort, p.err, lim);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      Ring st, raw;
      int used = 0, raw_used = 0;
      bool ok = true;
      const int soff = mx_code_bytes(p.K);
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const Tile t = decode_tile(ctl.tab, p, tile);
        // A as one box of 128 rows, or the boxes of 32 that the group reaches:
        // each load costs the producer about 40 cycles, each box the memory
        // its rows
        const int nrows = min(MM, t.row_end - t.row0);
        const bool whole = nrows > MM - 32;
        const int box = whole ? MM : 32, boxes = whole ? 1 : cdiv(nrows, 32);
        const CUtensorMap *mapA = whole ? &tmA1 : &tmA, *mapR = whole ? &tmR1 : &tmR;
        const CUtensorMap* mapB = t.nc > p.ct.chunks ? &tmB1 : &tmB;
        const int brow = t.g * p.b_rows + t.c0 * 64;
        const uint8_t* bs =
            p.b_scales + (static_cast<int64_t>(t.g) * p.b_chunks + t.c0) * nkb * kAtom;
        const uint32_t bytes = boxes * box * kRowB + t.nc * (64 * kRowB + kAtom);
        for (int kb = 0; kb < nkb; ++kb) {
          // the first uses of a stage need no wait (one takes 170 cycles even
          // when the barrier is complete)
          if (used < ST) {
            ++used;
          } else if (!wait(ctl.empty[st.slot], st.phase ^ 1u)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&ctl.full[st.slot]);
          const uint32_t sa = sbase + st.slot * kStageBytes;
          mbar_arrive_expect_tx(fb, bytes);
          tma_load_2d(sa + kABytes, mapB, kb * kRowB, brow, fb);
          bulk_load(sa + kOffSfb, bs + static_cast<int64_t>(kb) * t.nc * kAtom, t.nc * kAtom, fb);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(sa + b * 32 * kRowB, mapA, kb * kRowB, t.row0 + b * 32, fb);
          if ((kb & 1) == 0) {  // A's scales of two k-blocks
            if (raw_used < kRaw) {
              ++raw_used;
            } else if (!wait(ctl.raw_empty[raw.slot], raw.phase ^ 1u)) {
              ok = false;
              break;
            }
            const uint32_t rb = smem_u32(&ctl.raw_full[raw.slot]);
            mbar_arrive_expect_tx(rb, boxes * box * 16);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(sbase + kOffRaw + raw.slot * 2048 + b * 32 * 16, mapR, soff + kb * 8,
                          t.row0 + b * 32, rb);
            raw.next(kRaw);
          }
          st.next(ST);
        }
      }
      // wait until every stage filled has been released
      for (int i = 0; i < ST; ++i, st.next(ST))
        if (!mbar_wait_bounded(smem_u32(&ctl.empty[st.slot]), st.phase ^ 1u, &never, p.err, lim)) break;
      for (int i = 0; i < kRaw; ++i, raw.next(kRaw))
        if (!mbar_wait_bounded(smem_u32(&ctl.raw_empty[raw.slot]), raw.phase ^ 1u, &never, p.err, lim)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (elect_one()) {
      Ring st, acc;
      bool ok = true;
      const uint64_t adesc0 = smem_desc_sw128(sbase);
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const int nc = p.ct.count(tile % p.ct.tiles);
        const uint32_t id0 = idesc_mxf4(MM, 64 * nc, 0), id1 = idesc_mxf4(MM, 64 * nc, 2);
        if (!wait(ctl.acc_empty[acc.slot], acc.phase ^ 1u)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc.slot * kAccCols);
        for (int kb = 0; kb < nkb; ++kb) {
          // committed by a thread that has waited for the stage's operands
          if (!wait(ctl.sf_full[st.slot], st.phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = adesc0 + st.slot * (kStageBytes >> 4), bd = ad + (kABytes >> 4);
          const uint32_t tsfa = tmem_base + kSfCol + st.slot * kSfCols, tsfb = tsfa + kSfaCols;
          const int mmas = min(4, cdiv(kp - kb * kMxKBlock, 64));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk >= mmas) break;
            mma_mxf4(d_tmem, ad + 2 * kk, bd + 2 * kk, (kk & 1) ? id1 : id0, tsfa + 4 * (kk >> 1),
                     tsfb + 2 * nc * (kk >> 1), (kb | kk) != 0 ? 1u : 0u);
          }
          tc_commit(smem_u32(&ctl.empty[st.slot]));
          st.next(ST);
        }
        if (!ok) break;
        tc_commit(smem_u32(&ctl.acc_full[acc.slot]));
        acc.next(kAccs);
      }
      // every MMA issued has completed before TMEM is freed
      tc_commit(smem_u32(&ctl.drain));
      mbar_wait_bounded(smem_u32(&ctl.drain), 0, &never, p.err, lim);
    }
  } else if (warp == 3) {
    // ------------------------------------------- scales from shared memory to TMEM
    if (elect_one()) {
      Ring st;
      bool ok = true;
      const uint64_t sf0 = smem_desc_atom(sbase + kOffSfa);
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const int nc = p.ct.count(tile % p.ct.tiles);
        for (int kb = 0; kb < nkb; ++kb) {
          if (!wait(ctl.full[st.slot], st.phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t sfa = sf0 + st.slot * (kStageBytes >> 4), sfb = sfa + (2 * kAtom >> 4);
          const uint32_t tsfa = tmem_base + kSfCol + st.slot * kSfCols, tsfb = tsfa + kSfaCols;
          tmem_cp_atom(tsfa, sfa);
          tmem_cp_atom(tsfa + 4, sfa + (kAtom >> 4));
#pragma unroll
          for (int c = 0; c < kMxTileChunks; ++c)
            if (c < nc) tmem_cp_atom(tsfb + 4 * c, sfb + c * (kAtom >> 4));
          tc_commit(smem_u32(&ctl.sf_full[st.slot]));
          st.next(ST);
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------ scales of A
    // From the records' order into the atoms': lane i moves rows i, i + 32,
    // i + 64, i + 96, whose words make up one lane of an atom.
    Ring st, raw;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      uint4 v[4];
      for (int kb = 0; kb < nkb; ++kb) {
        if ((kb & 1) == 0) {
          if (!wait_warp(ctl.raw_full[raw.slot], raw.phase)) {
            ok = false;
            break;
          }
          const uint4* src = reinterpret_cast<const uint4*>(smem + kOffRaw + raw.slot * 2048) + lane;
#pragma unroll
          for (int h = 0; h < 4; ++h) v[h] = src[32 * h];
        }
        if (!wait_warp(ctl.empty[st.slot], st.phase ^ 1u)) {
          ok = false;
          break;
        }
        const uint32_t dst = sbase + st.slot * kStageBytes + kOffSfa + lane * 16;
        st_shared_v4m(dst, make_uint4(v[0].x, v[1].x, v[2].x, v[3].x));
        st_shared_v4m(dst + kAtom, make_uint4(v[0].y, v[1].y, v[2].y, v[3].y));
#pragma unroll
        for (int h = 0; h < 4; ++h) { v[h].x = v[h].z; v[h].y = v[h].w; }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&ctl.full[st.slot]));
          // only here: the stores have taken the values, so the loads are done
          // (an arrival right behind the loads let the next copy overtake them)
          if ((kb & 1) == 0) mbar_arrive(smem_u32(&ctl.raw_empty[raw.slot]));
        }
        if ((kb & 1) == 0) raw.next(kRaw);
        st.next(ST);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int w = warp - 4;
    Ring acc;
    bool live = true;  // false once a wait gave up: the rest without work
    int buf = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const Tile t = decode_tile(ctl.tab, p, tile);
      live = live && wait_warp(ctl.acc_full[acc.slot], acc.phase);
      tc_fence_after();
      epilogue_tile<SWIGLU, OUT>(p, &tmC, w, tmem_base + acc.slot * kAccCols, t.row0,
                                  min(MM, t.row_end - t.row0), t.c0, t.nc, sbase + kOffEpi, buf, live,
                                  [&] {
                                    tc_fence_before();
                                    __syncwarp();
                                    if (lane == 0) mbar_arrive(smem_u32(&ctl.acc_empty[acc.slot]));
                                  });
      acc.next(kAccs);
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

template <bool SWIGLU, int OUT>
cudaError_t launch_variant(unsigned grid, const CUtensorMap (&m)[7], const Params& p,
                           cudaStream_t st) {
  static int done[64] = {0};
  static std::mutex mu;
  const cudaError_t e =
      allow_smem(grouped_gemm_mxfp4_kernel<SWIGLU, OUT>, kSmemBytes<OUT>, done, mu);
  if (e != cudaSuccess) return e;
  return launch_pdl(kPdlGemm, grouped_gemm_mxfp4_kernel<SWIGLU, OUT>, dim3(grid), dim3(kThreads),
                    kSmemBytes<OUT>, st, m[0], m[1], m[2], m[3], m[4], m[5], m[6],
                    p);
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

}  // namespace mx

namespace {

// Single CTAs or pairs: the same bits.  Pairs move fewer operand bytes, but
// there are half as many of them, with tiles twice as high, and their first
// tile takes longer.  So they win where each pair has several tiles to walk and
// the groups fill them.  Products alone, equal groups, warm, us single / pair:
//   gate_up, K=1536, 6 column tiles: 1 group of 2048 rows 8.0 / 10.8, 16384 22.2 / 21.8,
//     65536 67.5 / 50.5; 8 groups, 8192 rows 14.2 / 17.4, 32768 38.5 / 31.7; 64 groups, 16384
//     rows 28.1 / 28.3, 24576 35.7 / 34.4, 65536 73.8 / 56.4 (Zipf(1.2) groups 76.2 / 56.4)
//   down, K=512, 8 tiles: 1 group of 8192 rows 10.4 / 12.0, 24576 23.0 / 21.1; 64 groups, 32768
//     rows 31.9 / 32.1, 65536 53.8 / 51.5
//   128 groups, down 448 -> 1280: 96 rows each 17.6 / 25.6, 160 25.7 / 26.0, 384 45.0 / 42.4
//   K=2048, A no longer kept (when the pair kernel had that form): 8 groups, 8192 rows
//     26.6 / 38.6, 98304 214 / 314
// Seven 256-row tiles a pair and 160 rows a group part these; the worst miss was
// the down product of 64 groups of 320 rows, 22.9 / 26.1 (a pair).
bool use_pairs(const MxGemmArgs& a, int sms) {
  if (mx_num_kblocks(a.K) > mx::kPairKBlocks) return false;
  const int forced = forced_gemm_kernel();
  if (forced >= 0) return forced == 1;
  const int64_t tiles = mx_col_tiles(mx_weight_rows(a.N, a.swiglu)).tiles;
  return a.M >= 160 * static_cast<int64_t>(a.G) && a.M * tiles >= 7ll * 256 * (sms / 2);
}

}  // namespace

cudaError_t launch_grouped_gemm_mxfp4(const MxGemmArgs& a, cudaStream_t st) {
  using namespace mx;
  if (a.M == 0 || a.G == 0) return cudaSuccess;
  if (a.G > kMaxGroups || a.K % 8 != 0 || a.N % 8 != 0 || (a.f32_out && a.swiglu))
    return cudaErrorInvalidValue;
  const int sms = num_sms_for_current_device();
  if (use_pairs(a, sms)) return launch_grouped_gemm_mxfp4_pair(a, st);
  Params p = make_params(a);
  const uint64_t cb = static_cast<uint64_t>(mx_code_bytes(a.K));
  const uint64_t M = static_cast<uint64_t>(a.M), wrows = static_cast<uint64_t>(a.G) * p.b_rows;
  CUtensorMap m[7];
  if (!make_code_map(&m[0], a.rows, M, cb, p.a_row_bytes, 32) ||
      !make_code_map(&m[1], a.rows, M, cb, p.a_row_bytes, MM) ||
      !make_code_map(&m[2], a.weight, wrows, cb, cb, 64 * p.ct.chunks) ||
      !make_code_map(&m[3], a.weight, wrows, cb, cb, 64 * (p.ct.chunks + 1)) ||
      !make_raw_map(&m[4], a.rows, M, p.a_row_bytes, 32) ||
      !make_raw_map(&m[5], a.rows, M, p.a_row_bytes, MM))
    return cudaErrorInvalidValue;
  if (a.quantized_out)
    m[6] = m[0];  // not used
  else if (!make_out_map(&m[6], a.out, M, static_cast<uint64_t>(a.N), a.f32_out != 0))
    return cudaErrorInvalidValue;
  const int64_t max_tiles = (cdiv64(a.M, MM) + a.G) * p.ct.tiles;
  const unsigned grid = static_cast<unsigned>(max_tiles < sms ? max_tiles : sms);
  if (a.f32_out) return launch_variant<false, kF32>(grid, m, p, st);
  if (!a.swiglu) return launch_variant<false, kBf16>(grid, m, p, st);
  if (a.quantized_out) return launch_variant<true, kRecords>(grid, m, p, st);
  return launch_variant<true, kBf16>(grid, m, p, st);
}

}  // namespace hmoe
