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
#include <cuda.h>
#include <mutex>

#include "internal.h"
#include "mxfp4.cuh"

namespace hmoe {
namespace {

constexpr int MM = 128;           // rows per tile
constexpr int kRowB = 128;        // bytes of codes per operand row and stage
constexpr int kMxMaxGroups = 1024;
constexpr int kMxThreads = 384;   // 4 control warps, 8 epilogue warps
constexpr int kEpiBox = 32 * 32 * 2;
constexpr int kAtom = 512;        // scales of 128 rows x 128 elements
constexpr int kAccs = 2;
constexpr int kTmemCols = 512;

template <int BN>
struct MxTile {
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
struct MxCtl {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t acc_full[kAccs];
  uint64_t acc_empty[kAccs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int num_m_tiles;
  int pad_;
  int group_rows[kMxMaxGroups + 1];
  int tile_prefix[kMxMaxGroups + 1];
};

template <int BN>
constexpr size_t mx_smem_bytes() {
  return 1024 + static_cast<size_t>(MxTile<BN>::kStages) * MxTile<BN>::kStageBytes +
         8 * kEpiBox + sizeof(MxCtl<MxTile<BN>::kStages>);
}
static_assert(mx_smem_bytes<128>() <= 232448, "shared memory budget of one sm_100 CTA");

struct MxParams {
  const uint8_t* a_rows;   // records
  const uint8_t* b_scales; // atoms
  const int32_t* counts;
  int G;
  int64_t M;
  int N;            // output columns
  int K;
  int a_row_bytes;
  int a_box_rows;   // rows of one A load
  int n_tiles;
  int b_rows;       // packed rows per group
  int b_chunks;     // 128-row scale chunks per group
  void* out;        // bf16 [M, N] or records
  int* err;
  unsigned long long wait_limit_ns;
};

__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                         uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], "
      "p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows x 16 bytes of shared memory to four TMEM columns of all four lane
// quadrants.
__device__ __forceinline__ void tmem_cp_atom(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
// Scale atom in shared memory: no swizzle, 8-row core matrices of 128
// contiguous bytes.
__device__ __forceinline__ uint64_t smem_desc_atom(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 16;
  d |= static_cast<uint64_t>(128u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  return d;
}
// Instruction descriptor of the block-scaled kinds: bits [4,6) B scale id,
// [7,10) A type (1 = e2m1), [10,12) B type, [17,23) N >> 3, 23 scale type
// (1 = e8m0), [27,29) M >> 7, [29,31) A scale id.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n, int sf_id) {
  return (static_cast<uint32_t>(sf_id) << 4) | (1u << 7) | (1u << 10) |
         (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(m >> 7) << 27) | (static_cast<uint32_t>(sf_id) << 29);
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared_v4m(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

struct MxTilePos {
  int g, row0, row_end, n;
};
template <class Ctl>
__device__ __forceinline__ MxTilePos decode_tile(const Ctl& ctl, int G, int n_tiles, int tile) {
  MxTilePos t;
  const int mt = tile / n_tiles;
  t.n = tile - mt * n_tiles;
  int lo = 0, hi = G;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ctl.tile_prefix[mid] <= mt) lo = mid; else hi = mid;
  }
  t.g = lo;
  t.row0 = ctl.group_rows[lo] + (mt - ctl.tile_prefix[lo]) * MM;
  t.row_end = ctl.group_rows[lo + 1];
  return t;
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}

template <int BN, bool SWIGLU, bool QOUT>
__global__ void __launch_bounds__(kMxThreads, 1)
grouped_gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA,
                          const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const MxParams p) {
  using T = MxTile<BN>;
  constexpr int ST = T::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  auto& ctl = *reinterpret_cast<MxCtl<ST>*>(smem + ST * T::kStageBytes + 8 * kEpiBox);
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
    // prefix sums of the groups' rows and tiles; rows past M are cut off, so
    // that no count, however wrong, leads outside the operands
    const int per = cdiv(G, 32);
    const int g0 = min(G, lane * per), g1 = min(G, g0 + per);
    int64_t rows = 0;
    for (int g = g0; g < g1; ++g) rows += max(0, p.counts[g]);
    int64_t rin = rows;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t ro = __shfl_up_sync(0xffffffffu, rin, off);
      if (lane >= off) rin += ro;
    }
    int64_t rr = rin - rows;
    int tiles = 0;
    for (int g = g0; g < g1; ++g) {
      const int a = static_cast<int>(rr < p.M ? rr : p.M);
      rr += max(0, p.counts[g]);
      const int b = static_cast<int>(rr < p.M ? rr : p.M);
      ctl.group_rows[g] = a;
      ctl.tile_prefix[g] = tiles;
      tiles += cdiv(b - a, MM);
    }
    int tin = tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int to = __shfl_up_sync(0xffffffffu, tin, off);
      if (lane >= off) tin += to;
    }
    for (int g = g0; g < g1; ++g) ctl.tile_prefix[g] += tin - tiles;
    if (lane == 31) {
      ctl.group_rows[G] = static_cast<int>(rin < p.M ? rin : p.M);
      ctl.tile_prefix[G] = tin;
      ctl.num_m_tiles = tin;
    }
  } else if (warp == 1) {
    tmem_alloc(smem_u32(&ctl.tmem_base), kTmemCols);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();

  const uint32_t tmem_base = ctl.tmem_base;
  const int num_tiles = ctl.num_m_tiles * p.n_tiles;
  const int kp = mx_padded_k(p.K);
  const int nkb = cdiv(kp, kMxKBlock);
  volatile int* abort = &ctl.abort;
  int never = 0;
  const unsigned long long lim = p.wait_limit_ns;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const MxTilePos t = decode_tile(ctl, G, p.n_tiles, tile);
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
    if (lane == 0) {
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
      const MxTilePos t = decode_tile(ctl, G, p.n_tiles, tile);
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
    const int out_row_bytes = QOUT ? mx_row_bytes(p.N) : 0;
    const int out_cb = mx_code_bytes(p.N), out_ns = mx_num_scales(p.N);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const MxTilePos t = decode_tile(ctl, G, p.n_tiles, tile);
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
          {
            uint32_t ra[32];
            tmem_ld_32cols(trow + (SWIGLU ? 64 : 32) * c, ra);
            if (SWIGLU) {
              uint32_t ua[32];
              tmem_ld_32cols(trow + 64 * c + 32, ua);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i)
                v[i] = silu_mul(__uint_as_float(ra[i]), __uint_as_float(ua[i]));
            } else {
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(ra[i]);
            }
          }
          if constexpr (QOUT) {
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
            const uint32_t s = mx_scale_code(amax);
            const float inv = mx_inv_scale(s);
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              q[i] = mx_cvt8(v[8 * i] * inv, v[8 * i + 1] * inv, v[8 * i + 2] * inv,
                             v[8 * i + 3] * inv, v[8 * i + 4] * inv, v[8 * i + 5] * inv,
                             v[8 * i + 6] * inv, v[8 * i + 7] * inv);
            if (row_ok) {
              uint8_t* orow = static_cast<uint8_t*>(p.out) + grow * out_row_bytes;
              *reinterpret_cast<uint4*>(orow + col0 / 2) = make_uint4(q[0], q[1], q[2], q[3]);
              orow[out_cb + col0 / 32] = static_cast<uint8_t>(s);
              if (col0 / 32 == out_ns - 1)
                for (int b = out_cb + out_ns; b < out_row_bytes; ++b) orow[b] = 0;
            }
          } else {
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) packed[i] = cvt_bf16x2(v[2 * i], v[2 * i + 1]);
            if (quad_full) {
              // a whole 32 x 32 box: staged and stored with TMA
              if (lane == 0) bulk_wait_group_read<0>();
              __syncwarp();
              const uint32_t dst = stg + lane * 64;
              const uint32_t sw = (lane >> 1) & 3;
#pragma unroll
              for (int c4 = 0; c4 < 4; ++c4)
                st_shared_v4m(dst + ((c4 ^ sw) << 4),
                              make_uint4(packed[4 * c4], packed[4 * c4 + 1], packed[4 * c4 + 2],
                                         packed[4 * c4 + 3]));
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&tmC, col0, t.row0 + quad * 32, stg);
                bulk_commit_group();
              }
            } else if (row_ok) {
              uint16_t* orow = static_cast<uint16_t*>(p.out) + grow * p.N;
#pragma unroll
              for (int c4 = 0; c4 < 4; ++c4)
                if (col0 + c4 * 8 + 8 <= p.N)
                  *reinterpret_cast<uint4*>(orow + col0 + c4 * 8) =
                      make_uint4(packed[4 * c4], packed[4 * c4 + 1], packed[4 * c4 + 2],
                                 packed[4 * c4 + 3]);
            }
          }
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
typedef CUresult (*EncodeTiledFnM)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFnM encode_fn_m() {
  static EncodeTiledFnM fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFnM>(ptr);
  });
  return fn;
}

// Bytes [rows, cols] with a row stride, boxes of box_rows x 128 bytes.
bool make_code_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols,
                   uint64_t stride, uint32_t box_rows) {
  EncodeTiledFnM enc = encode_fn_m();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {stride};
  const cuuint32_t box[2] = {kRowB, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_out_map(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols) {
  EncodeTiledFnM enc = encode_fn_m();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {cols * 2};
  const cuuint32_t box[2] = {32, 32};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool SWIGLU, bool QOUT>
cudaError_t launch_variant(unsigned grid, const CUtensorMap& ma, const CUtensorMap& mb,
                           const CUtensorMap& mc, const MxParams& p, cudaStream_t st) {
  static int done[64] = {0};
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      e = cudaFuncSetAttribute(grouped_gemm_mxfp4_kernel<BN, SWIGLU, QOUT>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(mx_smem_bytes<BN>()));
      if (e != cudaSuccess) return e;
      done[dev] = 1;
    }
  }
  return launch_pdl(kPdlGemm, grouped_gemm_mxfp4_kernel<BN, SWIGLU, QOUT>, dim3(grid),
                    dim3(kMxThreads), mx_smem_bytes<BN>(), st, ma, mb, mc, p);
}

}  // namespace

cudaError_t launch_grouped_gemm_mxfp4(const MxGemmArgs& a, cudaStream_t st) {
  if (a.M == 0 || a.G == 0) return cudaSuccess;
  if (a.G > kMxMaxGroups || a.K % 8 != 0 || a.N % 8 != 0) return cudaErrorInvalidValue;
  constexpr int BN = 128;
  const uint8_t* w = static_cast<const uint8_t*>(a.weight);
  MxParams p;
  p.a_rows = static_cast<const uint8_t*>(a.rows);
  p.b_scales = w + mx_weight_scale_offset(a.G, a.N, a.K, a.swiglu);
  p.counts = a.counts;
  p.G = a.G;
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.a_row_bytes = mx_row_bytes(a.K);
  p.a_box_rows = a.M > 64 * static_cast<int64_t>(a.G) ? 128 : 32;
  p.b_rows = mx_weight_rows(a.N, a.swiglu);
  p.b_chunks = cdiv(p.b_rows, 128);
  p.n_tiles = cdiv(p.b_rows, BN);
  p.out = a.out;
  p.err = a.err;
  p.wait_limit_ns = kWaitLimitNs;
  const uint64_t cb = static_cast<uint64_t>(mx_code_bytes(a.K));
  CUtensorMap ma, mb, mc;
  if (!make_code_map(&ma, a.rows, static_cast<uint64_t>(a.M), cb, p.a_row_bytes, p.a_box_rows) ||
      !make_code_map(&mb, w, static_cast<uint64_t>(a.G) * p.b_rows, cb, cb, BN))
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
