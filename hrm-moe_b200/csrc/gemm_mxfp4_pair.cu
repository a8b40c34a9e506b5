// MXFP4 grouped GEMM on CTA pairs (tcgen05.mma.cta_group::2), for groups of
// many rows; same results as grouped_gemm_mxfp4_kernel.
//
// Two CTAs of a cluster share a 256-row x (up to) 192-column tile.  Each
// stages its own 128 rows of A and half of the tile's rows of B; the scales of
// A are its own rows', the scales of B are the whole tile's in both CTAs (each
// CTA's tensor core applies them from its own TMEM).
//
// At the 4-bit rate (4 x bf16) operand traffic is what a plain tile loop is
// bound by, so A stays: a pair takes a 256-row block and walks its column
// tiles with the block's A in shared memory (a ring of six 256-element
// k-blocks: K <= 1536, longer K is the single-CTA kernel's), and a k-block's
// slot is refilled for the next row block as soon as the last column tile has
// used it.  B streams through a ring of its own.
// XL gate_up at T=16384: 0.54 GB of operands to the SMs instead of 0.86 GB.
//
// TMEM (512 columns): two 192-column accumulators, six slots of A scales
// (8 columns) and of B scales (12).  192 columns rather than 256: two
// accumulators of 256 would leave no column for the scales.  A slot's scales
// live as long as its codes, under the same barriers.
//
// Work is shared out as whole row blocks, round after round, and the rest as
// runs of tiles.  (All of it as runs of tiles balanced as well, but the pairs
// then worked far apart in memory: the down product, bound by its writes,
// took 117 instead of 92 us.)
//
// Measured on XL 64x8 at T=16384 (131072 rows): gate_up with quantised output
// 92.6 us for equal groups (4.5 PFLOP/s, tensor pipes 56 % active), where an MMA
// with fresh scales takes 107 cycles for its nominal 85 (average tile) and the
// first loads, the change from one row block to the next and the output stores
// leave the pipes idle the rest; down 93.6 us with bf16 output (466 MB, 0.77 of
// the copy bandwidth) and 193 us with fp32 output (868 MB, 0.70), where neither
// the tensor pipes (28 %) nor DRAM (54 %, 50 %) are full: the stores of the
// epilogue do not drain faster.
#include "gemm_mxfp4.cuh"

namespace hmoe {
namespace mx {
namespace {

constexpr int QA = kPairKBlocks;  // k-blocks of A
constexpr int QB = 6;             // k-blocks of B
constexpr int QR = 3;             // pairs of k-blocks of A's scales: as they come, and as atoms
constexpr int kABytes = MM * kRowB;
constexpr int kBChunkBytes = 32 * kRowB;  // a CTA's half of a chunk
constexpr int kBBytes = kMxTileChunks * kBChunkBytes;
constexpr int kSfaCol = kAccs * kAccCols;
constexpr int kSfbCol = kSfaCol + kSfaCols * QA;
static_assert(kSfbCol + kSfbCols * QB <= kTmemCols, "TMEM columns");

struct Ctl {
  uint64_t a_full[QA], a_empty[QA];
  uint64_t b_full[QB], b_empty[QB];
  uint64_t sf_full[QB];  // the k-block's scales are in TMEM
  uint64_t raw_full[QR];
  uint64_t sfa_full[QR], sfa_empty[QR];
  uint64_t acc_full[kAccs], acc_empty[kAccs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  GroupTables tab;
};

constexpr int kOffSfa = QA * kABytes;
constexpr int kOffB = kOffSfa + QR * 2048;
constexpr int kOffSfb = kOffB + QB * kBBytes;
constexpr int kOffRaw = kOffSfb + QB * kSfbBytes;  // [128 rows][16 scales]
constexpr int kOffEpi = kOffRaw + QR * 2048;
template <int OUT>
constexpr int kOffCtl = kOffEpi + epi_bytes<OUT>();
template <int OUT>
constexpr size_t kSmemBytes = 1024 + kOffCtl<OUT> + sizeof(Ctl);
static_assert(kSmemBytes<kBf16> <= 232448 && kSmemBytes<kRecords> <= 232448,
              "shared memory budget of one sm_100 CTA");

// Arrive on the leader's barrier: this thread's (and, through the fence, its
// warp's) shared-memory writes are visible to whoever waits with cluster scope.
__device__ __forceinline__ void arrive_release_cluster(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster)
               : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// mbar_wait_bounded with cluster-scope acquire.
__device__ __forceinline__ bool wait_cluster_bounded(uint32_t bar, uint32_t parity,
                                                     volatile int* abort, int* err,
                                                     unsigned long long limit_ns) {
  if (try_wait_cluster(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (true) {
    if (try_wait_cluster(bar, parity)) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *abort = 1;
      record_error(err, kDevTimeout);
      return false;
    }
  }
}

// The four MMAs of a k-block (accumulating into `d` unless `acc` is 0), with
// two mbarriers' state asked for in front of them and returned behind them:
// bit 0 bar0, bit 1 bar1.  One block of PTX, so that nothing waits for the
// answers in between.  Scale ids 0 and 2 take turns (two scales an MMA, four
// to a TMEM word); tsfb_step: TMEM columns of B's scales of 128 elements.
constexpr uint32_t kSfId2 = (2u << 4) | (2u << 29);
__host__ __device__ constexpr uint64_t smem_desc_sw128_hi() {
  return (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
         (static_cast<uint64_t>(2u) << 61);
}
__device__ __forceinline__ uint32_t mma_kblock(uint32_t d, uint32_t ad, uint32_t bd, uint32_t id0,
                                               uint32_t tsfa, uint32_t tsfb, uint32_t tsfb_step,
                                               uint32_t acc, uint32_t bar0, uint32_t parity0,
                                               uint32_t bar1, uint32_t parity1) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, t, q0, q1;\n\t"
      ".reg .b32 id2, sfa2, sfb2, r1, x1, x2, x3, y1, y2, y3;\n\t"
      ".reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q0, [%9], %10;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q1, [%11], %12;\n\t"
      "setp.ne.b32 p, %8, 0;\n\t"
      "setp.eq.b32 t, %8, %8;\n\t"
      "or.b32 id2, %4, %13;\n\t"
      "add.u32 sfa2, %5, 4;\n\tadd.u32 sfb2, %6, %7;\n\t"
      "add.u32 x1, %2, 2;\n\tadd.u32 x2, %2, 4;\n\tadd.u32 x3, %2, 6;\n\t"
      "add.u32 y1, %3, 2;\n\tadd.u32 y2, %3, 4;\n\tadd.u32 y3, %3, 6;\n\t"
      "mov.b64 a0, {%2, %14};\n\tmov.b64 a1, {x1, %14};\n\tmov.b64 a2, {x2, %14};\n\tmov.b64 a3, {x3, %14};\n\t"
      "mov.b64 b0, {%3, %14};\n\tmov.b64 b1, {y1, %14};\n\tmov.b64 b2, {y2, %14};\n\tmov.b64 b3, {y3, %14};\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%1], a0, b0, %4, [%5], [%6], p;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%1], a1, b1, id2, [%5], [%6], t;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%1], a2, b2, %4, [sfa2], [sfb2], t;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%1], a3, b3, id2, [sfa2], [sfb2], t;\n\t"
      "selp.u32 %0, 1, 0, q0;\n\t"
      "selp.u32 r1, 2, 0, q1;\n\t"
      "or.b32 %0, %0, r1;\n\t}"
      : "=&r"(r)
      : "r"(d), "r"(ad), "r"(bd), "r"(id0), "r"(tsfa), "r"(tsfb), "r"(tsfb_step), "r"(acc), "r"(bar0),
        "r"(parity0), "r"(bar1), "r"(parity1), "n"(kSfId2),
        "n"(static_cast<uint32_t>(smem_desc_sw128_hi() >> 32))
      : "memory");
  return r;
}

// A pair's share as a walk over units, a unit being column tiles [t0, t1) of
// one row block.  Whole rounds first (row blocks pair, pair + npairs, ...: the
// pairs work side by side on neighbouring rows), then the row blocks left
// over, their tiles dealt out as runs of equal length.
struct Walk {
  int block, blocks_end, step;  // whole row blocks
  int tile, tile_end;           // the rest
};
struct Unit : RowBlock {
  int t0, t1;
};
__device__ __forceinline__ Walk share_of(const Ctl& ctl, int tiles, int pair, int npairs) {
  const int blocks = ctl.tab.num_m_tiles;
  const int whole = blocks / npairs * npairs;
  const int64_t rest = static_cast<int64_t>(blocks - whole) * tiles;
  Walk w;
  w.block = pair;
  w.blocks_end = whole;
  w.step = npairs;
  w.tile = whole * tiles + static_cast<int>(rest * pair / npairs);
  w.tile_end = whole * tiles + static_cast<int>(rest * (pair + 1) / npairs);
  return w;
}
// The walk's next unit; false at its end.
__device__ __forceinline__ bool next_unit(const Ctl& ctl, int G, int tiles, Walk& w, Unit& un) {
  int mt;
  if (w.block < w.blocks_end) {
    mt = w.block;
    w.block += w.step;
    un.t0 = 0;
    un.t1 = tiles;
  } else if (w.tile < w.tile_end) {
    mt = w.tile / tiles;
    un.t0 = w.tile - mt * tiles;
    un.t1 = min(tiles, un.t0 + w.tile_end - w.tile);
    w.tile += un.t1 - un.t0;
  } else {
    return false;
  }
  static_cast<RowBlock&>(un) = find_block(ctl.tab, G, mt, 2 * MM);
  return true;
}

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

template <bool SWIGLU, int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
grouped_gemm_mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tmA,
                               const __grid_constant__ CUtensorMap tmB,
                               const __grid_constant__ CUtensorMap tmB1,
                               const __grid_constant__ CUtensorMap tmS,
                               const __grid_constant__ CUtensorMap tmS1,
                               const __grid_constant__ CUtensorMap tmR,
                               const __grid_constant__ CUtensorMap tmC, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Ctl& ctl = *reinterpret_cast<Ctl*>(smem + kOffCtl<OUT>);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.G;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  // ---------------------------------------------------------------- setup
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < QA; ++s) {
        mbar_init(smem_u32(&ctl.a_full[s]), 1);   // the leader's arm
        mbar_init(smem_u32(&ctl.a_empty[s]), 1);  // one commit per use
      }
      for (int s = 0; s < QB; ++s) {
        mbar_init(smem_u32(&ctl.b_full[s]), 1);
        mbar_init(smem_u32(&ctl.b_empty[s]), 1);
        mbar_init(smem_u32(&ctl.sf_full[s]), 1);
      }
      for (int s = 0; s < QR; ++s) {
        mbar_init(smem_u32(&ctl.raw_full[s]), 1);
        mbar_init(smem_u32(&ctl.sfa_full[s]), 2);   // both CTAs' scale warps
        mbar_init(smem_u32(&ctl.sfa_empty[s]), 1);
      }
      for (int a = 0; a < kAccs; ++a) {
        mbar_init(smem_u32(&ctl.acc_full[a]), 1);
        mbar_init(smem_u32(&ctl.acc_empty[a]), 2 * kEpiWarps);  // both CTAs' epilogue warps
      }
      mbar_init(smem_u32(&ctl.drain), 1);
      ctl.abort = 0;
      fence_mbar_init();
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmB1);
      tma_prefetch_desc(&tmS);
      tma_prefetch_desc(&tmS1);
      tma_prefetch_desc(&tmR);
      tma_prefetch_desc(&tmC);
    }
    __syncwarp();
    grid_dependency_wait();  // launched early (launch_pdl): the counts are written before this
    build_tables(ctl.tab, p.counts, G, p.M, 2 * MM);
  } else if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl.tmem_base), kTmemCols);  // both CTAs, same warp
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barrier inits visible to the peer CTA before any remote signal
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();

  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl.tmem_base, 0);  // uniform, and seen to be
  const Walk share = share_of(ctl, p.ct.tiles, pair, npairs);
  const int kp = mx_padded_k(p.K);
  const int nkb = cdiv(kp, kMxKBlock);
  volatile int* abort = &ctl.abort;
  int never = 0;
  const unsigned long long lim = p.wait_limit_ns;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      Ring a, b;
      bool ok = true;
      Walk walk = share;
      Unit un{};
      while (ok && next_unit(ctl, G, p.ct.tiles, walk, un)) {
        const int my_row0 = un.row0 + static_cast<int>(rank) * MM;
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const bool longer = t < p.ct.extra;
          const CUtensorMap *mapB = longer ? &tmB1 : &tmB, *mapS = longer ? &tmS1 : &tmS;
          const int c0 = p.ct.first(t), nc = p.ct.count(t);
          const int brow = un.g * p.b_rows + c0 * 64 + static_cast<int>(rank) * nc * 32;
          const int srow = (un.g * p.b_chunks + c0) * nkb;
          const uint32_t bytes = 2 * nc * (kBChunkBytes + kAtom);  // both CTAs'
          const bool load_a = t == un.t0;
          for (int kb = 0; kb < nkb; ++kb) {
            if (load_a) {
              if (!mbar_wait_bounded(smem_u32(&ctl.a_empty[a.slot]), a.phase ^ 1u, abort, p.err, lim)) {
                ok = false;
                break;
              }
              const uint32_t fb = smem_u32(&ctl.a_full[a.slot]);
              if (leader) mbar_arrive_expect_tx(fb, 2 * kABytes);
              tma_load_2d_pair(sbase + a.slot * kABytes, &tmA, kb * kRowB, my_row0,
                               map_to_rank(fb, 0));
              a.next(QA);
            }
            if (!mbar_wait_bounded(smem_u32(&ctl.b_empty[b.slot]), b.phase ^ 1u, abort, p.err, lim)) {
              ok = false;
              break;
            }
            const uint32_t fb = smem_u32(&ctl.b_full[b.slot]);
            const uint32_t fb_leader = map_to_rank(fb, 0);
            if (leader) mbar_arrive_expect_tx(fb, bytes);
            tma_load_2d_pair(sbase + kOffB + b.slot * kBBytes, mapB, kb * kRowB, brow, fb_leader);
            tma_load_2d_pair(sbase + kOffSfb + b.slot * kSfbBytes, mapS, 0, srow + kb * nc, fb_leader);
            b.next(QB);
          }
        }
      }
      // wait until the MMAs have released every slot this CTA filled: no copy
      // and no commit is in flight when it leaves
      for (int i = 0; i < QA; ++i, a.next(QA))
        if (!mbar_wait_bounded(smem_u32(&ctl.a_empty[a.slot]), a.phase ^ 1u, &never, p.err, lim)) break;
      for (int i = 0; i < QB; ++i, b.next(QB))
        if (!mbar_wait_bounded(smem_u32(&ctl.b_empty[b.slot]), b.phase ^ 1u, &never, p.err, lim)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    // Even a wait on a barrier that is complete takes about 170 cycles here,
    // two MMAs' time, and the MMA queue is not much longer.  So the state of the
    // next k-block's barrier, and of the next accumulator's, is asked for in
    // front of this k-block's MMAs and looked at behind them (mma_kblock).
    if (leader && elect_one()) {
      Ring a, b, acc;
      bool ok = true;
      uint32_t ready = 0;  // bit 0: the next k-block, bit 1: the next accumulator
      // low words of the operands' descriptors (the high words are constant)
      const uint32_t adesc0 = static_cast<uint32_t>(smem_desc_sw128(sbase));
      const uint32_t bdesc0 = static_cast<uint32_t>(smem_desc_sw128(sbase + kOffB));
      const uint32_t a_empty = smem_u32(ctl.a_empty), b_empty = smem_u32(ctl.b_empty);
      const uint32_t sf_full = smem_u32(ctl.sf_full);
      const uint32_t acc_full = smem_u32(ctl.acc_full), acc_empty = smem_u32(ctl.acc_empty);
      const int full_kb = kp / kMxKBlock;           // k-blocks of four MMAs
      const int tail = cdiv(kp % kMxKBlock, 64);    // MMAs of the last, shorter one
      Walk walk = share;
      Unit un{};
      while (ok && next_unit(ctl, G, p.ct.tiles, walk, un)) {
        const int first = a.slot;  // the row block's first slot
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const int nc = p.ct.count(t);
          const bool load_a = t == un.t0;
          const bool free_a = t == un.t1 - 1;
          const uint32_t id0 = idesc_mxf4(2 * MM, 64 * nc, 0);
          if (!(ready & 2u) &&
              !mbar_wait_bounded(acc_empty + 8 * acc.slot, acc.phase ^ 1u, abort, p.err, lim)) {
            ok = false;
            break;
          }
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc.slot * kAccCols);
          Ring acc_next = acc;
          acc_next.next(kAccs);
          const uint32_t next_acc_empty = acc_empty + 8 * acc_next.slot;
          const uint32_t next_acc_parity = acc_next.phase ^ 1u;
          int sa = load_a ? a.slot : first;
          for (int kb = 0; kb < nkb; ++kb) {
            // committed by a thread that has waited for the k-block's A and B
            if (!(ready & 1u) && !mbar_wait_bounded(sf_full + 8 * b.slot, b.phase, abort, p.err, lim)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t ad = adesc0 + sa * (kABytes >> 4), bd = bdesc0 + b.slot * (kBBytes >> 4);
            const uint32_t tsfa = tmem_base + kSfaCol + kSfaCols * sa;
            const uint32_t tsfb = tmem_base + kSfbCol + kSfbCols * b.slot;
            const uint32_t done = b_empty + 8 * b.slot;
            b.next(QB);
            if (kb < full_kb) {
              ready = mma_kblock(d_tmem, ad, bd, id0, tsfa, tsfb, 2 * nc, kb, sf_full + 8 * b.slot,
                                 b.phase, next_acc_empty, next_acc_parity);
            } else {
              constexpr uint64_t kHi = smem_desc_sw128_hi();
              for (int kk = 0; kk < tail; ++kk)
                mma_mxf4_pair(d_tmem, kHi | (ad + 2 * kk), kHi | (bd + 2 * kk),
                              id0 | ((kk & 1) ? kSfId2 : 0u), tsfa + 4 * (kk >> 1),
                              tsfb + 2 * nc * (kk >> 1), (kb | kk) != 0 ? 1u : 0u);
              ready = 0;
            }
            tc_commit_pair_both(done);
            if (free_a) tc_commit_pair_both(a_empty + 8 * sa);
            if (load_a) a.next(QA);
            if (++sa == QA) sa = 0;
          }
          if (!ok) break;
          tc_commit_pair_both(acc_full + 8 * acc.slot);
          acc = acc_next;
        }
      }
      // every MMA issued has completed, and both CTAs' epilogues have released
      // every accumulator, before the pair tears down
      tc_commit_pair(smem_u32(&ctl.drain));
      mbar_wait_bounded(smem_u32(&ctl.drain), 0, &never, p.err, lim);
      for (int i = 0; i < kAccs; ++i, acc.next(kAccs))
        if (!mbar_wait_bounded(smem_u32(&ctl.acc_empty[acc.slot]), acc.phase ^ 1u, &never, p.err, lim))
          break;
    }
  } else if (warp == 3) {
    // ------------------------------------------- scales from shared memory to TMEM
    // A thread of its own, so that its waits are not in the MMA thread's way.
    // sf_full (commit, mbarrier, fence) hands a k-block on to the MMA thread.
    if (leader && elect_one()) {
      Ring a, sa, b;
      bool ok = true;
      const uint64_t sfa0 = smem_desc_atom(sbase + kOffSfa), sfb0 = smem_desc_atom(sbase + kOffSfb);
      Walk walk = share;
      Unit un{};
      while (ok && next_unit(ctl, G, p.ct.tiles, walk, un)) {
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const int nc = p.ct.count(t);
          const bool load_a = t == un.t0;
          for (int kb = 0; kb < nkb; ++kb) {
            if (load_a) {
              // a_full: the slot's TMEM columns are free as its codes are
              if (((kb & 1) == 0 && !wait_cluster_bounded(smem_u32(&ctl.sfa_full[sa.slot]), sa.phase,
                                                          abort, p.err, lim)) ||
                  !mbar_wait_bounded(smem_u32(&ctl.a_full[a.slot]), a.phase, abort, p.err, lim)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t tsfa = tmem_base + kSfaCol + kSfaCols * a.slot;
              const uint64_t d = sfa0 + ((sa.slot * 2048 + (kb & 1) * 1024) >> 4);
              tmem_cp_atom_pair(tsfa, d);
              tmem_cp_atom_pair(tsfa + 4, d + (kAtom >> 4));
              a.next(QA);
              if ((kb & 1) != 0 || kb == nkb - 1) {
                tc_commit_pair_both(smem_u32(&ctl.sfa_empty[sa.slot]));
                sa.next(QR);
              }
            }
            if (!mbar_wait_bounded(smem_u32(&ctl.b_full[b.slot]), b.phase, abort, p.err, lim)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t tsfb = tmem_base + kSfbCol + kSfbCols * b.slot;
            const uint64_t d = sfb0 + b.slot * (kSfbBytes >> 4);
#pragma unroll
            for (int c = 0; c < kMxTileChunks; ++c)
              if (c < nc) tmem_cp_atom_pair(tsfb + 4 * c, d + c * (kAtom >> 4));
            tc_commit_pair(smem_u32(&ctl.sf_full[b.slot]));
            b.next(QB);
          }
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------ scales of A
    // From the records' order into the atoms': lane i moves this CTA's rows
    // i, i + 32, i + 64, i + 96, whose words make up one lane of an atom.  Two
    // k-blocks at a time, ahead of the codes: the release at cluster scope
    // takes about 900 cycles.  (Loading the scales straight from global memory
    // was slower: the proxy fence waits for the loads in flight behind it.)
    // The warp loads its landing ring itself, QR steps ahead, and asks for the
    // step's A codes in L2: the units' A loads come in one burst from every
    // pair when a unit's last tile ends.
    struct Step {  // two k-blocks of a unit's A
      Walk walk;
      int kb, row0;
      bool live;
    };
    const auto start = [&](Step& st) {
      Unit un{};
      st.live = next_unit(ctl, G, p.ct.tiles, st.walk, un);
      st.kb = 0;
      st.row0 = un.row0 + static_cast<int>(rank) * MM;
    };
    const auto advance = [&](Step& st) {
      st.kb += 2;
      if (st.kb >= nkb) start(st);
    };
    const int soff = mx_code_bytes(p.K);
    Ring in, raw, sa;
    Step ahead, now;
    ahead.walk = share;
    start(ahead);
    now = ahead;
    const auto fetch = [&] {
      if (!ahead.live) return;
      if (elect_one()) {
        const uint32_t fb = smem_u32(&ctl.raw_full[in.slot]);
        mbar_arrive_expect_tx(fb, 2048);
        tma_load_2d(sbase + kOffRaw + in.slot * 2048, &tmR, soff + ahead.kb * 8, ahead.row0, fb);
        tma_prefetch_2d(&tmA, ahead.kb * kRowB, ahead.row0);
        if (ahead.kb + 1 < nkb) tma_prefetch_2d(&tmA, (ahead.kb + 1) * kRowB, ahead.row0);
      }
      __syncwarp();
      in.next(QR);
      advance(ahead);
    };
    for (int i = 0; i < QR; ++i) fetch();
    for (; now.live; advance(now)) {
      if (!mbar_wait_warp(smem_u32(&ctl.raw_full[raw.slot]), raw.phase, abort, p.err, lim)) break;
      const uint4* src = reinterpret_cast<const uint4*>(smem + kOffRaw + raw.slot * 2048) + lane;
      uint4 v[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) v[h] = src[32 * h];
      if (!mbar_wait_warp(smem_u32(&ctl.sfa_empty[sa.slot]), sa.phase ^ 1u, abort, p.err, lim)) break;
      const uint32_t dst = sbase + kOffSfa + sa.slot * 2048 + lane * 16;
      st_shared_v4m(dst, make_uint4(v[0].x, v[1].x, v[2].x, v[3].x));
      st_shared_v4m(dst + kAtom, make_uint4(v[0].y, v[1].y, v[2].y, v[3].y));
      st_shared_v4m(dst + 1024, make_uint4(v[0].z, v[1].z, v[2].z, v[3].z));
      st_shared_v4m(dst + 1024 + kAtom, make_uint4(v[0].w, v[1].w, v[2].w, v[3].w));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive_release_cluster(map_to_rank(smem_u32(&ctl.sfa_full[sa.slot]), 0));
      raw.next(QR);
      sa.next(QR);
      // only here may the landing slot be filled again: the stores have taken
      // the values, so the loads are done
      fetch();
    }
    // no copy into the landing ring is in flight when the CTA leaves (after an
    // early end), and no commit on its way to its barriers
    for (; raw.slot != in.slot || raw.phase != in.phase; raw.next(QR))
      if (!mbar_wait_warp(smem_u32(&ctl.raw_full[raw.slot]), raw.phase, &never, p.err, lim)) break;
    for (int i = 0; i < QR; ++i, sa.next(QR))
      if (!mbar_wait_warp(smem_u32(&ctl.sfa_empty[sa.slot]), sa.phase ^ 1u, &never, p.err, lim)) break;
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int w = warp - 4;
    Ring acc;
    bool live = true;  // false once a wait gave up: the rest without work
    int buf = 0;
    Walk walk = share;
    Unit un{};
    while (next_unit(ctl, G, p.ct.tiles, walk, un)) {
      const int my_row0 = un.row0 + static_cast<int>(rank) * MM;
      const int nrows = min(MM, un.row_end - my_row0);  // may be <= 0: nothing to store
      for (int t = un.t0; t < un.t1; ++t) {
        live = live && mbar_wait_warp(smem_u32(&ctl.acc_full[acc.slot]), acc.phase, abort, p.err, lim);
        tc_fence_after();
        epilogue_tile<SWIGLU, OUT>(
            p, &tmC, w, tmem_base + acc.slot * kAccCols, my_row0, nrows, p.ct.first(t), p.ct.count(t),
            sbase + kOffEpi, buf, live, [&] {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&ctl.acc_empty[acc.slot]), 0));
            });
        acc.next(kAccs);
      }
    }
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  // --------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the pair's MMAs or the peer use it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <bool SWIGLU, int OUT>
cudaError_t launch_variant(unsigned grid, const CUtensorMap& ma, const CUtensorMap& mb,
                           const CUtensorMap& mb1, const CUtensorMap& ms, const CUtensorMap& ms1,
                           const CUtensorMap& mr, const CUtensorMap& mc, const Params& p,
                           cudaStream_t st) {
  static int done[64] = {0};
  static std::mutex mu;
  const cudaError_t e =
      allow_smem(grouped_gemm_mxfp4_pair_kernel<SWIGLU, OUT>, kSmemBytes<OUT>, done, mu);
  if (e != cudaSuccess) return e;
  return launch_pdl(kPdlGemm, grouped_gemm_mxfp4_pair_kernel<SWIGLU, OUT>, dim3(grid),
                    dim3(kThreads), kSmemBytes<OUT>, st, ma, mb, mb1, ms, ms1, mr, mc, p);
}

}  // namespace
}  // namespace mx

cudaError_t launch_grouped_gemm_mxfp4_pair(const MxGemmArgs& a, cudaStream_t st) {
  using namespace mx;
  Params p = make_params(a);
  const uint64_t cb = static_cast<uint64_t>(mx_code_bytes(a.K));
  const uint64_t wrows = static_cast<uint64_t>(a.G) * p.b_rows;
  const uint64_t atoms = static_cast<uint64_t>(mx_weight_scale_atoms(a.G, a.N, a.K, a.swiglu));
  CUtensorMap ma, mb, mb1, ms, ms1, mr, mc;
  if (!make_code_map(&ma, a.rows, static_cast<uint64_t>(a.M), cb, p.a_row_bytes, MM) ||
      !make_code_map(&mb, a.weight, wrows, cb, cb, 32 * p.ct.chunks) ||
      !make_code_map(&mb1, a.weight, wrows, cb, cb, 32 * (p.ct.chunks + 1)) ||
      !make_scale_map(&ms, p.b_scales, atoms, p.ct.chunks) ||
      !make_scale_map(&ms1, p.b_scales, atoms, p.ct.chunks + 1) ||
      !make_raw_map(&mr, a.rows, static_cast<uint64_t>(a.M), p.a_row_bytes, MM))
    return cudaErrorInvalidValue;
  if (a.quantized_out)
    mc = ma;  // not used
  else if (!make_out_map(&mc, a.out, static_cast<uint64_t>(a.M), static_cast<uint64_t>(a.N),
                         a.f32_out != 0))
    return cudaErrorInvalidValue;
  const int sms = num_sms_for_current_device();
  const int64_t max_tiles = (cdiv64(a.M, 2 * MM) + a.G) * p.ct.tiles;
  int pairs = static_cast<int>(max_tiles < sms / 2 ? max_tiles : sms / 2);
  if (pairs < 1) pairs = 1;
  if (a.f32_out) return launch_variant<false, kF32>(2 * pairs, ma, mb, mb1, ms, ms1, mr, mc, p, st);
  if (!a.swiglu) return launch_variant<false, kBf16>(2 * pairs, ma, mb, mb1, ms, ms1, mr, mc, p, st);
  if (a.quantized_out) return launch_variant<true, kRecords>(2 * pairs, ma, mb, mb1, ms, ms1, mr, mc, p, st);
  return launch_variant<true, kBf16>(2 * pairs, ma, mb, mb1, ms, ms1, mr, mc, p, st);
}

}  // namespace hmoe
