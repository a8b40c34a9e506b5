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
// k-blocks, K <= 1536; longer K reloads A per column tile through the same
// ring), and a k-block's slot is refilled for the next row block as soon as
// the last column tile has used it.  B streams through a ring of its own.
// XL gate_up at T=16384: 0.54 GB of operands to the SMs instead of 0.86 GB.
//
// TMEM (512 columns): two 192-column accumulators, six slots of A scales
// (8 columns), five of B scales (16).  192 columns rather than 256: two
// accumulators of 256 would leave no column for the scales.  A slot's scales
// live as long as its codes, under the same barriers.
//
// Column tiles are runs of 64-column chunks, balanced (16 chunks: 3, 3, 3, 3,
// 2, 2).  The row blocks of all groups, each split into `parts` runs of
// column tiles, are the units the pairs take in turn; parts is the count that
// gives the shortest schedule for the actual row counts, found on the device.
#include "gemm_mxfp4.cuh"

namespace hmoe {
namespace mx {
namespace {

constexpr int QA = 6;             // k-blocks of A
constexpr int QB = 5;             // k-blocks of B
constexpr int kTileChunks = 3;    // 64-column chunks of a tile
constexpr int kAccCols = 64 * kTileChunks;
constexpr int kAccs = 2;
constexpr int kABytes = MM * kRowB;
constexpr int kBChunkBytes = 32 * kRowB;  // a CTA's half of a chunk
constexpr int kBBytes = kTileChunks * kBChunkBytes;
constexpr int kEpiWarps = 12;
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kSfaCol = kAccs * kAccCols;
constexpr int kSfbCol = kSfaCol + 8 * QA;
static_assert(kSfbCol + 16 * QB <= kTmemCols, "TMEM columns");

struct Ctl {
  uint64_t a_full[QA], a_empty[QA];
  uint64_t b_full[QB], b_empty[QB];
  uint64_t sf_full[QB];  // the k-block's scales are in TMEM
  uint64_t acc_full[kAccs], acc_empty[kAccs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int parts;
  GroupTables tab;
};

constexpr int kOffSfa = QA * kABytes;
constexpr int kOffB = kOffSfa + QA * 1024;
constexpr int kOffSfb = kOffB + QB * kBBytes;
constexpr int kOffEpi = kOffSfb + QB * 2048;
constexpr int kOffCtl = kOffEpi + kEpiWarps * kEpiBox;
constexpr size_t kSmemBytes = 1024 + kOffCtl + sizeof(Ctl);
static_assert(kSmemBytes <= 232448, "shared memory budget of one sm_100 CTA");

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

struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++slot == size) { slot = 0; phase ^= 1u; }
  }
};

// A unit: a row block and its column tiles [t0, t1).
struct Unit : RowBlock {
  int t0, t1;
};
__device__ __forceinline__ Unit find_unit(const Ctl& ctl, int G, int n_tiles, int u) {
  const int mt = u / ctl.parts;
  const int part = u - mt * ctl.parts;
  Unit r;
  static_cast<RowBlock&>(r) = find_block(ctl.tab, G, mt, 2 * MM);
  r.t0 = part * n_tiles / ctl.parts;
  r.t1 = (part + 1) * n_tiles / ctl.parts;
  return r;
}
// Column tile t: its first 64-column chunk and its number of chunks.
struct ColTile {
  int c0, nc;
};
__device__ __forceinline__ ColTile col_tile(const Params& p, int t) {
  return ColTile{t * p.tile_chunks + min(t, p.tile_extra), p.tile_chunks + (t < p.tile_extra)};
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                                 int c2, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

template <bool SWIGLU, bool QOUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
grouped_gemm_mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tmA,
                               const __grid_constant__ CUtensorMap tmB,
                               const __grid_constant__ CUtensorMap tmB1,
                               const __grid_constant__ CUtensorMap tmS,
                               const __grid_constant__ CUtensorMap tmC, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Ctl& ctl = *reinterpret_cast<Ctl*>(smem + kOffCtl);
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
        mbar_init(smem_u32(&ctl.a_full[s]), 3);   // the leader's arm, both CTAs' scale warps
        mbar_init(smem_u32(&ctl.a_empty[s]), 1);  // one commit per use
      }
      for (int s = 0; s < QB; ++s) {
        mbar_init(smem_u32(&ctl.b_full[s]), 1);
        mbar_init(smem_u32(&ctl.b_empty[s]), 1);
        mbar_init(smem_u32(&ctl.sf_full[s]), 1);
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
      tma_prefetch_desc(&tmC);
    }
    __syncwarp();
    grid_dependency_wait();  // launched early (launch_pdl): the counts are written before this
    build_tables(ctl.tab, p.counts, G, p.M, 2 * MM);
    __syncwarp();
    if (lane == 0) {
      // shortest schedule: rounds of units, a unit being its column tiles and
      // an eighth of one for its own start
      const int mt = ctl.tab.num_m_tiles;
      int best = 1;
      int64_t best_cost = INT64_MAX;
      for (int parts = 1; parts <= min(p.n_tiles, 64); ++parts) {
        const int64_t cost = cdiv64(static_cast<int64_t>(mt) * parts, npairs) *
                             (8 * cdiv(p.n_tiles, parts) + 1);
        if (cost < best_cost) { best_cost = cost; best = parts; }
      }
      ctl.parts = best;
    }
  } else if (warp == 1) {
    tmem_alloc_pair(smem_u32(&ctl.tmem_base), kTmemCols);  // both CTAs, same warp
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barrier inits visible to the peer CTA before any remote signal
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();

  const uint32_t tmem_base = ctl.tmem_base;
  const int units = ctl.tab.num_m_tiles * ctl.parts;
  const int kp = mx_padded_k(p.K);
  const int nkb = cdiv(kp, kMxKBlock);
  const bool resident = nkb <= QA;
  volatile int* abort = &ctl.abort;
  int never = 0;
  const unsigned long long lim = p.wait_limit_ns;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      Ring a, b;
      bool ok = true;
      for (int u = pair; ok && u < units; u += npairs) {
        const Unit un = find_unit(ctl, G, p.n_tiles, u);
        const int my_row0 = un.row0 + static_cast<int>(rank) * MM;
        // the next unit's A into L2: its loads come in one burst from every
        // pair as this unit's last tile ends
        if (resident && u + npairs < units) {
          const int next_row0 =
              find_unit(ctl, G, p.n_tiles, u + npairs).row0 + static_cast<int>(rank) * MM;
          for (int kb = 0; kb < nkb; ++kb) tma_prefetch_2d(&tmA, kb * kRowB, next_row0);
        }
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const ColTile ct = col_tile(p, t);
          const CUtensorMap* mapB = t < p.tile_extra ? &tmB1 : &tmB;
          const int brow = un.g * p.b_rows + ct.c0 * 64 + static_cast<int>(rank) * ct.nc * 32;
          const int srow = un.g * p.b_chunks + (ct.c0 >> 1);
          const uint32_t bytes = 2 * (ct.nc * kBChunkBytes + 2048);  // both CTAs'
          const bool load_a = t == un.t0 || !resident;
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
            tma_load_3d_pair(sbase + kOffSfb + b.slot * 2048, &tmS, 0, kb, srow, fb_leader);
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
    if (leader && elect_one()) {
      Ring a, b, acc;
      bool ok = true;
      const uint64_t adesc0 = smem_desc_sw128(sbase), bdesc0 = smem_desc_sw128(sbase + kOffB);
      for (int u = pair; ok && u < units; u += npairs) {
        const Unit un = find_unit(ctl, G, p.n_tiles, u);
        const int first = a.slot;  // the row block's first slot (resident)
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const ColTile ct = col_tile(p, t);
          const bool load_a = t == un.t0 || !resident;
          const bool free_a = t == un.t1 - 1 || !resident;
          const uint32_t id0 = idesc_mxf4(2 * MM, 64 * ct.nc, 0), id1 = idesc_mxf4(2 * MM, 64 * ct.nc, 2);
          // a tile that starts in the middle of a scale atom: two columns in
          const uint32_t sfb0 = tmem_base + kSfbCol + 2 * (ct.c0 & 1);
          if (!mbar_wait_bounded(smem_u32(&ctl.acc_empty[acc.slot]), acc.phase ^ 1u, abort, p.err, lim)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc.slot * kAccCols);
          int sa = first;
          for (int kb = 0; kb < nkb; ++kb) {
            if (load_a) {
              sa = a.slot;
              if (!wait_cluster_bounded(smem_u32(&ctl.a_full[sa]), a.phase, abort, p.err, lim)) {
                ok = false;
                break;
              }
              a.next(QA);
            }
            if (!mbar_wait_bounded(smem_u32(&ctl.b_full[b.slot]), b.phase, abort, p.err, lim) ||
                !mbar_wait_bounded(smem_u32(&ctl.sf_full[b.slot]), b.phase, abort, p.err, lim)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t ad = adesc0 + sa * (kABytes >> 4), bd = bdesc0 + b.slot * (kBBytes >> 4);
            const uint32_t tsfa = tmem_base + kSfaCol + 8 * sa, tsfb = sfb0 + 16 * b.slot;
            const int mmas = min(4, cdiv(kp - kb * kMxKBlock, 64));
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              if (kk >= mmas) break;
              mma_mxf4_pair(d_tmem, ad + 2 * kk, bd + 2 * kk, (kk & 1) ? id1 : id0,
                            tsfa + 4 * (kk >> 1), tsfb + 8 * (kk >> 1), (kb | kk) != 0 ? 1u : 0u);
            }
            tc_commit_pair_both(smem_u32(&ctl.b_empty[b.slot]));
            b.next(QB);
            if (free_a) tc_commit_pair_both(smem_u32(&ctl.a_empty[sa]));
            if (++sa == QA) sa = 0;
          }
          if (!ok) break;
          tc_commit_pair_both(smem_u32(&ctl.acc_full[acc.slot]));
          acc.next(kAccs);
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
    // A thread of its own: the copies of the next k-blocks run, and are
    // issued, beside this one's MMAs (in the MMA thread they took longer to
    // issue than the MMAs, 154 -> 138 us for XL gate_up with everything else
    // as it is).  The MMA thread waits for them through sf_full; b_full and
    // a_full, which it waits for too, order the slot's reuse.
    if (leader && elect_one()) {
      Ring a, b;
      bool ok = true;
      const uint64_t sfa0 = smem_desc_atom(sbase + kOffSfa), sfb0 = smem_desc_atom(sbase + kOffSfb);
      for (int u = pair; ok && u < units; u += npairs) {
        const Unit un = find_unit(ctl, G, p.n_tiles, u);
        for (int t = un.t0; ok && t < un.t1; ++t) {
          const ColTile ct = col_tile(p, t);
          const bool load_a = t == un.t0 || !resident;
          const bool two = (ct.c0 & 1) + ct.nc > 2;  // atoms of 128 rows that the tile reaches
          for (int kb = 0; kb < nkb; ++kb) {
            if (load_a) {
              if (!wait_cluster_bounded(smem_u32(&ctl.a_full[a.slot]), a.phase, abort, p.err, lim)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t tsfa = tmem_base + kSfaCol + 8 * a.slot;
              const uint64_t d = sfa0 + a.slot * (1024 >> 4);
              tmem_cp_atom_pair(tsfa, d);
              tmem_cp_atom_pair(tsfa + 4, d + (kAtom >> 4));
              a.next(QA);
            }
            if (!mbar_wait_bounded(smem_u32(&ctl.b_full[b.slot]), b.phase, abort, p.err, lim)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t tsfb = tmem_base + kSfbCol + 16 * b.slot;
            const uint64_t d = sfb0 + b.slot * (2048 >> 4);
            tmem_cp_atom_pair(tsfb, d);
            tmem_cp_atom_pair(tsfb + 8, d + (kAtom >> 4));
            if (two) {
              tmem_cp_atom_pair(tsfb + 4, d + (1024 >> 4));
              tmem_cp_atom_pair(tsfb + 12, d + ((1024 + kAtom) >> 4));
            }
            tc_commit_pair(smem_u32(&ctl.sf_full[b.slot]));
            b.next(QB);
          }
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------ scales of A
    // Lane i brings this CTA's rows i, i + 32, i + 64, i + 96: batches of four
    // k-blocks, the next batch's loads in flight while this one is stored.
    const int r0 = static_cast<int>(rank) * MM + lane;
    const int soff = mx_code_bytes(p.K);
    Ring a;
    uint2 cur[4][4], nxt[4][4];
    auto load = [&](const Unit& un, int kb0, uint2 (&v)[4][4]) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int row = un.row0 + r0 + 32 * h;
        const uint8_t* src = p.a_rows + static_cast<int64_t>(row) * p.a_row_bytes + soff;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[h][i] = row < un.row_end && kb0 + i < nkb
                        ? *reinterpret_cast<const uint2*>(src + (kb0 + i) * 8)
                        : make_uint2(0, 0);
      }
    };
    int u = pair, kb0 = 0, t = 0;
    Unit un;
    bool ok = true;
    if (u < units) {
      un = find_unit(ctl, G, p.n_tiles, u);
      t = un.t0;
      load(un, 0, cur);
    }
    while (ok && u < units) {
      int nkb0 = kb0 + 4;
      if (nkb0 >= nkb) {
        nkb0 = 0;
        t = resident ? un.t1 : t + 1;
        if (t >= un.t1) {
          u += npairs;
          if (u < units) {
            un = find_unit(ctl, G, p.n_tiles, u);
            t = un.t0;
          }
        }
      }
      if (u < units) load(un, nkb0, nxt);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (kb0 + i >= nkb) break;
        if (!mbar_wait_bounded(smem_u32(&ctl.a_empty[a.slot]), a.phase ^ 1u, abort, p.err, lim)) {
          ok = false;
          break;
        }
        const uint32_t dst = sbase + kOffSfa + a.slot * 1024 + lane * 16;
        // the atom's 16 bytes of a lane: its four rows' words
        st_shared_v4m(dst, make_uint4(cur[0][i].x, cur[1][i].x, cur[2][i].x, cur[3][i].x));
        st_shared_v4m(dst + kAtom, make_uint4(cur[0][i].y, cur[1][i].y, cur[2][i].y, cur[3][i].y));
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) arrive_release_cluster(map_to_rank(smem_u32(&ctl.a_full[a.slot]), 0));
        a.next(QA);
      }
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) cur[h][i] = nxt[h][i];
      kb0 = nkb0;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    const int third = (warp - 4) >> 2;
    const int r_in_tile = quad * 32 + lane;
    const uint32_t stg = sbase + kOffEpi + (warp - 4) * kEpiBox;
    Ring acc;
    bool ok = true;
    for (int u = pair; ok && u < units; u += npairs) {
      const Unit un = find_unit(ctl, G, p.n_tiles, u);
      const int my_row0 = un.row0 + static_cast<int>(rank) * MM;
      const int nrows = min(MM, un.row_end - my_row0);  // may be <= 0: nothing to store
      const int64_t grow = static_cast<int64_t>(my_row0) + r_in_tile;
      const bool row_ok = r_in_tile < nrows;
      const bool quad_full = (quad + 1) * 32 <= nrows;
      for (int t = un.t0; t < un.t1; ++t) {
        const ColTile ct = col_tile(p, t);
        if (!mbar_wait_bounded(smem_u32(&ctl.acc_full[acc.slot]), acc.phase, abort, p.err, lim)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t trow = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) +
                              static_cast<uint32_t>(acc.slot * kAccCols);
        constexpr int kPer = SWIGLU ? 1 : 2;  // 32-column outputs of a chunk
        if (quad * 32 < nrows) {
#pragma unroll 1
          for (int c = third; c < ct.nc * kPer; c += 3) {
            const int col0 = (ct.c0 * kPer + c) * 32;
            if (col0 >= p.N) break;
            float v[32];
            load_chunk<SWIGLU>(trow + (SWIGLU ? 64 : 32) * c, v);
            store_chunk<QOUT>(v, p, &tmC, col0, grow, my_row0 + quad * 32, row_ok, quad_full, stg);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&ctl.acc_empty[acc.slot]), 0));
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

template <bool SWIGLU, bool QOUT>
cudaError_t launch_variant(unsigned grid, const CUtensorMap& ma, const CUtensorMap& mb,
                           const CUtensorMap& mb1, const CUtensorMap& ms, const CUtensorMap& mc,
                           const Params& p, cudaStream_t st) {
  static int done[64] = {0};
  static std::mutex mu;
  const cudaError_t e =
      allow_smem(grouped_gemm_mxfp4_pair_kernel<SWIGLU, QOUT>, kSmemBytes, done, mu);
  if (e != cudaSuccess) return e;
  return launch_pdl(kPdlGemm, grouped_gemm_mxfp4_pair_kernel<SWIGLU, QOUT>, dim3(grid),
                    dim3(kThreads), kSmemBytes, st, ma, mb, mb1, ms, mc, p);
}

}  // namespace
}  // namespace mx

cudaError_t launch_grouped_gemm_mxfp4_pair(const MxGemmArgs& a, cudaStream_t st) {
  using namespace mx;
  Params p = make_params(a);
  const int chunks = cdiv(p.b_rows, 64);
  p.n_tiles = cdiv(chunks, kTileChunks);
  p.tile_chunks = chunks / p.n_tiles;
  p.tile_extra = chunks % p.n_tiles;
  const uint64_t cb = static_cast<uint64_t>(mx_code_bytes(a.K));
  const uint64_t nkb = cdiv(mx_padded_k(a.K), kMxKBlock);
  const uint64_t wrows = static_cast<uint64_t>(a.G) * p.b_rows;
  CUtensorMap ma, mb, mb1, ms, mc;
  if (!make_code_map(&ma, a.rows, static_cast<uint64_t>(a.M), cb, p.a_row_bytes, MM) ||
      !make_code_map(&mb, a.weight, wrows, cb, cb, 32 * p.tile_chunks) ||
      !make_code_map(&mb1, a.weight, wrows, cb, cb, 32 * (p.tile_chunks + 1)) ||
      !make_scale_map(&ms, p.b_scales, static_cast<uint64_t>(a.G) * p.b_chunks, nkb))
    return cudaErrorInvalidValue;
  if (a.quantized_out)
    mc = ma;  // not used
  else if (!make_out_map(&mc, a.out, static_cast<uint64_t>(a.M), static_cast<uint64_t>(a.N)))
    return cudaErrorInvalidValue;
  const int sms = num_sms_for_current_device();
  const int64_t max_tiles = (cdiv64(a.M, 2 * MM) + a.G) * p.n_tiles;
  int pairs = static_cast<int>(max_tiles < sms / 2 ? max_tiles : sms / 2);
  if (pairs < 1) pairs = 1;
  if (!a.swiglu) return launch_variant<false, false>(2 * pairs, ma, mb, mb1, ms, mc, p, st);
  if (a.quantized_out) return launch_variant<true, true>(2 * pairs, ma, mb, mb1, ms, mc, p, st);
  return launch_variant<true, false>(2 * pairs, ma, mb, mb1, ms, mc, p, st);
}

}  // namespace hmoe
