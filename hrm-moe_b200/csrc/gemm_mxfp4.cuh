// Shared pieces of the MXFP4 grouped GEMMs: block-scaled MMA wrappers, tile
// tables, the epilogue of 32 output columns, tensor maps.
#pragma once

#include <cuda.h>
#include <mutex>

#include "internal.h"
#include "mxfp4.cuh"

namespace hmoe {
namespace mx {

constexpr int MM = 128;      // rows of one CTA's tile
constexpr int kRowB = 128;   // bytes of codes per operand row and k-block
constexpr int kMaxGroups = 1024;
constexpr int kAtom = 512;   // scales of 128 rows x 128 elements
constexpr int kEpiBox = 32 * 32 * 2;
constexpr int kTmemCols = 512;
constexpr int kAccCols = 64 * kMxTileChunks;
constexpr int kAccs = 2;
constexpr int kEpiWarps = 12;  // three per lane quadrant
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kPairKBlocks = 6;  // the most that the CTA-pair kernel takes
constexpr int kSfaCols = 8;                  // TMEM columns of a k-block's scales
constexpr int kSfbCols = 4 * kMxTileChunks;
constexpr int kSfbBytes = kMxTileChunks * kAtom;

struct Params {
  const uint8_t* a_rows;    // records
  const uint8_t* b_scales;  // atoms
  const int32_t* counts;
  int G;
  int64_t M;
  int N;            // output columns
  int K;
  int a_row_bytes;
  MxColTiles ct;    // column tiles
  int b_rows;       // packed rows per group
  int b_chunks;     // 64-row chunks per group
  void* out;        // bf16 or fp32 [M, N], or records
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
__device__ __forceinline__ void mma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                              uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], "
      "p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows x 16 bytes of shared memory to four TMEM columns of all four lane
// quadrants (the pair form: in both CTAs, each from its own shared memory).
__device__ __forceinline__ void tmem_cp_atom(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
__device__ __forceinline__ void tmem_cp_atom_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
               : "memory");
}
// One lane of a converged warp, chosen by the hardware.  Around the issue of
// TMA and tcgen05 instructions this, not a test of the lane index: the
// compiler then knows that a single lane is active and emits each instruction
// once, instead of a loop over the active lanes (measured in the pair kernel:
// 110 -> 50 cycles per tcgen05 instruction issued).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
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
__device__ __forceinline__ void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared_v4m(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// mbar_wait_bounded by a whole warp, with one answer for all its lanes: the
// lanes read the barrier, the abort flag and the clock each for itself and may
// differ near the limit, and a lane that left alone would leave the others at
// the warp's next synchronisation without a bound.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort,
                                               int* err, unsigned long long limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort, err, limit_ns));
}

// A place in a ring of barriers, and the parity of its phase.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++slot == size) { slot = 0; phase ^= 1u; }
  }
};

struct GroupTables {
  int group_rows[kMaxGroups + 1];
  int tile_prefix[kMaxGroups + 1];  // prefix of row blocks
  int num_m_tiles;
};

// One warp: the groups' first rows and row blocks from the device counts.
// Rows past M are cut off, so that no count, however wrong, leads outside the
// operands.
__device__ __forceinline__ void build_tables(GroupTables& t, const int32_t* counts, int G, int64_t M,
                                             int block_rows) {
  const int lane = threadIdx.x & 31;
  const int per = cdiv(G, 32);
  const int g0 = min(G, lane * per), g1 = min(G, g0 + per);
  // up to 128 groups: a lane's counts are loaded at once and kept
  constexpr int kKeep = 4;
  int c[kKeep];
#pragma unroll
  for (int i = 0; i < kKeep; ++i) c[i] = g0 + i < g1 ? max(0, counts[g0 + i]) : 0;
  int64_t rows = 0;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) rows += c[i];
  for (int g = g0 + kKeep; g < g1; ++g) rows += max(0, counts[g]);
  int64_t rin = rows;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t ro = __shfl_up_sync(0xffffffffu, rin, off);
    if (lane >= off) rin += ro;
  }
  int64_t rr = rin - rows;
  int tiles = 0;
  const auto place = [&](int g, int count) {
    const int a = static_cast<int>(rr < M ? rr : M);
    rr += count;
    const int b = static_cast<int>(rr < M ? rr : M);
    t.group_rows[g] = a;
    t.tile_prefix[g] = tiles;
    tiles += cdiv(b - a, block_rows);
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (g0 + i < g1) place(g0 + i, c[i]);
  for (int g = g0 + kKeep; g < g1; ++g) place(g, max(0, counts[g]));
  int tin = tiles;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int to = __shfl_up_sync(0xffffffffu, tin, off);
    if (lane >= off) tin += to;
  }
  for (int g = g0; g < g1; ++g) t.tile_prefix[g] += tin - tiles;
  if (lane == 31) {
    t.group_rows[G] = static_cast<int>(rin < M ? rin : M);
    t.tile_prefix[G] = tin;
    t.num_m_tiles = tin;
  }
}

struct RowBlock {
  int g, row0, row_end;
};
__device__ __forceinline__ RowBlock find_block(const GroupTables& t, int G, int mt, int block_rows) {
  int lo = 0, hi = G;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.tile_prefix[mid] <= mt) lo = mid; else hi = mid;
  }
  RowBlock r;
  r.g = lo;
  r.row0 = t.group_rows[lo] + (mt - t.tile_prefix[lo]) * block_rows;
  r.row_end = t.group_rows[lo + 1];
  return r;
}

// Two fp32 products (sums) in one instruction, each rounded to nearest.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// silu(g) * u in fp32.  With a = 2^(-|g| log2 e) <= 1, the sigmoid of g is
// 1 / (1 + a), or a / (1 + a) where g < 0: nothing overflows, and far on the
// negative side it keeps a's subnormals (1 / (1 + 2^(|g| log2 e)) is zero from
// g = -87.4 on, where silu(g) is still a normal number, times any u).
// Approximate exponential and reciprocal, 2^-22 relative each.
__device__ __forceinline__ float2 silu_mul2(float2 g, float2 u) {
  const float2 x = mul2(make_float2(fabsf(g.x), fabsf(g.y)),
                        make_float2(-1.4426950408889634f, -1.4426950408889634f));
  float2 a, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(a.x) : "f"(x.x));
  asm("ex2.approx.f32 %0, %1;" : "=f"(a.y) : "f"(x.y));
  const float2 d = add2(a, make_float2(1.0f, 1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  const float2 n = make_float2(g.x < 0.0f ? g.x * a.x : g.x, g.y < 0.0f ? g.y * a.y : g.y);
  return mul2(mul2(n, r), u);
}

// 32 output columns of one row, as a warp: rounded to bf16 and stored as a
// whole 32 x 32 box by TMA where all 32 rows are the group's, else row by row.
__device__ __forceinline__ void store_bf16(const float (&v)[32], const Params& p,
                                           const CUtensorMap* tmC, int col0, int64_t row,
                                           int box_row, bool row_ok, bool box_full, uint32_t stg) {
  const int lane = threadIdx.x & 31;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = cvt_bf16x2(v[2 * i], v[2 * i + 1]);
  if (box_full) {
    if (lane == 0) bulk_wait_group_read<0>();
    __syncwarp();
    const uint32_t dst = stg + lane * 64;
    const uint32_t sw = (lane >> 1) & 3;
#pragma unroll
    for (int c4 = 0; c4 < 4; ++c4)
      st_shared_v4m(dst + ((c4 ^ sw) << 4),
                    make_uint4(w[4 * c4], w[4 * c4 + 1], w[4 * c4 + 2], w[4 * c4 + 3]));
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tmC, col0, box_row, stg);
      bulk_commit_group();
    }
  } else if (row_ok) {
    uint16_t* orow = static_cast<uint16_t*>(p.out) + row * p.N;
#pragma unroll
    for (int c4 = 0; c4 < 4; ++c4)
      if (col0 + c4 * 8 + 8 <= p.N)
        *reinterpret_cast<uint4*>(orow + col0 + c4 * 8) =
            make_uint4(w[4 * c4], w[4 * c4 + 1], w[4 * c4 + 2], w[4 * c4 + 3]);
  }
}

// The same in fp32, as two boxes of 16 columns through the warp's one buffer.
__device__ __forceinline__ void store_f32(const float (&v)[32], const Params& p,
                                          const CUtensorMap* tmC, int col0, int64_t row,
                                          int box_row, bool row_ok, bool box_full, uint32_t stg) {
  const int lane = threadIdx.x & 31;
  if (box_full) {
    const uint32_t dst = stg + lane * 64;
    const uint32_t sw = (lane >> 1) & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (col0 + 16 * h >= p.N) break;
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const float* f = v + 16 * h + 4 * c4;
        st_shared_v4m(dst + ((c4 ^ sw) << 4),
                      make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                 __float_as_uint(f[3])));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(tmC, col0 + 16 * h, box_row, stg);
        bulk_commit_group();
      }
    }
  } else if (row_ok) {
    float* orow = static_cast<float*>(p.out) + row * p.N + col0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col0 + 4 * i < p.N)  // N is a multiple of 8
        *reinterpret_cast<float4*>(orow + 4 * i) =
            make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
}

// A block of 32 values of one row -> its codes and scale.
__device__ __forceinline__ uint4 quantize_block(const float (&v)[32], uint32_t& s) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max3_abs(v[2 * i], v[2 * i + 1], m);
  s = mx_scale_code(__float_as_uint(m));
  const float inv = mx_inv_scale(s);
  const float2 inv2 = make_float2(inv, inv);
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = mul2(make_float2(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]), inv2);
    q[i] = mx_cvt8(f[0].x, f[0].y, f[1].x, f[1].y, f[2].x, f[2].y, f[3].x, f[3].y);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}
__device__ __forceinline__ uint32_t ld_shared_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// 32 output columns out of TMEM: 32 accumulator columns, or (SWIGLU) the 32
// gate columns and the 32 up columns behind them.  The wait names the
// registers, so that no use of them can move above it.
template <bool SWIGLU>
__device__ __forceinline__ void load_chunk(uint32_t taddr, float (&v)[32]) {
  uint32_t ra[32];
  tmem_ld_32cols(taddr, ra);
  if constexpr (SWIGLU) {
    uint32_t ua[32];
    tmem_ld_32cols(taddr + 32, ua);
    tc_wait_ld_regs(ra);
    tc_wait_ld_regs(ua);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float2 h = silu_mul2(make_float2(__uint_as_float(ra[i]), __uint_as_float(ra[i + 1])),
                                 make_float2(__uint_as_float(ua[i]), __uint_as_float(ua[i + 1])));
      v[i] = h.x;
      v[i + 1] = h.y;
    }
  } else {
    tc_wait_ld_regs(ra);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(ra[i]);
  }
}

// What the epilogue writes (kF32: plain product only).
enum Out { kBf16 = 0, kRecords = 1, kF32 = 2 };

// Shared memory of the epilogue: a 2 KiB box per warp (bf16, fp32), or per row
// quadrant two buffers of 32 rows x 48 bytes of codes and 4 of scales.
constexpr int kQuadBuf = 32 * (16 * kMxTileChunks + 4);
template <int OUT>
__host__ __device__ constexpr int epi_bytes() {
  return OUT == kRecords ? (4 * 2 * kQuadBuf + 1023) / 1024 * 1024 : kEpiWarps * kEpiBox;
}

// One CTA's 128 rows of a finished tile, for epilogue warp `w` of kEpiWarps
// (row quadrant = warp index mod 4; three warps share a quadrant's columns).
// release() is called once by every warp, as soon as it has its last values
// out of TMEM.
//
// Quantised output: a warp holds 32 rows of one block each, and storing those
// straight from registers touches 32 lines with each instruction.  So the
// three warps of a quadrant collect the tile's codes and scales in shared
// memory and store them row by row, up to 48 bytes a row from neighbouring
// lanes (XL gate_up at T=16384: 92.4 instead of 95.8 us).  One named barrier a tile (the
// two buffers alternate); a warp whose wait gave up (`live` false) still goes
// through it.
template <bool SWIGLU, int OUT, class Release>
__device__ __forceinline__ void epilogue_tile(const Params& p, const CUtensorMap* tmC, int w,
                                              uint32_t acc_tmem, int row0, int nrows, int chunk0,
                                              int chunks, uint32_t epi, int& buf, bool live,
                                              Release release) {
  const int quad = w & 3, third = w >> 2;
  const int lane = threadIdx.x & 31;
  const int r = quad * 32 + lane;
  const uint32_t tquad = acc_tmem + (static_cast<uint32_t>(quad * 32) << 16);
  if (quad * 32 >= nrows) {
    release();
    return;
  }
  if constexpr (OUT == kRecords) {
    static_assert(SWIGLU && kEpiWarps / 4 >= kMxTileChunks, "a chunk a warp");
    const uint32_t codes = epi + (quad * 2 + buf) * kQuadBuf;
    buf ^= 1;  // per tile that the quadrant takes part in: the barrier is between two uses
    const uint32_t scales = codes + 32 * 16 * kMxTileChunks;
    if (third < chunks && live) {
      float v[32];
      load_chunk<true>(tquad + 64 * third, v);
      release();
      uint32_t s;
      const uint4 q = quantize_block(v, s);
      st_shared_v4m(codes + lane * (16 * kMxTileChunks) + third * 16, q);
      asm volatile("st.shared.u8 [%0], %1;" ::"r"(scales + lane * 4 + third), "r"(s) : "memory");
    } else {
      release();
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + quad), "n"(8 * kEpiWarps) : "memory");
    // piece i: 16 bytes of codes, and the scale, of row i / chunks
    const int i = third * 32 + lane;
    if (i < 32 * chunks && live) {
      const int row = chunks == 3 ? i / 3 : chunks == 2 ? i >> 1 : i;
      const int col = i - row * chunks;
      const int blk = chunk0 + col;  // block of the output row
      if (quad * 32 + row < nrows && blk * 32 < p.N) {
        const int row_bytes = mx_row_bytes(p.N), cb = mx_code_bytes(p.N), ns = mx_num_scales(p.N);
        uint8_t* orow = static_cast<uint8_t*>(p.out) +
                        (static_cast<int64_t>(row0) + quad * 32 + row) * row_bytes;
        *reinterpret_cast<uint4*>(orow + blk * 16) =
            ld_shared_v4(codes + row * (16 * kMxTileChunks) + col * 16);
        orow[cb + blk] = static_cast<uint8_t>(ld_shared_u8(scales + row * 4 + col));
        if (blk == ns - 1)
          for (int b = cb + ns; b < row_bytes; ++b) orow[b] = 0;
      }
    }
  } else {
    constexpr int kPer = SWIGLU ? 1 : 2;  // 32-column outputs of a chunk
    const int end = live ? min(chunks * kPer, cdiv(p.N, 32) - chunk0 * kPer) : 0;
    if (third >= end) release();
#pragma unroll 1
    for (int c = third; c < end; c += kEpiWarps / 4) {
      float v[32];
      load_chunk<SWIGLU>(tquad + (SWIGLU ? 64 : 32) * c, v);
      if (c + kEpiWarps / 4 >= end) release();
      const int col0 = (chunk0 * kPer + c) * 32;
      const int64_t row = static_cast<int64_t>(row0) + r;
      const bool full = (quad + 1) * 32 <= nrows;
      if constexpr (OUT == kF32)
        store_f32(v, p, tmC, col0, row, row0 + quad * 32, r < nrows, full, epi + w * kEpiBox);
      else
        store_bf16(v, p, tmC, col0, row, row0 + quad * 32, r < nrows, full, epi + w * kEpiBox);
    }
  }
}

// ------------------------------------------------------------ host side ----
bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t rows,
              uint64_t cols, uint64_t stride, uint32_t box_rows, uint32_t box_cols,
              CUtensorMapSwizzle swizzle);
// Codes [rows, cols bytes] with a row stride, boxes of box_rows x 128 bytes.
inline bool make_code_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols,
                          uint64_t stride, uint32_t box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, cols, stride, box_rows, kRowB,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}
// Whole records, boxes of box_rows x 16 bytes (the scales of two k-blocks).
inline bool make_raw_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t row_bytes,
                         uint32_t box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, row_bytes, row_bytes, box_rows, 16,
                  CU_TENSOR_MAP_SWIZZLE_NONE);
}
// Scale atoms of 512 bytes, boxes of several.
inline bool make_scale_map(CUtensorMap* map, const void* base, uint64_t atoms, uint32_t box) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, atoms, 128, 512, box, 128,
                  CU_TENSOR_MAP_SWIZZLE_NONE);
}
// Output [rows, cols], boxes of 32 rows x 64 bytes.
inline bool make_out_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, bool f32) {
  return make_map(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base,
                  rows, cols, cols * (f32 ? 4 : 2), 32, f32 ? 16 : 32, CU_TENSOR_MAP_SWIZZLE_64B);
}
inline Params make_params(const MxGemmArgs& a) {
  Params p;
  p.a_rows = static_cast<const uint8_t*>(a.rows);
  p.b_scales = static_cast<const uint8_t*>(a.weight) +
               mx_weight_scale_offset(a.G, a.N, a.K, a.swiglu);
  p.counts = a.counts;
  p.G = a.G;
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.a_row_bytes = mx_row_bytes(a.K);
  p.b_rows = mx_weight_rows(a.N, a.swiglu);
  p.b_chunks = cdiv(p.b_rows, 64);
  p.ct = mx_col_tiles(p.b_rows);
  p.out = a.out;
  p.err = a.err;
  p.wait_limit_ns = kWaitLimitNs;
  return p;
}

// Once per kernel and device: the shared-memory opt-in.
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, size_t bytes, int (&done)[64], std::mutex& mu) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (!done[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes));
    if (e != cudaSuccess) return e;
    done[dev] = 1;
  }
  return cudaSuccess;
}

}  // namespace mx

// 256-row tiles on CTA pairs (gemm_mxfp4_pair.cu), K of at most kPairKBlocks.
cudaError_t launch_grouped_gemm_mxfp4_pair(const MxGemmArgs& args, cudaStream_t st);

}  // namespace hmoe
