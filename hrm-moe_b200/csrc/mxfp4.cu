// MXFP4 rows: quantise, dequantise, pack weights, and the combine of the
// quantised expert path.  All are single passes bound by HBM (or, for a few
// rows, by the launch).
#include "internal.h"
#include "mxfp4.cuh"

namespace hmoe {
namespace {

constexpr int kQThreads = 256;

// One thread per block of 32: the maximum and the scale are the thread's own,
// its 16 bytes of codes are one store.  The kernels are short of instruction
// slots before they are short of bandwidth, so the work is kept in packed
// bf16 pairs.  (Four lanes to a block, 8 elements each, took 126 instructions
// per 8 elements and 20 us for [16384, 1536] bf16; the way back, element by
// element, 238 and 28 us.  Now both in a row take 19.8 us for 127 MB, at the
// copy bandwidth: the codes stay in L2.)  A CTA takes whole rows, so that one
// 32-bit multiply finds a block's row.
struct RowSplit {
  int rows_per_cta, blocks;  // blocks of a row
  uint32_t magic;            // ceil(2^32 / blocks)
};
RowSplit row_split(int blocks) {
  RowSplit r;
  r.blocks = blocks;
  r.rows_per_cta = blocks < kQThreads ? kQThreads / blocks : 1;
  r.magic = static_cast<uint32_t>(((1ull << 32) + blocks - 1) / blocks);
  return r;
}
// Row of block i of a CTA.  Exact: with several rows to a CTA, i * blocks <
// 2 * kQThreads^2 < 2^32; with one row it is 0, and with one block to a row
// (whose magic number does not fit) it is i.
__device__ __forceinline__ int block_row(const RowSplit& sp, int i) {
  if (sp.rows_per_cta == 1) return 0;
  return sp.blocks == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), sp.magic));
}

// WIDE: whole blocks, rows 32-byte aligned (two or four 32-byte loads a block);
// else 16-byte loads, each of which may lie behind K (a multiple of 8).
template <bool BF16, bool WIDE>
__global__ void __launch_bounds__(kQThreads)
quantize_kernel(const void* x, int64_t rows, int K, int64_t x_stride, RowSplit sp, uint8_t* out,
                int* clear_err) {
  grid_dependency_wait();  // launched early (launch_pdl)
  grid_launch_dependents();
  if (clear_err && blockIdx.x == 0 && threadIdx.x == 0) *clear_err = 0;
  const int row_bytes = mx_row_bytes(K), cb = mx_code_bytes(K);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * sp.rows_per_cta;
  const int nrows = static_cast<int>(rows - row0 < sp.rows_per_cta ? rows - row0 : sp.rows_per_cta);
  const int total = nrows * sp.blocks;
  for (int i = threadIdx.x; i < total; i += kQThreads) {
    const int r = block_row(sp, i);
    const int b = i - r * sp.blocks;
    uint32_t s;
    const uint4 q = mx_quantize_row_block<BF16, WIDE>(
        static_cast<const uint8_t*>(x) + (row0 + r) * x_stride * (BF16 ? 2 : 4), b, K, s);
    uint8_t* o = out + (row0 + r) * row_bytes;
    reinterpret_cast<uint4*>(o)[b] = q;
    o[cb + b] = static_cast<uint8_t>(s);
    if (b == sp.blocks - 1)
      for (int z = cb + sp.blocks; z < row_bytes; ++z) o[z] = 0;
  }
}

// Four codes (the low 16 bits of w) -> their values as two bf16 pairs: the
// bytes of the eight magnitudes are looked up by byte permutes, the sign bits
// likewise.
__device__ __forceinline__ void values4(uint32_t w, uint32_t& v01, uint32_t& v23) {
  const uint32_t sel = w & 0x7777u;
  // 0, .5, 1, 1.5, 2, 3, 4, 6: 0x0000 3f00 3f80 3fc0 4000 4040 4080 40c0
  const uint32_t lo = __byte_perm(0xc0800000u, 0xc0804000u, sel);
  const uint32_t hi = __byte_perm(0x3f3f3f00u, 0x40404040u, sel) |
                      __byte_perm(0x00008000u, 0u, (w >> 3) & 0x1111u);
  v01 = __byte_perm(lo, hi, 0x5140u);
  v23 = __byte_perm(lo, hi, 0x7362u);
}

// WIDE: whole blocks, 32-byte aligned output rows.
template <bool BF16, bool WIDE>
__global__ void __launch_bounds__(kQThreads)
dequantize_kernel(const uint8_t* rows_in, int64_t rows, int K, RowSplit sp, void* out) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int row_bytes = mx_row_bytes(K), cb = mx_code_bytes(K);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * sp.rows_per_cta;
  const int nrows = static_cast<int>(rows - row0 < sp.rows_per_cta ? rows - row0 : sp.rows_per_cta);
  const int total = nrows * sp.blocks;
  for (int i = threadIdx.x; i < total; i += kQThreads) {
    const int r = block_row(sp, i);
    const int b = i - r * sp.blocks;
    const uint8_t* row = rows_in + (row0 + r) * row_bytes;
    const uint4 c = ld_16bytes(row + 16 * b);
    const uint32_t s = row[cb + b];
    // the scale in bf16: 2^-127 is a subnormal, 255 is NaN
    const uint32_t sb = s == 255u ? 0x7fc0u : s == 0u ? 0x0040u : s << 7;
    const uint32_t s2 = sb | sb << 16;
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t v[16];  // exact: two significant bits, and 2^-128 is a bf16 subnormal
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      values4(w[j], v[4 * j], v[4 * j + 1]);
      values4(w[j] >> 16, v[4 * j + 2], v[4 * j + 3]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = mul_bf16x2(v[j], s2);
    constexpr int ES = BF16 ? 2 : 4;
    uint8_t* dst = static_cast<uint8_t*>(out) + ((row0 + r) * K + b * kMxBlock) * ES;
    constexpr int kParts = BF16 ? 4 : 8;  // 16-byte stores
#pragma unroll
    for (int h = 0; h < kParts; h += 2) {
      uint4 q[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (BF16)
          q[g] = make_uint4(v[4 * ((h + g) % 4)], v[4 * ((h + g) % 4) + 1], v[4 * ((h + g) % 4) + 2],
                            v[4 * ((h + g) % 4) + 3]);
        else
          q[g] = make_uint4(v[2 * (h + g)] << 16, v[2 * (h + g)] & 0xffff0000u,
                            v[2 * (h + g) + 1] << 16, v[2 * (h + g) + 1] & 0xffff0000u);
      }
      if (WIDE) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 16 * h),
                     "r"(q[0].x), "r"(q[0].y), "r"(q[0].z), "r"(q[0].w), "r"(q[1].x), "r"(q[1].y),
                     "r"(q[1].z), "r"(q[1].w)
                     : "memory");
      } else {
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (b * kMxBlock + (h + g) * (16 / ES) < K)
            *reinterpret_cast<uint4*>(dst + 16 * (h + g)) = q[g];
      }
    }
  }
}

// Packed row n' of a group -> the source row it comes from, -1 for padding.
__device__ __forceinline__ int packed_source_row(int np, int N, int swiglu) {
  if (!swiglu) return np;
  const int f = (np >> 6) * 32 + (np & 31);  // feature; rows alternate 32 gate, 32 up
  if (f >= N) return -1;
  return (np & 32) ? N + f : f;
}

// Once per weight: codes row by row, 16 bytes a thread, then the scale atoms
// byte by byte.
__global__ void __launch_bounds__(kQThreads)
pack_weight_kernel(const uint8_t* __restrict__ codes, int64_t code_stride,
                   const uint8_t* __restrict__ scales, int64_t scale_stride, int G, int N, int K,
                   int swiglu, uint8_t* __restrict__ out_codes, uint8_t* __restrict__ out_scales) {
  const int np_rows = mx_weight_rows(N, swiglu), src_rows = swiglu ? 2 * N : N;
  const int cb = mx_code_bytes(K), ns = mx_num_scales(K);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kQThreads;
  const int chunks = cb / 16;
  const int64_t ncode = static_cast<int64_t>(G) * np_rows * chunks;
  for (int64_t i = first; i < ncode; i += step) {
    const int64_t gr = i / chunks;
    const int c = static_cast<int>(i - gr * chunks);
    const int64_t g = gr / np_rows;
    const int src = packed_source_row(static_cast<int>(gr - g * np_rows), N, swiglu);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (src >= 0)
      v = *reinterpret_cast<const uint4*>(codes + (g * src_rows + src) * code_stride + c * 16);
    reinterpret_cast<uint4*>(out_codes)[i] = v;
  }
  const MxColTiles ct = mx_col_tiles(np_rows);
  const int nkb = mx_num_kblocks(K);
  const int atoms = cdiv(np_rows, 64) * nkb;  // of a group
  const int64_t nscale = static_cast<int64_t>(G) * atoms * 512;
  for (int64_t i = first; i < nscale; i += step) {
    const int byte = static_cast<int>(i & 511);
    const int64_t g = (i >> 9) / atoms;
    const int r = static_cast<int>((i >> 9) - g * atoms);
    // tile, k-block and atom of the tile's atoms of that k-block
    const int split = ct.extra * (ct.chunks + 1) * nkb;  // atoms of the longer tiles
    const int t = r < split ? r / ((ct.chunks + 1) * nkb) : ct.extra + (r - split) / (ct.chunks * nkb);
    const int nc = ct.count(t);
    const int rt = r - ct.first(t) * nkb;
    const int kb = rt / nc;
    const int col = (rt - kb * nc) * 4 + ((byte >> 2) & 3);  // TMEM column of the tile
    const int j = col / (2 * nc);                             // which 128 elements
    const int np = ct.first(t) * 64 + (col - j * 2 * nc) * 32 + (byte >> 4);
    const int k0 = kb * 8 + j * 4 + (byte & 3);
    uint8_t v = 0;
    if (np < np_rows && k0 < ns) {
      const int src = packed_source_row(np, N, swiglu);
      if (src >= 0) v = scales[(g * src_rows + src) * scale_stride + k0];
    }
    out_scales[i] = v;
  }
}

// y[t] = [final[t] +] sum over j of w[t, j] * row pos[t, j], in fp32, rounded
// once.  Unlike combine_kernel, which repeats the roundings of the
// reference's bf16 products and running sums, nothing here has a bf16
// intermediate: the rows are the products' fp32 sums.  A warp per 32 chunks of
// 8 columns of a token's row; four rows of a chunk are loaded before they are
// summed, in slot order.  Bound by reading the rows: XL 64x8 at
// T=16384 856 MB in 139 us, 0.96 of the copy bandwidth.
// Four CTAs an SM, 64 registers a thread, five words of them spilled: with
// three and no spills the whole path takes 62 instead of 63 us at T=1000, 164
// instead of 155 at T=4200 and the same at 16384.
__global__ void __launch_bounds__(kQThreads, 4)
combine_f32_kernel(const float* rows, const int32_t* pos, const void* topk_w, int topk_w_is_f32,
                   int64_t T, int row_chunks, int k, int warps_per_token, const uint4* final_in,
                   uint4* out) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * (kQThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = wid / warps_per_token;
  if (t >= T) return;
  const int cw = static_cast<int>(wid - t * warps_per_token);
  int p = -1;
  float w = 0.0f;
  if (lane < k) {
    p = pos[t * k + lane];
    w = topk_w_is_f32 ? static_cast<const float*>(topk_w)[t * k + lane]
                      : bf16_bits_to_f32(static_cast<const uint16_t*>(topk_w)[t * k + lane]);
  }
  constexpr int kBatch = 4;
  for (int c0 = cw * 32; c0 < row_chunks; c0 += warps_per_token * 32) {
    const int c = c0 + lane;
    const bool live = c < row_chunks;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    if (final_in && live) {
      const uint4 u = final_in[t * row_chunks + c];
      const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { acc[2 * i] = bf16_lo(q[i]); acc[2 * i + 1] = bf16_hi(q[i]); }
    }
    for (int j0 = 0; j0 < k; j0 += kBatch) {
      uint4 v[kBatch][2];
      float ws[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int pj = __shfl_sync(0xffffffffu, p, (j0 + b) & 31);
        ws[b] = __shfl_sync(0xffffffffu, w, (j0 + b) & 31);
        const bool use = j0 + b < k && pj >= 0;
        if (!use) ws[b] = 0.0f;  // a dropped assignment adds nothing, whatever its weight
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[b][h] = live && use
                        ? ld_16bytes(rows + (static_cast<int64_t>(pj) * row_chunks + c) * 8 + 4 * h)
                        : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t q[4] = {v[b][h].x, v[b][h].y, v[b][h].z, v[b][h].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[4 * h + i] = fmaf(ws[b], __uint_as_float(q[i]), acc[4 * h + i]);
        }
      }
    }
    if (live)
      out[t * row_chunks + c] = make_uint4(cvt_bf16x2(acc[0], acc[1]), cvt_bf16x2(acc[2], acc[3]),
                                           cvt_bf16x2(acc[4], acc[5]), cvt_bf16x2(acc[6], acc[7]));
  }
}

unsigned stream_blocks(int64_t threads) {
  const int64_t want = cdiv64(threads, kQThreads);
  const int64_t most = static_cast<int64_t>(num_sms_for_current_device()) * 64;
  return static_cast<unsigned>(want < most ? (want > 0 ? want : 1) : most);
}

}  // namespace

cudaError_t launch_mx_quantize(const void* x, int64_t rows, int K, int64_t x_stride, int dtype,
                               void* out, int* clear_err, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const RowSplit sp = row_split(mx_num_scales(K));
  const int64_t ctas = cdiv64(rows, sp.rows_per_cta);
  if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
  const bool bf16 = dtype == kDtypeBF16;
  const bool wide = K % kMxBlock == 0 && reinterpret_cast<uintptr_t>(x) % 32 == 0 &&
                    x_stride * (bf16 ? 2 : 4) % 32 == 0;
  const auto kernel = bf16 ? (wide ? quantize_kernel<true, true> : quantize_kernel<true, false>)
                           : (wide ? quantize_kernel<false, true> : quantize_kernel<false, false>);
  return launch_pdl(kPdlDispatch, kernel, dim3(static_cast<unsigned>(ctas)), dim3(kQThreads), 0, st,
                    x, rows, K, x_stride, sp, static_cast<uint8_t*>(out), clear_err);
}

cudaError_t launch_mx_dequantize(const void* rows_in, int64_t rows, int K, int dtype, void* out,
                                 cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const RowSplit sp = row_split(mx_num_scales(K));
  const int64_t ctas = cdiv64(rows, sp.rows_per_cta);
  if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
  const bool bf16 = dtype == kDtypeBF16;
  const bool wide = K % kMxBlock == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  const auto kernel = bf16 ? (wide ? dequantize_kernel<true, true> : dequantize_kernel<true, false>)
                           : (wide ? dequantize_kernel<false, true> : dequantize_kernel<false, false>);
  return launch_pdl(kPdlDispatch, kernel, dim3(static_cast<unsigned>(ctas)), dim3(kQThreads), 0, st,
                    static_cast<const uint8_t*>(rows_in), rows, K, sp, out);
}

cudaError_t launch_mx_pack_weight(const void* codes, int64_t code_stride, const void* scales,
                                  int64_t scale_stride, int G, int N, int K, int swiglu, void* out,
                                  cudaStream_t st) {
  uint8_t* o = static_cast<uint8_t*>(out);
  const int64_t threads = static_cast<int64_t>(G) * mx_weight_rows(N, swiglu) *
                          (mx_code_bytes(K) / 16);
  pack_weight_kernel<<<stream_blocks(threads), kQThreads, 0, st>>>(
      static_cast<const uint8_t*>(codes), code_stride, static_cast<const uint8_t*>(scales),
      scale_stride, G, N, K, swiglu, o, o + mx_weight_scale_offset(G, N, K, swiglu));
  return cudaGetLastError();
}

cudaError_t launch_combine_f32(const float* rows, const int32_t* pos, const void* topk_w,
                               int topk_w_is_f32, int64_t T, int d, int k, const void* final_in,
                               void* out, cudaStream_t st) {
  if (T == 0) return cudaSuccess;
  const int row_chunks = d / 8;
  // a row over several warps, so that enough loads are in flight (with the
  // dispatch's rows likewise, the experts of XL 64x8: T=300 55.7 -> 45.8 us,
  // 2000 94.8 -> 86.7, 16384 459 -> 454)
  const int wpt = cdiv(row_chunks, 32);
  const int64_t blocks = cdiv64(T * wpt, kQThreads / 32);
  return launch_pdl(kPdlCombine, combine_f32_kernel, dim3(static_cast<unsigned>(blocks)),
                    dim3(kQThreads), 0, st, rows, pos, topk_w, topk_w_is_f32, T, row_chunks, k, wpt,
                    static_cast<const uint4*>(final_in), static_cast<uint4*>(out));
}

}  // namespace hmoe
