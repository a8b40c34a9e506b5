// MXFP4 rows: quantise, dequantise, pack weights, and the combine of the
// quantised expert path.  All are single passes bound by HBM (or, for a few
// rows, by the launch).
#include "internal.h"
#include "mxfp4.cuh"

namespace hmoe {
namespace {

constexpr int kQThreads = 256;

// |x| of two bf16 as bits: the maximum of bf16 magnitudes orders as unsigned
// 16-bit integers, NaN above everything.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __vmaxu2(a, b);
}

// One thread per 8 elements (a 16-byte load of bf16, two of fp32), four lanes
// per block of 32: the block's maximum is two shuffles, a lane's 8 codes are
// one 32-bit word, and lane 0 of the four stores the scale byte.  Elements
// past K are zeros; the lanes past the last block fill the record's padding.
template <bool BF16>
__global__ void __launch_bounds__(kQThreads)
quantize_kernel(const void* __restrict__ x, int64_t rows, int K, int64_t x_stride,
                uint8_t* __restrict__ out) {
  grid_dependency_wait();  // launched early (launch_pdl)
  grid_launch_dependents();
  const int row_bytes = mx_row_bytes(K);
  const int cb = mx_code_bytes(K), ns = mx_num_scales(K);
  const int lanes_per_row = 4 * ns;  // 8 elements each
  const int64_t total = rows * lanes_per_row;
  // every lane of a warp runs the same trip count (the shuffles see all lanes)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kQThreads + (threadIdx.x & ~31);
       base < total; base += static_cast<int64_t>(gridDim.x) * kQThreads) {
    const int64_t i = base + (threadIdx.x & 31);
    const bool live = i < total;
    const int64_t r = live ? i / lanes_per_row : 0;
    const int c = live ? static_cast<int>(i - r * lanes_per_row) : 0;  // 8-element chunk of the row
    float v[8];
    uint32_t amax = 0;
    if (live && c * 8 < K) {  // K is a multiple of 8
      if (BF16) {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) +
                                                        r * x_stride + c * 8);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
        const uint32_t m = max_u16x2(max_u16x2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                     max_u16x2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
        amax = max(m >> 16, m & 0xffffu) << 16;
      } else {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) +
                                                          r * x_stride + c * 8);
        const float4 a = p[0], b = p[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (!live) continue;  // whole groups of four lanes: total is a multiple of 4
    const uint32_t s = mx_scale_code(amax);
    const float inv = mx_inv_scale(s);
    uint8_t* row = out + r * row_bytes;
    reinterpret_cast<uint32_t*>(row)[c] =
        mx_cvt8(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, v[4] * inv, v[5] * inv, v[6] * inv,
                v[7] * inv);
    if ((c & 3) == 0) {
      row[cb + (c >> 2)] = static_cast<uint8_t>(s);
      if ((c >> 2) == ns - 1)
        for (int b = cb + ns; b < row_bytes; ++b) row[b] = 0;
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(kQThreads)
dequantize_kernel(const uint8_t* __restrict__ rows_in, int64_t rows, int K,
                  void* __restrict__ out) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int row_bytes = mx_row_bytes(K), cb = mx_code_bytes(K);
  const int chunks = K / 8;
  const int64_t total = rows * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kQThreads) {
    const int64_t r = i / chunks;
    const int c = static_cast<int>(i - r * chunks);
    const uint8_t* row = rows_in + r * row_bytes;
    const uint32_t w = reinterpret_cast<const uint32_t*>(row)[c];
    const uint32_t s = row[cb + (c >> 2)];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mx_value((w >> (4 * j)) & 15u, s);
    if (BF16) {
      // exact: two significant bits, and 2^-128 is a bf16 subnormal
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + r * K + c * 8) =
          make_uint4(cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3]), cvt_bf16x2(v[4], v[5]),
                     cvt_bf16x2(v[6], v[7]));
    } else {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + r * K + c * 8);
      p[0] = make_float4(v[0], v[1], v[2], v[3]);
      p[1] = make_float4(v[4], v[5], v[6], v[7]);
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
// intermediate to repeat.  One warp per (token, block of 32 16-byte columns);
// the k rows of a column block are loaded before they are summed, in slot
// order.
__global__ void __launch_bounds__(kQThreads, 4)
combine_f32_kernel(const uint4* __restrict__ rows, const int32_t* __restrict__ pos,
                   const void* __restrict__ topk_w, int topk_w_is_f32, int64_t T, int row_chunks,
                   int k, int warps_per_token, const uint4* final_in, uint4* out) {
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
  constexpr int kBatch = 8;
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
      uint4 v[kBatch];
      float ws[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int pj = j0 + b < k ? __shfl_sync(0xffffffffu, p, (j0 + b) & 31) : -1;
        ws[b] = __shfl_sync(0xffffffffu, w, (j0 + b) & 31);
        v[b] = live && pj >= 0 ? __ldg(rows + static_cast<int64_t>(pj) * row_chunks + c)
                               : make_uint4(0, 0, 0, 0);
        if (pj < 0) ws[b] = 0.0f;  // a dropped assignment adds nothing, whatever its weight
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const uint32_t q[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[2 * i] = fmaf(ws[b], bf16_lo(q[i]), acc[2 * i]);
          acc[2 * i + 1] = fmaf(ws[b], bf16_hi(q[i]), acc[2 * i + 1]);
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
                               void* out, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const dim3 grid(stream_blocks(rows * 4 * mx_num_scales(K)));
  if (dtype == kDtypeBF16)
    return launch_pdl(kPdlDispatch, quantize_kernel<true>, grid, dim3(kQThreads), 0, st, x, rows, K,
                      x_stride, static_cast<uint8_t*>(out));
  return launch_pdl(kPdlDispatch, quantize_kernel<false>, grid, dim3(kQThreads), 0, st, x, rows, K,
                    x_stride, static_cast<uint8_t*>(out));
}

cudaError_t launch_mx_dequantize(const void* rows_in, int64_t rows, int K, int dtype, void* out,
                                 cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const dim3 grid(stream_blocks(rows * (K / 8)));
  if (dtype == kDtypeBF16)
    return launch_pdl(kPdlDispatch, dequantize_kernel<true>, grid, dim3(kQThreads), 0, st,
                      static_cast<const uint8_t*>(rows_in), rows, K, out);
  return launch_pdl(kPdlDispatch, dequantize_kernel<false>, grid, dim3(kQThreads), 0, st,
                    static_cast<const uint8_t*>(rows_in), rows, K, out);
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

cudaError_t launch_combine_f32(const void* rows, const int32_t* pos, const void* topk_w,
                               int topk_w_is_f32, int64_t T, int d, int k, const void* final_in,
                               void* out, cudaStream_t st) {
  if (T == 0) return cudaSuccess;
  const int row_chunks = d * 2 / 16;
  // small T: a row over several warps, so that enough loads are in flight
  const int wpt = T < 4096 ? cdiv(row_chunks, 32) : 1;
  const int64_t blocks = cdiv64(T * wpt, kQThreads / 32);
  return launch_pdl(kPdlCombine, combine_f32_kernel, dim3(static_cast<unsigned>(blocks)),
                    dim3(kQThreads), 0, st, static_cast<const uint4*>(rows), pos, topk_w,
                    topk_w_is_f32, T, row_chunks, k, wpt, static_cast<const uint4*>(final_in),
                    static_cast<uint4*>(out));
}

}  // namespace hmoe
