// MXFP4 (OCP Microscaling Formats v1.0): e2m1 elements, one e8m0 scale per
// block of 32 along K.
//
// Activation rows are records: the codes (K' / 2 bytes, low nibble first,
// K' = K filled up to whole blocks), then one scale byte per block, the scale
// section filled up to 8 bytes and the record to 16 with zeros.  A record
// moves as one row copy (dispatch), its codes are 16-byte aligned for TMA, and
// the 8 scale bytes of a 256-element k-block are one aligned load.
//
// Packed weights: the codes [G, N', K' / 2] (for gate_up weights N' =
// 2 * ceil(I / 32) * 32 with 32 gate rows, then the 32 up rows of the same
// features, and so on, so that a column tile holds matching gate and up
// columns), then, 1024-byte aligned, the scales in the order of the GEMMs'
// column tiles.  A tile is a run of up to three 64-row chunks (the chunks of a
// group shared out evenly); its scales of a 256-element k-block are 4 TMEM
// columns a chunk: the columns of the first 128 elements (32 rows each, a
// 32-bit word of 4 scales per row), then those of the second.  Four columns
// are an atom of 512 bytes, 16 bytes for each of 32 lanes.
#pragma once

#include "common.cuh"

namespace hmoe {

constexpr int kMxBlock = 32;   // elements per scale
constexpr int kMxKBlock = 256;  // elements per 128-byte swizzled row of codes

__host__ __device__ inline int mx_padded_k(int K) { return (K + 31) / 32 * 32; }
__host__ __device__ inline int mx_code_bytes(int K) { return mx_padded_k(K) / 2; }
__host__ __device__ inline int mx_num_scales(int K) { return mx_padded_k(K) / 32; }
__host__ __device__ inline int mx_scale_bytes(int K) { return (mx_num_scales(K) + 7) / 8 * 8; }
__host__ __device__ inline int mx_row_bytes(int K) {
  return (mx_code_bytes(K) + mx_scale_bytes(K) + 15) / 16 * 16;
}
// Rows of one group's packed weight for N output columns.
__host__ __device__ inline int mx_weight_rows(int N, int swiglu) {
  return swiglu ? 2 * mx_padded_k(N) : N;
}
// Column tiles of a group: `tiles` runs of 64-row chunks, the first `extra`
// of them one longer than `chunks`.
constexpr int kMxTileChunks = 3;
struct MxColTiles {
  int tiles, chunks, extra;
  __host__ __device__ int first(int t) const { return t * chunks + (t < extra ? t : extra); }
  __host__ __device__ int count(int t) const { return chunks + (t < extra ? 1 : 0); }
};
__host__ __device__ inline MxColTiles mx_col_tiles(int rows) {
  const int chunks = cdiv(rows, 64);
  MxColTiles t;
  t.tiles = cdiv(chunks, kMxTileChunks);
  t.chunks = chunks / t.tiles;
  t.extra = chunks % t.tiles;
  return t;
}
__host__ __device__ inline int mx_num_kblocks(int K) { return cdiv(mx_padded_k(K), kMxKBlock); }
inline int64_t mx_weight_scale_offset(int G, int N, int K, int swiglu) {
  const int64_t codes = static_cast<int64_t>(G) * mx_weight_rows(N, swiglu) * mx_code_bytes(K);
  return (codes + 1023) / 1024 * 1024;
}
inline int64_t mx_weight_scale_atoms(int G, int N, int K, int swiglu) {
  return static_cast<int64_t>(G) * cdiv(mx_weight_rows(N, swiglu), 64) * mx_num_kblocks(K);
}
inline int64_t mx_weight_bytes(int G, int N, int K, int swiglu) {
  return mx_weight_scale_offset(G, N, K, swiglu) + mx_weight_scale_atoms(G, N, K, swiglu) * 512;
}

// Scale byte of a block whose largest magnitude has the fp32 bits `amax`
// (sign cleared): floor(log2 amax) - 2, the exponent of e2m1's largest power
// of two being 2, at least 2^-127; 255 (NaN) when the block holds an infinity
// or a NaN.  The maximum is taken on the bits: they order as the values do,
// and NaN comes out above everything.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale (exact: a power of two between 2^-125 and 2^127; 0 for NaN).
__device__ __forceinline__ float mx_inv_scale(uint32_t code) {
  return code == 255u ? 0.0f : __uint_as_float((254u - code) << 23);
}

// Eight values -> eight e2m1 codes in one word (v0 in the low nibble), round to
// nearest even, saturating at 6.
__device__ __forceinline__ uint32_t mx_cvt8(float v0, float v1, float v2, float v3, float v4,
                                            float v5, float v6, float v7) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
  return r;
}

// max(|a|, |b|, |c|), NaN if any is.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Loads of what the kernel before may have written: volatile, so that the
// compiler moves none of them above griddepcontrol.wait, whatever the
// qualifiers of the pointer that a kernel passes in.
__device__ __forceinline__ void ld_32bytes(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
        "=r"(w[7])
      : "l"(p)
      : "memory");
}
__device__ __forceinline__ uint4 ld_16bytes(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n\t.reg .b32 x;\n\tabs.bf16x2 x, %2;\n\tmax.NaN.bf16x2 %0, %1, x;\n\t}"
      : "=r"(r)
      : "r"(a), "r"(b));
  return r;
}

// Block b of a row of K values: codes, and the scale in s.  WIDE: whole blocks,
// 32-byte aligned rows; else 16-byte loads, each of which may lie behind K (a
// multiple of 8).
template <bool BF16, bool WIDE>
__device__ __forceinline__ uint4 mx_quantize_row_block(const uint8_t* row, int b, int K, uint32_t& s) {
  constexpr int kWords = BF16 ? 16 : 32;
  constexpr int ES = BF16 ? 2 : 4;
  uint32_t w[kWords];
  const uint8_t* src = row + b * (kMxBlock * ES);
  if (WIDE) {
#pragma unroll
    for (int h = 0; h < kWords / 8; ++h) ld_32bytes(src + 32 * h, w + 8 * h);
  } else {
#pragma unroll
    for (int h = 0; h < kWords / 4; ++h) {
      const uint4 q = b * kMxBlock + h * (16 / ES) < K ? ld_16bytes(src + 16 * h)
                                                      : make_uint4(0, 0, 0, 0);
      w[4 * h] = q.x; w[4 * h + 1] = q.y; w[4 * h + 2] = q.z; w[4 * h + 3] = q.w;
    }
  }
  uint32_t amax;
  if (BF16) {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int j = 1; j < 16; ++j) m = max_abs_bf16x2(m, w[j]);
    amax = max_abs_bf16x2(m, m >> 16) << 16;
  } else {
    float m = fabsf(__uint_as_float(w[0]));
#pragma unroll
    for (int j = 1; j < 31; j += 2)
      m = max3_abs(__uint_as_float(w[j % kWords]), __uint_as_float(w[(j + 1) % kWords]), m);
    amax = __float_as_uint(max3_abs(__uint_as_float(w[kWords - 1]), m, m));
  }
  s = mx_scale_code(amax);
  const float inv = mx_inv_scale(s);
  uint32_t q[4];
  if (BF16) {
    // x / s in bf16: exact (a power of two), or so small that its code is 0
    const uint32_t inv2 = cvt_bf16x2(inv, inv);
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = mul_bf16x2(w[j], inv2);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[j] = mx_cvt8(bf16_lo(w[4 * j]), bf16_hi(w[4 * j]), bf16_lo(w[4 * j + 1]),
                     bf16_hi(w[4 * j + 1]), bf16_lo(w[4 * j + 2]), bf16_hi(w[4 * j + 2]),
                     bf16_lo(w[4 * j + 3]), bf16_hi(w[4 * j + 3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[(8 * j + e) % kWords]) * inv;
      q[j] = mx_cvt8(f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]);
    }
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

}  // namespace hmoe
