// Microscaled 4-bit floats: blocks of 32 values along a row share a power of two (a byte, 127 + e; 255: not a number), a value is 2^e times
// an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, 8 being the sign). Rows lie as the tensor cores read them:
//   codes   [rows, K / 2]: two to a byte, the even one in the low half;
//   scales  [tiles][chunks(K)][512]: a tile is 128 rows, a chunk 128 values, and row r's byte of block b of a chunk at
//           (r % 32) 16 + r / 32 * 4 + b: lanes of tensor memory are r % 32, columns r / 32 (tcgen05.cp 32x128b.warpx4). Chunks are an
//           even number, those past K are zeros. Rows of several experts begin a tile each, so tile numbers follow from the plan's offsets.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace mx {

constexpr int BLOCK = 32, TILE = 128, CHUNK = 128, ATOM = 512;

__host__ __device__ constexpr int chunks(int k) { return (k + 2 * CHUNK - 1) / (2 * CHUNK) * 2; }
// where a row of a tile has its bytes
__host__ __device__ constexpr int row_at(int r) { return (r % 32) * 16 + r / 32 * 4; }

// The scale's byte of a block whose largest magnitude has these bits: floor(log2) - 2, and 255 for infinities and what is not a number.
__device__ __forceinline__ uint32_t scale_of(uint32_t top_bits) {
  const uint32_t e = top_bits >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^-e of a scale's byte (255: anything): exact as a float, and so is its product with a value that does not become zero as a code
__device__ __forceinline__ float inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }
// 2^-e from the bits of the block's largest magnitude: inverse(scale_of(top_bits)), but for what is not finite, where anything will do
__device__ __forceinline__ float inverse_of(uint32_t top_bits) { return __uint_as_float(min(0x80000000u - (top_bits & 0x7f800000u), 0x7f000000u)); }
__device__ __forceinline__ float value_of(uint32_t scale) {
  return __uint_as_float(scale == 0 ? 0x00400000u : scale == 255 ? 0x7fffffffu : scale << 23);
}
// eight values to codes, nearest with ties to even, 6 at most
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// what eight codes stand for
__device__ __forceinline__ void values8(uint32_t codes, float scale, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n.reg .b8 a, b, c, d;\n"
      "mov.b32 {a, b, c, d}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
  }
}

// Eight values as they are read, their largest magnitude's bits as a float's, and themselves as floats.
template <typename T> struct Eight;
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ uint32_t top() const {
    float v[8];
    floats(v);
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(v[i]) & 0x7fffffffu);
    return t;
  }
};
template <> struct Eight<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ uint32_t top() const {       // two 16-bit halves at a time: bits of magnitudes are in the order of the magnitudes
    constexpr uint32_t M = 0x7fff7fffu;
    const uint32_t t = __vmaxu2(__vmaxu2(w.x & M, w.y & M), __vmaxu2(w.z & M, w.w & M));
    return max(t & 0xffff0000u, t << 16);
  }
};

// A warp's span of 256 values, eight a lane: the lane's codes, and its block's scale (four lanes have a block).
template <typename T> __device__ __forceinline__ uint32_t quantize(const Eight<T>& x, uint32_t& scale) {
  uint32_t top = x.top();
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  scale = scale_of(top);
  const float by = inverse_of(top);
  float v[8];
  x.floats(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= by;
  return codes8(v);
}
// The scales of the four blocks of this half of the warp as a word.
__device__ __forceinline__ uint32_t four_scales(uint32_t scale, int lane) {
  uint32_t word = scale << (lane / 4 % 4 * 8);
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  return word | __shfl_xor_sync(0xffffffffu, word, 8);
}

// The tile of a row of expert-sorted rows and its place there, by a whole warp; `offsets` null: one run of rows. False: behind the last expert's rows.
__device__ __forceinline__ bool place_of(const int* offsets, int experts, int row, int& tile, int& at) {
  if (!offsets) {
    tile = row / TILE;
    at = row_at(row % TILE);
    return true;
  }
  const int lane = threadIdx.x & 31;
  int tiles = 0, first = 0;
  for (int e = lane; e < experts; e += 32) {
    const int a = offsets[e], b = offsets[e + 1];
    if (b <= row) tiles += (b - a + TILE - 1) / TILE;
    else if (a <= row) first = a + 1;
  }
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  const int found = (int)__reduce_max_sync(0xffffffffu, first);
  first = row - found + 1;
  tile = tiles + first / TILE;
  at = row_at(first % TILE);
  return found > 0;
}

}  // namespace mx
