// Codes of four bits as operands of mma.sync, without a conversion. A bfloat16 with the bits 0000 0000 0cccc is the denormal
// c * 2^-133, and one with the bits 0000 0000 cccc0000 is 16 c * 2^-133 (its lowest exponent bit has the weight that the next
// mantissa bit would have), so a word of eight codes is four pairs after four ANDs and one shift; the other operand is multiplied by
// 2^64 (2^60 against the second kind), which is exact, and the float32 sum is that of the integers times 2^-69. Products with
// denormals are exact on the tensor cores. (128 + c in the mantissa and a subtraction: 11 instructions a word instead of 5.)
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "mma.cuh"

namespace fb {

constexpr unsigned LOW = 0x000f000fu, HIGH = 0x00f000f0u;      // pairs of codes: times 1 and times 16
// a sum of products of 2^64 x and codes, put back to its size
constexpr float UNSCALE = 590295810358705651712.f;             // 2^69

__device__ __forceinline__ unsigned times(unsigned pair, unsigned by) {
  unsigned r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(by));
  return r;
}
// a pair of bfloat16 times 2^64 or 2^60
__device__ __forceinline__ unsigned raised(unsigned pair, bool by_60) { return times(pair, by_60 ? 0x5d805d80u : 0x5f805f80u); }
// c[0..3] += rows (word_a: rows lane / 4, word_b: rows + 8) of 32 codes a row, eight a lane, times eight columns: x holds the lane's
// eight elements of its column (lane / 4), raised by 64, 60, 64, 60
__device__ __forceinline__ void mma_codes(float (&c)[4], unsigned word_a, unsigned word_b, const uint4& x) {
  const unsigned a0[4] = {word_a & LOW, word_b & LOW, word_a & HIGH, word_b & HIGH};
  hb::mma_bf16(c, a0, x.x, x.y);
  word_a >>= 8;
  word_b >>= 8;
  const unsigned a1[4] = {word_a & LOW, word_b & LOW, word_a & HIGH, word_b & HIGH};
  hb::mma_bf16(c, a1, x.z, x.w);
}
// the first products of a sum
__device__ __forceinline__ void mma_first(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_codes_first(float (&c)[4], unsigned word_a, unsigned word_b, const uint4& x) {
  const unsigned a0[4] = {word_a & LOW, word_b & LOW, word_a & HIGH, word_b & HIGH};
  mma_first(c, a0, x.x, x.y);
  word_a >>= 8;
  word_b >>= 8;
  const unsigned a1[4] = {word_a & LOW, word_b & LOW, word_a & HIGH, word_b & HIGH};
  hb::mma_bf16(c, a1, x.z, x.w);
}
__device__ __forceinline__ uint4 raised(const uint4& x) {
  return make_uint4(raised(x.x, false), raised(x.y, true), raised(x.z, false), raised(x.w, true));
}

// ---- blocks of 16 cached rows (tokens) of one key/value head, G groups of 32 dims: 640 G bytes
//   keys' codes    [16 rows][4 lanes][G words]: the word holds dims 8 lane .. 8 lane + 7 of its group, even dims in the lower half
//   values' codes  [2][8 lanes][4 pairs of rows][G words]: dims 4 lane .. 4 lane + 3 of its group of the even row in the lower half
//   scales         [16 rows][keys' G, values' G] bfloat16
//   keys' lows     [16 rows][G] bfloat16
//   values' lows   [G][16 rows] bfloat16
constexpr int GROUP = 32, BLOCK_ROWS = 16;
template <int G> struct Block {
  static constexpr int K = 0, V = 256 * G, SCALES = 512 * G, K_LOW = 576 * G, V_LOW = 608 * G, BYTES = 640 * G;
  static __host__ __device__ constexpr int key_word(int row, int lane, int group) { return K + ((row * 4 + lane) * G + group) * 4; }
  static __host__ __device__ constexpr int value_word(int row, int lane, int group) {
    return V + (((row >> 3) * 32 + lane * 4 + ((row >> 1) & 3)) * G + group) * 4;
  }
  static __host__ __device__ constexpr int scale(int row, int is_v, int group) { return SCALES + (row * 2 * G + is_v * G + group) * 2; }
  static __host__ __device__ constexpr int key_low(int row, int group) { return K_LOW + (row * G + group) * 2; }
  static __host__ __device__ constexpr int value_low(int row, int group) { return V_LOW + (group * 16 + row) * 2; }
};

}  // namespace fb
