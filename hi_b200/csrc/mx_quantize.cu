// Rows to microscaled 4-bit floats (mx.cuh) and back. Bound by memory: x is read once, codes and scales are a quarter of bfloat16.
#include "api.h"
#include "common.cuh"
#include "mx.cuh"

namespace {

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&two);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int SPAN = 256;          // values a warp takes at a time, eight a lane
constexpr int THREADS = 256;

// Row blockIdx.x (of `rows` in the order of `sorted_entry`, if there is one), SPANs blockIdx.y * 8 + warp, ... Four lanes have a block of 32.
template <typename T>
__global__ void __launch_bounds__(THREADS)
mx_quantize_kernel(const T* __restrict__ x, long long x_ld, int k, const int* __restrict__ sorted_entry, int top_k,
                   const int* __restrict__ offsets, int experts, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int span = blockIdx.y * (THREADS / 32) + warp, all = mx::chunks(k);
  if (span * 2 >= all) return;
  const size_t from = sorted_entry ? sorted_entry[row] / top_k : row;
  int tile, at;
  mx::place_of(offsets, experts, row, tile, at);
  const int k0 = span * SPAN + lane * 8;
  float v[8] = {};
  if (k0 < k) hb::load8(x + from * x_ld + k0, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t scale = mx::scale_of(top);
  const float by = scale == 255 ? 0.f : mx::inverse(scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = scale == 255 ? 0.f : v[i] * by;
  if (k0 < k) *reinterpret_cast<uint32_t*>(codes + (size_t)row * (k / 2) + k0 / 2) = mx::codes8(v);
  // the four blocks of 16 lanes: a word of scales
  uint32_t word = scale << (lane / 4 % 4 * 8);
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (lane % 16 == 0)
    *reinterpret_cast<uint32_t*>(scales + ((size_t)tile * all + span * 2 + lane / 16) * mx::ATOM + at) = word;
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
mx_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int k, const int* __restrict__ offsets, int experts,
                 T* __restrict__ out) {
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int span = blockIdx.y * (THREADS / 32) + warp, all = mx::chunks(k);
  if (span * 2 >= all) return;
  int tile, at;
  mx::place_of(offsets, experts, row, tile, at);
  const int k0 = span * SPAN + lane * 8;
  if (k0 >= k) return;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + (size_t)row * (k / 2) + k0 / 2);
  const float scale = mx::value_of(scales[((size_t)tile * all + span * 2 + lane / 16) * mx::ATOM + at + lane / 4 % 4]);
  float v[8];
  mx::values8(word, scale, v);
  store8(out + (size_t)row * k + k0, v);
}

}  // namespace

// x [*, K] (rows x_ld elements apart, 16-byte aligned) -> codes, scales of `rows` rows: row i of x, or with sorted_entry (and the plan's offsets
// of its experts) row sorted_entry[i] / top_k. K a multiple of 32.
extern "C" int hb_mx_quantize(const void* x, int dtype, long long x_ld, int rows, int K, const int* sorted_entry, int top_k, const int* offsets,
                              int experts, void* codes, void* scales, cudaStream_t stream) {
  if (!x || !codes || !scales || rows < 0 || K <= 0 || (sorted_entry && (!offsets || top_k < 1 || experts < 1)) ||
      (dtype != HB_DTYPE_F32 && dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK || (reinterpret_cast<uintptr_t>(x) & 15) || x_ld * (dtype == HB_DTYPE_F32 ? 4 : 2) % 16) return HB_ERR_UNSUPPORTED;
  if (rows == 0) return HB_OK;
  const dim3 grid(rows, (mx::chunks(K) / 2 + THREADS / 32 - 1) / (THREADS / 32));
  if (dtype == HB_DTYPE_F32)
    mx_quantize_kernel<<<grid, THREADS, 0, stream>>>((const float*)x, x_ld, K, sorted_entry, top_k, offsets, experts, (uint8_t*)codes, (uint8_t*)scales);
  else
    mx_quantize_kernel<<<grid, THREADS, 0, stream>>>((const __nv_bfloat16*)x, x_ld, K, sorted_entry, top_k, offsets, experts, (uint8_t*)codes,
                                                     (uint8_t*)scales);
  HB_LAUNCH_CHECK();
  return HB_OK;
}

// The values that rows stand for, [rows, K] in out_dtype.
extern "C" int hb_mx_values(const void* codes, const void* scales, int rows, int K, const int* offsets, int experts, void* out, int out_dtype,
                            cudaStream_t stream) {
  if (!codes || !scales || !out || rows < 0 || K <= 0 || (offsets && experts < 1) || (out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK) return HB_ERR_UNSUPPORTED;
  if (rows == 0) return HB_OK;
  const dim3 grid(rows, (mx::chunks(K) / 2 + THREADS / 32 - 1) / (THREADS / 32));
  if (out_dtype == HB_DTYPE_F32)
    mx_values_kernel<<<grid, THREADS, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, K, offsets, experts, (float*)out);
  else
    mx_values_kernel<<<grid, THREADS, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, K, offsets, experts, (__nv_bfloat16*)out);
  HB_LAUNCH_CHECK();
  return HB_OK;
}
