// Rows to microscaled 4-bit floats (mx.cuh) and back: x is read once, codes and scales are a quarter of bfloat16. A warp has four spans of 256 values on
// their way, a lane eight values of each, four lanes a block of 32. What bounds it: HBM for float32 (8,001 x 8,192 43.9 us, 1.03 of the copy rate), for
// bfloat16 instructions too (8,192 x 16,384 59.9 us, 0.87; with one span a warp and maxima of floats instead of 16-bit halves 89.8); back, HBM (52.8 us, 0.98).
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
constexpr int THREADS = 256, WARPS = THREADS / 32;

// A warp takes MANY spans of 256 values of a row. Four lanes have a block of 32.
template <typename T, int MANY>
__global__ void __launch_bounds__(THREADS)
mx_quantize_kernel(const T* __restrict__ x, long long x_ld, int rows, int k, const int* __restrict__ sorted_entry, int top_k,
                   const int* __restrict__ offsets, int experts, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  asm volatile("griddepcontrol.launch_dependents;");       // the product behind this launch may begin to bring its weights
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all = mx::chunks(k), groups = (all / 2 + MANY - 1) / MANY;
  const long long item = (long long)blockIdx.x * WARPS + warp;
  const int row = (int)(item / groups), first = (int)(item % groups) * MANY;
  if (row >= rows) return;
  // (behind the last expert's rows stands anything; x is asked for all the same, before the offsets are there)
  const size_t from = sorted_entry ? min((unsigned)sorted_entry[row], (unsigned)(rows - 1)) / (unsigned)top_k : row;
  const T* const in = x + from * x_ld + lane * 8;
  mx::Eight<T> x8[MANY];
#pragma unroll
  for (int m = 0; m < MANY; ++m) {
    const int k0 = (first + m) * SPAN + lane * 8;
    if (k0 < k) x8[m].load(in + (first + m) * SPAN);
    else x8[m].zero();
  }
  int tile, at;
  if (!mx::place_of(offsets, experts, row, tile, at)) return;
  uint8_t* const to = codes + (size_t)row * (k / 2) + lane * 4;
  uint8_t* const scale_to = scales + (size_t)tile * all * mx::ATOM + at;
#pragma unroll
  for (int m = 0; m < MANY; ++m) {
    const int span = first + m, k0 = span * SPAN + lane * 8;
    if (span * 2 >= all) break;
    uint32_t scale;
    const uint32_t eight = mx::quantize(x8[m], scale);
    if (k0 < k) *reinterpret_cast<uint32_t*>(to + span * (SPAN / 2)) = eight;
    const uint32_t word = mx::four_scales(scale, lane);
    if (lane % 16 == 0) *reinterpret_cast<uint32_t*>(scale_to + (size_t)(span * 2 + lane / 16) * mx::ATOM) = word;
  }
}

template <typename T, int MANY>
__global__ void __launch_bounds__(THREADS)
mx_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int k, const int* __restrict__ offsets,
                 int experts, T* __restrict__ out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all = mx::chunks(k), groups = (all / 2 + MANY - 1) / MANY;
  const long long item = (long long)blockIdx.x * WARPS + warp;
  const int row = (int)(item / groups), first = (int)(item % groups) * MANY;
  if (row >= rows) return;
  int tile, at;
  if (!mx::place_of(offsets, experts, row, tile, at)) return;
  const uint8_t* const from = codes + (size_t)row * (k / 2) + lane * 4;
  const uint8_t* const scale_from = scales + (size_t)tile * all * mx::ATOM + at + lane / 4 % 4;
  uint32_t word[MANY], scale[MANY];
#pragma unroll
  for (int m = 0; m < MANY; ++m) {
    const bool there = (first + m) * SPAN + lane * 8 < k;
    word[m] = there ? *reinterpret_cast<const uint32_t*>(from + (first + m) * (SPAN / 2)) : 0u;
    scale[m] = there ? scale_from[(size_t)((first + m) * 2 + lane / 16) * mx::ATOM] : 0u;
  }
#pragma unroll
  for (int m = 0; m < MANY; ++m) {
    const int k0 = (first + m) * SPAN + lane * 8;
    if (k0 >= k) break;
    float v[8];
    mx::values8(word[m], mx::value_of(scale[m]), v);
    store8(out + (size_t)row * k + k0, v);
  }
}

// Four spans a warp where that still gives every SM 32 warps, else one: a few rows want as many warps as they can have (1 x 5,120 1.4 us).
int blocks_of(int rows, int k, int many) {
  const long long items = (long long)rows * ((mx::chunks(k) / 2 + many - 1) / many), blocks = (items + WARPS - 1) / WARPS;
  return blocks > 0x7fffffffll ? 0 : (int)blocks;
}
bool much(int rows, int k) { return (long long)rows * (mx::chunks(k) / 2) >= 4 * 148 * 32; }

template <typename T, int MANY>
void quantize(const void* x, long long x_ld, int rows, int k, const int* sorted_entry, int top_k, const int* offsets, int experts, void* codes,
              void* scales, int blocks, cudaStream_t stream) {
  mx_quantize_kernel<T, MANY><<<blocks, THREADS, 0, stream>>>((const T*)x, x_ld, rows, k, sorted_entry, top_k, offsets, experts, (uint8_t*)codes,
                                                              (uint8_t*)scales);
}
template <typename T, int MANY>
void values(const void* codes, const void* scales, int rows, int k, const int* offsets, int experts, void* out, int blocks, cudaStream_t stream) {
  mx_values_kernel<T, MANY><<<blocks, THREADS, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, rows, k, offsets, experts, (T*)out);
}

}  // namespace

// x [*, K] (rows x_ld elements apart, 16-byte aligned) -> codes, scales of `rows` rows: row i of x, or with sorted_entry (and the plan's offsets
// of its experts) row sorted_entry[i] / top_k; with offsets, rows from offsets[experts] on are left as they are. K a multiple of 32.
extern "C" int hb_mx_quantize(const void* x, int dtype, long long x_ld, int rows, int K, const int* sorted_entry, int top_k, const int* offsets,
                              int experts, void* codes, void* scales, cudaStream_t stream) {
  if (!x || !codes || !scales || rows < 0 || K <= 0 || (sorted_entry && (!offsets || top_k < 1 || experts < 1)) ||
      (dtype != HB_DTYPE_F32 && dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK || (reinterpret_cast<uintptr_t>(x) & 15) || x_ld * (dtype == HB_DTYPE_F32 ? 4 : 2) % 16) return HB_ERR_UNSUPPORTED;
  if (rows == 0) return HB_OK;
  const bool four = much(rows, K);
  const int blocks = blocks_of(rows, K, four ? 4 : 1);
  if (blocks == 0) return HB_ERR_UNSUPPORTED;
  auto* launch = dtype == HB_DTYPE_F32 ? (four ? quantize<float, 4> : quantize<float, 1>) : (four ? quantize<__nv_bfloat16, 4> : quantize<__nv_bfloat16, 1>);
  launch(x, x_ld, rows, K, sorted_entry, top_k, offsets, experts, codes, scales, blocks, stream);
  HB_LAUNCH_CHECK();
  return HB_OK;
}

// The values that rows stand for, [rows, K] in out_dtype; with offsets, rows from offsets[experts] on are left as they are.
extern "C" int hb_mx_values(const void* codes, const void* scales, int rows, int K, const int* offsets, int experts, void* out, int out_dtype,
                            cudaStream_t stream) {
  if (!codes || !scales || !out || rows < 0 || K <= 0 || (offsets && experts < 1) || (out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK) return HB_ERR_UNSUPPORTED;
  if (rows == 0) return HB_OK;
  const bool four = much(rows, K);
  const int blocks = blocks_of(rows, K, four ? 4 : 1);
  if (blocks == 0) return HB_ERR_UNSUPPORTED;
  auto* launch = out_dtype == HB_DTYPE_F32 ? (four ? values<float, 4> : values<float, 1>) : (four ? values<__nv_bfloat16, 4> : values<__nv_bfloat16, 1>);
  launch(codes, scales, rows, K, offsets, experts, out, blocks, stream);
  HB_LAUNCH_CHECK();
  return HB_OK;
}
