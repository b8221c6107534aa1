// Products with weights of four bits: out[t, n] = sum_k x[t, k] s[n, k / group] (c[n, k] - 8) (+ bias[n]), x bfloat16, codes c 0 .. 15,
// scales s bfloat16, float32 sums. The weights lie in blocks of 16 rows x 128 k, row tile after row tile:
//   codes   [16 rows][4 lanes][4 words]: word i of lane q holds k = 32 i + 8 q .. + 7, even k in the lower half
//   scales  [16 rows][128 / group] bfloat16
// (rows and k past the matrix: code 8, scale 0), 1,024 + 32 (128 / group) bytes a block.
//
// Few tokens (up to 16): the time is the weights' way out of HBM. A word of codes goes into mma.sync as it is (four_bit.cuh; the products
// of whole numbers with x are exact), weights as the 16 rows and tokens as 8 columns; the eight's share comes off as the sum's start, -8
// times the sum of x over the group, which the same instruction computes once from codes of 8; then the group's scale multiplies its sum
// in float32. No product is rounded. A block is up to 16 warps that share K in turns of a block of weights; x waits in shared memory in
// the fragments' order, raised by 2^64 once, each warp's own part; the row tiles of a block follow one another and the loads run ahead
// over their ends, three blocks a warp, asked for again where they were used (before the use, into copies, with addresses worked out
// anew: 163 instructions a block of weights, 8 x 16,384 x 5,120 14.5 us instead of 13.1). The warps' sums meet in shared memory in a fixed order.
// 8 x 16,384 x 5,120 3.2 TB/s (13.5 us), 1 x 2,048 x 2,048 2.9 us of which 2 are the launch; what bounds it is each warp's chain of loads, unpacking and
// products (a warp takes 900 cycles a block of weights, 8.4 an instruction), not HBM (0.5 of its rate) nor the tensor cores (0.19). Measured
// and not kept, 8 x 16,384 x 5,120 / 1 x 5,120 x 8,192: a ring of bulk copies a warp and two row tiles at a time 15.3 / 19.7, two or four sums a group
// of their own 14.9 / 11.6, sums joined by the warps in turn without a barrier 13.5 / 11.6, clusters that share K 19.7 / 13.9.
#include "api.h"
#include "common.cuh"
#include "four_bit.cuh"

namespace {

constexpr int ROWS = 16, KB = 128;      // of a block of weights
constexpr int AHEAD = 3;                // blocks a warp has in flight
constexpr int MOST_WARPS = 16, MOST_TILES = 16;
constexpr int MOST_SMEM = 200 * 1024;

struct Few {
  const __nv_bfloat16* x;
  long long x_ld;
  const uint8_t* w;
  const __nv_bfloat16* bias;
  void* out;
  int out_f32, tokens, n_out, K, chunks, panel;      // panel: blocks of K that x is held for at a time
};

template <int GPC> __device__ __forceinline__ uint2 load_scales(const uint8_t* p) {
  if constexpr (GPC == 1) return make_uint2(__ldcs(reinterpret_cast<const unsigned short*>(p)), 0u);
  else if constexpr (GPC == 2) return make_uint2(__ldcs(reinterpret_cast<const unsigned*>(p)), 0u);
  else return __ldcs(reinterpret_cast<const uint2*>(p));
}
__device__ __forceinline__ float scale_of(uint2 v, int i) {
  const unsigned w = i < 2 ? v.x : v.y;
  return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}

// The outputs of a block's row tiles that are NaN, by the definition, one product after the other: an input of 2^64 and more, raised, is infinite, and
// the eights' share with it, so that its token's outputs are NaN where they have a value or an infinity. (Inputs looked at as they come in, and the
// tokens remembered until the end: 8 x 16,384 x 5,120 17.0 us instead of 14.4, as calls.)
template <int GPC> __device__ __forceinline__ void redo(const Few& a, int tiles) {
  constexpr int BYTES = 1024 + ROWS * 2 * GPC;
  for (int t = 0; t < a.tokens; ++t) {
    const __nv_bfloat16* x = a.x + (size_t)t * a.x_ld;
    bool nan = false;
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) nan = nan || __hisnan(x[k]);
    if (__syncthreads_or(nan)) continue;                          // they are what they should be
    for (int j = threadIdx.x; j < tiles * ROWS; j += blockDim.x) {
      const int row = (blockIdx.x + j / ROWS * gridDim.x) * ROWS + j % ROWS;
      if (row >= a.n_out) continue;
      const size_t to = (size_t)t * a.n_out + row;
      const float was = a.out_f32 ? reinterpret_cast<const float*>(a.out)[to] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.out)[to]);
      if (was == was) continue;
      float sum = 0.f;
#pragma unroll 1
      for (int k = 0; k < a.K && sum == sum; ++k) {
        const uint8_t* block = a.w + ((size_t)(row / ROWS) * a.chunks + k / KB) * BYTES;
        const int at = k % KB, e = at % 8;
        const unsigned word = reinterpret_cast<const unsigned*>(block)[(row % ROWS * 4 + at % 32 / 8) * 4 + at / 32];
        const int code = (int)(word >> (e % 2 * 16 + e / 2 * 4) & 15u) - 8;
        const float scale = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(block + 1024)[row % ROWS * GPC + at * GPC / KB]);
        sum = fmaf(__bfloat162float(x[k]), (float)code * scale, sum);
      }
      if (a.bias) sum += __bfloat162float(a.bias[row]);
      if (a.out_f32) reinterpret_cast<float*>(a.out)[to] = sum;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[to] = __float2bfloat16_rn(sum);
    }
  }
}

// NT: tiles of 8 tokens; GPC: groups in a block of weights' 128 k
template <int NT, int GPC>
__global__ void __launch_bounds__(MOST_WARPS * 32, 1) four_bit_few_kernel(const Few a) {
  constexpr int BYTES = 1024 + ROWS * 2 * GPC, TILE = ROWS * 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, q4 = lane & 3;
  uint4* xs = reinterpret_cast<uint4*>(smem);                                     // [panel][NT][4][32 lanes]
  float2* start = reinterpret_cast<float2*>(xs + (size_t)a.panel * NT * 128);     // [panel][GPC][NT][4]: what the eights come to, negative
  float* red = reinterpret_cast<float*>(start + (size_t)a.panel * GPC * NT * 4);  // [2][warps][TILE]
  float* kept = red + 2 * warps * TILE;                                           // [tiles][TILE], of earlier panels
  __shared__ int any_nan;
  if (threadIdx.x == 0) any_nan = 0;
  const int tokens = a.tokens;
  const int row_tiles = (a.n_out + ROWS - 1) / ROWS;
  const int tiles = (row_tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;
  int turn = 0;
  for (int c0 = 0; c0 < a.chunks; c0 += a.panel) {
    const int n_chunks = min(a.panel, a.chunks - c0), per = (n_chunks - warp + warps - 1) / warps;
    const int total = tiles * per;                                // blocks of weights of this warp
    uint4 lo[AHEAD], hi[AHEAD];
    uint2 s_lo[AHEAD], s_hi[AHEAD];
    int l_i = 0, left = total;
    const uint8_t* b = a.w + ((size_t)blockIdx.x * a.chunks + c0 + warp) * BYTES + lane * 16;
    const int to_scales = 1024 + g * 2 * GPC - lane * 16, next_block = warps * BYTES;
    const long long next_tile = ((long long)gridDim.x * a.chunks - (long long)per * warps) * BYTES;
    auto load = [&](int u) {
      if (left <= 0) return;
      lo[u] = __ldcs(reinterpret_cast<const uint4*>(b));
      hi[u] = __ldcs(reinterpret_cast<const uint4*>(b + 512));
      s_lo[u] = load_scales<GPC>(b + to_scales);
      s_hi[u] = load_scales<GPC>(b + to_scales + 16 * GPC);
      --left;
      b += next_block;
      if (++l_i == per) { l_i = 0; b += next_tile; }
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load(u);
    __syncwarp();
    for (int i = 0; i < per; ++i) {                               // this warp's x
      const int c = warp + i * warps;
      uint4* to = xs + (size_t)c * NT * 128 + lane;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int token = n * 8 + g;
        const __nv_bfloat16* from = a.x + (size_t)min(token, tokens - 1) * a.x_ld;
        float eights[GPC][4];
#pragma unroll
        for (int k = 0; k < GPC; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) eights[k][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = (c0 + c) * KB + 32 * j + 8 * q4;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (token < tokens && k < a.K) v = fb::raised(__ldg(reinterpret_cast<const uint4*>(from + k)));
          to[(n * 4 + j) * 32] = v;
          fb::mma_codes(eights[j * GPC / 4], 0x88888888u, 0x88888888u, v);
        }
        if (g == 0)
#pragma unroll
          for (int k = 0; k < GPC; ++k) start[((size_t)c * GPC + k) * NT * 4 + n * 4 + q4] = make_float2(-eights[k][0], -eights[k][1]);
      }
    }
    __syncwarp();
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    int tile = 0, i = 0;
    auto finish = [&]() {                                         // the warps' sums of a row tile meet
      float* mine = red + (turn * warps + warp) * TILE;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mine[(n * 8 + 2 * q4 + (e & 1)) * ROWS + g + 8 * (e >> 1)] = acc[n][e];
          acc[n][e] = 0.f;
        }
      __syncthreads();
      for (int j = threadIdx.x; j < TILE; j += blockDim.x) {
        float sum = 0.f;
        for (int w = 0; w < warps; ++w) sum += red[(turn * warps + w) * TILE + j];
        if (c0 > 0) sum += kept[tile * TILE + j];
        if (c0 + a.panel < a.chunks) {
          kept[tile * TILE + j] = sum;
          continue;
        }
        const int t = j / ROWS, row = (blockIdx.x + tile * gridDim.x) * ROWS + j % ROWS;
        if (t >= tokens || row >= a.n_out) continue;
        sum *= fb::UNSCALE;
        if (a.bias) sum += __bfloat162float(a.bias[row]);
        if (sum != sum) any_nan = 1;
        const size_t at = (size_t)t * a.n_out + row;
        if (a.out_f32) reinterpret_cast<float*>(a.out)[at] = sum;
        else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(sum);
      }
      turn ^= 1;
      ++tile;
      i = 0;
    };
    const uint4* xc = xs + (size_t)warp * NT * 128 + lane;
    const float2* st = start + (size_t)warp * GPC * NT * 4 + q4;
    for (int it = 0; it < total; it += AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (it + u >= total) break;
#pragma unroll
        for (int k = 0; k < GPC; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 begin = st[(k * NT + n) * 4];
            float part[4] = {begin.x, begin.y, begin.x, begin.y};
#pragma unroll
            for (int j = k * 4 / GPC; j < (k + 1) * 4 / GPC; ++j)
              fb::mma_codes(part, j == 0 ? lo[u].x : j == 1 ? lo[u].y : j == 2 ? lo[u].z : lo[u].w,
                            j == 0 ? hi[u].x : j == 1 ? hi[u].y : j == 2 ? hi[u].z : hi[u].w, xc[(n * 4 + j) * 32]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = fmaf(part[e], scale_of(e < 2 ? s_lo[u] : s_hi[u], k), acc[n][e]);
          }
        load(u);
        xc += warps * NT * 128;
        st += warps * GPC * NT * 4;
        if (++i == per) {
          xc -= per * warps * NT * 128;
          st -= per * warps * GPC * NT * 4;
          finish();
        }
      }
    }
    if (per <= 0)
      for (int j = 0; j < tiles; ++j) finish();
    __syncthreads();                                              // `kept` and the last sums are in place
  }
  if (any_nan) redo<GPC>(a, tiles);
}

template <int NT, int GPC>
int launch_few(Few a, cudaStream_t stream) {
  const int row_tiles = (a.n_out + ROWS - 1) / ROWS;
  // as many warps as share K evenly: the fewest turns, then the fewest warps
  int warps = a.chunks < MOST_WARPS ? a.chunks : MOST_WARPS;
  const int turns = (a.chunks + warps - 1) / warps;
  warps = (a.chunks + turns - 1) / turns;
  const int fixed = 2 * warps * ROWS * 8 * NT * 4, each = NT * 2048 + GPC * NT * 32;
  int blocks = row_tiles < 148 ? row_tiles : 148;
  int kept = 0;
  a.panel = a.chunks;
  if (fixed + a.panel * each > MOST_SMEM) {
    kept = MOST_TILES * ROWS * 8 * NT * 4;
    a.panel = (MOST_SMEM - fixed - kept) / each / warps * warps;
    blocks = max(blocks, (row_tiles + MOST_TILES - 1) / MOST_TILES);
  }
  const int smem = fixed + kept + a.panel * each;
  auto* kernel = four_bit_few_kernel<NT, GPC>;
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = hb::allow_smem(kernel, MOST_SMEM + 16 * 1024, allowed);
  if (e != cudaSuccess) return (int)e;
  kernel<<<blocks, warps * 32, smem, stream>>>(a);
  HB_LAUNCH_CHECK();
  return HB_OK;
}

}  // namespace

// x [tokens, K] with rows x_ld elements apart, up to 16 of them, w blocks as above, bias [n_out] bfloat16 or null, out [tokens, n_out] contiguous.
extern "C" int hb_four_bit_linear(const void* x, long long x_ld, const void* w, const void* bias, void* out, int out_dtype, int tokens,
                                  int n_out, int K, int group, cudaStream_t stream) {
  if (!x || !w || !out || tokens < 0 || n_out < 0 || K < 0 || (out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (tokens > 16 || (group != 32 && group != 64 && group != 128) || K % group || K == 0 || x_ld % 8 ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15))
    return HB_ERR_UNSUPPORTED;
  if (tokens == 0 || n_out == 0) return HB_OK;
  const Few a{(const __nv_bfloat16*)x, x_ld, (const uint8_t*)w, (const __nv_bfloat16*)bias, out, out_dtype == HB_DTYPE_F32, tokens,
              n_out, K, (K + KB - 1) / KB, 0};
  if (tokens <= 8)
    return group == 128 ? launch_few<1, 1>(a, stream) : group == 64 ? launch_few<1, 2>(a, stream) : launch_few<1, 4>(a, stream);
  return group == 128 ? launch_few<2, 1>(a, stream) : group == 64 ? launch_few<2, 2>(a, stream) : launch_few<2, 4>(a, stream);
}
