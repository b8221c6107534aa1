// What the products of microscaled 4-bit floats share (mx_gemm_tc.cu: many rows, mx_gemm_few_tc.cu: few rows and experts).
#pragma once
#include <cuda.h>

#include "api.h"
#include "common.cuh"
#include "mx.cuh"
#include "tc.cuh"

namespace mx {

constexpr int KB = 256;                           // k of a stage
constexpr int SCALES = KB / CHUNK * ATOM;         // of 128 rows, a stage

// What is not a number stays so (fminf and fmaxf take the other one): the sums of a row or a weight with a block that is none.
__device__ __forceinline__ float least(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float most(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The unit in float32, by the fast exponential and division. By their documented errors it is off by at most (5 + 1.2 |gate|) 2^-23 of the result
// (of which the gate's part goes away above zero), the clamped unit, whose 1.702 gate is rounded too, by (6 + 3.7 |gate|) 2^-23. The most that was
// found, over 2^24 gates a range, in units of 2^-23: 1.8 above -1, 4.7 from there to -8, 8.5 to -16, 33 to -80; clamped 2.4, 10.8, 20.4, 55.
// Denominators past 2^126 give 0.
template <bool CLAMPED> __device__ __forceinline__ float unit(float gate, float up, float limit) {
  if constexpr (CLAMPED) {
    const float g = least(gate, limit), u = least(most(up, -limit), limit);
    return __fdividef(g, 1.f + __expf(-1.702f * g)) * (u + 1.f);
  }
  return __fdividef(gate, 1.f + __expf(-gate)) * up;
}
__device__ __forceinline__ float unit(float gate, float up, float limit) {
  return limit > 0.f ? unit<true>(gate, up, limit) : unit<false>(gate, up, limit);
}

struct Params {
  const uint8_t *x_scales, *w_scales;
  const int* offsets;            // [experts + 1] first row of every expert, or null: one
  const int* sorted_entry;       // GLU, with scores: the entry of a row
  const float* scores;           // GLU: a factor of a row's sums, or null
  const __nv_bfloat16* bias;
  void* out;                     // plain: [rows, n_out]; GLU: codes [rows, n_out / 4]
  uint8_t* out_scales;           // GLU
  int* status;
  int out_f32, rows, experts, n_out, chunks, w_tiles;   // chunks of K; tiles of 128 weight rows an expert
  float limit;
  int behind;                    // right behind the launch that quantises x, which weights do not wait for
  const void* raw;               // up to FEWEST rows that the blocks quantise themselves (raw_ld apart, of K values), or null
  long long raw_ld;
  int raw_f32, K;
};
constexpr int FEWEST = 16, FEWEST_K = 10240;      // rows and values of a row that a block can quantise itself: what its shared memory holds beside the weights

struct Call {
  const void *x, *x_scales, *w, *w_scales;
  int K, scale_tiles;            // of x
  cudaStream_t stream;
};

__device__ __forceinline__ float score_of(const Params& p, int row) {
  return p.scores ? p.scores[p.sorted_entry ? p.sorted_entry[row] : row] : 1.f;
}

// First row, tile of 128 rows and unit of `rows_each` rows of every expert, [experts + 1] each, by one warp.
__device__ __forceinline__ void place_experts(const Params& p, int rows_each, int* first_row, int* first_tile, int* first_unit) {
  const int lane = threadIdx.x & 31;
  int tiles_before = 0, units_before = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    const bool there = e < p.experts;
    const int a = there && p.offsets ? p.offsets[e] : 0, b = there ? (p.offsets ? p.offsets[e + 1] : p.rows) : 0;
    const int tiles = (b - a + TILE - 1) / TILE, units = (b - a + rows_each - 1) / rows_each;
    int tile_sum = tiles, unit_sum = units;
    for (int o = 1; o < 32; o <<= 1) {
      const int left = __shfl_up_sync(0xffffffffu, tile_sum, o), also = __shfl_up_sync(0xffffffffu, unit_sum, o);
      if (lane >= o) { tile_sum += left; unit_sum += also; }
    }
    if (there) {
      first_row[e] = a;
      first_tile[e] = tiles_before + tile_sum - tiles;
      first_unit[e] = units_before + unit_sum - units;
      if (e == p.experts - 1) {
        first_row[p.experts] = b;
        first_tile[p.experts] = tiles_before + tile_sum;
        first_unit[p.experts] = units_before + unit_sum;
      }
    }
    tiles_before += __shfl_sync(0xffffffffu, tile_sum, 31);
    units_before += __shfl_sync(0xffffffffu, unit_sum, 31);
  }
}
// The expert of tile `at` in the order (expert, feature tile, unit of rows): units fastest, so that neighbours share weights. By a whole warp.
__device__ __forceinline__ int expert_of(const Params& p, const int* first_unit, int f_tiles, int at) {
  const int lane = threadIdx.x & 31;
  int e = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32)
    e += __popc(__ballot_sync(0xffffffffu, e0 + lane < p.experts && first_unit[min(e0 + lane, p.experts - 1) + 1] * f_tiles <= at));
  return e;
}

// A launch in clusters of `cluster` blocks; behind a launch that quantises, as soon as that lets it.
template <typename Kernel, typename Maps>
int start(Kernel* kernel, const Maps& maps, const Params& p, int threads, int blocks, int cluster, size_t smem, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.behind) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  config.attrs = attr;
  config.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, maps, p);
  return e == cudaSuccess ? HB_OK : (int)e;
}

}  // namespace mx

// Few rows, and experts: `splits` blocks share K (1: none do), up to `most` rows a tile.
int hb_mx_clusters(int size);      // clusters of so many blocks that live at a time
int hb_mx_gemm_few(const mx::Call& c, const mx::Params& p, bool glu, int splits, int most);
