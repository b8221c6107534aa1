// Products of microscaled 4-bit rows and weights (mx.cuh) on the 5th-generation tensor cores, which multiply both as they are
// (tcgen05.mma kind::mxf4, scales from tensor memory, float32 sums there):
//     C[r, f] = sum_k X[r, k] W[e(r), f, k]      for rows in the order of their experts (one run of rows: one expert)
// 128 rows are the MMA's M, BN weight rows its N, so that a thread of the epilogue has neighbouring features of one row:
//   plain  C (+ bias) in bfloat16 or float32;
//   GLU    weight rows are 32 of gate and 32 of up in turn: silu(s g) (s u) or the clamped unit, s the row's score, of 32 features is a
//          block, which leaves as codes and a scale: the down product's operand.
// Persistent blocks walk the tiles (expert, BN features, 128 rows; rows fastest: neighbours share weights):
//   warp 0       brings a stage of 256 k: rows and weights by TMA (128-byte rows, swizzled), the scales' atoms as bulk copies;
//   warp 1       copies the scales to tensor memory (tcgen05.cp runs in order with the products) and issues the products, four of 64 k;
//   warps 2 .. 9 read sums back (two warps a quarter of the rows, each half of the columns) and write results, while the next tile's sums
//                go to the other half of tensor memory.
// Rows of a tile past its expert's last and weight rows past n_out are computed from whatever is there, and not stored.
// Every wait is bounded; a block that gave up says where in `status` and leaves by the common exit.
#include <cuda.h>

#include "api.h"
#include "common.cuh"
#include "mx.cuh"
#include "tc.cuh"

namespace {

constexpr int BM = 128, KB = 256;                 // rows of a tile, k of a stage
constexpr int A_BYTES = BM * KB / 2, SCALES = KB / mx::CHUNK * mx::ATOM;        // SCALES: of 128 rows, a stage
constexpr int EPILOGUE = 8, THREADS = 64 + 32 * EPILOGUE;
constexpr int MOST_EXPERTS = 1024;

// hb::clamped_glu with a division that has no second path (its denominator is 1 at least; past 2^126 the result is 0)
__device__ __forceinline__ float clamped(float gate, float up, float limit) {
  const float g = fminf(gate, limit), u = fminf(fmaxf(up, -limit), limit);
  return __fdividef(g, 1.f + expf(-1.702f * g)) * (u + 1.f);
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
};
struct Maps {
  CUtensorMap x[4];              // boxes of 16, 32, 64 and 128 rows
  CUtensorMap w;
};
struct Tile { int expert, row0, rows, scale_tile, f0; };

template <int BN> constexpr int stage_bytes() { return A_BYTES + BN * KB / 2 + SCALES + BN / 128 * SCALES; }

template <bool GLU, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS, 1)
mx_gemm_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int B_BYTES = BN * KB / 2, STAGE = stage_bytes<BN>(), W_TILES = BN / 128;
  constexpr int B_AT = A_BYTES, SA_AT = B_AT + B_BYTES, SB_AT = SA_AT + SCALES;
  constexpr int TMEM_COLS = 512, SCALE_AT = 2 * BN, SA_COLS = 8, SET_COLS = SA_COLS + BN / 32 * 2;
  static_assert(SCALE_AT + 2 * SET_COLS <= TMEM_COLS, "two tiles' sums and two stages' scales");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;            // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  int* first_row = reinterpret_cast<int*>(tmem_slot + 2);        // [experts + 1]
  int* first_tile = first_row + p.experts + 1;                   // [experts + 1] tiles of rows before an expert's

  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], EPILOGUE); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tc::alloc(tmem_slot, TMEM_COLS);
  if (warp == 2) {
    int before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int a = e < p.experts ? (p.offsets ? p.offsets[e] : 0) : 0, b = e < p.experts ? (p.offsets ? p.offsets[e + 1] : p.rows) : 0;
      int tiles = (b - a + BM - 1) / BM, sum = tiles;
      for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += left;
      }
      if (e < p.experts) {
        first_row[e] = a;
        first_tile[e] = before + sum - tiles;
        if (e == p.experts - 1) { first_row[p.experts] = b; first_tile[p.experts] = before + sum; }
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  const int f_tiles = (p.n_out + BN - 1) / BN, all = first_tile[p.experts] * f_tiles, stages = p.chunks / 2;
  // tile i of this block, by a whole warp
  auto tile_at = [&](int i, Tile& t) {
    const int at = blockIdx.x + i * gridDim.x;
    if (at >= all) return false;
    int e = 0;                                    // experts whose tiles come before
    for (int e0 = 0; e0 < p.experts; e0 += 32)
      e += __popc(__ballot_sync(0xffffffffu, e0 + lane < p.experts && first_tile[min(e0 + lane, p.experts - 1) + 1] * f_tiles <= at));
    const int tiles = first_tile[e + 1] - first_tile[e], here = at - first_tile[e] * f_tiles, f = here / tiles, m = here - f * tiles;
    t.expert = e;
    t.row0 = first_row[e] + m * BM;
    t.rows = min(BM, first_row[e + 1] - t.row0);
    t.scale_tile = first_tile[e] + m;
    t.f0 = f * BN;
    return true;
  };

  Tile t;
  if (warp == 0) {                                // ---- what a stage needs
    int s = 0, turn = 1, issued = 0;
    bool ok = true;
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem), bars = tc::smem_u32(full);
    for (int i = 0; ok && tile_at(i, t); ++i) {
      const int box = tc::uniform(t.rows <= 16 ? 0 : t.rows <= 32 ? 1 : t.rows <= 64 ? 2 : 3);
      const int row = tc::uniform(t.row0), w_row = tc::uniform(t.expert * p.n_out + t.f0), w_tile = tc::uniform(t.f0 / 128);
      const int more = W_TILES > 1 ? min(W_TILES, p.w_tiles - w_tile) : 1;
      const uint8_t* xs = p.x_scales + (size_t)t.scale_tile * p.chunks * mx::ATOM;
      const uint8_t* ws = p.w_scales + ((size_t)t.expert * p.w_tiles + w_tile) * p.chunks * mx::ATOM;
      const uint32_t bytes = (16u << box) * (KB / 2) + B_BYTES + SCALES + more * SCALES;
      for (int kb = 0; kb < stages; ++kb) {
        if (!tc::mbar_wait_warp(&empty[s], turn)) {
          if (lane == 0) atomicExch(p.status, 91);
          ok = false;
          break;
        }
        const uint32_t st = ring + s * STAGE, bar = bars + s * 8;
        if (mine) tc::mbar_expect_tx(&full[s], bytes);
        tc::tma_load_2d_if(mine, st + B_AT, &maps.w, kb * (KB / 2), w_row, bar);
        tc::tma_load_2d_if(mine, st, &maps.x[box], kb * (KB / 2), row, bar);
        tc::bulk_load_if(mine, st + SA_AT, xs + (size_t)kb * SCALES, SCALES, bar);
        tc::bulk_load_if(mine, st + SB_AT, ws + (size_t)kb * SCALES, SCALES, bar);
        if constexpr (W_TILES > 1)
          if (more > 1) tc::bulk_load_if(mine, st + SB_AT + SCALES, ws + ((size_t)p.chunks * mx::ATOM + (size_t)kb * SCALES), SCALES, bar);
        if (++s == STAGES) { s = 0; turn ^= 1; }
        ++issued;
      }
    }
    // the block ends when nothing reaches for its memory: the last commits have arrived, or, where a wait ran out, the copies on their way
    if (ok) {
      for (int i = 0; i < STAGES && tc::mbar_wait_warp(&empty[s], turn); ++i)
        if (++s == STAGES) { s = 0; turn ^= 1; }
    } else {
      for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {                         // ---- products
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem);
    const uint64_t operands = tc::desc_kmajor(ring), atoms = tc::desc_scales(ring);
    int s = 0, turn = 0, set = 0;
    bool ok = true;
    for (int i = 0; ok && tile_at(i, t); ++i) {
      const int b = i & 1;
      if (i >= 2 && !tc::mbar_wait_warp(&acc_empty[b], (i / 2 - 1) & 1)) {
        if (lane == 0) atomicExch(p.status, 94);
        break;
      }
      tc::fence_after();
      const uint32_t acc = tmem + b * BN;
      for (int kb = 0; kb < stages; ++kb) {
        if (!tc::mbar_wait_warp(&full[s], turn)) {
          if (lane == 0) atomicExch(p.status, 92);
          ok = false;
          break;
        }
        tc::fence_after();
        const uint32_t sa = tmem + SCALE_AT + set * SET_COLS, sb = sa + SA_COLS;
        const uint64_t a = operands + (s * STAGE >> 4), w = a + (B_AT >> 4), from = atoms + (s * STAGE >> 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc::copy_scales_if(mine, sa + c * 4, from + ((SA_AT + c * mx::ATOM) >> 4));
#pragma unroll
          for (int j = 0; j < W_TILES; ++j)
            tc::copy_scales_if(mine, sb + c * (BN / 32) + j * 4, from + ((SB_AT + j * SCALES + c * mx::ATOM) >> 4));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc::mma_mx_if(mine, acc, a + (k * 32 >> 4), w + (k * 32 >> 4), tc::idesc_mxf4(BM, BN, k % 2 * 2), sa + k / 2 * 4, sb + k / 2 * (BN / 32),
                        kb | k);
        tc::commit_if(mine, &empty[s]);
        if (++s == STAGES) { s = 0; turn ^= 1; }
        set ^= 1;
      }
      tc::commit_if(mine, &acc_full[b]);
    }
  } else {                                        // ---- results
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    for (int i = 0; tile_at(i, t); ++i) {
      const int b = i & 1, r = quarter * 32 + lane;
      const bool live = r < t.rows;
      const size_t row = (size_t)t.row0 + (live ? r : 0);
      const float score = GLU && p.scores && live ? p.scores[p.sorted_entry ? p.sorted_entry[row] : row] : 1.f;
      if (!tc::mbar_wait_warp(&acc_full[b], (i / 2) & 1)) {
        if (lane == 0) atomicExch(p.status, 93);
        break;
      }
      tc::fence_after();
      const uint32_t from = tmem + b * BN + ((uint32_t)(quarter * 32) << 16);
      if (quarter * 32 < t.rows) {
        if constexpr (GLU) {
          const int groups = p.n_out / 64, out_chunks = mx::chunks(p.n_out / 2);
          uint8_t* scale_row = p.out_scales + (size_t)t.scale_tile * out_chunks * mx::ATOM + mx::row_at(r);
#pragma unroll 1
          for (int c = half * 64; c < BN; c += 128) {
            const int g0 = (t.f0 + c) / 64;       // the group of 32 features
            if (g0 >= groups) break;
            uint32_t g[32], u[32];
            tc::ld32_nowait(from + c, g);
            tc::ld32_nowait(from + c + 32, u);
            tc::wait_ld();
            float act[32];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float gs = score * __uint_as_float(g[j]), us = score * __uint_as_float(u[j]);
              act[j] = p.limit > 0.f ? clamped(gs, us, p.limit) : __fdividef(gs, 1.f + expf(-gs)) * us;
              top = max(top, __float_as_uint(act[j]) & 0x7fffffffu);
            }
            const uint32_t scale = mx::scale_of(top);
            const float by = scale == 255 ? 0.f : mx::inverse(scale);
            uint32_t word[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = scale == 255 ? 0.f : act[q * 8 + j] * by;
              word[q] = mx::codes8(v);
            }
            if (live) {
              *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + row * (p.n_out / 4) + g0 * 16) = make_uint4(word[0], word[1], word[2], word[3]);
              scale_row[(g0 / 4) * mx::ATOM + g0 % 4] = (uint8_t)scale;
              if (g0 == groups - 1)
                for (int q = groups; q < out_chunks * 4; ++q) scale_row[(q / 4) * mx::ATOM + q % 4] = 0;
            }
          }
        } else {
#pragma unroll 1
          for (int c = half * 32; c < BN; c += 64) {
            const int f = t.f0 + c;
            if (f >= p.n_out) break;
            float v[32];
            tc::ld32(from + c, v);
            if (!live) continue;
            if (p.bias) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (f + j < p.n_out) v[j] += __bfloat162float(p.bias[f + j]);
            }
            const size_t at = row * p.n_out + f;
            if (p.out_f32) {
              float* o = reinterpret_cast<float*>(p.out) + at;
              if (p.n_out % 4 == 0 && f + 32 <= p.n_out) {
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (f + j < p.n_out) o[j] = v[j];
              }
            } else {
              __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
              if (p.n_out % 8 == 0 && f + 32 <= p.n_out) {
#pragma unroll
                for (int j = 0; j < 32; j += 8)
                  *reinterpret_cast<uint4*>(o + j) = make_uint4(tc::pack16<false>(v[j], v[j + 1]), tc::pack16<false>(v[j + 2], v[j + 3]),
                                                                tc::pack16<false>(v[j + 4], v[j + 5]), tc::pack16<false>(v[j + 6], v[j + 7]));
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (f + j < p.n_out) o[j] = __float2bfloat16_rn(v[j]);
              }
            }
          }
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&acc_empty[b]);
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc(tmem, TMEM_COLS);
  }
}

template <bool GLU, int BN, int STAGES>
int launch(const void* x, const void* w, int K, const Params& p, int blocks, cudaStream_t stream) {
  Maps maps;
  for (int b = 0; b < 4; ++b)
    if (!tc::make_map_bytes(&maps.x[b], x, (uint64_t)p.rows, (uint64_t)K / 2, 16u << b)) return HB_ERR_UNSUPPORTED;
  if (!tc::make_map_bytes(&maps.w, w, (uint64_t)p.experts * p.n_out, (uint64_t)K / 2, BN)) return HB_ERR_UNSUPPORTED;
  const size_t smem = (size_t)STAGES * stage_bytes<BN>() + 1024 + 256 + 8 * ((size_t)p.experts + 1);
  if (smem > 227 * 1024) return HB_ERR_UNSUPPORTED;
  auto* kernel = mx_gemm_kernel<GLU, BN, STAGES>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e = hb::allow_smem(kernel, 227 * 1024, allowed);
  if (e != cudaSuccess) return (int)e;
  kernel<<<blocks, THREADS, smem, stream>>>(maps, p);
  HB_LAUNCH_CHECK();
  return HB_OK;
}

}  // namespace

// Rows (codes, scales; `offsets` the plan's, or null with experts 1) by weights [experts, n_out, K]. glu 0: out [rows, n_out] in out_dtype, bias
// bfloat16 [n_out] or null. glu 1: n_out is twice the features, gate and up in turn by 32; out codes and out_scales of the features; scores
// (with sorted_entry: by entry, else by row) or null, limit > 0 for the clamped unit. status: one int on the device, nonzero after a wait that ran out.
extern "C" int hb_mx_gemm(const void* x, const void* x_scales, int rows, const int* offsets, int experts, const void* w, const void* w_scales,
                          int n_out, int K, const void* bias, const int* sorted_entry, const float* scores, int glu, float limit, void* out,
                          int out_dtype, void* out_scales, int* status, cudaStream_t stream) {
  if (!x || !x_scales || !w || !w_scales || !out || !status || rows < 0 || n_out < 0 || K <= 0 || experts < 1 || (!offsets && experts != 1) ||
      (glu ? !out_scales || bias : out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK || experts > MOST_EXPERTS || (glu && n_out % 64) || (long long)experts * n_out > 0x7fffffffll ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales) |
        reinterpret_cast<uintptr_t>(out)) & 15))
    return HB_ERR_UNSUPPORTED;
  if (rows == 0 || n_out == 0) return HB_OK;
  const Params p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, offsets, sorted_entry, scores, (const __nv_bfloat16*)bias, out,
                 (uint8_t*)out_scales, status, out_dtype == HB_DTYPE_F32, rows, experts, n_out, mx::chunks(K), (n_out + 127) / 128, limit};
  const long long tiles = ((long long)(rows + BM - 1) / BM + (experts < rows ? experts : rows) - 1) * ((n_out + 127) / 128);
  const int blocks = (int)(tiles < 148 ? tiles : 148);
  return glu ? launch<true, 128, 6>(x, w, K, p, blocks, stream) : launch<false, 128, 6>(x, w, K, p, blocks, stream);
}
