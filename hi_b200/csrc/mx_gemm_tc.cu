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

constexpr int BM = 128, KB = 256;                 // rows of a block's tile, k of a stage
constexpr int SCALES = KB / mx::CHUNK * mx::ATOM;        // SCALES: of 128 rows, a stage
constexpr int EPILOGUE = 8, THREADS = 64 + 32 * EPILOGUE;
constexpr int MOST_EXPERTS = 1024, MOST_SPLITS = 8;

// The unit in float32, by the fast exponential and division (2^-21 of the result, and where the gate is far below zero as much of it; denominators
// past 2^126 give 0).
template <bool CLAMPED> __device__ __forceinline__ float unit(float gate, float up, float limit) {
  if constexpr (CLAMPED) {
    const float g = fminf(gate, limit), u = fminf(fmaxf(up, -limit), limit);
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
};
struct Maps {
  CUtensorMap x[4];              // boxes of 16, 32, 64 and 128 rows
  CUtensorMap w, x_scales, w_scales;
};
struct Tile { int expert, row0, rows, scale_tile, f0; };      // rows: this block's, none or less perhaps

template <bool PAIR, int BN> constexpr int stage_bytes() {
  return BM * KB / 2 + (PAIR ? BN / 2 : BN) * KB / 2 + SCALES + (BN + 127) / 128 * SCALES;
}

// 32 neighbouring features of 32 rows, one a lane: four lanes trade words, so that they store 64 bytes of a row together.
__device__ __forceinline__ void store_rows(const Params& p, int lane, int quarter, const Tile& t, int f, float (&v)[32]) {
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (f + j < p.n_out) v[j] += __bfloat162float(p.bias[f + j]);
  }
  const int r = quarter * 32 + lane, first = quarter * 32 + (lane & ~3), word = lane & 3;
  const bool whole = f + 32 <= p.n_out;
  if (p.out_f32) {
    float* const o = reinterpret_cast<float*>(p.out) + (size_t)t.row0 * p.n_out + f;
    if (whole && p.n_out % 4 == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          w[q] = make_uint4(__float_as_uint(v[h * 16 + q * 4]), __float_as_uint(v[h * 16 + q * 4 + 1]), __float_as_uint(v[h * 16 + q * 4 + 2]),
                            __float_as_uint(v[h * 16 + q * 4 + 3]));
        tc::trade_rows(w, lane);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (first + q < t.rows) *reinterpret_cast<uint4*>(o + (size_t)(first + q) * p.n_out + h * 16 + word * 4) = w[q];
      }
    } else if (r < t.rows) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (f + j < p.n_out) o[(size_t)r * p.n_out + j] = v[j];
    }
  } else {
    __nv_bfloat16* const o = reinterpret_cast<__nv_bfloat16*>(p.out) + (size_t)t.row0 * p.n_out + f;
    if (whole && p.n_out % 8 == 0) {
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = make_uint4(tc::pack16<false>(v[q * 8], v[q * 8 + 1]), tc::pack16<false>(v[q * 8 + 2], v[q * 8 + 3]),
                          tc::pack16<false>(v[q * 8 + 4], v[q * 8 + 5]), tc::pack16<false>(v[q * 8 + 6], v[q * 8 + 7]));
      tc::trade_rows(w, lane);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (first + q < t.rows) *reinterpret_cast<uint4*>(o + (size_t)(first + q) * p.n_out + word * 8) = w[q];
    } else if (r < t.rows) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (f + j < p.n_out) o[(size_t)r * p.n_out + j] = __float2bfloat16_rn(v[j]);
    }
  }
}

// A block of 32 results of one row, `group` of them before it: codes and scale; behind the last one, zeros for the blocks past its end.
__device__ __forceinline__ void store_block(const Params& p, const Tile& t, int r, int group, const float (&act)[32]) {
  const int groups = p.n_out / 64, out_chunks = mx::chunks(p.n_out / 2);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(act[j]) & 0x7fffffffu);
  const uint32_t scale = mx::scale_of(top);
  const float by = mx::inverse(scale);            // (what is multiplied by the scale 255 does not matter)
  uint32_t word[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act[q * 8 + j] * by;
    word[q] = mx::codes8(v);
  }
  if (r >= t.rows) return;
  *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + (size_t)(t.row0 + r) * (p.n_out / 4) + group * 16) =
      make_uint4(word[0], word[1], word[2], word[3]);
  uint8_t* scale_row = p.out_scales + (size_t)t.scale_tile * out_chunks * mx::ATOM + mx::row_at(r);
  scale_row[(group / 4) * mx::ATOM + group % 4] = (uint8_t)scale;
  if (group == groups - 1)
    for (int q = groups; q < out_chunks * 4; ++q) scale_row[(q / 4) * mx::ATOM + q % 4] = 0;
}

__device__ __forceinline__ float score_of(const Params& p, const Tile& t, int r) {
  if (!p.scores || r >= t.rows) return 1.f;
  const int row = t.row0 + r;
  return p.scores[p.sorted_entry ? p.sorted_entry[row] : row];
}

template <bool GLU, bool PAIR, bool SPLIT, int BN, int STAGES>
__global__ void __launch_bounds__(THREADS, 1)
mx_gemm_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int B_ROWS = PAIR ? BN / 2 : BN, B_BYTES = B_ROWS * KB / 2, STAGE = stage_bytes<PAIR, BN>(), W_TILES = (BN + 127) / 128;
  constexpr int B_AT = BM * KB / 2, SA_AT = B_AT + B_BYTES, SB_AT = SA_AT + SCALES;
  // Tensor memory: two tiles' sums, which share 64 columns where 512 are not enough, then two stages' scales.
  constexpr bool SHARED = BN == 256;
  constexpr int TMEM_COLS = 512, SLOT1 = SHARED ? 192 : BN, SCALE_AT = SLOT1 + BN, SA_COLS = 8, CHUNK_COLS = W_TILES * 4, SET_COLS = SA_COLS + 2 * CHUNK_COLS;
  static_assert(!(PAIR && SPLIT) && SCALE_AT + 2 * SET_COLS <= TMEM_COLS && STAGE % 1024 == 0, "a form at a time, all within tensor memory");
  constexpr int UNIT = PAIR ? 2 : 1;              // blocks that share a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;            // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint64_t* acc_shared = acc_empty + 2;           // SHARED: the columns that both tiles' sums take have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_shared + 1);
  int* first_row = reinterpret_cast<int*>(tmem_slot + 2);        // [experts + 1]
  int* first_tile = first_row + p.experts + 1;                   // [experts + 1] tiles of 128 rows before an expert's
  int* first_unit = PAIR ? first_tile + p.experts + 1 : first_tile;      // and of a unit's

  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = PAIR || SPLIT ? (int)tc::cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], UNIT * EPILOGUE); }
    tc::mbar_init(acc_shared, UNIT * EPILOGUE / 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) tc::alloc_pair(tmem_slot, TMEM_COLS);
    else tc::alloc(tmem_slot, TMEM_COLS);
  }
  if (warp == 3 && lane < (PAIR ? 3 : 1)) {
    const CUtensorMap* map = lane == 0 ? &maps.w : lane == 1 ? &maps.x_scales : &maps.w_scales;
    tc::prefetch_map(map);
  }
  if (warp == 2) {
    int tiles_before = 0, units_before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const bool there = e < p.experts;
      const int a = there && p.offsets ? p.offsets[e] : 0, b = there ? (p.offsets ? p.offsets[e + 1] : p.rows) : 0;
      const int tiles = (b - a + BM - 1) / BM, units = (tiles + UNIT - 1) / UNIT;
      int tile_sum = tiles, unit_sum = units;
      for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, tile_sum, o), also = __shfl_up_sync(0xffffffffu, unit_sum, o);
        if (lane >= o) { tile_sum += left; unit_sum += also; }
      }
      if (there) {
        first_row[e] = a;
        first_tile[e] = tiles_before + tile_sum - tiles;
        if (PAIR) first_unit[e] = units_before + unit_sum - units;
        if (e == p.experts - 1) {
          first_row[p.experts] = b;
          first_tile[p.experts] = tiles_before + tile_sum;
          if (PAIR) first_unit[p.experts] = units_before + unit_sum;
        }
      }
      tiles_before += __shfl_sync(0xffffffffu, tile_sum, 31);
      units_before += __shfl_sync(0xffffffffu, unit_sum, 31);
    }
  }
  tc::fence_before();
  if constexpr (PAIR) tc::cluster_meet();         // (the other block's barriers are ready too)
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  int splits = 1;
  if constexpr (SPLIT) asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(splits));
  const int group = PAIR ? 2 : splits, unit_id = blockIdx.x / group, unit_count = gridDim.x / group;
  const int f_tiles = (p.n_out + BN - 1) / BN, all = first_unit[p.experts] * f_tiles, stages = p.chunks / 2;
  const int share = (stages + splits - 1) / splits, kb0 = SPLIT ? min(stages, rank * share) : 0, kb1 = SPLIT ? min(stages, kb0 + share) : stages;
  // tile i of this block, by a whole warp; rows fastest: neighbours share weights
  auto tile_at = [&](int i, Tile& t) {
    const int at = unit_id + i * unit_count;
    if (at >= all) return false;
    int e = 0;                                    // experts whose tiles come before
    for (int e0 = 0; e0 < p.experts; e0 += 32)
      e += __popc(__ballot_sync(0xffffffffu, e0 + lane < p.experts && first_unit[min(e0 + lane, p.experts - 1) + 1] * f_tiles <= at));
    const int units = first_unit[e + 1] - first_unit[e], here = at - first_unit[e] * f_tiles, f = here / units, m = (here - f * units) * UNIT;
    t.expert = e;
    t.row0 = first_row[e] + (m + (PAIR ? rank : 0)) * BM;
    t.rows = max(0, min(BM, first_row[e + 1] - t.row0));
    t.scale_tile = first_tile[e] + m + (PAIR ? rank : 0);
    t.f0 = f * BN;
    return true;
  };

  Tile t;
  if (warp == 0) {                                // ---- what a stage needs
    int s = 0, turn = 1, issued = 0;
    bool ok = true;
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem), bars = PAIR ? tc::even_block(full) : tc::smem_u32(full);
    auto load = [&](uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
      if constexpr (PAIR) tc::tma_load_2d_pair_if(mine, to, map, x, y, bar);
      else tc::tma_load_2d_if(mine, to, map, x, y, bar);
    };
    for (int i = 0; ok && tile_at(i, t); ++i) {
      const int box = PAIR ? 3 : tc::uniform(t.rows <= 16 ? 0 : t.rows <= 32 ? 1 : t.rows <= 64 ? 2 : 3);
      const int row = tc::uniform(t.row0), w_row = tc::uniform(t.expert * p.n_out + t.f0 + (PAIR ? rank * B_ROWS : 0));
      const int xs = tc::uniform(t.scale_tile * p.chunks), ws = tc::uniform((t.expert * p.w_tiles + t.f0 / 128) * p.chunks);
      const uint32_t bytes = UNIT * ((16u << box) * (KB / 2) + B_BYTES + SCALES + W_TILES * SCALES);
      auto weights = [&](int at, int kb) {
        const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
        if (mine && (rank == 0 || !PAIR)) tc::mbar_expect_tx(&full[at], bytes);
        load(st + B_AT, &maps.w, kb * (KB / 2), w_row, bar);
        if constexpr (PAIR) {
#pragma unroll
          for (int j = 0; j < W_TILES; ++j) load(st + SB_AT + j * SCALES, &maps.w_scales, 0, ws + j * p.chunks + kb * 2, bar);
        } else {
          tc::bulk_load_if(mine, st + SB_AT, p.w_scales + ((size_t)ws + kb * 2) * mx::ATOM, SCALES, bar);
        }
      };
      auto activations = [&](int at, int kb) {
        const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
        load(st, &maps.x[box], kb * (KB / 2), row, bar);
        if constexpr (PAIR) load(st + SA_AT, &maps.x_scales, 0, xs + kb * 2, bar);
        else tc::bulk_load_if(mine, st + SA_AT, p.x_scales + ((size_t)xs + kb * 2) * mx::ATOM, SCALES, bar);
      };
      int kb = tc::uniform(kb0);
      if (i == 0 && p.behind) {                   // the first stages' weights come while the rows are still being quantised
        const int ahead = tc::uniform(min(STAGES, kb1 - kb0));
        for (int q = 0; q < ahead; ++q) weights(q, kb + q);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int q = 0; q < ahead; ++q) activations(q, kb + q);
        kb += ahead;
        issued = ahead;
        if (ahead == STAGES) turn ^= 1;
        else s = ahead;
      }
      for (; kb < kb1; ++kb) {
        if (!tc::mbar_wait_warp(&empty[s], turn)) {
          if (lane == 0) atomicExch(p.status, 91);
          ok = false;
          break;
        }
        weights(s, kb);
        activations(s, kb);
        if (++s == STAGES) { s = 0; turn ^= 1; }
        ++issued;
      }
    }
    // the block ends when nothing reaches for its memory: the last commits have arrived, or, where a wait ran out, the copies on their way
    if (ok) {
      for (int i = 0; i < STAGES && tc::mbar_wait_warp(&empty[s], turn); ++i)
        if (++s == STAGES) { s = 0; turn ^= 1; }
    } else if (rank == 0 || !PAIR) {
      for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {                         // ---- products
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem);
    const uint64_t operands = tc::desc_kmajor(ring), atoms = tc::desc_scales(ring);
    auto copy = [&](uint32_t to, uint64_t from) {
      if constexpr (PAIR) tc::copy_scales_pair_if(mine, to, from);
      else tc::copy_scales_if(mine, to, from);
    };
    // PAIR: a stage's scales are copied before the products of the stage before it, so that no product waits for the copies issued with it
    // (8,192 x 16,384 x 5,120 262 -> 252 us; a tile of few rows waits longer for its first product so, 2,048 x 2,048 5.9 -> 6.1).
    int s = 0, turn = 0, set = 0;
    bool ok = true;
    auto scales = [&](int at, int parity, int to) {
      if (!tc::mbar_wait_warp(&full[at], parity)) {
        if (lane == 0) atomicExch(p.status, 92);
        return false;
      }
      tc::fence_after();
      const uint32_t sa = tmem + SCALE_AT + to * SET_COLS, sb = sa + SA_COLS;
      const uint64_t from = atoms + (at * STAGE >> 4);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        copy(sa + c * 4, from + ((SA_AT + c * mx::ATOM) >> 4));
#pragma unroll
        for (int j = 0; j < W_TILES; ++j) copy(sb + c * CHUNK_COLS + j * 4, from + ((SB_AT + j * SCALES + c * mx::ATOM) >> 4));
      }
      return true;
    };
    const bool issues = rank == 0 || !PAIR;
    if (PAIR && issues && unit_id < all) ok = scales(0, 0, 0);
    for (int i = 0; issues && ok && tile_at(i, t); ++i) {
      const int b = i & 1;
      if ((SHARED && i >= 1 && !tc::mbar_wait_warp(acc_shared, (i - 1) & 1)) || (i >= 2 && !tc::mbar_wait_warp(&acc_empty[b], (i / 2 - 1) & 1))) {
        if (lane == 0) atomicExch(p.status, 94);
        break;
      }
      tc::fence_after();
      const uint32_t acc = tmem + b * SLOT1;
      const bool another = unit_id + (i + 1) * unit_count < all;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int next = s + 1 == STAGES ? 0 : s + 1, next_turn = s + 1 == STAGES ? turn ^ 1 : turn;
        if (PAIR ? (kb + 1 < kb1 || another) && !scales(next, next_turn, set ^ 1) : !scales(s, turn, set)) {
          ok = false;
          break;
        }
        const uint32_t sa = tmem + SCALE_AT + set * SET_COLS, sb = sa + SA_COLS;
        const uint64_t a = operands + (s * STAGE >> 4), w = a + (B_AT >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t idesc = tc::idesc_mxf4(UNIT * BM, BN, k % 2 * 2), more = (kb - kb0) | k;
          if constexpr (PAIR) tc::mma_mx_pair_if(mine, acc, a + (k * 32 >> 4), w + (k * 32 >> 4), idesc, sa + k / 2 * 4, sb + k / 2 * CHUNK_COLS, more);
          else tc::mma_mx_if(mine, acc, a + (k * 32 >> 4), w + (k * 32 >> 4), idesc, sa + k / 2 * 4, sb + k / 2 * CHUNK_COLS, more);
        }
        if constexpr (PAIR) tc::commit_pair_if(mine, &empty[s]);
        else tc::commit_if(mine, &empty[s]);
        s = next;
        turn = next_turn;
        set ^= 1;
      }
      if constexpr (PAIR) tc::commit_pair_if(mine, &acc_full[b]);
      else tc::commit_if(mine, &acc_full[b]);
    }
  } else if constexpr (!SPLIT) {                  // ---- results
    const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
    auto arrive = [&](uint64_t* bar) {
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) tc::arrive_even(tc::even_block(bar));
        else tc::mbar_arrive(bar);
      }
    };
    for (int i = 0; tile_at(i, t); ++i) {
      const int b = i & 1;
      const float score = GLU ? score_of(p, t, r) : 1.f;
      if (!tc::mbar_wait_warp(&acc_full[b], (i / 2) & 1)) {
        if (lane == 0) atomicExch(p.status, 93);
        break;
      }
      tc::fence_after();
      const uint32_t from = tmem + b * SLOT1 + ((uint32_t)(quarter * 32) << 16);
      const bool live = quarter * 32 < t.rows;
      constexpr int TURNS = (BN + 127) / 128;     // groups of 64 columns of this warp: the shared one first
#pragma unroll
      for (int j = 0; j < TURNS; ++j) {
        const int g = SHARED && b == 0 ? BN / 64 - 1 - half - 2 * j : half + 2 * j, f = t.f0 + g * 64;
        const bool some = live && f < p.n_out;
        uint32_t lo[32], hi[32];
        if (some) {
          tc::ld32_nowait(from + g * 64, lo);
          tc::ld32_nowait(from + g * 64 + 32, hi);
          tc::wait_ld();
        }
        if (SHARED && j == 0 && half == 0) arrive(acc_shared);
        if (j == TURNS - 1) arrive(&acc_empty[b]);
        if (!some) continue;
        if constexpr (GLU) {
          float act[32];
          if (p.limit > 0.f) {
#pragma unroll
            for (int q = 0; q < 32; ++q) act[q] = unit<true>(score * __uint_as_float(lo[q]), score * __uint_as_float(hi[q]), p.limit);
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q) act[q] = unit<false>(score * __uint_as_float(lo[q]), score * __uint_as_float(hi[q]), 0.f);
          }
          store_block(p, t, r, f / 64, act);
        } else {
          float v[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(lo[q]);
          store_rows(p, lane, quarter, t, f, v);
          if (f + 32 < p.n_out) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(hi[q]);
            store_rows(p, lane, quarter, t, f + 32, v);
          }
        }
      }
    }
  }
  if constexpr (SPLIT) {
    // The cluster's one tile: every block sends its sums of a run of rows to the block that finishes those, which adds them in the blocks' order.
    constexpr int PITCH = BN + 4;                 // floats: neighbouring rows' words lie in different banks
    const bool there = tile_at(0, t);
    if (there && kb0 < kb1 && warp >= 2 && !tc::mbar_wait_warp(&acc_full[0], 0) && lane == 0) atomicExch(p.status, 93);
    tc::fence_after();
    __syncwarp();
    tc::cluster_meet();                           // every block's ring is free
    const int run = there ? (t.rows + splits - 1) / splits : 1;
    if (there && kb0 < kb1 && warp >= 2) {
      const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
      if (quarter * 32 < t.rows) {
        uint32_t to = 0;
        if (r < t.rows)
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(tc::smem_u32(smem) + (uint32_t)((rank * run + r % run) * PITCH * 4)), "r"(r / run));
#pragma unroll
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
          uint32_t v[32];
          tc::ld32_nowait(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
          tc::wait_ld();
          if (r < t.rows) {
#pragma unroll
            for (int q = 0; q < 32; q += 4)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c + q) * 4), "r"(v[q]), "r"(v[q + 1]), "r"(v[q + 2]), "r"(v[q + 3])
                           : "memory");
          }
        }
      }
    }
    __syncwarp();
    tc::cluster_meet();
    const int mine = there ? max(0, min(run, t.rows - rank * run)) : 0, parts = (stages + share - 1) / share;      // (of the blocks that had a part of K)
    const float* sums = reinterpret_cast<const float*>(smem);
    constexpr int WIDTH = GLU ? 64 : 32;
    for (int i = warp; i < mine * (BN / WIDTH); i += THREADS / 32) {
      const int row = i / (BN / WIDTH), c = i % (BN / WIDTH) * WIDTH, r = rank * run + row, f = t.f0 + c;
      if (f >= p.n_out) continue;
      const float* at = sums + row * PITCH + c + lane;
      float a = 0.f, b = 0.f;
      for (int q = 0; q < parts; ++q) {
        a += at[q * run * PITCH];
        if constexpr (GLU) b += at[q * run * PITCH + 32];
      }
      if constexpr (GLU) {
        const float score = score_of(p, t, r);
        float act = unit(score * a, score * b, p.limit);
        const uint32_t scale = mx::scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(act) & 0x7fffffffu));
        act *= mx::inverse(scale);
        float v[8] = {act};
#pragma unroll
        for (int j = 1; j < 8; ++j) v[j] = __shfl_down_sync(0xffffffffu, act, j);
        const int feature = f / 2;                // of the unit's first
        const size_t out_row = (size_t)(t.row0 + r) * (p.n_out / 4);
        if (lane % 8 == 0) *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + out_row + feature / 2 + lane / 2) = mx::codes8(v);
        const int groups = p.n_out / 64, out_chunks = mx::chunks(p.n_out / 2), q = f / 64 + lane;      // lane 0: the block's; behind the last block, zeros
        if (lane == 0 || (f / 64 == groups - 1 && q < out_chunks * 4))
          p.out_scales[((size_t)t.scale_tile * out_chunks + q / 4) * mx::ATOM + mx::row_at(r) + q % 4] = lane == 0 ? (uint8_t)scale : 0;
      } else if (f + lane < p.n_out) {
        if (p.bias) a += __bfloat162float(p.bias[f + lane]);
        const size_t o = (size_t)(t.row0 + r) * p.n_out + f + lane;
        if (p.out_f32) reinterpret_cast<float*>(p.out)[o] = a;
        else reinterpret_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(a);
      }
    }
  }
  tc::fence_before();
  __syncwarp();
  if constexpr (PAIR) tc::cluster_meet();         // neither block's barriers or tensor memory are reached for any more
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    if constexpr (PAIR) tc::dealloc_pair(tmem, TMEM_COLS);
    else tc::dealloc(tmem, TMEM_COLS);
  }
}

struct Call {
  const void *x, *x_scales, *w, *w_scales;
  int K, scale_tiles;            // of x
  cudaStream_t stream;
};

template <bool GLU, bool PAIR, bool SPLIT, int BN, int STAGES>
int launch(const Call& c, const Params& p, int blocks, int cluster) {
  Maps maps;
  // a map costs the host 0.3 us: those that tiles of these rows ask for
  const int rest = p.rows % BM, last = rest == 0 ? 3 : rest <= 16 ? 0 : rest <= 32 ? 1 : rest <= 64 ? 2 : 3;
  for (int b = 0; b < 4; ++b) {
    const bool asked = PAIR ? b == 3 : p.offsets ? b == 0 || p.rows > 8 << b : b == last || (b == 3 && p.rows >= BM);
    if (asked && !tc::make_map_bytes(&maps.x[b], c.x, (uint64_t)p.rows, (uint64_t)c.K / 2, 16u << b)) return HB_ERR_UNSUPPORTED;
  }
  if (!tc::make_map_bytes(&maps.w, c.w, (uint64_t)p.experts * p.n_out, (uint64_t)c.K / 2, PAIR ? BN / 2 : BN)) return HB_ERR_UNSUPPORTED;
  if (PAIR && (!tc::make_map_scales(&maps.x_scales, c.x_scales, (uint64_t)c.scale_tiles * p.chunks, KB / mx::CHUNK) ||
               !tc::make_map_scales(&maps.w_scales, c.w_scales, (uint64_t)p.experts * p.w_tiles * p.chunks, KB / mx::CHUNK)))
    return HB_ERR_UNSUPPORTED;
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256, "the barriers fit");
  static_assert(STAGES * stage_bytes<PAIR, BN>() + 1280 + 12 * 128 <= 227 * 1024, "128 experts at least");
  const size_t smem = (size_t)STAGES * stage_bytes<PAIR, BN>() + 1024 + 256 + (PAIR ? 12 : 8) * ((size_t)p.experts + 1);
  if (smem > 227 * 1024) return HB_ERR_UNSUPPORTED;
  auto* kernel = mx_gemm_kernel<GLU, PAIR, SPLIT, BN, STAGES>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e = hb::allow_smem(kernel, 227 * 1024, allowed);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = c.stream;
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
  e = cudaLaunchKernelEx(&config, kernel, maps, p);
  return e == cudaSuccess ? HB_OK : (int)e;
}

// The form by a model of the time in us: a stage takes a single block 0.275 and a pair, which does four times as much, 0.34 in the first round and 0.44
// in others (the card is at its power limit then), but a tile at least what its results take, 3 and 6; starting, the first stage's way and the last results 3.7
// and 6.5. Blocks that share K meet in 1.5 and 0.07 a row
// more. Rows of experts are taken to be equally many. Measured, as pairs / single blocks: 512 x 16,384 x 5,120 24.1 / 25.9, 700 x 5,120 x 8,192 18.7 / 20.4,
// 2,048 x 16,384 x 5,120 68.4 / 81.5, 2,048 x 5,120 x 8,192 46.6 / 49.4, 99 x 5,120 x 8,192 17.6 / 12.5, 12,288 rows of 64
// experts of 2,048 x 2,048 67.4 / 52.8; 8 x 5,120 x 8,192 11.7, in two parts 10.0.
template <bool GLU>
int gemm(const Call& c, const Params& p) {
  const int runs = p.experts < p.rows ? p.experts : p.rows, each = (p.rows + runs - 1) / runs, stages = p.chunks / 2;
  const int f_tiles = (p.n_out + 127) / 128;
  const long long most = ((p.rows + BM - 1) / BM + runs - 1LL) * f_tiles;              // tiles that there may be, and pairs of them
  const long long most_pairs = ((p.rows + 2 * BM - 1) / (2 * BM) + runs - 1LL) * ((p.n_out + 255) / 256);
  const long long likely = (long long)runs * ((each + BM - 1) / BM) * f_tiles, likely_pairs = (long long)runs * ((each + 2 * BM - 1) / (2 * BM)) * ((p.n_out + 255) / 256);
  const float single = 3.7f + (likely + 147) / 148 * fmaxf(3.f, stages * 0.275f);
  const float pair = 6.5f + (likely_pairs + 73) / 74 * fmaxf(6.f, stages * 0.44f) - stages * 0.1f;
  int splits = 1;
  float best = single < pair ? single : pair;
  for (int n = 2; n <= MOST_SPLITS && n <= stages && n * most <= 148; ++n) {
    const float shared = 5.2f + 0.07f * each + (stages + n - 1) / n * 0.275f;
    if (shared < best) { best = shared; splits = n; }
  }
  if (splits > 1) return launch<GLU, false, true, 128, 6>(c, p, (int)most * splits, splits);
  if (pair < single) return launch<GLU, true, false, 256, 6>(c, p, 2 * (int)(most_pairs < 74 ? most_pairs : 74), 2);
  return launch<GLU, false, false, 128, 6>(c, p, (int)(most < 148 ? most : 148), 1);
}

}  // namespace

// Rows (codes, scales; `offsets` the plan's, or null with experts 1) by weights [experts, n_out, K]. raw not null: they are quantised first, as
// hb_mx_quantize does (raw_dtype, raw_ld; with offsets in the order of sorted_entry, entries / top_k). glu 0: out [rows, n_out] in out_dtype, bias
// bfloat16 [n_out] or null. glu 1: n_out is twice the features, gate and up in turn by 32; out codes and out_scales of the features; scores
// (with sorted_entry: by entry, else by row) or null, limit > 0 for the clamped unit. status: one int on the device, nonzero after a wait that ran out.
extern "C" int hb_mx_gemm(const void* raw, int raw_dtype, long long raw_ld, int top_k, void* x, void* x_scales, int rows, const int* offsets,
                          int experts, const void* w, const void* w_scales, int n_out, int K, const void* bias, const int* sorted_entry,
                          const float* scores, int glu, float limit, void* out, int out_dtype, void* out_scales, int* status, cudaStream_t stream) {
  if (!x || !x_scales || !w || !w_scales || !out || !status || rows < 0 || n_out < 0 || K <= 0 || experts < 1 || (!offsets && experts != 1) ||
      (glu ? !out_scales || bias : out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if (K % mx::BLOCK || experts > MOST_EXPERTS || (glu && n_out % 64) || (long long)experts * n_out > 0x7fffffffll ||
      (long long)experts * ((n_out + 127) / 128) * mx::chunks(K) > 0x7fffffffll ||
      ((long long)(rows + BM - 1) / BM + experts) * mx::chunks(K) > 0x7fffffffll ||
      ((long long)(rows + BM - 1) / BM + experts) * ((n_out + 127) / 128) > 0x7fffffffll ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales) |
        reinterpret_cast<uintptr_t>(out)) & 15))
    return HB_ERR_UNSUPPORTED;
  if (rows == 0 || n_out == 0) return HB_OK;
  if (raw) {
    const int e = hb_mx_quantize(raw, raw_dtype, raw_ld, rows, K, offsets ? sorted_entry : nullptr, top_k, offsets, experts, x, x_scales, stream);
    if (e != HB_OK) return e;
  }
  const Params p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, offsets, sorted_entry, scores, (const __nv_bfloat16*)bias, out, (uint8_t*)out_scales, status, out_dtype == HB_DTYPE_F32, rows,
                 experts, n_out, mx::chunks(K), (n_out + 127) / 128, limit, raw != nullptr};
  const Call c{x, x_scales, w, w_scales, K, (rows + BM - 1) / BM + (experts < rows ? experts : rows) - 1, stream};
  return glu ? gemm<true>(c, p) : gemm<false>(c, p);
}
