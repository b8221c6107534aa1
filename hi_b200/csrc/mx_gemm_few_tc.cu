// Products of microscaled 4-bit floats for few rows, and for experts, of which each has its own few (mx_gemm.cuh; many rows: mx_gemm_tc.cu):
//     C[r, f] = sum_k X[r, k] W[e(r), f, k]      for rows in the order of their experts (one run of rows: one expert)
// The product is taken transposed: 128 weight rows are the MMA's M, an expert's rows, up to BT of them, its N, rounded up to 16, so that what an
// expert costs goes by the rows it has and its weights come once for all of them. What bounds it is HBM, which brings the weights (units of 64 tokens, 1 of
// 16 experts of 5,120 x 8,192: 97 us, 1.05 of the copy rate), and where a launch does not fill the SMs the issue of copies and products, 0.2 us a stage, behind
// 1.7 to 2 us until the first weights are there (8 x 2,048 x 2,048 5.0 us, 8 x 5,120 x 8,192 8.5, where HBM alone would take 0.3 and 3.4).
// Blocks walk the tiles (expert, 128 features, BT rows; rows fastest: neighbours share weights):
//   warp 0       brings a stage of 256 k: weights and rows by TMA (128-byte rows, swizzled), the scales' atoms as bulk copies; the first stages before
//                the block's warps meet, and their weights before the launch that quantises the rows has ended;
//   warp 1       copies the scales to tensor memory (tcgen05.cp runs in order with the products) and issues the products, four of 64 k;
//   warps 2 .. 17 read sums back, a lane a feature (four warps a quarter of the features, runs of 16 rows in turn), and write results, while the next
//                tile's sums go to the other slot of tensor memory. GLU: a quarter of gate features and one of up features trade halves of their
//                rows, so that both have whole units; 32 lanes are a block: its largest magnitude by one reduction, its codes by a transposition of
//                eight lanes' words of eight rows.
// SPLIT: a cluster's blocks share out K, one tile a cluster; each sends its sums to the block that finishes those rows, which adds them in the
// blocks' order.
// Rows past an expert's last and weight rows past n_out are computed from whatever is there, and not stored.
// Every wait is bounded; a block that gave up says where in `status` and leaves by the common exit.
#include <type_traits>

#include "mx_gemm.cuh"

namespace {

using mx::Call;
using mx::KB;
using mx::Params;
using mx::SCALES;

constexpr int BF = 128, A_BYTES = BF * KB / 2;    // weight rows of a tile
constexpr int EPILOGUE = 16, THREADS = 64 + 32 * EPILOGUE;
constexpr int X_STAGE = mx::FEWEST * KB / 2;       // RAW: a stage's rows
constexpr int TRADE = EPILOGUE * 8 * 32 * 4;      // GLU: room for what warps trade

struct Maps {
  CUtensorMap x[4];              // boxes of 16, 32, 64 and 128 rows
  CUtensorMap w;
};
struct Tile { int expert, row0, rows, scale_tile, off, f0; };      // its first row is row `off` of the tile of scales

template <bool RAW, int BT> constexpr int stage_bytes() { return A_BYTES + SCALES + (RAW ? 0 : BT * KB / 2 + (BT + 127) / 128 * SCALES); }

// Eight lanes' words of eight codes, one a row: lane i has the row's i % 8 then, eight neighbouring features.
__device__ __forceinline__ uint32_t transpose(uint32_t x, int lane) {
  uint32_t y = __shfl_xor_sync(0xffffffffu, x, 4);
  x = lane & 4 ? (y >> 16) | (x & 0xffff0000u) : (x & 0xffffu) | (y << 16);
  y = __shfl_xor_sync(0xffffffffu, x, 2);
  x = lane & 2 ? ((y >> 8) & 0x00ff00ffu) | (x & 0xff00ff00u) : (x & 0x00ff00ffu) | ((y & 0x00ff00ffu) << 8);
  y = __shfl_xor_sync(0xffffffffu, x, 1);
  return lane & 1 ? ((y >> 4) & 0x0f0f0f0fu) | (x & 0xf0f0f0f0u) : (x & 0x0f0f0f0fu) | ((y & 0x0f0f0f0fu) << 4);
}

// The rows of the stages kb0 .. kb1 - 1, quantised by the warps behind the first two to where the products read them: `x` a stage's 16 rows of 128
// bytes, swizzled, `scales` its atoms, of which 16 rows are written.
template <typename T>
__device__ __forceinline__ void quantize_rows(const Params& p, uint8_t* x, uint8_t* scales, int kb0, int kb1, int warp, int lane) {
  constexpr int MANY = 8;                         // loads of a lane on their way
  const int each = EPILOGUE / p.rows, row = (warp - 2) % p.rows, first = (warp - 2) / p.rows;       // warps of a row
  if (first >= each) return;
  const T* const from = reinterpret_cast<const T*>(p.raw) + (size_t)row * p.raw_ld + lane * 8;
  x += row * 128 + ((lane / 4 ^ (row & 7)) << 4) + lane % 4 * 4;
  scales += lane / 16 * mx::ATOM + row * 16;
  for (int s0 = first; s0 < kb1 - kb0; s0 += each * MANY) {
    mx::Eight<T> v[MANY];
#pragma unroll
    for (int m = 0; m < MANY; ++m) {
      const int k = (kb0 + s0 + m * each) * KB;
      if (s0 + m * each < kb1 - kb0 && k + lane * 8 < p.K) v[m].load(from + k);
      else v[m].zero();
    }
#pragma unroll
    for (int m = 0; m < MANY; ++m) {
      const int s = s0 + m * each;
      if (s >= kb1 - kb0) break;
      uint32_t scale;
      const uint32_t codes = mx::quantize(v[m], scale), word = mx::four_scales(scale, lane);
      *reinterpret_cast<uint32_t*>(x + s * X_STAGE) = codes;
      if (lane % 16 == 0) *reinterpret_cast<uint32_t*>(scales + s * SCALES) = word;
    }
  }
}

// RAW: up to 16 rows come as they are.
template <bool GLU, bool SPLIT, bool RAW, int BT, int STAGES>
__global__ void __launch_bounds__(THREADS, 1)
mx_gemm_few_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int STAGE = stage_bytes<RAW, BT>(), X_TILES = (BT + 127) / 128;
  constexpr int X_AT = A_BYTES, SA_AT = RAW ? A_BYTES : X_AT + BT * KB / 2, SX_AT = SA_AT + SCALES;
  // Tensor memory: two tiles' sums, which share 64 columns where 512 are not enough, then two stages' scales.
  constexpr bool SHARED = BT == 256;
  constexpr int TMEM_COLS = 512, SLOT1 = SHARED ? 192 : BT, SCALE_AT = SLOT1 + BT, SA_COLS = 8, CHUNK_COLS = X_TILES * 4, SET_COLS = SA_COLS + 2 * CHUNK_COLS;
  static_assert(SCALE_AT + 2 * SET_COLS <= TMEM_COLS && STAGE % 1024 == 0 && BT % 64 == 0 && BT <= 256, "all within tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int resident = RAW ? p.chunks / 2 : 0;    // RAW: stages of rows that there is room for
  uint8_t *x_rows = smem + STAGES * STAGE, *x_scales = x_rows + resident * X_STAGE, *behind_ring = x_scales + resident * SCALES;
  float* trade = reinterpret_cast<float*>(behind_ring);          // GLU: [EPILOGUE][8][32]
  uint64_t* full = reinterpret_cast<uint64_t*>(behind_ring + (GLU && !SPLIT ? TRADE : 0));
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;            // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint64_t* acc_shared = acc_empty + 2;           // SHARED: the columns that both tiles' sums take have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_shared + 1);
  int* first_row = reinterpret_cast<int*>(tmem_slot + 2);        // [experts + 1] each
  int* first_tile = first_row + p.experts + 1;
  int* first_unit = first_tile + p.experts + 1;

  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int rank = 0, splits = 1;
  if constexpr (SPLIT) {
    rank = (int)tc::cluster_rank();
    asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(splits));
  }
  const int unit_id = blockIdx.x / splits, unit_count = gridDim.x / splits, f_tiles = (p.n_out + BF - 1) / BF, stages = p.chunks / 2;
  const int share = (stages + splits - 1) / splits, kb0 = SPLIT ? min(stages, rank * share) : 0, kb1 = SPLIT ? min(stages, kb0 + share) : stages;
  // tile i of this block, by a whole warp
  auto tile_at = [&](int i, Tile& t) {
    const int at = unit_id + i * unit_count;
    if (!p.offsets) {                             // one run of rows: no table (the first copies leave 0.4 us earlier)
      const int units = (p.rows + BT - 1) / BT, f = units == 1 ? at : at / units, m = at - f * units;
      if (f >= f_tiles) return false;
      t = {0, m * BT, min(BT, p.rows - m * BT), m * BT / mx::TILE, m * BT % mx::TILE, f * BF};
      return true;
    }
    if (at >= first_unit[p.experts] * f_tiles) return false;
    const int e = mx::expert_of(p, first_unit, f_tiles, at), row = first_row[e];
    const int units = first_unit[e + 1] - first_unit[e], here = at - first_unit[e] * f_tiles, f = here / units, m = here - f * units;
    t = {e, row + m * BT, min(BT, first_row[e + 1] - row - m * BT), first_tile[e] + m * BT / mx::TILE, m * BT % mx::TILE, f * BF};
    return true;
  };
  const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem), bars = tc::smem_u32(full);
  auto weights = [&](const Tile& t, int at, int kb) {      // and what the stage waits for
    const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
    const int box = t.rows <= 16 ? 0 : t.rows <= 32 ? 1 : t.rows <= 64 ? 2 : 3;
    const int more = BT > 128 && t.rows > 128 ? (BT - 128) * (KB / 2) : 0, two = BT > 128 && t.off + t.rows > 128;
    if (mine) tc::mbar_expect_tx(&full[at], RAW ? A_BYTES + SCALES : A_BYTES + (16u << box) * (KB / 2) + more + SCALES + (SCALES << two));
    tc::tma_load_2d_if(mine, st, &maps.w, kb * (KB / 2), t.expert * p.n_out + t.f0, bar);
    tc::bulk_load_if(mine, st + SA_AT, p.w_scales + ((size_t)(t.expert * p.w_tiles + t.f0 / 128) * p.chunks + kb * 2) * mx::ATOM, SCALES, bar);
  };
  auto rows = [&](const Tile& t, int at, int kb) {
    if constexpr (RAW) return;
    const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
    const int box = t.rows <= 16 ? 0 : t.rows <= 32 ? 1 : t.rows <= 64 ? 2 : 3;
    const uint8_t* from = p.x_scales + ((size_t)t.scale_tile * p.chunks + kb * 2) * mx::ATOM;
    tc::tma_load_2d_if(mine, st + X_AT, &maps.x[box], kb * (KB / 2), t.row0, bar);
    tc::bulk_load_if(mine, st + SX_AT, from, SCALES, bar);
    if (BT > 128 && t.rows > 128)
      tc::tma_load_2d_if(mine, st + X_AT + 128 * KB / 2, &maps.x[BT == 192 ? 2 : 3], kb * (KB / 2), t.row0 + 128, bar);
    if (BT > 128 && t.off + t.rows > 128) tc::bulk_load_if(mine, st + SX_AT + SCALES, from + (size_t)p.chunks * mx::ATOM, SCALES, bar);
  };

  Tile t;
  int ahead = 0;                                  // warp 0: stages on their way before the warps meet
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < STAGES; ++s) tc::mbar_init(&full[s], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (p.offsets) mx::place_experts(p, BT, first_row, first_tile, first_unit);
    __syncwarp();
    if (tile_at(0, t)) {
      ahead = min(STAGES, kb1 - kb0);
      if (p.behind) {
        for (int q = 0; q < ahead; ++q) weights(t, q, kb0 + q);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int q = 0; q < ahead; ++q) rows(t, q, kb0 + q);
      } else {
        for (int q = 0; q < ahead; ++q) {
          weights(t, q, kb0 + q);
          rows(t, q, kb0 + q);
        }
      }
    } else if (p.behind) {                        // (where no block has a tile, the launch still ends behind the other one)
      asm volatile("griddepcontrol.wait;" ::: "memory");
    }
  }
  if (warp == 1) tc::alloc(tmem_slot, TMEM_COLS);
  if (warp == 2 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) tc::mbar_init(&empty[s], 1);
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], EPILOGUE); }
    tc::mbar_init(acc_shared, EPILOGUE);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if constexpr (RAW) {                            // while the first weights are on their way
    if (warp >= 2) {
      if (p.raw_f32) quantize_rows<float>(p, x_rows, x_scales, kb0, kb1, warp, lane);
      else quantize_rows<__nv_bfloat16>(p, x_rows, x_scales, kb0, kb1, warp, lane);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  if (warp == 0) {                                // ---- what a stage needs
    int s = ahead == STAGES ? 0 : ahead, turn = ahead == STAGES ? 0 : 1, issued = ahead;
    for (int i = 0; ok && tile_at(i, t); ++i)
      for (int kb = kb0 + (i == 0 ? ahead : 0); kb < kb1; ++kb) {
        if (!tc::mbar_wait_warp(&empty[s], turn)) {
          if (lane == 0) atomicExch(p.status, 91);
          ok = false;
          break;
        }
        weights(t, s, kb);
        rows(t, s, kb);
        if (++s == STAGES) { s = 0; turn ^= 1; }
        ++issued;
      }
    // the block ends when nothing reaches for its memory: the last commits have arrived, or, where a wait ran out, the copies on their way
    if (ok) {
      for (int i = 0; i < STAGES && tc::mbar_wait_warp(&empty[s], turn); ++i)
        if (++s == STAGES) { s = 0; turn ^= 1; }
    } else {
      for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {                         // ---- products
    const uint64_t operands = tc::desc_kmajor(ring), atoms = tc::desc_scales(ring);
    int s = 0, turn = 0, set = 0;
    const uint64_t resident_x = tc::desc_kmajor(tc::smem_u32(x_rows)), resident_atoms = tc::desc_scales(tc::smem_u32(x_scales));
    for (int i = 0; ok && tile_at(i, t); ++i) {
      const int b = i & 1;
      if ((SHARED && i >= 1 && !tc::mbar_wait_warp(acc_shared, (i - 1) & 1)) || (i >= 2 && !tc::mbar_wait_warp(&acc_empty[b], (i / 2 - 1) & 1))) {
        if (lane == 0) atomicExch(p.status, 94);
        break;
      }
      tc::fence_after();
      const uint32_t acc = tmem + b * SLOT1, idesc = tc::idesc_mxf4(BF, tc::uniform((t.rows + 15) & ~15), 0);
      const bool two = BT > 128 && tc::uniform(t.off + t.rows) > 128;
      const uint32_t off = tc::uniform(t.off / 32);        // columns of the scales before the tile's
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!tc::mbar_wait_warp(&full[s], turn)) {
          if (lane == 0) atomicExch(p.status, 92);
          ok = false;
          break;
        }
        tc::fence_after();
        const uint32_t sa = tmem + SCALE_AT + set * SET_COLS, sx = sa + SA_COLS;
        const uint64_t a = operands + (s * STAGE >> 4), from = atoms + (s * STAGE >> 4);
        const uint64_t x = RAW ? resident_x + ((kb - kb0) * X_STAGE >> 4) : a + (X_AT >> 4);
        const uint64_t from_x = RAW ? resident_atoms + ((kb - kb0) * SCALES >> 4) : from + (SX_AT >> 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tc::copy_scales_if(mine, sa + c * 4, from + ((SA_AT + c * mx::ATOM) >> 4));
          tc::copy_scales_if(mine, sx + c * CHUNK_COLS, from_x + (c * mx::ATOM >> 4));
          if (two) tc::copy_scales_if(mine, sx + c * CHUNK_COLS + 4, from + ((SX_AT + SCALES + c * mx::ATOM) >> 4));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc::mma_mx_if(mine, acc, a + (k * 32 >> 4), x + (k * 32 >> 4), idesc | tc::idesc_mxf4(0, 0, k % 2 * 2), sa + k / 2 * 4, sx + k / 2 * CHUNK_COLS + off,
                        (kb - kb0) | k);
        tc::commit_if(mine, &empty[s]);
        if (++s == STAGES) { s = 0; turn ^= 1; }
        set ^= 1;
      }
      tc::commit_if(mine, &acc_full[b]);
    }
  } else if constexpr (!SPLIT) {                  // ---- results
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    auto arrive = [&](uint64_t* bar) {
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar);
    };
    for (int i = 0; tile_at(i, t); ++i) {
      const int b = i & 1, f = t.f0 + quarter * 32 + lane;
      constexpr int TURNS = BT / 64;              // runs of 16 rows of this warp, those in the shared columns first
      auto run_at = [&](int j) { return part * 16 + (SHARED && b == 0 ? TURNS - 1 - j : j) * 64; };
      float score = 1.f;                          // GLU: lane 8 j + q has that of row q of the warp's eight of run j
      if (GLU && p.scores) {
        const int r = run_at(lane / 8) + (quarter & 1 ? 8 : 0) + lane % 8;
        if (lane / 8 < TURNS && r < t.rows) score = mx::score_of(p, t.row0 + r);
      }
      if (ok && !tc::mbar_wait_warp(&acc_full[b], (i / 2) & 1)) {        // (goes on without waiting: warps trade)
        if (lane == 0) atomicExch(p.status, 93);
        ok = false;
      }
      tc::fence_after();
      const uint32_t from = tmem + b * SLOT1 + ((uint32_t)(quarter * 32) << 16);
      const bool there = GLU ? t.f0 + quarter / 2 * 64 < p.n_out : t.f0 + quarter * 32 < p.n_out;
      const float bias = !GLU && p.bias && f < p.n_out ? __bfloat162float(p.bias[f]) : 0.f;
#pragma unroll 1
      for (int j = 0; j < TURNS; ++j) {
        const int c = run_at(j);
        const bool some = there && c < t.rows;
        // GLU: gate's warp keeps the run's first 8 rows and gives the others to up's, which keeps those
        const bool up = GLU && (quarter & 1);
        uint32_t v[16];
        __syncwarp();                             // (lanes part where rows or features end; the loads want the warp together)
        if (some) {
          if constexpr (GLU) {
            tc::ld8_nowait(from + c + (up ? 8 : 0), reinterpret_cast<uint32_t(&)[8]>(v[0]));
            tc::ld8_nowait(from + c + (up ? 0 : 8), reinterpret_cast<uint32_t(&)[8]>(v[8]));
          } else {
            tc::ld16_nowait(from + c, v);
          }
          tc::wait_ld();
        }
        if (SHARED && j == 0) arrive(acc_shared);
        if (j == TURNS - 1) arrive(&acc_empty[b]);
        if (!some) continue;
        if constexpr (GLU) {
          float* const give = trade + (warp - 2) * 256 + lane;
          const float* const take = trade + ((warp ^ 1) - 2) * 256 + lane;
          const int r = c + (up ? 8 : 0) + lane % 8;
#pragma unroll
          for (int q = 0; q < 8; ++q) give[q * 32] = __uint_as_float(v[8 + q]);
          asm volatile("bar.sync %0, 64;" ::"r"(1 + part * 2 + quarter / 2) : "memory");
          float act[8];
          auto units = [&](auto clamped) {
            constexpr bool CLAMPED = decltype(clamped)::value;
            if (up) {
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float s = __shfl_sync(0xffffffffu, score, j * 8 + q);
                act[q] = mx::unit<CLAMPED>(s * take[q * 32], s * __uint_as_float(v[q]), p.limit);
              }
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float s = __shfl_sync(0xffffffffu, score, j * 8 + q);
                act[q] = mx::unit<CLAMPED>(s * __uint_as_float(v[q]), s * take[q * 32], p.limit);
              }
            }
          };
          if (p.limit > 0.f) units(std::true_type{});
          else units(std::false_type{});
          asm volatile("bar.sync %0, 64;" ::"r"(1 + part * 2 + quarter / 2) : "memory");
          const int block = t.f0 / 64 + quarter / 2, blocks = p.n_out / 64, out_chunks = mx::chunks(p.n_out / 2);
          uint32_t top[8], mine_top = 0;
#pragma unroll
          for (int q = 0; q < 8; ++q) top[q] = __reduce_max_sync(0xffffffffu, __float_as_uint(act[q]) & 0x7fffffffu);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            act[q] *= mx::inverse_of(top[q]);
            if (lane % 8 == q) mine_top = top[q];
          }
          const uint32_t word = transpose(mx::codes8(act), lane);
          if (r < t.rows) *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + (size_t)(t.row0 + r) * (p.n_out / 4) + block * 16 + lane / 8 * 4) = word;
          if (r < t.rows && lane < 8) {
            uint8_t* const to = p.out_scales + (size_t)(t.scale_tile + (t.off + r) / mx::TILE) * out_chunks * mx::ATOM + mx::row_at((t.off + r) % mx::TILE);
            to[block / 4 * mx::ATOM + block % 4] = (uint8_t)mx::scale_of(mine_top);
            if (block == blocks - 1)
              for (int q = blocks; q < out_chunks * 4; ++q) to[q / 4 * mx::ATOM + q % 4] = 0;
          }
        } else {
          const size_t at = (size_t)(t.row0 + c) * p.n_out + f;
          const int count = t.rows - c;
          if (p.out_f32) {
            float* const o = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
            for (int q = 0; q < 16; ++q)
              if (q < count && f < p.n_out) o[(size_t)q * p.n_out] = __uint_as_float(v[q]) + bias;
          } else if (p.n_out % 2 == 0) {          // a lane stores two features, even lanes of one row and odd lanes of the next
            __nv_bfloat16* const o = reinterpret_cast<__nv_bfloat16*>(p.out) + at - (lane & 1);
#pragma unroll
            for (int q = 0; q < 16; q += 2) {
              const float a = __uint_as_float(v[q]) + bias, d = __uint_as_float(v[q + 1]) + bias;
              const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? a : d, 1);
              const int row = q + (lane & 1);
              if (row < count && f < p.n_out)
                *reinterpret_cast<uint32_t*>(o + (size_t)row * p.n_out) = lane & 1 ? tc::pack16<false>(other, d) : tc::pack16<false>(a, other);
            }
          } else {
            __nv_bfloat16* const o = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
            for (int q = 0; q < 16; ++q)
              if (q < count && f < p.n_out) o[(size_t)q * p.n_out] = __float2bfloat16_rn(__uint_as_float(v[q]) + bias);
          }
        }
      }
    }
  }
  if constexpr (SPLIT) {
    const bool there = tile_at(0, t);
    const int run = there ? (t.rows + splits - 1) / splits : 1;
    const float score = GLU && there && lane < run && rank * run + lane < t.rows ? mx::score_of(p, t.row0 + rank * run + lane) : 1.f;
    if (there && kb0 < kb1 && warp >= 2 && !tc::mbar_wait_warp(&acc_full[0], 0) && lane == 0) atomicExch(p.status, 93);
    tc::fence_after();
    __syncwarp();
    tc::cluster_meet();                           // every block's ring is free
    if (there && kb0 < kb1 && warp >= 2) {
      const int quarter = warp & 3;
      int turn = (warp - 2) >> 2;                 // four warps a quarter, in turn
#pragma unroll 1
      for (int r = 0; r < splits; ++r) {
        uint32_t to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to)
            : "r"(ring + (uint32_t)((rank * run * BF + quarter * 32 + lane) * 4)), "r"(r));
        const int end = min(t.rows, (r + 1) * run);
#pragma unroll 1
        for (int c = r * run; c < end; c += 16) {
          if (turn-- > 0) continue;
          turn = 3;
          uint32_t v[16];
          tc::ld16_nowait(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
          tc::wait_ld();
#pragma unroll
          for (int q = 0; q < 16; ++q)
            if (c + q < end) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + (c - r * run + q) * BF * 4), "r"(v[q]) : "memory");
        }
      }
    }
    __syncwarp();
    tc::cluster_meet();
    const int own = there ? max(0, min(run, t.rows - rank * run)) : 0, parts = (stages + share - 1) / share;      // (of the blocks that had a part of K)
    const float* sums = reinterpret_cast<const float*>(smem);
    constexpr int WIDTH = GLU ? 64 : 32;
    for (int i = warp; i < own * (BF / WIDTH); i += THREADS / 32) {
      const int row = i / (BF / WIDTH), c = i % (BF / WIDTH) * WIDTH, r = rank * run + row, f = t.f0 + c;
      if (f >= p.n_out) continue;
      const float* at = sums + row * BF + c + lane;
      float a = 0.f, b = 0.f;
      for (int q = 0; q < parts; ++q) {
        a += at[q * run * BF];
        if constexpr (GLU) b += at[q * run * BF + 32];
      }
      if constexpr (GLU) {
        const float known = __shfl_sync(0xffffffffu, score, row & 31), one = row < 32 ? known : mx::score_of(p, t.row0 + r);
        float act = mx::unit(one * a, one * b, p.limit);
        const uint32_t scale = mx::scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(act) & 0x7fffffffu));
        act *= mx::inverse(scale);
        float w[8] = {act};
#pragma unroll
        for (int j = 1; j < 8; ++j) w[j] = __shfl_down_sync(0xffffffffu, act, j);
        if (lane % 8 == 0)
          *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + (size_t)(t.row0 + r) * (p.n_out / 4) + f / 4 + lane / 2) = mx::codes8(w);
        const int blocks = p.n_out / 64, out_chunks = mx::chunks(p.n_out / 2), q = f / 64 + lane;      // lane 0: the block's; behind the last block, zeros
        if (lane == 0 || (f / 64 == blocks - 1 && q < out_chunks * 4))
          p.out_scales[((size_t)(t.scale_tile + r / mx::TILE) * out_chunks + q / 4) * mx::ATOM + mx::row_at(r % mx::TILE) + q % 4] = lane == 0 ? (uint8_t)scale : 0;
      } else if (f + lane < p.n_out) {
        if (p.bias) a += __bfloat162float(p.bias[f + lane]);
        const size_t o = (size_t)(t.row0 + r) * p.n_out + f + lane;
        if (p.out_f32) reinterpret_cast<float*>(p.out)[o] = a;
        else reinterpret_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(a);
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc(tmem, TMEM_COLS);
  }
}

template <bool GLU, bool SPLIT, bool RAW, int BT, int STAGES>
int launch(const Call& c, const Params& p, int blocks, int cluster) {
  Maps maps;
  if constexpr (!RAW) {
    // A map costs the host 0.3 us: those that tiles of these rows ask for, in the others' places the last of them.
    auto box_of = [](int rows) { return rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3; };
    const int rest = p.rows % BT ? p.rows % BT : BT;         // rows of one run's last tile; a tile of 192 has 64 of them as a second box
    int made = -1;
    for (int b = 3; b >= 0; --b) {
      const bool asked = p.offsets ? b <= box_of(p.rows < BT ? p.rows : BT) : b == box_of(rest) || (p.rows >= BT && b == box_of(BT)) || (BT == 192 && b == 2);
      if (asked && !tc::make_map_bytes(&maps.x[b], c.x, (uint64_t)p.rows, (uint64_t)c.K / 2, BT < (16 << b) ? BT : 16 << b)) return HB_ERR_UNSUPPORTED;
      if (asked) made = b;
    }
    for (int b = 0; b < 4; ++b) {
      const bool asked = p.offsets ? b <= box_of(p.rows < BT ? p.rows : BT) : b == box_of(rest) || (p.rows >= BT && b == box_of(BT)) || (BT == 192 && b == 2);
      if (!asked) maps.x[b] = maps.x[made];
    }
  }
  if (!tc::make_map_bytes(&maps.w, c.w, (uint64_t)p.experts * p.n_out, (uint64_t)c.K / 2, BF)) return HB_ERR_UNSUPPORTED;
  constexpr int TRADED = GLU && !SPLIT ? TRADE : 0;
  constexpr int RESIDENT = RAW ? mx::FEWEST_K / KB * (X_STAGE + SCALES) : 0;
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256 && STAGES * stage_bytes<RAW, BT>() + RESIDENT + TRADED + 1280 + 12 * (RAW ? 2 : 385) <= 227 * 1024,
                "with 384 experts");
  const size_t smem = (size_t)STAGES * stage_bytes<RAW, BT>() + (RAW ? p.chunks / 2 * (X_STAGE + SCALES) : 0) + TRADED + 1024 + 256 + 12 * ((size_t)p.experts + 1);
  if (smem > 227 * 1024) return HB_ERR_UNSUPPORTED;
  auto* kernel = mx_gemm_few_kernel<GLU, SPLIT, RAW, BT, STAGES>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e = hb::allow_smem(kernel, 227 * 1024, allowed);
  if (e != cudaSuccess) return (int)e;
  return mx::start(kernel, maps, p, THREADS, blocks, cluster, smem, c.stream);
}

template <bool GLU>
int few(const Call& c, const Params& p, int splits, int most) {
  auto grid = [&](int bt) {        // tiles that there may be
    const long long units = (p.rows + bt - 1) / bt + (p.experts < p.rows ? p.experts : p.rows) - 1LL;
    return units * ((p.n_out + BF - 1) / BF);
  };
  auto blocks = [&](int bt) { return (int)(grid(bt) < 148 ? grid(bt) : 148); };
  if (p.raw) return splits > 1 ? launch<GLU, true, true, 64, 5>(c, p, (int)grid(64) * splits, splits) : launch<GLU, false, true, 64, 5>(c, p, blocks(64), 1);
  if (splits > 1) return launch<GLU, true, false, 128, 6>(c, p, (int)grid(128) * splits, splits);
  if (most <= 64) return launch<GLU, false, false, 64, 7>(c, p, blocks(64), 1);
  if (most <= 128) return launch<GLU, false, false, 128, 6>(c, p, blocks(128), 1);
  if (most <= 192) return launch<GLU, false, false, 192, GLU ? 4 : 5>(c, p, blocks(192), 1);
  return launch<GLU, false, false, 256, 4>(c, p, blocks(256), 1);
}

}  // namespace

// How many clusters of `size` blocks live at a time on the current device; without one, as many as its blocks would make.
int hb_mx_clusters(int size) {
  static std::atomic<int> known[64][16];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device > 63 || size > 15) return 148 / size;
  int n = known[device][size].load(std::memory_order_relaxed);
  if (n > 0) return n;
  auto* kernel = mx_gemm_few_kernel<false, true, false, 128, 6>;
  constexpr size_t smem = 6 * stage_bytes<false, 128>() + 1280 + 24;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return 148 / size;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(size * 148);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n <= 0) return 148 / size;
  known[device][size].store(n, std::memory_order_relaxed);
  return n;
}

// splits: blocks that share K (1: none do); most: rows of a tile, 64 (where there are no more in all), 128, 192 or 256.
int hb_mx_gemm_few(const Call& c, const Params& p, bool glu, int splits, int most) {
  return glu ? few<true>(c, p, splits, most) : few<false>(c, p, splits, most);
}
