// Products of many rows of microscaled 4-bit floats (mx_gemm.cuh) on the 5th-generation tensor cores, which multiply rows and weights as they
// are (tcgen05.mma kind::mxf4, scales from tensor memory, float32 sums there):
//     C[r, f] = sum_k X[r, k] W[e(r), f, k]      for rows in the order of their experts (one run of rows: one expert)
// Two blocks of a cluster on 256 rows x 256 weight rows (cta_group::2), each with its 128 rows and half of the weight rows; a thread of the epilogue
// has neighbouring features of one row:
//   plain  C (+ bias) in bfloat16 or float32;
//   GLU    weight rows are 32 of gate and 32 of up in turn: silu(s g) (s u) or the clamped unit, s the row's score, of 32 features is a
//          block, which leaves as codes and a scale: the down product's operand.
// Persistent pairs walk the tiles (expert, 256 features, 256 rows; rows fastest: neighbours share weights):
//   warp 0       brings a stage of 256 k by TMA: its rows, its weight rows (128-byte rows, swizzled), and the scales of its rows and of all weight rows;
//   warp 1       of the even block copies the scales to both blocks' tensor memory, a stage ahead of its products (8,192 x 16,384 x 5,120 262 ->
//                252 us), and issues the products, four of 64 k;
//   warps 2 .. 9 read sums back (two warps a quarter of the rows, 64 columns in turn) and write results, while the next tile's sums go to the other slot
//                of tensor memory. The slots share 64 columns, which are read first.
// What bounds it: 2,048 x 16,384 x 5,120 takes 66 us, 5.2 PFLOP/s, 90,100 cycles, of which products are 75,000; for a second or more the card's power limit
// lowers the clock and it takes 78. A stage is 530 cycles (products 512); between two tiles the products wait 1,000 to 1,200 for the sums' first 64 columns.
// Rows of a tile past its expert's last and weight rows past n_out are computed from whatever is there, and not stored.
// Every wait is bounded; a block that gave up says where in `status` and leaves by the common exit.
#include "mx_gemm.cuh"

namespace {

using mx::Call;
using mx::KB;
using mx::Params;
using mx::SCALES;
using mx::unit;

constexpr int BM = 128, BN = 256, STAGES = 6;     // rows of a block's tile, features of a pair's
constexpr int A_BYTES = BM * KB / 2, B_BYTES = BN / 2 * KB / 2, STAGE = A_BYTES + B_BYTES + SCALES + BN / 128 * SCALES;
constexpr int EPILOGUE = 8, THREADS = 64 + 32 * EPILOGUE;
constexpr int MOST_EXPERTS = 384, MOST_SPLITS = 8;       // experts: whose tables shared memory holds beside the stages

struct Maps { CUtensorMap x, w, x_scales, w_scales; };
struct Tile { int expert, row0, rows, scale_tile, f0; };      // rows: this block's, none or less perhaps

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
  const float by = mx::inverse_of(top);
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

template <bool GLU>
__global__ void __launch_bounds__(THREADS, 1)
mx_gemm_kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int B_AT = A_BYTES, SA_AT = B_AT + B_BYTES, SB_AT = SA_AT + SCALES, W_TILES = BN / 128;
  // Tensor memory: two tiles' sums, which share 64 columns, then two stages' scales.
  constexpr int TMEM_COLS = 512, SLOT1 = 192, SCALE_AT = SLOT1 + BN, SA_COLS = 8, CHUNK_COLS = W_TILES * 4, SET_COLS = SA_COLS + 2 * CHUNK_COLS;
  static_assert(SCALE_AT + 2 * SET_COLS <= TMEM_COLS && STAGE % 1024 == 0, "all within tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;            // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint64_t* acc_shared = acc_empty + 2;           // the columns that both tiles' sums take have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_shared + 1);
  int* first_row = reinterpret_cast<int*>(tmem_slot + 2);        // [experts + 1] each
  int* first_tile = first_row + p.experts + 1;
  int* first_unit = first_tile + p.experts + 1;

  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, rank = (int)tc::cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], 2 * EPILOGUE); }
    tc::mbar_init(acc_shared, EPILOGUE);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tc::alloc_pair(tmem_slot, TMEM_COLS);
  if (warp == 3 && lane < 4) tc::prefetch_map(lane == 0 ? &maps.w : lane == 1 ? &maps.x : lane == 2 ? &maps.x_scales : &maps.w_scales);
  if (warp == 2) mx::place_experts(p, 2 * BM, first_row, first_tile, first_unit);
  tc::fence_before();
  tc::cluster_meet();                             // (the other block's barriers are ready too)
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  const int pair_id = blockIdx.x / 2, pair_count = gridDim.x / 2;
  const int f_tiles = (p.n_out + BN - 1) / BN, all = first_unit[p.experts] * f_tiles, stages = p.chunks / 2;
  // tile i of this pair, by a whole warp
  auto tile_at = [&](int i, Tile& t) {
    const int at = pair_id + i * pair_count;
    if (at >= all) return false;
    const int e = mx::expert_of(p, first_unit, f_tiles, at);
    const int units = first_unit[e + 1] - first_unit[e], here = at - first_unit[e] * f_tiles, f = here / units, m = (here - f * units) * 2 + rank;
    t.expert = e;
    t.row0 = first_row[e] + m * BM;
    t.rows = max(0, min(BM, first_row[e + 1] - t.row0));
    t.scale_tile = first_tile[e] + m;
    t.f0 = f * BN;
    return true;
  };

  Tile t;
  if (warp == 0) {                                // ---- what a stage needs
    int s = 0, turn = 1, issued = 0;
    bool ok = true;
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem), bars = tc::even_block(full);
    if (p.behind && pair_id >= all) asm volatile("griddepcontrol.wait;" ::: "memory");      // (where no block has a tile, the launch still ends behind the other one)
    for (int i = 0; ok && tile_at(i, t); ++i) {
      const int row = tc::uniform(t.row0), w_row = tc::uniform(t.expert * p.n_out + t.f0 + rank * (BN / 2));
      const int xs = tc::uniform(t.scale_tile * p.chunks), ws = tc::uniform((t.expert * p.w_tiles + t.f0 / 128) * p.chunks);
      auto weights = [&](int at, int kb) {
        const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
        if (mine && rank == 0) tc::mbar_expect_tx(&full[at], 2 * STAGE);
        tc::tma_load_2d_pair_if(mine, st + B_AT, &maps.w, kb * (KB / 2), w_row, bar);
#pragma unroll
        for (int j = 0; j < W_TILES; ++j) tc::tma_load_2d_pair_if(mine, st + SB_AT + j * SCALES, &maps.w_scales, 0, ws + j * p.chunks + kb * 2, bar);
      };
      auto activations = [&](int at, int kb) {
        const uint32_t st = ring + at * STAGE, bar = bars + at * 8;
        tc::tma_load_2d_pair_if(mine, st, &maps.x, kb * (KB / 2), row, bar);
        tc::tma_load_2d_pair_if(mine, st + SA_AT, &maps.x_scales, 0, xs + kb * 2, bar);
      };
      int kb = 0;
      if (i == 0 && p.behind) {                   // the first stages' weights come while the rows are still being quantised
        const int ahead = min(STAGES, stages);
        for (int q = 0; q < ahead; ++q) weights(q, q);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int q = 0; q < ahead; ++q) activations(q, q);
        kb = issued = ahead;
        if (ahead == STAGES) turn ^= 1;
        else s = ahead;
      }
      for (; kb < stages; ++kb) {
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
    } else if (rank == 0) {
      for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait_warp(&full[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {                         // ---- products
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem);
    const uint64_t operands = tc::desc_kmajor(ring), atoms = tc::desc_scales(ring);
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
        tc::copy_scales_pair_if(mine, sa + c * 4, from + ((SA_AT + c * mx::ATOM) >> 4));
#pragma unroll
        for (int j = 0; j < W_TILES; ++j) tc::copy_scales_pair_if(mine, sb + c * CHUNK_COLS + j * 4, from + ((SB_AT + j * SCALES + c * mx::ATOM) >> 4));
      }
      return true;
    };
    if (rank == 0 && pair_id < all) ok = scales(0, 0, 0);
    for (int i = 0; rank == 0 && ok && tile_at(i, t); ++i) {
      const int b = i & 1;
      if ((i >= 1 && !tc::mbar_wait_warp(acc_shared, (i - 1) & 1)) || (i >= 2 && !tc::mbar_wait_warp(&acc_empty[b], (i / 2 - 1) & 1))) {
        if (lane == 0) atomicExch(p.status, 94);
        break;
      }
      tc::fence_after();
      const uint32_t acc = tmem + b * SLOT1;
      const bool another = pair_id + (i + 1) * pair_count < all;
      for (int kb = 0; kb < stages; ++kb) {
        const int next = s + 1 == STAGES ? 0 : s + 1, next_turn = s + 1 == STAGES ? turn ^ 1 : turn;
        const bool more = kb + 1 < stages || another;
        if (kb > 0 && more && !scales(next, next_turn, set ^ 1)) {
          ok = false;
          break;
        }
        const uint32_t sa = tmem + SCALE_AT + set * SET_COLS, sb = sa + SA_COLS;
        const uint64_t a = operands + (s * STAGE >> 4), w = a + (B_AT >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc::mma_mx_pair_if(mine, acc, a + (k * 32 >> 4), w + (k * 32 >> 4), tc::idesc_mxf4(2 * BM, BN, k % 2 * 2), sa + k / 2 * 4, sb + k / 2 * CHUNK_COLS,
                             kb | k);
        tc::commit_pair_if(mine, &empty[s]);
        if (kb == 0 && more && !scales(next, next_turn, set ^ 1)) {        // (a tile's first products have waited long enough)
          ok = false;
          break;
        }
        s = next;
        turn = next_turn;
        set ^= 1;
      }
      tc::commit_pair_if(mine, &acc_full[b]);
    }
  } else {                                        // ---- results
    const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
    // What has been read is in registers when the warp arrives; a release towards the cluster would wait for the results' stores, 1,700 cycles a tile.
    auto arrive = [&](uint64_t* bar) {
      tc::fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(tc::even_block(bar)) : "memory");
    };
    for (int i = 0; tile_at(i, t); ++i) {
      const int b = i & 1;
      const float score = GLU && r < t.rows ? mx::score_of(p, t.row0 + r) : 1.f;
      if (!tc::mbar_wait_warp(&acc_full[b], (i / 2) & 1)) {
        if (lane == 0) atomicExch(p.status, 93);
        break;
      }
      tc::fence_after();
      const uint32_t from = tmem + b * SLOT1 + ((uint32_t)(quarter * 32) << 16);
      const bool live = quarter * 32 < t.rows;
#pragma unroll
      for (int j = 0; j < 2; ++j) {               // 64 columns of this warp at a time, the shared ones first
        const int g = b == 0 ? 3 - half - 2 * j : half + 2 * j, f = t.f0 + g * 64;
        const bool some = live && f < p.n_out;
        uint32_t lo[32], hi[32];
        __syncwarp();                             // (lanes part where rows or features end; the loads want the warp together)
        if (some) {
          tc::ld32_nowait(from + g * 64, lo);
          tc::ld32_nowait(from + g * 64 + 32, hi);
          tc::wait_ld();
        }
        if (j == 0 && half == 0) arrive(acc_shared);
        if (j == 1) arrive(&acc_empty[b]);
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
  tc::fence_before();
  __syncwarp();
  tc::cluster_meet();                             // neither block's barriers or tensor memory are reached for any more
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::dealloc_pair(tmem, TMEM_COLS);
  }
}

template <bool GLU>
int pairs(const Call& c, const Params& p, int pairs) {
  Maps maps;
  if (!tc::make_map_bytes(&maps.x, c.x, (uint64_t)p.rows, (uint64_t)c.K / 2, BM) ||
      !tc::make_map_bytes(&maps.w, c.w, (uint64_t)p.experts * p.n_out, (uint64_t)c.K / 2, BN / 2) ||
      !tc::make_map_scales(&maps.x_scales, c.x_scales, (uint64_t)c.scale_tiles * p.chunks, KB / mx::CHUNK) ||
      !tc::make_map_scales(&maps.w_scales, c.w_scales, (uint64_t)p.experts * p.w_tiles * p.chunks, KB / mx::CHUNK))
    return HB_ERR_UNSUPPORTED;
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256 && STAGES * STAGE + 1280 + 12 * (MOST_EXPERTS + 1) <= 227 * 1024, "the barriers and tables fit");
  const size_t smem = (size_t)STAGES * STAGE + 1024 + 256 + 12 * ((size_t)p.experts + 1);
  auto* kernel = mx_gemm_kernel<GLU>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e = hb::allow_smem(kernel, 227 * 1024, allowed);
  if (e != cudaSuccess) return (int)e;
  return mx::start(kernel, maps, p, THREADS, 2 * pairs, 2, smem, c.stream);
}

// The form by a model of the time in us. Few rows (mx_gemm_few_tc.cu): a stage of 128 weight rows by n rows takes a block 0.12 + 0.0014 n, 0.2 at least,
// and the first stage's way and the last results 3.4; n blocks that share K 4.3, 0.07 a tile, 0.17 a stage and 0.02 + 0.05 / n a row. Pairs: a stage 0.34
// in the first round and 0.44 in others (the card is at its power limit then), 6.5 besides. A tile takes what its results take at least: 0.4 + 0.022 n, of a
// gated unit 0.5 + 0.035 n, a pair 5. An expert's last tile is taken to be half full. For several experts' rows fractions of a round count, which is right for
// many tiles and too little for fewer than there are SMs: clusters share K for one run of rows and for a single routed row only (two rows of 16
// experts of 2,048 x 8,192 would take 9.8 by these constants, 4.8 by the rule, 7.9 in four parts). Measured (us):
//   pairs / single blocks: 512 x 16,384 x 5,120 22.3 / 24.0, 700 x 5,120 x 8,192 17.9 / 18.1, 2,048 x 16,384 x 5,120 66 / 73, units of 700 x 8,192 x 5,120
//   28.8 / 34.0, 99 x 5,120 x 8,192 17.0 / 11.8; 16 experts of 5,120 x 8,192, 4,096 rows: up 210 / 216, down 121 / 117, 2,048 rows: 155 / 148, 83 / 79; 12,288 rows of 64
//   experts of 2,048 x 1,024: 49 / 57, 45 / 36;
//   one, two, four and eight parts: 1 x 256 x 8,192 7.9 / 6.7 / 5.9 / 5.5, 16 x 2,048 x 8,192 9.0 / 8.7 / 7.5 / 12.4 (more clusters than live at a
//   time), 60 x 2,048 x 4,096 6.8 / 9.1 / 7.9 / 13.3; one and three: 1 x 5,120 x 8,192 9.5 / 8.6, 60 x 5,120 x 8,192 10.2 / 10.8;
//   tiles of up to 64, 128 and 256 rows: 8 x 7,168 x 5,120 7.5 / 7.8 / 9.4; of 128, 192 and 256: 256 x 5,120 x 8,192 12.4 / 15.3 / 17.9, 512 x 5,120 x
//   8,192 19.6 / 15.5 / 18.4, 160 x 16,384 x 5,120 15.1 / 13.4 / 14.6, 700 x 16,384 x 5,120 33.6 / 32.7 / 31.2; experts' up and down with 64 rows each 116,
//   63 / 123, 69 / 124, 74, with 128 each 165, 79 / 166, 79 / 148, 82 (for a second or more 307 / 318 / 313 the two together), with 256 each 261, 117 / 235,
//   128 / 216, 124.
// A single block's tile of n rows: its stages, or its results where those take longer.
float tile_us(int stages, float n, bool glu) { return fmaxf(stages * fmaxf(0.2f, 0.12f + 0.0014f * n), glu ? 0.5f + 0.035f * n : 0.4f + 0.022f * n); }
// `runs`: experts that may have rows. splits 0: pairs of blocks; else single ones, so many of them on a tile, with up to `most_rows` rows of it.
struct Form { int splits, most_rows; };
Form form(int rows, int experts, int n_out, int chunks, bool glu) {
  const int runs = experts < rows ? experts : rows, each = (rows + runs - 1) / runs, stages = chunks / 2;
  const long long f_tiles = (n_out + 127) / 128, f_pairs = (n_out + BN - 1) / BN;
  int most_rows = 64;
  float single = 3.4e38f, pair;
  if (runs == 1) {
    for (int t = rows <= 64 ? 64 : 128; t <= (rows <= 64 ? 64 : 256); t += 64) {
      const int tiles = (rows + t - 1) / t;
      const float us = 3.4f + (f_tiles * tiles + 147) / 148 * tile_us(stages, (float)rows / tiles, glu);
      if (us < single) { single = us; most_rows = t; }
    }
    pair = 6.5f + ((rows + 2 * BM - 1) / (2 * BM) * f_pairs + 73) / 74 * fmaxf(5.f, stages * 0.44f) - stages * 0.1f;
  } else {
    if (rows > 64) most_rows = each <= 128 ? 128 : 256;
    const float tiles = runs * (each > most_rows ? (float)each / most_rows + 0.5f : 1.f), pairs = runs * ((float)each / (2 * BM) + 0.5f);
    single = 3.4f + f_tiles / 148.f * tiles * tile_us(stages, rows / tiles, glu);
    pair = 6.5f + f_pairs / 74.f * pairs * fmaxf(5.f, stages * 0.44f);
  }
  Form best{single <= pair ? 1 : 0, most_rows};
  float least = fminf(single, pair);
  const long long most = ((rows + BM - 1) / BM + runs - 1LL) * f_tiles;                // tiles that there may be
  for (int n = 2; n <= MOST_SPLITS && n <= stages && n * most <= 148; ++n) {
    const float shared = 4.3f + 0.07f * most + (stages + n - 1) / n * 0.17f + each * (0.02f + 0.05f / n);
    if (shared < least && most <= hb_mx_clusters(n)) { least = shared; best = {n, 128}; }
  }
  return best;
}

int gemm(const Call& c, const Params& p, bool glu) {
  const Form f = form(p.rows, p.experts, p.n_out, p.chunks, glu);
  if (f.splits || p.raw) return hb_mx_gemm_few(c, p, glu, f.splits ? f.splits : 1, f.most_rows);
  const int runs = p.experts < p.rows ? p.experts : p.rows;
  const long long most = ((p.rows + 2 * BM - 1) / (2 * BM) + runs - 1LL) * ((p.n_out + BN - 1) / BN);      // tiles that there may be
  const int n = (int)(most < 74 ? most : 74);
  return glu ? pairs<true>(c, p, n) : pairs<false>(c, p, n);
}

}  // namespace

// Rows (codes, scales; `offsets` the plan's, or null with experts 1) by weights [experts, n_out, K]. raw not null: they are quantised first, as
// hb_mx_quantize does (raw_dtype, raw_ld; with offsets in the order of sorted_entry, entries / top_k), or with x null, up to 16 rows of up to 10,240
// values of one run, by the product's own blocks. glu 0: out [rows, n_out] in out_dtype, bias
// bfloat16 [n_out] or null. glu 1: n_out is twice the features, gate and up in turn by 32; out codes and out_scales of the features; scores
// (with sorted_entry: by entry, else by row) or null, limit > 0 for the clamped unit. status: one int on the device, nonzero after a wait that ran out.
extern "C" int hb_mx_gemm(const void* raw, int raw_dtype, long long raw_ld, int top_k, void* x, void* x_scales, int rows, const int* offsets,
                          int experts, const void* w, const void* w_scales, int n_out, int K, const void* bias, const int* sorted_entry,
                          const float* scores, int glu, float limit, void* out, int out_dtype, void* out_scales, int* status, cudaStream_t stream) {
  const bool direct = raw && !x;
  if (direct && (offsets || rows > mx::FEWEST || K > mx::FEWEST_K)) return HB_ERR_BAD_ARG;
  if ((!direct && (!x || !x_scales)) || !w || !w_scales || !out || !status || rows < 0 || n_out < 0 || K <= 0 || experts < 1 || (!offsets && experts != 1) ||
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
  if (direct && (K % mx::BLOCK || (reinterpret_cast<uintptr_t>(raw) & 15) || raw_ld * (raw_dtype == HB_DTYPE_F32 ? 4 : 2) % 16 ||
                 (raw_dtype != HB_DTYPE_F32 && raw_dtype != HB_DTYPE_BF16)))
    return HB_ERR_UNSUPPORTED;
  if (raw && !direct) {
    const int e = hb_mx_quantize(raw, raw_dtype, raw_ld, rows, K, offsets ? sorted_entry : nullptr, top_k, offsets, experts, x, x_scales, stream);
    if (e != HB_OK) return e;
  }
  const Params p{(const uint8_t*)x_scales, (const uint8_t*)w_scales, offsets, sorted_entry, scores, (const __nv_bfloat16*)bias, out, (uint8_t*)out_scales, status, out_dtype == HB_DTYPE_F32, rows,
                 experts, n_out, mx::chunks(K), (n_out + 127) / 128, limit, raw && !direct, direct ? raw : nullptr, raw_ld, raw_dtype == HB_DTYPE_F32, K};
  const Call c{x, x_scales, w, w_scales, K, (rows + BM - 1) / BM + (experts < rows ? experts : rows) - 1, stream};
  return gemm(c, p, glu != 0);
}

// The form that hb_mx_gemm takes: 0 pairs of blocks, else 1000 times the blocks that share a tile's K and the rows of a tile.
extern "C" int hb_mx_gemm_form(int rows, int experts, int n_out, int K, int glu) {
  if (rows < 1 || experts < 1 || n_out < 1 || K < 1) return -1;
  const Form f = form(rows, experts, n_out, mx::chunks(K), glu != 0);
  return f.splits ? f.splits * 1000 + f.most_rows : 0;
}
