// Products of many tokens with weights of four bits on the 5th-generation tensor cores (tcgen05): out[t, n] = sum_k x[t, k] w[n, k]
// (+ bias[n]), w in the blocks of four_bit_linear.cu, x bfloat16, float32 sums in tensor memory.
//
// The product is taken transposed as in grouped_gemm_tc.cu: 128 weight rows are the MMA's M, up to 256 tokens its N. The operand in shared
// memory has to be bfloat16, so here, unlike for a few tokens, scale * (code - 8) is rounded to it (2^-8 of a weight at most, as a bfloat16
// checkpoint's weights are; the group's scale cannot wait for the sum, which runs over all groups in tensor memory). A stage is 128 k, one
// block of weights a row tile of 16:
//   warp 0        brings the tokens' tile by TMA (two boxes of 64 k, 128-byte swizzle)
//   warp 2        brings the 8 row tiles' blocks of codes as one bulk copy each, stages ahead, into a ring of their own
//   warps 3 .. 18 unpack: eight of them the stage's first 64 k, the others the rest, each a row tile
//   warp 1        issues the products, eight of 16 k a stage, and the commits
//   warps 19 .. 22 read the sums back, add the bias and store: the next tile accumulates into the other half of tensor memory
// A pair of codes is a pair of denormals after an AND (four_bit.cuh), and code * 2^-133 times scale * 2^73 minus 8 scale * 2^-60 is one
// instruction with one rounding: the tile holds 2^-60 of the weights, the results are multiplied by 2^60. 9 instructions a word of eight codes
// (code in the mantissa of 128, minus 136, times the scale: 15).
// Every row tile is unpacked once per tile of tokens, and where its weights wait decides what a stage takes. Up to 128 tokens: in tensor
// memory, from which the products read them: a warp stores its 16 rows x 64 k as one instruction, 64 columns a stage behind the sums, and shared
// memory has the tokens alone to bring to the tensor cores and room for 4 to 6 stages. (In shared memory, a 16-byte store a word, three
// stages, the same splits: 64 x 16,384 x 5,120 25.9 us instead of 22.5, 128 of 30.6 / 23.3, 99 x 7,168 x 5,120 21.1 / 17.9, 17 x 5,120 x 5,120 15.8 /
// 14.6, where the weights alone take 6.7, 6.7, 3.0 and 2.1.) What is left there is the unpacking warps' work, 0.43 us a stage, of which the
// products of 64 tokens take a fifth.
// PAIR: two blocks of a cluster on 256 rows x up to 256 tokens (cta_group::2), each with its 128 rows and half of the tokens, for
// many tokens, where the tokens' way from L2 would bound single blocks; weights in shared memory, swizzled, eight lanes with rows i and i + 4,
// which meet eight banks of 16 bytes (tensor memory holds two tiles' sums). 2,048 x 16,384 x 5,120 221 to 231 us, 1.48 to 1.55 PFLOP/s.
// SPLIT: few tiles: the blocks of a cluster share out K, one tile a cluster; each sends its sums to the block that finishes those
// tokens, which adds them in the order of the blocks. Which form when: `gemm`, below.
// Every wait is bounded; a block that gave up says where in `status` and leaves by the common exit.
#include <cuda.h>

#include "api.h"
#include "common.cuh"
#include "four_bit.cuh"
#include "tc.cuh"

namespace {

constexpr int BF = 128, KB = 128;                 // weight rows of a block, k of a stage
constexpr int A_BYTES = BF * KB * 2;
constexpr int UNPACK = 8, EPILOGUE = 4;           // warps: to unpack half a stage, to write results
constexpr int FIRST_UNPACK = 3, FIRST_EPILOGUE = FIRST_UNPACK + 2 * UNPACK, THREADS = 32 * (FIRST_EPILOGUE + EPILOGUE);
constexpr int RAW_BLOCK = 1152;                   // room for a block of codes and scales, the largest
constexpr int MOST_SPLITS = 8;                    // blocks that share out K
constexpr size_t stage_bytes(bool pair, int bt) { return (pair ? A_BYTES + bt / 2 * KB * 2 : bt * KB * 2); }

struct Params {
  const uint8_t* w;
  const __nv_bfloat16* bias;
  void* out;
  int* status;
  int out_f32, tokens, n_out, chunks, most;       // most: tokens of a tile, a multiple of 16
  int box;                                        // rows of a tokens' box: as many as a tile needs
  unsigned zero;                                  // 0, unknown to the compiler
};

// An arrival on the even block's barrier of what this block's own tensor cores read from its own shared memory: ordered within the block (a
// release towards the cluster took 1,500 cycles a stage).
__device__ __forceinline__ void arrive_pair(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint2 load8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(tc::smem_u32(p)) : "memory");
  return v;
}
// Four steps of 16 k of rows g and g + 8 into tensor memory, 32 columns of 16 lanes: a step is 8 columns, of which a lane has two neighbours.
__device__ __forceinline__ void store_rows(uint32_t taddr, const uint4& a0, const uint4& a1, const uint4& b0, const uint4& b1) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(a0.x), "r"(a0.y), "r"(b0.x), "r"(b0.y), "r"(a0.z), "r"(a0.w), "r"(b0.z), "r"(b0.w),
        "r"(a1.x), "r"(a1.y), "r"(b1.x), "r"(b1.y), "r"(a1.z), "r"(a1.w), "r"(b1.z), "r"(b1.w) : "memory");
}
template <int GPC> __device__ __forceinline__ uint2 row_scales(const uint8_t* p) {
  if constexpr (GPC == 1) return make_uint2(*reinterpret_cast<const unsigned short*>(p), 0u);
  else if constexpr (GPC == 2) return make_uint2(*reinterpret_cast<const unsigned*>(p), 0u);
  else return *reinterpret_cast<const uint2*>(p);
}
// Scale i of four, what it multiplies codes by in each place of a word, and what eight of it comes to; in both halves.
struct Factors { unsigned low, high, minus_eight; };
__device__ __forceinline__ Factors factors(uint2 v, int i) {
  const unsigned s = __byte_perm(i < 2 ? v.x : v.y, 0u, i & 1 ? 0x3232 : 0x1010);
  Factors f;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(f.low) : "r"(s), "r"(0x64006400u));             // 2^73
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(f.high) : "r"(s), "r"(0x62006200u));            // 2^69
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(f.minus_eight) : "r"(s), "r"(0xa300a300u));     // -2^-57
  return f;
}
constexpr float GROW = 1152921504606846976.f;     // 2^60, of the results
// eight codes as bfloat16 scale * (code - 8) * 2^-60
__device__ __forceinline__ uint4 unpack(unsigned w, const Factors& f) {
  unsigned r[4];
#pragma unroll
  for (int i = 0; i < 2; ++i, w >>= 8) {
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r[2 * i]) : "r"(w & fb::LOW), "r"(f.low), "r"(f.minus_eight));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r[2 * i + 1]) : "r"(w & fb::HIGH), "r"(f.high), "r"(f.minus_eight));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

template <bool PAIR, bool SPLIT, int BT, int STAGES, int RAW, int GPC>
__global__ void __launch_bounds__(THREADS, 1)
four_bit_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const Params p) {
  constexpr int XR = PAIR ? BT / 2 : BT;          // token rows of a stage
  constexpr int X_BYTES = XR * KB * 2, STAGE_BYTES = (PAIR ? A_BYTES : 0) + X_BYTES, X_AT = STAGE_BYTES - X_BYTES;
  constexpr int BLOCK_BYTES = 1024 + 32 * GPC;
  constexpr int SLOTS = SPLIT ? 1 : 2;
  constexpr int TMEM_COLS = 512, A_COLS = KB / 2;          // sums first, then, without PAIR, the stages' weights
  static_assert(!(PAIR && SPLIT) && SLOTS * BT + (PAIR ? 0 : STAGES * A_COLS) <= TMEM_COLS, "a form at a time, all within tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* raw = smem + STAGES * STAGE_BYTES;     // [RAW][UNPACK][RAW_BLOCK]
  uint64_t* full_x = reinterpret_cast<uint64_t*>(raw + RAW * UNPACK * RAW_BLOCK);
  uint64_t* full_a = full_x + STAGES;
  uint64_t* empty = full_a + STAGES;
  uint64_t* acc_full = empty + STAGES;            // [2]
  uint64_t* acc_empty = acc_full + 2;             // [2]
  uint64_t* raw_full = acc_empty + 2;             // [RAW]
  uint64_t* raw_empty = raw_full + RAW;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + RAW);

  const int warp = tc::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = PAIR || SPLIT ? (int)tc::cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(&full_x[s], 1);
      tc::mbar_init(&full_a[s], (PAIR ? 4 : 2) * UNPACK);
      tc::mbar_init(&empty[s], 1);
    }
    for (int r = 0; r < RAW; ++r) { tc::mbar_init(&raw_full[r], 1); tc::mbar_init(&raw_empty[r], 2 * UNPACK); }
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], PAIR ? 2 * EPILOGUE : EPILOGUE); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) tc::alloc_pair(tmem_slot, TMEM_COLS);
    else tc::alloc(tmem_slot, TMEM_COLS);
  }
  tc::fence_before();
  if constexpr (PAIR) tc::cluster_meet();         // (the other block's barriers are ready too)
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  constexpr int FEATURES = PAIR ? 2 * BF : BF;
  const int f_tiles = (p.n_out + FEATURES - 1) / FEATURES, t_tiles = (p.tokens + p.most - 1) / p.most, all = f_tiles * t_tiles;
  int splits = 1;
  if constexpr (SPLIT) asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(splits));
  const int group = PAIR ? 2 : splits, units = gridDim.x / group, unit = blockIdx.x / group;
  const int share = (p.chunks + splits - 1) / splits;
  const int c0 = SPLIT ? rank * share : 0, c1 = SPLIT ? min(p.chunks, c0 + share) : p.chunks;
  // tiles in order of weights: neighbours share their tokens
  auto tile_at = [&](int i, int& f0, int& t0, int& n) {
    const int t = unit + i * units;
    if (t >= all) return false;
    f0 = t % f_tiles * FEATURES;
    t0 = t / f_tiles * p.most;
    n = min(p.most, p.tokens - t0);
    return true;
  };

  if (warp == 0) {                                // ---- tokens
    int s = 0, turn = 1, issued = 0, f0, t0, n;
    bool ok = true;
    const uint32_t mine = tc::elect_one(), ring = tc::smem_u32(smem), bars = PAIR ? tc::even_block(full_x) : tc::smem_u32(full_x);
    for (int i = 0; ok && tile_at(i, f0, t0, n); ++i) {
      const int row = tc::uniform(t0 + (PAIR ? rank * ((n + 15) / 16 * 8) : 0));      // a pair's tokens are half in one block, half in the other
      for (int c = tc::uniform(c0); c < c1; ++c) {
        if (!tc::mbar_wait_warp(&empty[s], turn)) {
          if (lane == 0) atomicExch(p.status, 81);
          ok = false;
          break;
        }
        const uint32_t to = ring + s * STAGE_BYTES + X_AT, bar = bars + s * 8;
        if (mine && rank == 0 | !PAIR) tc::mbar_expect_tx(&full_x[s], (PAIR ? 2 : 1) * p.box * KB * 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (PAIR) tc::tma_load_2d_pair_if(mine, to + h * (X_BYTES / 2), &map_x, c * KB + h * 64, row, bar);
          else tc::tma_load_2d_if(mine, to + h * (X_BYTES / 2), &map_x, c * KB + h * 64, row, bar);
        }
        if (++s == STAGES) { s = 0; turn ^= 1; }
        ++issued;
      }
    }
    // nothing reaches for the block's memory when it ends: the last commits have arrived, which come behind the products and those behind
    // the copies; where a wait ran out they may never, and the copies on their way are waited for
    if (ok) {
      for (int i = 0; i < STAGES && tc::mbar_wait_warp(&empty[s], turn); ++i)
        if (++s == STAGES) { s = 0; turn ^= 1; }
    } else if (rank == 0 || !PAIR) {
      for (int i = max(0, issued - STAGES); i < issued; ++i) tc::mbar_wait_warp(&full_x[i % STAGES], (i / STAGES) & 1);
    }
  } else if (warp == 1) {                         // ---- products
    const uint32_t mine = tc::elect_one();
    const uint64_t ring = tc::desc_kmajor(tc::smem_u32(smem));
    int s = 0, turn = 0, f0, t0, n;
    bool ok = true;
    for (int i = 0; (rank == 0 || !PAIR) && ok && tile_at(i, f0, t0, n); ++i) {
      const int b = i % SLOTS;
      if (i >= SLOTS && !tc::mbar_wait_warp(&acc_empty[b], (i / SLOTS - 1) & 1)) {
        if (lane == 0) atomicExch(p.status, 84);
        break;
      }
      tc::fence_after();
      const uint32_t idesc = tc::idesc_bf16(FEATURES, tc::uniform((n + 15) & ~15), false), acc = tmem + b * BT;
      for (int c = c0; c < c1; ++c) {
        if (!tc::mbar_wait_warp(&full_x[s], turn) || !tc::mbar_wait_warp(&full_a[s], turn)) {
          if (lane == 0) atomicExch(p.status, 82);
          ok = false;
          break;
        }
        tc::fence_after();
        const uint64_t a = ring + s * (STAGE_BYTES >> 4), x = a + (X_AT >> 4);
        const uint32_t a_tmem = tmem + SLOTS * BT + s * A_COLS;
#pragma unroll
        for (int k = 0; k < KB / 16; ++k) {
          const uint64_t ka = a + ((k / 4 * (A_BYTES / 2) + k % 4 * 32) >> 4), kx = x + ((k / 4 * (X_BYTES / 2) + k % 4 * 32) >> 4);
          if constexpr (PAIR) tc::mma_pair_if(mine, acc, ka, kx, idesc, (c - c0) | k);
          else tc::mma_a_tmem_if(mine, acc, a_tmem + k * 8, kx, idesc, (c - c0) | k);
        }
        if constexpr (PAIR) tc::commit_pair_if(mine, &empty[s]);
        else tc::commit_if(mine, &empty[s]);
        if (++s == STAGES) { s = 0; turn ^= 1; }
      }
      if constexpr (PAIR) tc::commit_pair_if(mine, &acc_full[b]);
      else tc::commit_if(mine, &acc_full[b]);
    }
  } else if (warp == 2) {                         // ---- codes
    const int row_tiles = (p.n_out + 15) / 16;
    int r = 0, turn = 1, issued = 0, f0, t0, n;
    bool ok = true;
    for (int i = 0; ok && tile_at(i, f0, t0, n); ++i) {
      const int tile = f0 / 16 + rank * (PAIR ? UNPACK : 0), tiles = max(0, min(UNPACK, row_tiles - tile));
      const uint8_t* from = p.w + ((size_t)(tile + lane) * p.chunks + c0) * BLOCK_BYTES;
      for (int c = c0; c < c1; ++c, from += BLOCK_BYTES) {
        if (!tc::mbar_wait_warp(&raw_empty[r], turn)) {
          if (lane == 0) atomicExch(p.status, 86);
          ok = false;
          break;
        }
        if (lane == 0) tc::mbar_expect_tx(&raw_full[r], tiles * BLOCK_BYTES);
        __syncwarp();
        if (lane < tiles)
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(tc::smem_u32(raw + (r * UNPACK + lane) * RAW_BLOCK)), "l"(from), "r"(BLOCK_BYTES), "r"(tc::smem_u32(&raw_full[r]))
                       : "memory");
        if (++r == RAW) { r = 0; turn ^= 1; }
        ++issued;
      }
    }
    for (int i = max(0, issued - RAW); i < issued; ++i) tc::mbar_wait_warp(&raw_full[i % RAW], (i / RAW) & 1);      // no copy is under way at the end
  } else if (warp < FIRST_EPILOGUE) {             // ---- weights
    // PAIR: row tile `part`, rows g and g + 8 of lanes in an order for the stores. Else the warp's part of tensor memory: its quarter's first or
    // second 16 lanes, rows as the store's fragments have them.
    const int half = (warp - FIRST_UNPACK) / UNPACK, q4 = lane & 3;
    const int part = PAIR ? (warp - FIRST_UNPACK) % UNPACK : (warp & 3) * 2 + (warp - FIRST_UNPACK) / 4 % 2;
    const int g = PAIR ? lane >> 3 | (lane & 4) : lane >> 2;
    int f0, t0, n;
    const uint32_t bars = PAIR ? tc::even_block(full_a) : tc::smem_u32(full_a);
    uint8_t* const row = smem + half * (A_BYTES / 2) + (part * 16 + g) * 128;
    int tiles = 0;
    while (tile_at(tiles, f0, t0, n)) ++tiles;
    const int stages = c1 > c0 ? tiles * (c1 - c0) : 0;
    int s = 0, turn = 1, r = 0, r_turn = 0;
    uint4 a0, a1, b0, b1;                         // what goes into the next stage: rows g and g + 8, two words of 32 k each
    const unsigned pick = q4 & 1 ? 0x7351u : 0x6240u;
    auto next = [&]() {                           // false: the codes did not come
      if (!tc::mbar_wait_warp(&raw_full[r], r_turn)) {
        if (lane == 0) atomicExch(p.status, 87);
        return false;
      }
      const uint8_t* block = raw + (r * UNPACK + part) * RAW_BLOCK;        // (rows past the weight's: whatever is there; they are not written out)
      uint2 lo, hi;
      if constexpr (PAIR) {                       // k 8 q4 .. + 7 of each 32
        const uint8_t* words = block + (g * 4 + q4) * 16 + half * 8;
        lo = load8(words);
        hi = load8(words + 512);
      } else {                                    // k 4 q4 .. + 3 and 16 + 4 q4 .. + 3: a part of two words, one of k under 16 and one of the rest
        const uint8_t* words = block + (g * 4 + q4 / 2) * 16 + half * 8;
        const uint2 l0 = load8(words), l1 = load8(words + 32), h0 = load8(words + 512), h1 = load8(words + 544);
        lo = make_uint2(__byte_perm(l0.x, l1.x, pick), __byte_perm(l0.y, l1.y, pick));
        hi = make_uint2(__byte_perm(h0.x, h1.x, pick), __byte_perm(h0.y, h1.y, pick));
      }
      const uint2 s_lo = row_scales<GPC>(block + 1024 + g * 2 * GPC), s_hi = row_scales<GPC>(block + 1024 + (g + 8) * 2 * GPC);
      const int k0 = GPC == 1 ? 0 : GPC == 2 ? half : 2 * half, k1 = GPC == 4 ? k0 + 1 : k0;
      const Factors lo0 = factors(s_lo, k0), hi0 = factors(s_hi, k0);
      const Factors lo1 = GPC == 4 ? factors(s_lo, k1) : lo0, hi1 = GPC == 4 ? factors(s_hi, k1) : hi0;
      a0 = unpack(lo.x, lo0);
      a1 = unpack(lo.y, lo1);
      b0 = unpack(hi.x, hi0);
      b1 = unpack(hi.y, hi1);
      // The place is given back when the loads have come: the barrier's address waits for them. (An arrival right behind the loads, and one behind
      // their use as the source has it, overtook them at times, and the next codes were read.)
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&raw_empty[r] + ((lo.x ^ lo.y ^ hi.x ^ hi.y ^ s_lo.x ^ s_lo.y ^ s_hi.x ^ s_hi.y) & p.zero));
      if (++r == RAW) { r = 0; r_turn ^= 1; }
      return true;
    };
    bool ok = stages > 0 && next();
    for (int i = 0; ok && i < stages; ++i) {
      if (!tc::mbar_wait_warp(&empty[s], turn)) {
        if (lane == 0) atomicExch(p.status, 83);
        break;
      }
      if constexpr (PAIR) {
        uint8_t *at0 = row + s * STAGE_BYTES + ((q4 ^ g) << 4), *at1 = row + s * STAGE_BYTES + (((4 | q4) ^ g) << 4);
        *reinterpret_cast<uint4*>(at0) = a0;
        *reinterpret_cast<uint4*>(at1) = a1;
        *reinterpret_cast<uint4*>(at0 + 8 * 128) = b0;
        *reinterpret_cast<uint4*>(at1 + 8 * 128) = b1;
      } else {
        tc::fence_after();
        store_rows(tmem + SLOTS * BT + s * A_COLS + half * (A_COLS / 2) + ((uint32_t)(part * 16) << 16), a0, a1, b0, b1);
      }
      if (i + 1 < stages) ok = next();            // while the stores are on their way: the fence waits for them
      if constexpr (PAIR) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      } else {
        tc::wait_st();
        tc::fence_before();
      }
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) arrive_pair(bars + s * 8);
        else tc::mbar_arrive(&full_a[s]);
      }
      if (++s == STAGES) { s = 0; turn ^= 1; }
    }
  } else if constexpr (!SPLIT) {                  // ---- results
    const int quarter = warp & 3;
    int f0, t0, n;
    for (int i = 0; tile_at(i, f0, t0, n); ++i) {
      const int b = i % SLOTS, f = f0 + rank * BF + quarter * 32 + lane;
      const bool f_ok = f < p.n_out;
      const float bias = p.bias && f_ok ? __bfloat162float(p.bias[f]) : 0.f;
      if (!tc::mbar_wait_warp(&acc_full[b], (i / SLOTS) & 1)) {
        if (lane == 0) atomicExch(p.status, 85);
        break;
      }
      tc::fence_after();
#pragma unroll 1
      for (int c = 0; c < n; c += 32) {
        float v[32];
        tc::ld32(tmem + b * BT + ((uint32_t)(quarter * 32) << 16) + c, v);
        if (!f_ok) continue;
        const size_t at = (size_t)(t0 + c) * p.n_out + f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (c + j >= n) break;
          if (p.out_f32) reinterpret_cast<float*>(p.out)[at + (size_t)j * p.n_out] = fmaf(v[j], GROW, bias);
          else reinterpret_cast<__nv_bfloat16*>(p.out)[at + (size_t)j * p.n_out] = __float2bfloat16_rn(fmaf(v[j], GROW, bias));
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) tc::arrive_even(tc::even_block(&acc_empty[b]));
        else tc::mbar_arrive(&acc_empty[b]);
      }
    }
  }
  if constexpr (SPLIT) {
    // the cluster's one tile: every block sends its sums of a run of tokens to the block that finishes it
    int f0, t0, n;
    const bool there = tile_at(0, f0, t0, n);
    bool ok = true;
    if (there && c0 < c1 && warp >= FIRST_UNPACK) {
      ok = tc::mbar_wait_warp(&acc_full[0], 0);
      if (!ok && lane == 0) atomicExch(p.status, 85);
    }
    tc::fence_after();
    __syncwarp();
    tc::cluster_meet();                           // every block's ring is free
    const int run = (n + splits - 1) / splits;
    if (there && c0 < c1 && warp >= FIRST_UNPACK) {
      const int quarter = warp & 3, turns = (FIRST_EPILOGUE + EPILOGUE - FIRST_UNPACK) / 4;     // five warps a quarter of the rows, 32 tokens in turn
      int turn = (warp - FIRST_UNPACK) / 4;
#pragma unroll 1
      for (int r = 0; r < splits; ++r) {
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at)
            : "r"(tc::smem_u32(smem) + (uint32_t)((rank * run * BF + quarter * 32 + lane) * 4)), "r"(r));
        const int end = min(n, (r + 1) * run);
#pragma unroll 1
        for (int c = r * run; c < end; c += 32) {
          if (turn-- > 0) continue;
          turn = turns - 1;
          float v[32];
          tc::ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < end) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + (c - r * run + j) * BF * 4), "f"(v[j]) : "memory");
        }
      }
    }
    __syncwarp();
    tc::cluster_meet();
    const int mine = there ? min(run, n - rank * run) : 0;
    const float* sums = reinterpret_cast<const float*>(smem);
    for (int i = threadIdx.x; i < mine * BF; i += THREADS) {
      const int f = f0 + i % BF;
      if (f >= p.n_out) continue;
      float v = 0.f;
      for (int r = 0; r * share < p.chunks; ++r) v += sums[r * run * BF + i];      // (of the blocks that had a part of K)
      v = fmaf(v, GROW, p.bias ? __bfloat162float(p.bias[f]) : 0.f);
      const size_t at = (size_t)(t0 + rank * run + i / BF) * p.n_out + f;
      if (p.out_f32) reinterpret_cast<float*>(p.out)[at] = v;
      else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    }
  }
  tc::fence_before();
  __syncwarp();
  if constexpr (PAIR) tc::cluster_meet();         // no product of the pair reads this block any more
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    if constexpr (PAIR) tc::dealloc_pair(tmem, TMEM_COLS);
    else tc::dealloc(tmem, TMEM_COLS);
  }
}

// [rows, cols] bfloat16, rows ld elements apart
bool make_map_rows(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  tc::EncodeTiledFn fn = tc::encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld * 2};
  const cuuint32_t box[2] = {64, box_rows}, elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool PAIR, bool SPLIT, int BT, int STAGES, int RAW, int GPC>
int launch(const void* x, long long x_ld, int K, Params p, int blocks, int cluster, cudaStream_t stream) {
  CUtensorMap map;
  p.box = (p.most + 15) / 16 * (PAIR ? 8 : 16);
  if (!make_map_rows(&map, x, p.tokens, K, x_ld, p.box)) return HB_ERR_UNSUPPORTED;
  const size_t smem = STAGES * stage_bytes(PAIR, BT) + RAW * UNPACK * RAW_BLOCK + 1024 + 512;
  auto* kernel = four_bit_gemm_kernel<PAIR, SPLIT, BT, STAGES, RAW, GPC>;
  static std::atomic<unsigned long long> allowed{0};
  cudaError_t e = hb::allow_smem(kernel, (int)smem, allowed);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = cluster > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&config, kernel, map, p);
  return e == cudaSuccess ? HB_OK : (int)e;
}

// How many clusters of `size` blocks live at a time on the current device (0: the runtime does not say).
int clusters_of(int size) {
  static std::atomic<int> known[64][MOST_SPLITS + 1];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device > 63) return 0;
  int n = known[device][size].load(std::memory_order_relaxed);
  if (n > 0) return n;
  auto* kernel = four_bit_gemm_kernel<false, true, 128, 4, 8, 1>;
  constexpr size_t smem = stage_bytes(false, 128) * 4 + 8 * UNPACK * RAW_BLOCK + 1536;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return 0;
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
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n <= 0) return 0;
  known[device][size].store(n, std::memory_order_relaxed);
  return n;
}

// The form, the tokens of a tile and the splits of K by a model of the time in us, fitted to 14 sizes of weight and 7 counts of tokens: a block's
// stage takes 0.43 to 0.46 with 16 to 128 tokens (its unpacking, the products hide behind it), a pair's 0.48 to 0.68 with 32 to 256, in
// rounds of what lives at a time, and splits meet in 0.5 + 0.04 a token. Of 56 launches what it takes is 1.01 of the best form's time,
// 1.08 at worst. Measured, as pairs / single blocks / clusters of splits: 128 x 5,120 x 8,192 40.9 / 32.4 / 19.6 (three), 200 x 5,120 x 8,192
// 45.9 / 31.5 / -, 256 x 7,168 x 5,120 35.7 / 24.6 / -, 512 x 5,120 x 8,192 44.9 (176 tokens a tile; 50.6 with 256) / 60.4 / -, 512 x 16,384 x 5,120
// 65.4 / 77.7 / -, 512 x 1,024 x 8,192 41.3 / 32.2 / 16.9 (four), 17 x 1,024 x 8,192 - / 29.9 / 10.4 (eight).
template <int GPC>
int gemm(const void* x, long long x_ld, int K, Params p, cudaStream_t stream) {
  const int f_tiles = (p.n_out + BF - 1) / BF, fewest = (p.tokens + 255) / 256;
  struct { float us; bool pair; int most, splits; } best{3.4e38f, false, 0, 1};
  for (int t = fewest; t <= fewest + 8; ++t) {
    const int most = ((p.tokens + t - 1) / t + 15) / 16 * 16, tiles = (p.tokens + most - 1) / most;
    auto take = [&](float us, bool pair, int splits) {
      if (us < best.us) best = {us, pair, most, splits};
    };
    take(6.5f + ((f_tiles + 1) / 2 * (long long)tiles + 73) / 74 * p.chunks * (0.45f + 0.0009f * most), true, 1);
    if (most > 128) continue;
    const long long all = (long long)f_tiles * tiles;
    const float stage = 0.42f + 0.0003f * most;
    take(5.5f + (all + 147) / 148 * p.chunks * stage, false, 1);
    for (int s = 2; s <= MOST_SPLITS && s * all <= 148 && 2 * s <= p.chunks; ++s)
      if (all <= clusters_of(s)) take(6.f + 0.04f * most + (p.chunks + s - 1) / s * stage, false, s);
    if (most <= 16) break;
  }
  p.most = best.most;
  if (best.pair) {
    const long long pairs = (f_tiles + 1) / 2 * (long long)((p.tokens + p.most - 1) / p.most);
    return launch<true, false, 256, 3, 3, GPC>(x, x_ld, K, p, 2 * (int)(pairs < 74 ? pairs : 74), 2, stream);
  }
  const long long all = (long long)f_tiles * ((p.tokens + p.most - 1) / p.most);
  if (best.splits == 1) {
    const int blocks = (int)(all < 148 ? all : 148);
    return p.most <= 64 ? launch<false, false, 64, 6, 8, GPC>(x, x_ld, K, p, blocks, 1, stream)
                        : launch<false, false, 128, 4, 8, GPC>(x, x_ld, K, p, blocks, 1, stream);
  }
  const int blocks = (int)all * best.splits;
  return p.most <= 64 ? launch<false, true, 64, 6, 8, GPC>(x, x_ld, K, p, blocks, best.splits, stream)
                      : launch<false, true, 128, 4, 8, GPC>(x, x_ld, K, p, blocks, best.splits, stream);
}

}  // namespace

// Arguments as hb_four_bit_linear; x_ld at least K (a tensor map's rows); status: one int on the device, nonzero after a wait that ran out.
extern "C" int hb_four_bit_linear_tc(const void* x, long long x_ld, const void* w, const void* bias, void* out, int out_dtype,
                                     int tokens, int n_out, int K, int group, int* status, cudaStream_t stream) {
  if (!x || !w || !out || !status || tokens < 0 || n_out < 0 || K < 0 || (out_dtype != HB_DTYPE_F32 && out_dtype != HB_DTYPE_BF16))
    return HB_ERR_BAD_ARG;
  if ((group != 32 && group != 64 && group != 128) || K % group || K == 0 || x_ld % 8 || x_ld < K ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15))
    return HB_ERR_UNSUPPORTED;
  if (tokens == 0 || n_out == 0) return HB_OK;
  const Params p{(const uint8_t*)w, (const __nv_bfloat16*)bias, out, status, out_dtype == HB_DTYPE_F32, tokens, n_out, (K + KB - 1) / KB, 0, 0, 0u};
  return group == 128 ? gemm<1>(x, x_ld, K, p, stream) : group == 64 ? gemm<2>(x, x_ld, K, p, stream) : gemm<4>(x, x_ld, K, p, stream);
}
