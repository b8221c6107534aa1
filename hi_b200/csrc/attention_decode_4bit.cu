// Attention of single decoded tokens over the cache in four bits (four_bit.cuh has its blocks): with the key k_jd = s_jg c_jd + l_jg
// and the value v_jd = t_jg e_jd + m_jg of group g (32 dims),
//   score_ij = sum_g s_jg (sum_d q_d c_jd) + sum_g l_jg (sum_d q_d)            d over the group
//   o_d      = sum_j (p_j t_jg) (e_jd - 8) + sum_j p_j (m_jg + 8 t_jg)         p_j = exp(score - max), then over sum_j p_j
// so the codes enter the tensor cores as they are (whole numbers, exact), a key's scale multiplies the sum of its group, and a value's scale
// the weight it meets. Rounded to bfloat16 are the weights alone, once times the scale and once bare, beside the group's middle and in their
// sum: what they are off by is then relative to values of their own size. (With e_jd and m_jg as they are it was relative to the group's
// range: 0.0036 of the result's size over a long context instead of the 0.0024 that the bfloat16 cache's kernels have.)
//
// Both products are taken transposed, keys (then dims) as the 16 rows of mma.sync and the query heads of a kv head as its 8 columns, half
// the columns that heads as rows would leave empty; the weights change over with movmatrix. The rest is a few more products a
// block of 16 keys: l times the queries' sums in three pieces of bfloat16; for the values a matrix whose rows are the groups' lows, the
// groups' scales and ones, times the bare weights; and the eights, a row a group, times the scaled ones.
//
// Grid (split, kv head x tiles of 8 heads, token). A warp has steps of 32 keys of its own: 2 blocks, which lie side by side in a
// page of 32 and more, come as one bulk copy that the warp's own barrier counts, a few steps ahead; the warps meet at the end only,
// where their sums are joined. The splits of a token are a cluster, which reads one another's shared memory, or leave their rows to
// attention_merge. A step's copies leave out blocks behind the token's own.
// Rows of a block that the token may not read (not written yet, out of its window) hold anything, NaN as well: their scores, scales
// and lows are replaced, in a form of the step for those that have such rows. Every wait is bounded; on a time-out the kernel says so in
// `status` and its output is invalid.
#include "api.h"
#include "common.cuh"
#include "four_bit.cuh"
#include "tc.cuh"

namespace {

constexpr int STEP = 32;         // keys a warp takes at a time
constexpr int TILE = 64;         // splits are cut in these
constexpr int WARPS = 4;
constexpr int STAGES = 2;        // steps in flight a warp
constexpr int HEADS = 8;         // query heads of a block
constexpr int MOST_CLUSTER = 8;

struct Args {
  const __nv_bfloat16* q;
  const uint8_t* pages;
  const int* block_table;
  const int* seq_of_token;
  const int* positions;
  __nv_bfloat16* out;
  float* part_acc;
  float* part_ml;
  int* status;
  const long long* rows;         // the tokens of the launch among the step's, or null
  const float* sink_values;
  int step_tokens, table_stride, nh, nkv, page_size, page_shift, chunk, window, keep, split_tiles, splits, sink;      // page_shift: of a power of two, or -1
  float scale;
  unsigned zero;                 // 0, unknown to the compiler
};

__device__ __forceinline__ unsigned transpose8(unsigned v) {      // an 8 x 8 matrix of 16 bits over the warp
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <int G> struct Words;
template <> struct Words<4> {
  unsigned w[4];
  __device__ __forceinline__ explicit Words(const uint8_t* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
};
template <> struct Words<1> {
  unsigned w[1];
  __device__ __forceinline__ explicit Words(const uint8_t* p) { w[0] = *reinterpret_cast<const unsigned*>(p); }
};
template <> struct Words<2> {
  unsigned w[2];
  __device__ __forceinline__ explicit Words(const uint8_t* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  }
};
// two bfloat16 of a word as floats
__device__ __forceinline__ float low_half(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(unsigned w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ uint32_t in_block(const void* smem, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(smem)), "r"(rank));
  return at;
}
template <bool B> struct Const { static constexpr bool value = B; };

// CLUSTER: the splits of a token's heads are a cluster
template <int G, bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, 3) attn_decode_4bit_kernel(const Args a) {
  using B = fb::Block<G>;
  constexpr int HD = 32 * G, MT = STEP / 16;
  constexpr float RAISE = 18446744073709551616.f;                 // 2^64, of weights that meet codes (four_bit.cuh)
  extern __shared__ __align__(128) uint8_t ring_all[];            // [WARPS][STAGES][MT][B::BYTES]
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ float ml_s[WARPS][HEADS][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q4 = lane & 3;
  const int split = blockIdx.x, per = a.nh / a.nkv, head_tiles = (per + HEADS - 1) / HEADS;
  const int kvh = blockIdx.y / head_tiles, h0 = blockIdx.y % head_tiles * HEADS, heads = min(HEADS, per - h0);
  const int t = blockIdx.z;
  const long long chosen = a.rows ? a.rows[t] : t;
  if (chosen < 0 || chosen >= a.step_tokens) {
    if (threadIdx.x == 0) atomicExch(a.status, 32);
    return;
  }
  const int token = (int)chosen, own = a.positions[token];
  const int pos = (int)min((long long)own, (long long)a.table_stride * a.page_size - 1);      // the last key that the table has a page for
  const int* table = a.block_table + (size_t)a.seq_of_token[token] * a.table_stride;
  int lo = 0;
  if (a.chunk > 0) lo = own / a.chunk * a.chunk;
  if (a.window > 0) lo = max(lo, own - a.window + 1);
  // tiles of 64 positions: those of the first tokens that the window keeps, then lo's to the token's own
  const int t0 = lo / TILE, kept = min((a.keep + TILE - 1) / TILE, t0);
  const int n_tiles = pos < 0 ? 0 : kept + max(pos / TILE - t0 + 1, 0);
  const int first = split * a.split_tiles, mine = min(a.split_tiles, n_tiles - first);
  const size_t part0 = (size_t)t * a.nh + (size_t)kvh * per + h0, row0 = (size_t)token * a.nh + (size_t)kvh * per + h0;
  if (mine <= 0 && !CLUSTER) {                                    // the token has fewer splits
    if (a.splits > 1) {
      if (threadIdx.x < heads) {
        float* ml = a.part_ml + ((part0 + threadIdx.x) * a.splits + split) * 2;
        ml[0] = -INFINITY;
        ml[1] = 0.f;
      }
    } else {
      for (int i = threadIdx.x; i < heads * HD; i += WARPS * 32) a.out[row0 * HD + i] = __float2bfloat16_rn(0.f);
    }
    return;
  }

  uint8_t* ring = ring_all + warp * (STAGES * MT * B::BYTES);
  const uint32_t ring_at = tc::smem_u32(ring), full_at = tc::smem_u32(&full[warp][0]);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) tc::mbar_init(&full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  // steps of the split, dealt out in turn; step i covers the keys from key_of(i) on
  const int steps_all = max(mine, 0) * (TILE / STEP), steps = (steps_all - warp + WARPS - 1) / WARPS;
  auto key_of = [&](int i) {
    const int s = warp + i * WARPS, tile = first + s / (TILE / STEP);
    return (tile < kept ? tile : t0 + tile - kept) * TILE + s % (TILE / STEP) * STEP;
  };
  // Lane b brings block b of a step (lane 0 all of it from one page). Its page is looked up a step before the copy is asked for.
  const bool together = a.page_size >= STEP;
  const int n_copies = together ? 1 : MT;
  int next_page = -1, next_key = 0;
  auto look = [&](int i) {
    if (i >= steps) return;
    next_key = key_of(i);
    const int at = next_key + lane * 16;
    next_page = lane < n_copies && at <= pos ? table[a.page_shift >= 0 ? at >> a.page_shift : at / a.page_size] : -1;
  };
  // `after` is 0 and comes from what was read out of the stage last: the copy into it is not asked for before those loads have come.
  auto bring = [&](int i, unsigned after) {
    const int at = next_key + lane * 16, in_page = a.page_shift >= 0 ? at & (a.page_size - 1) : at % a.page_size;
    const int blocks = together ? min(MT, (pos - next_key) / fb::BLOCK_ROWS + 1) : 1;
    const uint32_t bytes = blocks * B::BYTES;
    const bool copies = next_page >= 0;
    const unsigned who = __ballot_sync(0xffffffffu, copies);
    if (lane == 0) tc::mbar_expect_tx(&full[warp][i % STAGES], __popc(who) * bytes);
    __syncwarp();
    if (copies)
      bulk_load(ring_at + (i % STAGES * MT + lane) * B::BYTES + after,
                a.pages + (((size_t)next_page * a.nkv + kvh) * (a.page_size / 16) + in_page / 16) * B::BYTES, bytes, full_at + i % STAGES * 8);
    look(i + 1);
  };
  look(0);
  for (int i = 0; i < min(STAGES, steps); ++i) bring(i, 0u);

  // the heads' queries as columns, raised; their sums over a group in three pieces. A row whose largest element is not 2^-30 .. 2^60 is brought there
  // by a power of two, which its scale takes back: smaller ones lost pieces of their sums, larger ones would be infinite where they are raised.
  uint4 qf[G];
  uint2 q_sums;
  float to_log2[2];                                               // of the lane's two heads
  {
    float sums[G];
    unsigned most = 0u;
#pragma unroll
    for (int c = 0; c < G; ++c) {
      qf[c] = make_uint4(0u, 0u, 0u, 0u);
      if (g < heads) qf[c] = *reinterpret_cast<const uint4*>(a.q + (row0 + g) * HD + c * 32 + q4 * 8);
      const unsigned w[4] = {qf[c].x, qf[c].y, qf[c].z, qf[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
    }
    most = max(most >> 16, most & 0xffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e_q = (int)(most >> 7) - 127;                       // (zero and numbers that are not normal: -127)
    const int down = most == 0u || e_q == 128 ? 0 : e_q < -30 ? e_q + 30 : max(0, e_q - 59);      // infinite: as it is
    const unsigned factor = (unsigned)(127 - down) << 7 | (unsigned)(127 - down) << 23;           // 2^-down, twice
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int theirs = min(__shfl_sync(0xffffffffu, down, (2 * q4 + h) * 4), 56);               // (2^(69 + 56) times the scale: a float)
      to_log2[h] = a.scale * 1.4426950408889634f * fb::UNSCALE * __int_as_float((127 + theirs) << 23);
    }
#pragma unroll
    for (int c = 0; c < G; ++c) {
      uint4 v = qf[c];
      if (down != 0) v = make_uint4(fb::times(v.x, factor), fb::times(v.y, factor), fb::times(v.z, factor), fb::times(v.w, factor));
      const unsigned w[4] = {v.x, v.y, v.z, v.w};
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += low_half(w[i]) + high_half(w[i]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sums[c] = sum / fb::UNSCALE;
      qf[c] = fb::raised(v);
    }
    unsigned p[3];
    if constexpr (G == 4) {
      const bool second = q4 & 1;
      hb::split3(second ? sums[2] : sums[0], second ? sums[3] : sums[1], p);
      q_sums = make_uint2(q4 < 2 ? p[0] : p[1], q4 < 2 ? p[2] : 0u);
    } else {
      hb::split3(sums[0], sums[1], p);
      q_sums = make_uint2(q4 == 0 ? p[0] : q4 == 1 ? p[1] : q4 == 2 ? p[2] : 0u, 0u);
    }
  }
  float m_run[2] = {-INFINITY, -INFINITY};
  float o[2 * G][4];                                              // dims 4 g + (0, 1) and (2, 3) of every group
  float low[4] = {0.f, 0.f, 0.f, 0.f};                            // rows g < G: lows' sums, G .. 2 G - 1: scales'; row 8: the weights'
  float eight[4] = {0.f, 0.f, 0.f, 0.f};                          // rows g < G: the eights'
#pragma unroll
  for (int c = 0; c < 2 * G; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[c][e] = 0.f;
  bool ok = true;
  int asked = min(STAGES, steps);

  for (int i = 0; i < steps; ++i) {
    if (!tc::mbar_wait_warp(&full[warp][i % STAGES], (i / STAGES) & 1)) {
      if (lane == 0) atomicExch(a.status, 31);
      ok = false;
      break;
    }
    const int key = key_of(i);
    const uint8_t* blocks = ring + i % STAGES * MT * B::BYTES;
    unsigned spent = 0u;
    auto seen = [&](int row) { return key + row <= pos && (key + row >= lo || key + row < a.keep); };
    auto step = [&](auto all_seen) {
    constexpr bool whole = decltype(all_seen)::value;
    float s[MT][4];
    float m_step[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const uint8_t* b = blocks + mt * B::BYTES;
      const Words<G> ka(b + B::key_word(g, q4, 0)), kb(b + B::key_word(g + 8, q4, 0));
      const int pair = G == 4 ? 2 * (q4 & 1) : 0;
      const unsigned la = *reinterpret_cast<const unsigned*>(b + B::key_low(g, pair)),
                     lb = *reinterpret_cast<const unsigned*>(b + B::key_low(g + 8, pair));
      const unsigned lows[4] = {la, lb, G == 4 ? la : 0u, G == 4 ? lb : 0u};
      const Words<G / 2> sa(b + B::scale(g, 0, 0)), sb(b + B::scale(g + 8, 0, 0));
      fb::mma_first(s[mt], lows, q_sums.x, q_sums.y);
#pragma unroll
      for (int c = 0; c < G; ++c) {
        float acc[4];
        fb::mma_codes_first(acc, ka.w[c], kb.w[c], qf[c]);
        const float fa = c & 1 ? high_half(sa.w[c / 2]) : low_half(sa.w[c / 2]), fb_ = c & 1 ? high_half(sb.w[c / 2]) : low_half(sb.w[c / 2]);
        s[mt][0] = fmaf(acc[0], fa, s[mt][0]);
        s[mt][1] = fmaf(acc[1], fa, s[mt][1]);
        s[mt][2] = fmaf(acc[2], fb_, s[mt][2]);
        s[mt][3] = fmaf(acc[3], fb_, s[mt][3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!whole && !seen(mt * 16 + g + 8 * (e >> 1))) s[mt][e] = -INFINITY;
        m_step[e & 1] = fmaxf(m_step[e & 1], s[mt][e]);
      }
    }
    // The weights are taken against `m_run`, which follows the maximum only when a head's has grown by more than a factor of 2, so that most
    // tiles leave the sums as they are. (At 2^8, where the largest weights are seldom 1 and rounded too, results were off by 0.0024 of their
    // size, 0.0021 so and where it follows at once.)
    bool grows = false;
    float m_new[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float m = m_step[h];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      m_new[h] = m * to_log2[h];                                     // (the scale is positive)
      grows = grows || m_new[h] > m_run[h] + 1.f;                 // (of a head that has seen nothing yet: any)
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m = fmaxf(m_new[h], m_run[h]), correct = m == m_run[h] ? 1.f : exp2_fast(m_run[h] - m);     // (the first: exp2(-inf) = 0)
        m_run[h] = m;
#pragma unroll
        for (int c = 0; c < 2 * G; ++c) { o[c][h] *= correct; o[c][2 + h] *= correct; }
        low[h] *= correct;
        low[2 + h] *= correct;
        eight[h] *= correct;
        eight[2 + h] *= correct;
      }
    }
    // a head that has seen nothing yet has a maximum of -inf; its weights are zeros
    const float base[2] = {m_run[0] == -INFINITY ? 0.f : -m_run[0], m_run[1] == -INFINITY ? 0.f : -m_run[1]};
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const uint8_t* b = blocks + mt * B::BYTES;
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = exp2_fast(fmaf(s[mt][e], to_log2[e & 1], base[e & 1]));
      // rows of the bare weights' product: a group's lows, a group's scales (columns of the records of 8 keys), at 8 ones
      unsigned la, lb;
      {
        const bool has = q4 < G;
        const unsigned ra = has ? *reinterpret_cast<const unsigned*>(b + B::scale(g, 0, 2 * q4)) : 0u,
                       rb = has ? *reinterpret_cast<const unsigned*>(b + B::scale(g + 8, 0, 2 * q4)) : 0u;
        la = transpose8(ra);
        lb = transpose8(rb);
        if (g < G) {
          la = *reinterpret_cast<const unsigned*>(b + B::value_low(2 * q4, g));
          lb = *reinterpret_cast<const unsigned*>(b + B::value_low(2 * q4 + 8, g));
        }
        if (!whole) {
          const int r = mt * 16 + 2 * q4;
          la &= (seen(r) ? 0xffffu : 0u) | (seen(r + 1) ? 0xffff0000u : 0u);
          lb &= (seen(r + 8) ? 0xffffu : 0u) | (seen(r + 9) ? 0xffff0000u : 0u);
        }
      }
      const unsigned ones = g == 0 ? 0x3f803f80u : 0u;
      const unsigned rest[4] = {la, ones, lb, ones};
      hb::mma_bf16(low, rest, transpose8(hb::pack_bf16(p[0], p[1])), transpose8(hb::pack_bf16(p[2], p[3])));
      const Words<G> va(b + B::value_word(2 * q4, g, 0)), vb(b + B::value_word(2 * q4 + 8, g, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] *= RAISE;
      const Words<G / 2> sa(b + B::scale(g, 1, 0)), sb(b + B::scale(g + 8, 1, 0));
      if (mt == MT - 1) spent = va.w[0] ^ vb.w[0] ^ sa.w[0] ^ sb.w[0] ^ la ^ lb;      // of every load
      const bool see_a = whole || seen(mt * 16 + g), see_b = whole || seen(mt * 16 + g + 8);
#pragma unroll
      for (int c = 0; c < G; ++c) {
        const float ta = c & 1 ? high_half(sa.w[c / 2]) : low_half(sa.w[c / 2]), tb = c & 1 ? high_half(sb.w[c / 2]) : low_half(sb.w[c / 2]);
        const float fa = see_a ? ta : 0.f, fb_ = see_b ? tb : 0.f;
        const unsigned x = transpose8(hb::pack_bf16(p[0] * fa, p[1] * fa)), y = transpose8(hb::pack_bf16(p[2] * fb_, p[3] * fb_));
        unsigned wa = va.w[c], wb = vb.w[c];
        const unsigned a0[4] = {wa & fb::LOW, wa & fb::HIGH, wb & fb::LOW, wb & fb::HIGH};
        hb::mma_bf16(o[2 * c], a0, x, y);
        wa >>= 8;
        wb >>= 8;
        const unsigned a1[4] = {wa & fb::LOW, wa & fb::HIGH, wb & fb::LOW, wb & fb::HIGH};
        hb::mma_bf16(o[2 * c + 1], a1, x, y);
        const unsigned eights = g == c ? 0x00080008u : 0u;
        const unsigned a2[4] = {eights, 0u, eights, 0u};
        hb::mma_bf16(eight, a2, x, y);
      }
    }
    };
    if (key + STEP - 1 <= pos && (key >= lo || key + STEP - 1 < a.keep)) step(Const<true>());
    else step(Const<false>());
    __syncwarp();                                                 // all lanes are through with the stage
    if (asked < steps) bring(asked++, spent & a.zero);
  }
  if (!ok) {                                                      // no copy is under way when the block ends
    for (int i = max(0, asked - STAGES); i < asked; ++i) tc::mbar_wait_warp(&full[warp][i % STAGES], (i / STAGES) & 1);
  }

  // this warp's sums in their size: o, and per head the sum of weights
  float l_run[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) l_run[h] = __shfl_sync(0xffffffffu, low[2 + h], q4);
#pragma unroll
  for (int c = 0; c < G; ++c) {
    float rest[2], eights[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float m = __shfl_sync(0xffffffffu, low[h], 4 * c + q4), t = __shfl_sync(0xffffffffu, low[h], 4 * (c + G) + q4);
      rest[h] = fmaf(8.f, t, m);
      eights[h] = __shfl_sync(0xffffffffu, eight[h], 4 * c + q4);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[2 * c + i][e] = fmaf(e < 2 ? o[2 * c + i][e] - eights[e & 1] : fmaf(o[2 * c + i][e], 1.f / 16.f, -eights[e & 1]), fb::UNSCALE, rest[e & 1]);
  }
  __syncthreads();                                                // every warp is through with its ring
  float* o_s = reinterpret_cast<float*>(ring_all);                // [WARPS][HEADS][HD]
  if (g == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ml_s[warp][2 * q4 + h][0] = m_run[h];
      ml_s[warp][2 * q4 + h][1] = l_run[h];
    }
  }
#pragma unroll
  for (int c = 0; c < G; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float4*>(o_s + (warp * HEADS + 2 * q4 + h) * HD + c * 32 + g * 4) =
          make_float4(o[2 * c][h], o[2 * c][2 + h], o[2 * c + 1][h], o[2 * c + 1][2 + h]);
  __syncthreads();
  float* joined = o_s + WARPS * HEADS * HD;                       // CLUSTER: [HEADS][HD], and (maximum, sum) of every head
  __shared__ float2 joined_ml[CLUSTER ? HEADS : 1];
  auto finish = [&](int h, int d, float m_nat, float l, const float4& sum) {
    if (a.sink && l > 0.f) l += expf((a.sink_values ? a.sink_values[kvh * per + h0 + h] : 0.f) - m_nat);
    const float inv = l > 0.f ? 1.f / l : l;                      // (a NaN stays one)
    *reinterpret_cast<uint2*>(a.out + (row0 + h) * HD + d) =
        make_uint2(hb::pack_bf16(sum.x * inv, sum.y * inv), hb::pack_bf16(sum.z * inv, sum.w * inv));
  };
  auto add = [](float4& sum, float& l, const float4& v, float w, float f) {
    l = fmaf(w, f, l);
    sum.x = fmaf(v.x, f, sum.x);
    sum.y = fmaf(v.y, f, sum.y);
    sum.z = fmaf(v.z, f, sum.z);
    sum.w = fmaf(v.w, f, sum.w);
  };
  for (int i = threadIdx.x; i < heads * (HD / 4); i += WARPS * 32) {
    const int h = i / (HD / 4), d = i % (HD / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, ml_s[w][h][0]);
    float l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      if (ml_s[w][h][1] != 0.f)                                   // (0: no key of its steps is the token's)
        add(sum, l, *reinterpret_cast<const float4*>(o_s + (w * HEADS + h) * HD + d), ml_s[w][h][1], exp2_fast(ml_s[w][h][0] - m));
    // of scores, not of their base-2 form; a row with a NaN says so in both numbers
    const float m_nat = l != l ? l : m * 0.6931471805599453f;
    if constexpr (CLUSTER) {
      *reinterpret_cast<float4*>(joined + h * HD + d) = sum;
      if (d == 0) joined_ml[h] = make_float2(m_nat, l);
    } else if (a.splits > 1) {
      const size_t at = (part0 + h) * a.splits + split;
      *reinterpret_cast<float4*>(a.part_acc + at * HD + d) = sum;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_nat, l);
    } else {
      finish(h, d, m_nat, l, sum);
    }
  }
  if constexpr (CLUSTER) {
    // the blocks share out the heads' rows and add the splits in their order
    tc::cluster_meet();
    for (int i = threadIdx.x * a.splits + split; i < heads * (HD / 4); i += WARPS * 32 * a.splits) {
      const int h = i / (HD / 4), d = i % (HD / 4) * 4;
      float m[MOST_CLUSTER], w[MOST_CLUSTER], top = -INFINITY;
      float4 v[MOST_CLUSTER];
#pragma unroll
      for (int r = 0; r < MOST_CLUSTER; ++r) {
        if (r >= a.splits) break;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[r]), "=f"(w[r]) : "r"(in_block(&joined_ml[h], r)) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w)
                     : "r"(in_block(joined + h * HD + d, r)) : "memory");
        top = fmaxf(top, m[r]);
      }
      float l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < MOST_CLUSTER; ++r) {
        if (r >= a.splits) break;
        if (w[r] != 0.f) add(sum, l, v[r], w[r], __expf(m[r] - top));
      }
      finish(h, d, top, l, sum);
    }
    tc::cluster_meet();                                           // a block's rows are there until all have read them
  }
}

}  // namespace

extern "C" int hb_attention_decode_4bit(const void* q, const void* pages, const int* block_table, int table_stride,
                                        const int* seq_of_token, const int* positions, void* out, int n_tokens, int nh, int nkv, int hd,
                                        int page_size, int chunk, int window, int keep, float scale, int sink,
                                        const float* sink_values, int split_tiles, int splits, int cluster, float* part_acc, float* part_ml,
                                        int* status, const long long* rows, int step_tokens, cudaStream_t stream) {
  if (!q || !pages || !block_table || !seq_of_token || !positions || !out || !status || n_tokens < 0 || nh <= 0 || nkv <= 0 ||
      nh % nkv || table_stride <= 0 || chunk < 0 || window < 0 || keep < 0 || (keep > 0 && chunk > 0) || split_tiles < 1 || splits < 1 || !(scale > 0.f) ||
      (cluster && (splits < 2 || splits > MOST_CLUSTER)) || (splits > 1 && !cluster && (!part_acc || !part_ml)))
    return HB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(out)) & 15) return HB_ERR_BAD_ARG;
  if ((hd != 64 && hd != 128) || !(page_size == 16 || page_size == 32 || (page_size > 0 && page_size % 64 == 0))) return HB_ERR_UNSUPPORTED;
  const int tiles = (nh / nkv + HEADS - 1) / HEADS;
  if (n_tokens > 65535 || (long long)nkv * tiles > 65535) return HB_ERR_UNSUPPORTED;
  if (n_tokens == 0) return HB_OK;
  const int shift = page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size);
  const Args a{(const __nv_bfloat16*)q, (const uint8_t*)pages, block_table, seq_of_token, positions, (__nv_bfloat16*)out, part_acc,
               part_ml, status, rows, sink_values, rows ? step_tokens : n_tokens, table_stride, nh, nkv, page_size, shift, chunk, window, keep,
               split_tiles, splits, sink, scale, 0u};
  const int smem = WARPS * STAGES * (STEP / 16) * 20 * hd;        // blocks of 20 hd bytes; the sums at the end take less
  auto* kernel = cluster ? (hd == 128 ? attn_decode_4bit_kernel<4, true> : attn_decode_4bit_kernel<2, true>)
                         : (hd == 128 ? attn_decode_4bit_kernel<4, false> : attn_decode_4bit_kernel<2, false>);
  static std::atomic<unsigned long long> allowed[4]{};
  cudaError_t e = hb::allow_smem(kernel, smem, allowed[2 * (hd == 128) + (cluster != 0)]);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(splits, nkv * tiles, n_tokens);
  config.blockDim = dim3(WARPS * 32);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = cluster ? 1 : 0;
  e = cudaLaunchKernelEx(&config, kernel, a);
  if (e != cudaSuccess) return (int)e;
  if (splits > 1 && !cluster)
    return hb_attention_merge_rows(part_acc, part_ml, out, HB_DTYPE_BF16, n_tokens * nh, hd, splits, sink, nh, sink_values, rows, step_tokens,
                                   stream);
  return HB_OK;
}
