// The cache in four bits: the append of a step's keys and values, and the expansion of pages for the kernels that read bfloat16.
//
// A row of a head is cut into groups of 32 dims. With y the row's values in bfloat16, as the bfloat16 cache would hold them:
//   low = min y, scale = bfloat16((max y - low) / 15), code = round((y - low) / scale) held to 0 .. 15;  y ~ scale * code + low
// (float32 division; a group of one value has scale 0 and codes 0). The scale is rounded to bfloat16 because it is kept so, 32 bits a
// group beside 128 of codes, and the codes are taken with the rounded one. A group that holds a value that is not finite is kept as
// low = NaN, so that it shows wherever it is read, as it would from a bfloat16 cache; its scale is 0, which keeps it out of the sums of
// other groups (attention_decode_4bit.cu).
//
// In decode steps both are bound by their launch. For prompts the append is bound by its instructions, some 400 a warp and row of keys or values
// (2,048 tokens, 40 heads of 128 on 8: 23.7 us, 27.4 with a division a code, where the bytes take 8.1; rotated 31.8), the expansion by the chains of
// short loads, so that its blocks are wide (2,048 rows of 8 heads of 128 in bfloat16: 5.1 us with 512 threads, 7.0 with 128; bytes 1.7).
// The append's stores are 2 and 4 bytes each, as the attention kernel's order of the codes has it (four_bit.cuh); they meet in L2.
#include "api.h"
#include "common.cuh"
#include "four_bit.cuh"
#include "tc.cuh"

namespace {

struct Post {
  const __nv_bfloat16* qkv;
  const float* inv_freq;
  const float* q_w;
  const float* k_w;
  const int* positions;
  const int* seq_of_token;
  const int* block_table;
  __nv_bfloat16* q_out;
  uint8_t* pages;
  int rot_pairs, interleaved, qk_norm, temp_on, norm_first, norm_dim, v_is_k;
  float qk_eps, floor_scale, attn_scale, rot_mul;
  int table_stride, page_size, write_kv, n_tokens, nh, nkv;
};

__device__ __forceinline__ float group_min(float v) {      // over 8 neighbouring lanes
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Four dims of a row a lane, eight lanes a group: codes, scale and low. Every lane of the warp calls it.
struct Quantised { unsigned codes; __nv_bfloat16 scale, low; };
__device__ __forceinline__ Quantised quantise(const float (&y)[4]) {
  const float low = group_min(fminf(fminf(y[0], y[1]), fminf(y[2], y[3])));
  const float high = -group_min(-fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) finite = finite && fabsf(y[i]) <= 3.4028234663852886e38f;
  // (a range that float32 does not hold counts as such)
  const unsigned all = __ballot_sync(0xffffffffu, finite && high - low <= 3.3e38f);
  const bool whole = (all >> (threadIdx.x & 24) & 0xffu) == 0xffu;
  Quantised r;
  r.scale = __float2bfloat16_rn((high - low) / 15.f);
  r.low = __float2bfloat16_rn(low);                        // exact
  // round((y - low) / step) by one division a group: y - low times the reciprocal is within 2.7e-6 of the float32 quotient (below 16; two
  // roundings of 2^-24, and the quotient's own), so the codes differ only beside a half. A warp with such a value, or with a step whose reciprocal
  // is not a normal number, divides. A sum with 1.5 * 2^23 rounds as rint does and leaves the code in its last bits.
  constexpr float MAGIC = 12582912.f;
  const float step = __bfloat162float(r.scale), inv = 1.f / step;
  bool sure = step >= 1e-30f;
  float code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = (y[i] - low) * inv;
    code[i] = fminf(c, 15.f) + MAGIC;
    sure = sure && fabsf(c - (code[i] - MAGIC)) < 0.49999f;
  }
  if (!__all_sync(0xffffffffu, sure || step == 0.f))
#pragma unroll
    for (int i = 0; i < 4; ++i) code[i] = fminf((y[i] - low) / step, 15.f) + MAGIC;
  r.codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.codes |= step > 0.f ? (__float_as_uint(code[i]) & 15u) << (4 * i) : 0u;
  if (!whole) {
    r.codes = 0;
    r.scale = __ushort_as_bfloat16(0u);
    r.low = __ushort_as_bfloat16(0x7fffu);
  }
  return r;
}

// A block is one token; a head is taken by hd / 4 lanes, four neighbouring dims each. The rotation's partners meet in shared memory.
template <int G>
__global__ void __launch_bounds__(256, 4) qkv_post_4bit_kernel(const Post a) {
  constexpr int HD = 32 * G, LPH = HD / 4, HPW = 32 / LPH;
  using B = fb::Block<G>;
  __shared__ float cs[HD / 2], sn[HD / 2];
  __shared__ float rows[8][HPW * HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int li = lane % LPH, t = blockIdx.x, pos = a.positions[t];
  for (int j = threadIdx.x; j < a.rot_pairs; j += blockDim.x) {
    float s, c;
    sincosf((float)pos * a.inv_freq[j], &s, &c);
    sn[j] = s * a.rot_mul;
    cs[j] = c * a.rot_mul;
  }
  __syncthreads();
  const int heads = a.nh + (a.v_is_k ? 1 : 2) * a.nkv, todo = a.write_kv ? heads : a.nh;
  int page = -1;
  if (a.write_kv && pos >= 0 && pos / a.page_size < a.table_stride)
    page = a.block_table[(size_t)a.seq_of_token[t] * a.table_stride + pos / a.page_size];
  float* row = rows[warp] + lane / LPH * HD;
  const int d0 = 4 * li, group = d0 / 32, rot = 2 * a.rot_pairs;
  const float mul = a.temp_on ? logf(floorf(((float)pos + 1.f) / a.floor_scale) + 1.f) * a.attn_scale + 1.f : 1.f;
  const int first = (blockIdx.y * warps + warp) * HPW, stride = gridDim.y * warps * HPW;
  const uint2* from = reinterpret_cast<const uint2*>(a.qkv + ((size_t)t * heads + lane / LPH) * HD + d0);
  auto load = [&](int h0) { return h0 + lane / LPH < todo ? __ldg(from + h0 * (HD / 4)) : make_uint2(0u, 0u); };
  uint2 next = load(first);                                  // the heads' rows come one ahead
  for (int h0 = first; h0 < todo; h0 += stride) {
    const int head = h0 + lane / LPH;
    const bool active = head < todo;
    const int kind = head < a.nh ? 0 : head < a.nh + a.nkv ? 1 : 2;
    float y[4], raw[4];
    {
      const uint2 v = next;
      next = load(h0 + stride);
      raw[0] = y[0] = __uint_as_float(v.x << 16);
      raw[1] = y[1] = __uint_as_float(v.x & 0xffff0000u);
      raw[2] = y[2] = __uint_as_float(v.y << 16);
      raw[3] = y[3] = __uint_as_float(v.y & 0xffff0000u);
    }
    if (a.norm_first && a.qk_norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += d0 + i < a.norm_dim ? y[i] * y[i] : 0.f;
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss / (float)a.norm_dim + a.qk_eps);
      const float* w = kind == 0 ? a.q_w : a.k_w;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= kind == 2 ? 1.f : inv * (w ? w[d0 + i] : 1.f);
    }
    __syncwarp();
    if (rot > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) row[d0 + i] = y[i];
      __syncwarp();
      if (kind != 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = d0 + i;
          if (d >= rot) continue;
          const int j = a.interleaved ? d >> 1 : d < a.rot_pairs ? d : d - a.rot_pairs;
          const bool second = a.interleaved ? d & 1 : d >= a.rot_pairs;
          const float other = row[a.interleaved ? d ^ 1 : second ? d - a.rot_pairs : d + a.rot_pairs];
          y[i] = second ? y[i] * cs[j] + other * sn[j] : y[i] * cs[j] - other * sn[j];
        }
      __syncwarp();
    }
    if (!a.norm_first && a.qk_norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss += d0 + i < a.norm_dim ? y[i] * y[i] : 0.f;
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss / (float)a.norm_dim + a.qk_eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= kind == 2 ? 1.f : inv;
    }
    if (kind == 0 && a.temp_on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] *= mul;
    }
    const uint2 packed = make_uint2(hb::pack_bf16(y[0], y[1]), hb::pack_bf16(y[2], y[3]));
    if (kind == 0 && active) *reinterpret_cast<uint2*>(a.q_out + ((size_t)t * a.nh + head) * HD + d0) = packed;
    if (!a.write_kv || __all_sync(0xffffffffu, kind == 0)) continue;
    y[0] = __uint_as_float(packed.x << 16);
    y[1] = __uint_as_float(packed.x & 0xffff0000u);
    y[2] = __uint_as_float(packed.y << 16);
    y[3] = __uint_as_float(packed.y & 0xffff0000u);
    const int kvh = kind == 0 ? 0 : kind == 1 ? head - a.nh : head - a.nh - a.nkv;
    const bool writes = active && kind != 0 && page >= 0;      // the host reserves pages before the step
    const int at = pos >= 0 ? pos % a.page_size : 0, r = at % fb::BLOCK_ROWS;
    uint8_t* block = a.pages + (((size_t)(writes ? page : 0) * a.nkv + kvh) * (a.page_size / fb::BLOCK_ROWS) + at / fb::BLOCK_ROWS) * B::BYTES;
    const Quantised z = quantise(y);
    // a key's word: even dims in the lower half; two lanes share it
    unsigned word = (z.codes & 0xfu) | (z.codes & 0xf0u) << 12 | (z.codes & 0xf00u) >> 4 | (z.codes & 0xf000u) << 8;
    if (li & 1) word <<= 8;
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    if (writes && kind == 1) {
      if (!(li & 1)) *reinterpret_cast<unsigned*>(block + B::key_word(r, (li % 8) / 2, group)) = word;
      if (li % 8 == 0) {
        *reinterpret_cast<__nv_bfloat16*>(block + B::scale(r, 0, group)) = z.scale;
        *reinterpret_cast<__nv_bfloat16*>(block + B::key_low(r, group)) = z.low;
      }
    }
    Quantised v = z;
    if (a.v_is_k) v = quantise(raw);                         // the key as projected is the value
    if (writes && (kind == 2 || a.v_is_k)) {
      *reinterpret_cast<uint16_t*>(block + B::value_word(r, li % 8, group) + (r & 1) * 2) = (uint16_t)v.codes;
      if (li % 8 == 0) {
        *reinterpret_cast<__nv_bfloat16*>(block + B::scale(r, 1, group)) = v.scale;
        *reinterpret_cast<__nv_bfloat16*>(block + B::value_low(r, group)) = v.low;
      }
    }
  }
}

// ---- pages of the step's portions as bfloat16. Request s needs its pages first_s .. last_s: from the oldest position that its first
// new token may read to its last one, and in front of them the pages of the first tokens that it keeps (`whole`: with kept tokens all pages
// from the request's first on); they lie side by side in the result, request after request, and `table` [n_seqs, table_stride]
// says where. Every other entry is -1, as that of a page which was given back: kernels that walk tiles larger than a page look at
// entries in front of first_s, and what they would multiply by weights of zero there has to be a page of the request or none. The grid is
// made from the host's copies of the requests' positions; where the device's ask for another number of pages, `status` says so
// (no entry names a page that is not in the result).
struct Expand {
  const uint8_t* pages;
  const int* block_table;
  const int* cu_seqlens;
  const int* positions;
  uint16_t* k;                     // bfloat16, or for the prefill kernels float16
  uint16_t* v;
  int* table;
  int n_seqs, table_stride, page_size, chunk, window, keep, whole, skip_single, nkv, total;
  // for the prefill kernels only
  const __nv_bfloat16* q;
  int n_tokens, nh;
  int4* most;                      // [n_seqs][nkv]: see most_4bit_kernel
  uint16_t* q_out;
  float* q_scale;                  // [n_tokens][nh]: of a row's scores, to units of log 2
  float scale_log2;
  float2* form;                    // [n_seqs][nkv]: what the values have been divided by, 1 for float16
  int* status;
};

// The pages of a request: `lead` of them from its first on, then those from `first` on, `count` in all.
struct Span {
  int lead, first, count;
  __host__ __device__ int page(int i) const { return i < lead ? i : first + i - lead; }
  __host__ __device__ bool has(int page) const { return page < lead || (page >= first && page < first + count - lead); }
};
template <typename I>              // int on the device, where divisions of 64 bits are slow
__host__ __device__ inline Span span_of(I start, I n, int page_size, int chunk, int window, int keep, int whole) {
  I low = 0;
  if (chunk > 0) low = start / chunk * chunk;
  else if (window > 0 && start - window + 1 > 0) low = start - window + 1;
  if (whole && keep > 0) low = 0;
  Span s;
  s.first = (int)(low / page_size);
  const int kept = keep / page_size + (keep % page_size != 0);
  s.lead = kept < s.first ? kept : s.first;
  s.count = s.lead + (int)((start + n - 1) / page_size) - s.first + 1;
  return s;
}
__device__ __forceinline__ Span span(const Expand& a, int s) {
  const int begin = a.cu_seqlens[s], n = a.cu_seqlens[s + 1] - begin;
  if (n <= 0 || (n == 1 && a.skip_single)) return Span{0, 0, 0};
  const int start = a.positions[begin];
  if (start < 0) return Span{0, 0, 0};
  return span_of(start, n, a.page_size, a.chunk, a.window, a.keep, a.whole);
}

// Whether the requests ask for as many pages as the grid has, by one warp. If not, `status` says so, and entries of pages behind the grid's are -1.
__device__ void check_total(const Expand& a) {
  int all = 0;
  for (int s = threadIdx.x; s < a.n_seqs; s += 32) all += span(a, s).count;
  if (__reduce_add_sync(0xffffffffu, all) == a.total) return;
  if (threadIdx.x == 0) atomicExch(a.status, 33);
  int before = 0;
  for (int s = 0; s < a.n_seqs; ++s) {
    const Span x = span(a, s);
    for (int i = max(0, a.total - before) + threadIdx.x; i < x.count && x.page(i) < a.table_stride; i += 32)
      a.table[(size_t)s * a.table_stride + x.page(i)] = -1;
    before += x.count;
  }
}

// The request and its page that page `out_page` of the result is; false: none (or the table has no such page). A whole block asks.
// `leads`: it is the request's first.
__device__ __forceinline__ bool find_page(const Expand& a, int out_page, int& seq, int& index, bool& leads) {
  __shared__ int found[3];
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {          // the requests' counts are summed 32 at a time
    int before = 0, who_seq = -1, at = 0, led = 0;
    for (int s0 = 0; s0 < a.n_seqs && who_seq < 0; s0 += 32) {
      Span x{0, 0, 0};
      if (s0 + lane < a.n_seqs) x = span(a, s0 + lane);
      int upto = x.count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > out_page);
      const int who = hit ? __ffs(hit) - 1 : 0;
      const int mine = out_page - (before + upto - x.count), here = __shfl_sync(0xffffffffu, x.page(mine), who);
      if (hit) { who_seq = s0 + who; at = here; led = __shfl_sync(0xffffffffu, mine, who) == 0; }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) { found[0] = who_seq; found[1] = at; found[2] = led; }
  }
  __syncthreads();
  seq = found[0];
  index = found[1];
  leads = found[2];
  return seq >= 0 && index < a.table_stride;
}
__device__ __forceinline__ float number(const uint8_t* p) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p)); }

// ---- for the tcgen05 prefill kernels: float16, which keeps 11 of a cached value's up to 13 bits where bfloat16 keeps 8. Keys and values of a
// request's kv head are divided by the least power of two above the largest of them, so float16 holds a group to 2^-11 of its largest
// magnitude where that is at least 2^-14 of the head's. A request with a smaller one, or with a largest one out of 2^-100 .. 2^100, is
// expanded to bfloat16 for that head instead, and its products are taken in it. What a request's result is rounded to depends on its own rows
// alone. A query's row of a head is multiplied by a power of two of its own, which the row's scale takes back: it keeps all bits of elements
// down to 2^-32 of its largest. Where its scores could pass 2^20 the mantissa of the scale goes into the row, rounded to float16 as the keys
// are: their maximum times a power of two is exact, and so are the differences to it. (Rounded, it would be off by more than float16's weights can grow.)
//
// The magnitudes of a request's kv head on the pages, of rows that are there (a group's ends: its low and fifteen steps above it): one atomic a
// block and number, and none where it changes nothing (29 us for 144 pages of 8 heads with one a warp, 7 so). `most` holds the bits of floats, whose
// order is theirs: keys' largest, keys' smallest group's above zero (taken from that of infinity, so that it only grows too), then values'; -1: none.
constexpr int EXPAND_THREADS = 512, MOST_THREADS = 128;

template <int G>
__global__ void __launch_bounds__(MOST_THREADS) most_4bit_kernel(const Expand a) {
  using B = fb::Block<G>;
  constexpr int INFINITE = 0x7f800000;
  const int kvh = blockIdx.y;
  int seq, index;
  bool leads;
  if (!find_page(a, blockIdx.x, seq, index, leads)) return;
  const int page = a.block_table[(size_t)seq * a.table_stride + index];
  if (page < 0) return;
  const int begin = a.cu_seqlens[seq], last = a.positions[begin] + a.cu_seqlens[seq + 1] - begin - 1;
  const int rows = min(a.page_size, last - index * a.page_size + 1);
  const uint8_t* from = a.pages + ((size_t)page * a.nkv + kvh) * (a.page_size / fb::BLOCK_ROWS) * B::BYTES;
  float k_most = 0.f, k_least = INFINITY, v_most = 0.f, v_least = INFINITY;
  auto take = [](float low, float scale, float& most, float& least) {
    const float size = fmaxf(fabsf(low), fabsf(fmaf(scale, 15.f, low)));      // (of a group of NaN: NaN)
    most = fmaxf(most, size);
    if (size > 0.f) least = fminf(least, size);
  };
  for (int i = threadIdx.x; i < rows * G; i += blockDim.x) {
    const int row = i / G, r = row % fb::BLOCK_ROWS, group = i % G;
    const uint8_t* block = from + row / fb::BLOCK_ROWS * B::BYTES;
    take(number(block + B::key_low(r, group)), number(block + B::scale(r, 0, group)), k_most, k_least);
    take(number(block + B::value_low(r, group)), number(block + B::scale(r, 1, group)), v_most, v_least);
  }
  __shared__ int all[4][MOST_THREADS / 32];
  const int mine[4] = {__reduce_max_sync(0xffffffffu, __float_as_int(k_most)), __reduce_max_sync(0xffffffffu, INFINITE - __float_as_int(k_least)),
                       __reduce_max_sync(0xffffffffu, __float_as_int(v_most)), __reduce_max_sync(0xffffffffu, INFINITE - __float_as_int(v_least))};
#pragma unroll
  for (int n = 0; n < 4; ++n)
    if (threadIdx.x % 32 == n) all[n][threadIdx.x / 32] = mine[n];
  __syncthreads();
  if (threadIdx.x < 4) {
    int most = 0;
    for (int w = 0; w < MOST_THREADS / 32; ++w) most = max(most, all[threadIdx.x][w]);
    int* to = reinterpret_cast<int*>(a.most + (size_t)seq * a.nkv + kvh) + threadIdx.x;
    if (most > *reinterpret_cast<volatile int*>(to)) atomicMax(to, most);      // it only grows
  }
}
// two to the power that is the least above a magnitude of these bits (of a normal float); of zero and none: 0
__device__ __forceinline__ int power_above(int bits) { return bits <= 0 ? 0 : (bits >> 23) - 126; }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((max(-126, min(e, 127)) + 127) << 23); }

// How a request's kv head is held: float16, keys and values divided by 2^k and 2^v, or (half false) bfloat16.
struct Held { bool half; int k, v; };
__device__ __forceinline__ Held held(const int4& most) {
  auto fits = [](int largest, int smallest) {                      // as `most` has them
    const int e = power_above(largest), least = 0x7f800000 - smallest;
    return largest <= 0 || (e >= -100 && e <= 100 && (largest >> 23) - (least >> 23) <= 13);
  };
  if (!fits(most.x, most.y) || !fits(most.z, most.w)) return Held{false, 0, 0};
  return Held{true, power_above(most.x), power_above(most.z)};
}
__device__ __forceinline__ uint32_t pack_as(bool half, float lo, float hi) { return half ? tc::pack16<true>(lo, hi) : tc::pack16<false>(lo, hi); }

constexpr int Q_TOKENS = 8;        // of a block that converts queries

// PREFILL: in the form that `most` asks for, and the queries beside it; else bfloat16
template <int G, bool PREFILL>
__global__ void __launch_bounds__(EXPAND_THREADS) expand_4bit_kernel(const Expand a) {
  constexpr int HD = 32 * G;
  using B = fb::Block<G>;
  const int out_page = blockIdx.x, kvh = blockIdx.y;
  if constexpr (PREFILL) {
    if (out_page >= a.total) {       // queries of this kv head
      __shared__ Held forms[Q_TOKENS];
      const int per = a.nh / a.nkv, t0 = (out_page - a.total) * Q_TOKENS, tokens = min(Q_TOKENS, min(a.n_tokens, a.cu_seqlens[a.n_seqs]) - t0);
      if ((int)threadIdx.x < tokens) {
        int s = 0, end = a.n_seqs;                                  // the last request that does not begin behind the token
        while (end - s > 1) {
          const int mid = (s + end) / 2;
          if (a.cu_seqlens[mid] <= t0 + (int)threadIdx.x) s = mid;
          else end = mid;
        }
        forms[threadIdx.x] = held(a.most[(size_t)s * a.nkv + kvh]);
      }
      __syncthreads();
      constexpr int WORDS = HD / 8;                                 // of a row, as many lanes
      const unsigned row_lanes = (WORDS == 16 ? 0xffffu : 0xffu) << (threadIdx.x & 31 & ~(WORDS - 1));
      for (int i = threadIdx.x; i < tokens * per * WORDS; i += blockDim.x) {
        const int token = i / WORDS / per, head = kvh * per + i / WORDS % per;
        const Held form = forms[token];
        const size_t row = (size_t)(t0 + token) * a.nh + head, at = row * HD + i % WORDS * 8;
        const uint4 raw = *reinterpret_cast<const uint4*>(a.q + at);
        float x[8], most = 0.f;
        hb::load8(a.q + at, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
        for (int o = WORDS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(row_lanes, most, o));
        const int e_q = max(-100, power_above(__float_as_int(most)));
        const float e_scale = power_of_two((__float_as_int(a.scale_log2) >> 23) - 127), rest = a.scale_log2 / e_scale;      // rest: 1 to 2
        const bool large = (float)HD * a.scale_log2 * power_of_two(e_q + form.k) > 1048576.f;
        const float up = large ? power_of_two(14 - e_q) * rest : power_of_two(15 - e_q);                   // (an infinity stays one)
        unsigned o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = tc::pack16<true>(x[2 * e] * up, x[2 * e + 1] * up);
        *reinterpret_cast<uint4*>(a.q_out + at) = form.half ? make_uint4(o[0], o[1], o[2], o[3]) : raw;
        if (i % WORDS == 0)
          a.q_scale[row] = !form.half ? a.scale_log2 : large ? power_of_two(e_q - 14 + form.k) * e_scale : power_of_two(e_q - 15 + form.k) * a.scale_log2;
      }
      return;
    }
  }
  int seq, index;
  bool leads;
  if (out_page == 0 && kvh == 0 && threadIdx.x < 32) check_total(a);
  if (!PREFILL && kvh == 0)          // the entries that no page of the result is for (with PREFILL: -1 already)
    for (long long i = (long long)out_page * blockDim.x + threadIdx.x; i < (long long)a.n_seqs * a.table_stride; i += (long long)a.total * blockDim.x) {
      if (!span(a, (int)(i / a.table_stride)).has((int)(i % a.table_stride))) a.table[i] = -1;
    }
  if (!find_page(a, out_page, seq, index, leads)) return;
  Held form{false, 0, 0};
  if constexpr (PREFILL) {
    form = held(a.most[(size_t)seq * a.nkv + kvh]);
    if (leads && threadIdx.x == 0) a.form[(size_t)seq * a.nkv + kvh] = make_float2(power_of_two(form.v), form.half ? 1.f : 0.f);
  }
  const float k_down = power_of_two(-form.k), v_down = power_of_two(-form.v);
  const int page = a.block_table[(size_t)seq * a.table_stride + index];
  if (kvh == 0 && threadIdx.x == 0) a.table[(size_t)seq * a.table_stride + index] = page < 0 ? -1 : out_page;
  const size_t out = ((size_t)out_page * a.nkv + kvh) * a.page_size * HD;
  if (page < 0) return;
  const uint8_t* from = a.pages + ((size_t)page * a.nkv + kvh) * (a.page_size / fb::BLOCK_ROWS) * B::BYTES;
  for (int i = threadIdx.x; i < a.page_size * 4 * G; i += blockDim.x) {      // eight dims of a key
    const int row = i / (4 * G), r = row % fb::BLOCK_ROWS, group = i % (4 * G) / 4, q = i % 4;
    const uint8_t* block = from + row / fb::BLOCK_ROWS * B::BYTES;
    const unsigned w = *reinterpret_cast<const unsigned*>(block + B::key_word(r, q, group));
    const float scale = number(block + B::scale(r, 0, group)) * k_down, low = number(block + B::key_low(r, group)) * k_down;
    unsigned o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = pack_as(form.half, fmaf(scale, (float)(w >> (4 * e) & 15), low), fmaf(scale, (float)(w >> (16 + 4 * e) & 15), low));
    *reinterpret_cast<uint4*>(a.k + out + (size_t)row * HD + group * 32 + q * 8) = make_uint4(o[0], o[1], o[2], o[3]);
  }
  for (int i = threadIdx.x; i < a.page_size / 2 * 8 * G; i += blockDim.x) {  // four dims of the values of two tokens
    const int row = i / (8 * G) * 2, r = row % fb::BLOCK_ROWS, group = i % (8 * G) / 8, g = i % 8;
    const uint8_t* block = from + row / fb::BLOCK_ROWS * B::BYTES;
    const unsigned w = *reinterpret_cast<const unsigned*>(block + B::value_word(r, g, group));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float scale = number(block + B::scale(r + e, 1, group)) * v_down, low = number(block + B::value_low(r + e, group)) * v_down;
      const unsigned c = w >> (16 * e);
      *reinterpret_cast<uint2*>(a.v + out + (size_t)(row + e) * HD + group * 32 + g * 4) = make_uint2(
          pack_as(form.half, fmaf(scale, (float)(c & 15), low), fmaf(scale, (float)(c >> 4 & 15), low)),
          pack_as(form.half, fmaf(scale, (float)(c >> 8 & 15), low), fmaf(scale, (float)(c >> 12 & 15), low)));
    }
  }
}

bool good_page(int page_size) { return page_size == 16 || page_size == 32 || (page_size > 0 && page_size % 64 == 0); }

}  // namespace

extern "C" int hb_qkv_post_4bit(const void* qkv, const float* inv_freq, int rot_pairs, int interleaved, int qk_norm, float qk_eps,
                                int temp_on, float floor_scale, float attn_scale, const float* q_norm_w, const float* k_norm_w,
                                int norm_first, int norm_dim, float rot_mul, int v_is_k, const int* positions,
                                const int* seq_of_token, const int* block_table, int table_stride, void* q_out, void* pages,
                                int page_size, int write_kv, int n_tokens, int nh, int nkv, int hd, cudaStream_t stream) {
  if (!qkv || !positions || !q_out || n_tokens < 0 || nh <= 0 || nkv <= 0 || ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 7))
    return HB_ERR_BAD_ARG;
  if (write_kv && (!pages || !block_table || !seq_of_token || table_stride <= 0)) return HB_ERR_BAD_ARG;
  if (!inv_freq) rot_pairs = 0;
  if (norm_dim <= 0) norm_dim = hd;
  if (rot_pairs < 0 || norm_dim > hd || 2 * rot_pairs > norm_dim || (temp_on && !(floor_scale > 0.f))) return HB_ERR_BAD_ARG;
  // a weightless norm after a rotation keeps its sum of squares only where the rotation keeps lengths
  if ((hd != 64 && hd != 128) || !good_page(page_size) || (qk_norm && !norm_first && (rot_mul != 1.f || q_norm_w || k_norm_w)))
    return HB_ERR_UNSUPPORTED;
  if (n_tokens == 0) return HB_OK;
  const Post a{(const __nv_bfloat16*)qkv, inv_freq, q_norm_w, k_norm_w, positions, seq_of_token, block_table, (__nv_bfloat16*)q_out,
               (uint8_t*)pages, rot_pairs, interleaved, qk_norm, temp_on, norm_first, norm_dim, v_is_k, qk_eps, floor_scale, attn_scale,
               rot_mul, table_stride, page_size, write_kv, n_tokens, nh, nkv};
  const int heads = nh + (v_is_k ? 1 : 2) * nkv, per_warp = hd == 64 ? 2 : 1;
  const int all = (heads + per_warp - 1) / per_warp;
  const dim3 grid(n_tokens, n_tokens < 148 ? (all + 7) / 8 : 1);      // few tokens: a warp a head, many: the sines are worth sharing
  if (hd == 128) qkv_post_4bit_kernel<4><<<grid, 256, 0, stream>>>(a);
  else qkv_post_4bit_kernel<2><<<grid, 256, 0, stream>>>(a);
  HB_LAUNCH_CHECK();
  return HB_OK;
}

namespace {
int expand(const Expand& a, int hd, bool prefill, cudaStream_t stream) {
  if (!a.pages || !a.block_table || !a.cu_seqlens || !a.positions || !a.table || !a.status || a.n_seqs < 0 || a.total < 0 || a.nkv <= 0 || a.table_stride <= 0 ||
      a.chunk < 0 || a.window < 0 || a.keep < 0 || (a.keep > 0 && a.chunk > 0) || (a.total > 0 && (!a.k || !a.v)))
    return HB_ERR_BAD_ARG;
  if ((hd != 64 && hd != 128) || !good_page(a.page_size) || a.nkv > 65535) return HB_ERR_UNSUPPORTED;
  if (a.n_seqs == 0 || a.total == 0) return HB_OK;
  const dim3 grid(a.total, a.nkv);
  if (prefill) {
    // the table's entries are -1, and (behind them) the magnitudes
    const cudaError_t e = cudaMemsetAsync(a.table, 0xff, (uint8_t*)(a.most + (size_t)a.n_seqs * a.nkv) - (uint8_t*)a.table, stream);
    if (e != cudaSuccess) return (int)e;
    const dim3 more(a.total + (a.n_tokens + Q_TOKENS - 1) / Q_TOKENS, a.nkv);
    if (hd == 128) most_4bit_kernel<4><<<grid, MOST_THREADS, 0, stream>>>(a);
    else most_4bit_kernel<2><<<grid, MOST_THREADS, 0, stream>>>(a);
    HB_LAUNCH_CHECK();
    if (hd == 128) expand_4bit_kernel<4, true><<<more, EXPAND_THREADS, 0, stream>>>(a);
    else expand_4bit_kernel<2, true><<<more, EXPAND_THREADS, 0, stream>>>(a);
  } else if (hd == 128) {
    expand_4bit_kernel<4, false><<<grid, EXPAND_THREADS, 0, stream>>>(a);
  } else {
    expand_4bit_kernel<2, false><<<grid, EXPAND_THREADS, 0, stream>>>(a);
  }
  HB_LAUNCH_CHECK();
  return HB_OK;
}
}  // namespace

extern "C" int hb_expand_pages_4bit(const void* pages, const int* block_table, int table_stride, const int* cu_seqlens,
                                    const int* positions, int n_seqs, int total, int page_size, int chunk, int window, int keep,
                                    int whole, int skip_single, int nkv, int hd, void* k, void* v, int* table, int* status,
                                    cudaStream_t stream) {
  return expand(Expand{(const uint8_t*)pages, block_table, cu_seqlens, positions, (uint16_t*)k, (uint16_t*)v, table, n_seqs,
                       table_stride, page_size, chunk, window, keep, whole, skip_single, nkv, total, nullptr, 0, 0, nullptr, nullptr, nullptr, 0.f, nullptr, status},
                hd, false, stream);
}

// What hb_prefill_attention_4bit needs of its workspace, in order, each part on 1,024 bytes.
namespace {
struct Room {
  size_t k, v, q, q_scale, table, most, form, part_acc, part_ml, all;
  Room(int total, int n_tokens, int n_seqs, int table_stride, int nh, int nkv, int hd, int page_size, int key_splits) {
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 1023) / 1024 * 1024; return here; };
    k = take((size_t)total * nkv * page_size * hd * 2);
    v = take((size_t)total * nkv * page_size * hd * 2);
    q = take((size_t)n_tokens * nh * hd * 2);
    q_scale = take((size_t)n_tokens * nh * 4);
    table = take((size_t)n_seqs * table_stride * 4);
    most = take((size_t)n_seqs * nkv * 16);
    form = take((size_t)n_seqs * nkv * 8);
    part_acc = take(key_splits > 1 ? (size_t)n_tokens * nh * key_splits * hd * 4 : 0);
    part_ml = take(key_splits > 1 ? (size_t)n_tokens * nh * key_splits * 8 : 0);
    all = at;
  }
};
}  // namespace

// How many pages the requests' new tokens may read, by what the host knows of them (cu_seqlens and positions on the device say the same);
// -1: a position lies outside a block table of `width` pages a request, or the mask is not one (first tokens are kept beside a sliding window, not beside chunks).
extern "C" long long hb_expand_total(const int* start_pos, const int* n_new, int n_seqs, int width, int page_size, int chunk, int window,
                                     int keep, int whole, int skip_single) {
  long long total = 0;
  if (!start_pos || !n_new || n_seqs < 0 || page_size <= 0 || chunk < 0 || window < 0 || keep < 0 || (keep > 0 && chunk > 0)) return -1;
  for (int s = 0; s < n_seqs; ++s) {
    const long long start = start_pos[s], n = n_new[s];
    if (n <= 0 || (n == 1 && skip_single)) continue;
    if (start < 0 || (start + n - 1) / page_size >= width) return -1;
    total += span_of(start, n, page_size, chunk, window, keep, whole).count;
  }
  return total;
}
extern "C" long long hb_prefill_attention_4bit_bytes(int total, int n_tokens, int n_seqs, int table_stride, int nh, int nkv, int hd,
                                                     int page_size, int key_splits) {
  return (long long)Room(total, n_tokens, n_seqs, table_stride, nh, nkv, hd, page_size, key_splits).all;
}

// Pages and queries in the form that each request's kv head is held in (float16 or bfloat16, above), then the tcgen05 prefill attention on them
// and the merge of shared keys.
extern "C" int hb_prefill_attention_4bit(const void* q, const void* pages, const int* block_table, int table_stride, const int* cu_seqlens,
                                         const int* positions, void* out, int n_tokens, int n_seqs, int max_new, int nh, int nkv, int hd,
                                         int page_size, int chunk, int window, int keep, float scale, int skip_single, int sink,
                                         const float* sink_values, int key_splits, int one_tile, int total, void* workspace,
                                         long long workspace_bytes, int* status, cudaStream_t stream) {
  if (!q || !workspace || n_tokens < 0 || nh <= 0 || nkv <= 0 || nh % nkv || total < 1 || key_splits < 1 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(workspace)) & 15))
    return HB_ERR_BAD_ARG;
  const Room room(total, n_tokens, n_seqs, table_stride, nh, nkv, hd, page_size, key_splits);
  if ((long long)room.all > workspace_bytes) return HB_ERR_BAD_ARG;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  float* q_scale = reinterpret_cast<float*>(w + room.q_scale);
  float2* form = reinterpret_cast<float2*>(w + room.form);
  int* table = reinterpret_cast<int*>(w + room.table);
  int code = expand(Expand{(const uint8_t*)pages, block_table, cu_seqlens, positions, (uint16_t*)(w + room.k), (uint16_t*)(w + room.v), table,
                           n_seqs, table_stride, page_size, chunk, window, keep, 0, skip_single, nkv, total, (const __nv_bfloat16*)q, n_tokens, nh,
                           (int4*)(w + room.most), (uint16_t*)(w + room.q), q_scale, scale * 1.4426950408889634f, form, status},
                    hd, true, stream);
  if (code != HB_OK) return code;
  float* part_acc = key_splits > 1 ? reinterpret_cast<float*>(w + room.part_acc) : nullptr;
  float* part_ml = key_splits > 1 ? reinterpret_cast<float*>(w + room.part_ml) : nullptr;
  code = hb_attention_prefill_tc_mixed(w + room.q, w + room.k, w + room.v, form, q_scale, table, table_stride, cu_seqlens, positions, out,
                                      n_tokens, total, n_seqs, max_new, nh, nkv, hd, page_size, chunk, window, keep, scale, skip_single,
                                      sink, sink_values, key_splits, part_acc, part_ml, one_tile, status, stream);
  if (code != HB_OK || key_splits == 1) return code;
  return hb_attention_merge(part_acc, part_ml, out, HB_DTYPE_BF16, n_tokens * nh, hd, key_splits, sink, nh, sink_values, stream);
}
