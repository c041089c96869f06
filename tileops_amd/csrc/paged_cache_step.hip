// The cache side of a serving step on gfx950: pages taken from and given back to a pool, the norm and rotation of query and
// key rows with the append of keys and values, and the read-back of 4-bit rows.
//
// The 4-bit cache ("fp4" below): 32 consecutive head elements form a block of e2m1 codes (two to a byte, the lower nibble
// first) with one power-of-two scale byte, x = code * 2^(byte - 127); byte 255 makes the block NaN.  Codes are
// [n_pages, heads_kv, page_size, dim / 2], scales [n_pages, heads_kv, page_size, dim / 32]: the rows of one (page, kv head)
// are contiguous, because a token-major pool would give every 64-byte row of a 128-byte line to another head's workgroup.
#include <climits>
#include <type_traits>

#include "common.h"
#include "device_utils.h"

namespace mi355 {

namespace {

// ------------------------------------------------------------------------------------------------- page allocation
// Sums of page counts saturate at INT_MAX (both operands are in [0, INT_MAX], so the unsigned sum does not wrap): a sum
// that saturates is more than any pool holds.
__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)INT_MAX); }

__device__ __forceinline__ int wave_sat_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x = sat_add(x, y);
  }
  return x;
}

__device__ __forceinline__ int pages_of(int tokens, int page_size) {  // tokens >= 0; the sum fits 32 unsigned bits
  return (int)(((uint32_t)tokens + (uint32_t)page_size - 1u) / (uint32_t)page_size);
}

constexpr int kAllocThreads = 1024;

// With c_b tokens cached and n_b to come, sequence b needs need_b = ceil((c_b + n_b) / page) - ceil(c_b / page) pages.  In batch
// order, page i of the call is free_pages[free - 1 - i] (the list is a stack); b is served if its tokens fit its table row and
// lie in the step, and need_b is 0 or sum_{a <= b} need_a <= free.  A new page's first token lies in this call, so the thread of that token
// writes the table entry, and token t's page is either an entry that this call leaves alone or a place in the list: no
// workgroup waits for another.  Every workgroup sums the needs of the sequences up to its own tokens itself (a few loads: 1024
// sequences a pass); the first one goes through all of them and writes what there is one of per sequence.
//
// Bound: the launch and a chain of four dependent loads.  A decode step of 64 sequences moves 2 KB (3.4 us), a prefill step 12 bytes a token
// (33 sequences with 135168 places for new tokens: 5.9 us).
template <bool kChunks>  // false: one new token per sequence, token t is sequence t's
__global__ __launch_bounds__(kAllocThreads) void kv_alloc_kernel(
    const int32_t* __restrict__ cached, const int32_t* __restrict__ cu_q, int32_t* __restrict__ block_table, int64_t bt_row_stride,
    const int32_t* __restrict__ free_pages, const int32_t* __restrict__ free_count, int64_t* __restrict__ slots,
    int32_t* __restrict__ positions, int32_t* __restrict__ seqlens_out, uint8_t* __restrict__ refused,
    int32_t* __restrict__ free_count_out, int batch, int total_q, int page_size, int max_pages, int n_pages) {
  __shared__ int s_cu[kAllocThreads + 1], s_cached[kAllocThreads], s_first[kAllocThreads];
  __shared__ int s_wave[kAllocThreads / 64];
  __shared__ int s_taken;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int tok = blockIdx.x * kAllocThreads + t;  // (the launcher keeps total_q below 2^31 - 1024)
  const int tok_end = min((int)(blockIdx.x + 1) * kAllocThreads, total_q);
  const int free0 = min(max(free_count[0], 0), n_pages);
  const int row_tokens = (int)min((int64_t)max_pages * page_size, (int64_t)INT_MAX);
  int64_t slot = -1;
  int pos = -1, carry = 0;
  if (t == 0) s_taken = 0;
  // the page of logical page lp of a served sequence whose first new page is number `first` of the call
  auto place = [&](int b, int c, int first, int at) __attribute__((always_inline)) {
    const int lp = at / page_size, off = at - lp * page_size, fresh = lp - pages_of(c, page_size);
    int page;
    if (fresh < 0) {
      page = block_table[(int64_t)b * bt_row_stride + lp];
    } else {
      page = free_pages[free0 - 1 - (first + fresh)];  // 0 <= first + fresh < free0: the sequence is served
      if (off == 0) block_table[(int64_t)b * bt_row_stride + lp] = page;
    }
    slot = (int64_t)page * page_size + off;
    pos = at;
  };
  for (int base = 0; base < batch; base += kAllocThreads) {
    const int nb = min(batch - base, kAllocThreads);
    if (blockIdx.x != 0 && (kChunks ? cu_q[base] : base) >= tok_end) break;  // the same for the whole workgroup
    const int b = base + t;
    int q0 = 0, c = 0;
    int64_t n = 0;
    if (t < nb) {
      q0 = kChunks ? cu_q[b] : b;
      n = kChunks ? (int64_t)cu_q[b + 1] - q0 : 1;
      c = cached[b];
    }
    // (tokens outside the step have no thread to write their pages' entries: their sequence is refused)
    const bool fits = n > 0 && c >= 0 && c + n <= row_tokens && (!kChunks || (q0 >= 0 && q0 + n <= total_q));
    const int need = fits ? pages_of(c + (int)n, page_size) - pages_of(c, page_size) : 0;
    int incl = wave_sat_scan(need);
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    int before = carry, total = carry;
#pragma unroll
    for (int w = 0; w < kAllocThreads / 64; w++) {
      if (w < wave) before = sat_add(before, s_wave[w]);
      total = sat_add(total, s_wave[w]);
    }
    incl = sat_add(before, incl);
    const bool served = fits && (need == 0 || incl <= free0);
    const int first = incl - need;
    if (blockIdx.x == 0) {
      if (t < nb) {
        seqlens_out[b] = served ? c + (int)n : c;
        refused[b] = n > 0 && !served;
      }
      if (served && need > 0) atomicMax(&s_taken, incl);
    }
    if constexpr (kChunks) {
      // (one writer per word: places behind the pass's sequences are nobody's but the end's, which thread nb - 1 writes)
      if (t < nb) {
        s_cu[t] = q0;
        s_cached[t] = c;
        s_first[t] = served ? first : -1;
      }
      if (t == nb - 1) s_cu[nb] = q0 + (int)max(n, (int64_t)0);
      __syncthreads();
      if (tok < total_q && tok >= s_cu[0] && tok < s_cu[nb]) {
        int lo = 0, hi = nb;  // the last sequence that starts at or before the token (empty ones start where the next does)
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_cu[mid] <= tok) lo = mid; else hi = mid;
        }
        const int64_t at = (int64_t)s_cached[lo] + (tok - s_cu[lo]);
        if (s_first[lo] >= 0 && at < row_tokens) place(base + lo, s_cached[lo], s_first[lo], (int)at);
      }
      __syncthreads();  // the arrays are written again
    } else {
      if (b == tok && t < nb && served) place(b, c, first, c);
      __syncthreads();
    }
    carry = total;
  }
  if (tok < total_q) {
    slots[tok] = slot;
    positions[tok] = pos;
  }
  if (blockIdx.x == 0) {
    __syncthreads();
    if (t == 0) free_count_out[0] = free0 - s_taken;
  }
}

// Pages of finished sequences back onto the list: entry j of sequence b's row goes to place free + (pages of the finished
// sequences before b) + j.  A workgroup of four waves takes four sequences, a wave each, and sums the pages of all sequences
// before them itself.  Bound: the launch (64 sequences 3.1 us, 515 with up to 1024 pages each 5.2 us).
constexpr int kReleaseWaves = 4;
__global__ __launch_bounds__(64 * kReleaseWaves) void kv_release_kernel(
    const uint8_t* __restrict__ finished, const int32_t* __restrict__ seqlens, const int32_t* __restrict__ block_table,
    int64_t bt_row_stride, int32_t* __restrict__ free_pages, const int32_t* __restrict__ free_count, int32_t* __restrict__ seqlens_out,
    int32_t* __restrict__ free_count_out, int batch, int page_size, int max_pages, int n_pages) {
  __shared__ int s_wave[kReleaseWaves], s_own[kReleaseWaves];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int b0 = blockIdx.x * kReleaseWaves;
  const int free0 = min(max(free_count[0], 0), n_pages);
  auto pages = [&](int b) { return finished[b] && seqlens[b] > 0 ? min(pages_of(seqlens[b], page_size), max_pages) : 0; };
  int sum = 0;
  for (int b = t; b < b0; b += 64 * kReleaseWaves) sum = sat_add(sum, pages(b));
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum = sat_add(sum, __shfl_xor(sum, m, 64));
  const int b = b0 + wave, n = b < batch ? pages(b) : 0;
  if (lane == 0) {
    s_wave[wave] = sum;
    s_own[wave] = n;
    if (b < batch) seqlens_out[b] = finished[b] ? 0 : seqlens[b];
  }
  __syncthreads();
  int first = free0, total = free0;
#pragma unroll
  for (int w = 0; w < kReleaseWaves; w++) {
    first = sat_add(first, s_wave[w]);
    total = sat_add(total, sat_add(s_wave[w], s_own[w]));
    if (w < wave) first = sat_add(first, s_own[w]);
  }
  const int32_t* row = block_table + (int64_t)b * bt_row_stride;
  const int fit = min(n, max(n_pages - first, 0));  // (never past the list, whatever the counts say)
  for (int j = lane; j < fit; j += 64) free_pages[first + j] = row[j];
  if (t == 0 && b0 + kReleaseWaves >= batch) free_count_out[0] = min(total, n_pages);
}

// ------------------------------------------------------------------------------------------------------- 4-bit blocks
// Scale byte of a block from the largest magnitude's bit pattern: the smallest e >= -126 with amax <= 6 * 2^e, plus 127.
// amax = m * 2^E with m in [1, 2), and 6 * 2^e = 1.5 * 2^(e + 2): e = E - 2 while m <= 1.5, else E - 1.  (As integers the
// patterns of magnitudes order like the magnitudes, and infinities and NaN come out above all finite ones.)
// e <= 126, and magnitudes are held to 3 * 2^126 first: a code of 4 would overflow 32 bits there.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const uint32_t bits = min(amax_bits, 0x7f400000u);  // 3 * 2^126
  const int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x400000u ? 2 : 1);
  return (uint32_t)(max(e, -126) + 127);
}

// N pairs of elements -> N bytes of codes (round to nearest, ties to the even code), the first in the lowest byte.  The scale is a power of
// two: dividing by it is exact.
template <int N>
__device__ __forceinline__ uint32_t fp4_pack(const float* x, uint32_t scale_byte) {
  const float lim = 0x1.8p127f, scale = __uint_as_float(scale_byte << 23);
  float c[2 * N];
#pragma unroll
  for (int e = 0; e < 2 * N; e++) c[e] = __builtin_amdgcn_fmed3f(x[e], -lim, lim);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[0], c[1], scale, 0);
  if constexpr (N == 4) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[2], c[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[4], c[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[6], c[7], scale, 3);
  }
  return scale_byte == 255u ? 0u : w;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// FP8 rows: scale = max(amax, 1e-4) / 448 from the largest magnitude's bit pattern, in whose order NaN and infinities come out on top: the
// scale says what the row holds.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) { return __uint_as_float(max(amax_bits, __float_as_uint(1e-4f))) / 448.0f; }
// v / scale as it is encoded.  (The clamp would make a number of a NaN; without a finite scale every quotient is NaN or zero.)
__device__ __forceinline__ float fp8_clamp(float z, float scale) { return scale < __builtin_inff() ? fminf(fmaxf(z, -448.0f), 448.0f) : z; }

// ------------------------------------------------------------------------------- norm + rotation + append of new rows
struct AppendParams {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens (heads are dim apart)
  const void *q_weight, *k_weight;       // null: no norm
  const void *cos_table, *sin_table;     // [max_position, rotary_dim / 2]
  const int32_t* positions;
  const int64_t* slots;
  uint16_t* q_out;
  void *k_cache, *v_cache, *k_scale, *v_scale;
  int64_t n_tokens;  // of the pool
  int tokens, heads, heads_kv, dim, rotary_dim, max_position, page_size;
  double eps;
  int weight_fp32, table_fp32, interleaved;
  int page_shift;  // log2 of page_size, -1 if it is no power of two
};

enum { kCache16 = 0, kCacheFp8 = 1, kCacheFp4 = 2 };

template <typename XT>
__device__ __forceinline__ float load_x(const uint16_t* p) {
  uint32_t raw[1] = {*p};
  float out[2];
  Unpack<XT, 2>::run(raw, out);
  return out[0];
}
template <typename XT>
__device__ __forceinline__ float load_side(const void* p, int64_t i, int fp32) {
  return fp32 ? ((const float*)p)[i] : load_x<XT>((const uint16_t*)p + i);
}

// Keys that become codes are normed and rotated in 64 bits and rounded once; queries, keys kept in 16 bits and values in 32.
// The general form, for rows that the vector form below does not take: one head of one token per wave, a pair of neighbouring
// elements per lane (two pairs at head dim 256).  R: the type that the norm and the rotation are formed in.
template <typename XT, typename R>
__device__ __forceinline__ void norm_rotate_pair(const AppendParams& p, const uint16_t* x, const void* weight, int64_t tpos, int d, R rstd, float* out) {
  auto normed = [&](int e) -> R {
    const R v = (R)load_x<XT>(x + e);
    return weight ? v * rstd * (R)load_side<XT>(weight, e, p.weight_fp32) : v;
  };
  const int half = p.rotary_dim >> 1;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int e = d + i;
    R y = normed(e);
    if (e < p.rotary_dim) {
      const int f = p.interleaved ? e >> 1 : (e < half ? e : e - half);
      const bool first = p.interleaved ? (e & 1) == 0 : e < half;
      const R other = normed(p.interleaved ? e ^ 1 : (first ? e + half : e - half));
      const R c = (R)load_side<XT>(p.cos_table, tpos * half + f, p.table_fp32), s = (R)load_side<XT>(p.sin_table, tpos * half + f, p.table_fp32);
      y = first ? y * c - other * s : y * c + other * s;
    }
    out[i] = (float)y;
  }
}

template <typename XT, typename R>
__device__ __forceinline__ R head_rstd(const AppendParams& p, const uint16_t* x, const void* weight, int lane) {
  if (!weight) return (R)1;
  R sum = 0;
  for (int d = 2 * lane; d < p.dim; d += 128) {
    const R a = (R)load_x<XT>(x + d), b = (R)load_x<XT>(x + d + 1);
    sum += a * a + b * b;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m, 64);
  return (R)1 / sqrt(sum / (R)p.dim + (R)p.eps);
}

template <typename XT, int CACHE>
__global__ __launch_bounds__(256) void qk_norm_rope_append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int unit = blockIdx.y * 4 + uni(threadIdx.x >> 6), t = blockIdx.x;
  if (unit >= p.heads + 2 * p.heads_kv) return;
  const bool is_q = unit < p.heads, is_k = !is_q && unit < p.heads + p.heads_kv;
  const int h = is_q ? unit : is_k ? unit - p.heads : unit - p.heads - p.heads_kv;
  const uint16_t* x = is_q ? p.q + t * p.q_stride : is_k ? p.k + t * p.k_stride : p.v + t * p.v_stride;
  x += (int64_t)h * p.dim;
  const int pos = p.rotary_dim ? p.positions[t] : 0;
  const int64_t tpos = min(max(pos, 0), p.max_position - 1);  // never outside the tables
  const int64_t slot = p.slots[t];
  if (!is_q && (slot < 0 || slot >= p.n_tokens)) return;
  const void* weight = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
  float y[2][2];
  const int pairs = p.dim >> 1;
  // keys that become codes: in 64 bits, rounded to 32 once, so that a value next to a rounding border gets the same code
  // whatever the order of a sum is
  if (is_k && CACHE != kCache16) {
    const double rstd = head_rstd<XT, double>(p, x, weight, lane);
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (lane + 64 * j < pairs) norm_rotate_pair<XT, double>(p, x, weight, tpos, 2 * (lane + 64 * j), rstd, y[j]);
  } else {
    const float rstd = head_rstd<XT, float>(p, x, weight, lane);
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (lane + 64 * j >= pairs) continue;
      if (is_q || is_k) {
        norm_rotate_pair<XT, float>(p, x, weight, tpos, 2 * (lane + 64 * j), rstd, y[j]);
      } else {
        y[j][0] = load_x<XT>(x + 2 * (lane + 64 * j));
        y[j][1] = load_x<XT>(x + 2 * (lane + 64 * j) + 1);
      }
    }
  }
  const int64_t token_row = slot * p.heads_kv + h;  // row of a token-major pool
  if (is_q || CACHE == kCache16) {
    uint16_t* dst = is_q ? p.q_out + ((int64_t)t * p.heads + h) * p.dim : (uint16_t*)(is_k ? p.k_cache : p.v_cache) + token_row * p.dim;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int i = lane + 64 * j;
      if (i < pairs) ((uint32_t*)dst)[i] = (uint32_t)f32_to_elem_bits<XT>(y[j][0]) | ((uint32_t)f32_to_elem_bits<XT>(y[j][1]) << 16);
    }
    return;
  }
  if (CACHE == kCacheFp8) {
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (lane + 64 * j < pairs) amax = max(amax, max(abs_bits(y[j][0]), abs_bits(y[j][1])));
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m, 64));
    const float sc = fp8_scale(amax);
    if (lane == 0) ((float*)(is_k ? p.k_scale : p.v_scale))[token_row] = sc;
    uint8_t* dst = (uint8_t*)(is_k ? p.k_cache : p.v_cache) + token_row * p.dim;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int i = lane + 64 * j;
      if (i >= pairs) continue;
      const float a = fp8_clamp(y[j][0] / sc, sc), b = fp8_clamp(y[j][1] / sc, sc);
      ((uint16_t*)dst)[i] = (uint16_t)(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0u, false) & 0xffff);
    }
    return;
  }
  // fp4: sixteen lanes hold a block
  const int64_t page = slot / p.page_size;
  const int64_t row = (page * p.heads_kv + h) * p.page_size + (slot - page * p.page_size);
  uint8_t* codes = (uint8_t*)(is_k ? p.k_cache : p.v_cache) + row * (p.dim >> 1);
  uint8_t* scales = (uint8_t*)(is_k ? p.k_scale : p.v_scale) + row * (p.dim >> 5);
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int i = lane + 64 * j;
    if (i >= pairs) continue;  // (whole groups of sixteen lanes: dim is a multiple of 32)
    uint32_t amax = max(abs_bits(y[j][0]), abs_bits(y[j][1]));
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, m, 64));
    const uint32_t byte = fp4_scale_byte(amax);
    codes[i] = (uint8_t)fp4_pack<1>(y[j], byte);
    if ((lane & 15) == 0) scales[i >> 4] = (uint8_t)byte;
  }
}

// The vector form: a lane has eight consecutive elements of a row (16 bytes), a wave 512 / dim rows at a time, rows of one kind (query,
// key, value) counted through all tokens so that few kv heads still fill the wave.  The other half of a rotated pair lies rotary_dim / 16
// lanes away: its raw elements come over as four dwords, and the lane norms them itself.  All rows of a wave are requested at its
// start; tables are read again only when the token changes.
// Takes: rotary_dim a multiple of 16 (interleaved: of 8), rows, tables and weights 16-byte aligned.
// Bound: memory.  32 query heads on 8, dim 128, 4-bit cache: 8192 tokens in 44.5 us, 4.1 TB/s of what a copy reaches 4.7 (general form: 189 us),
// 64 tokens in 3.7 us (5.0).  The kind of rotation is a template argument: its branches in the passes cost 7% (8192 tokens with four passes 52 us).
// Four values (16-bit or fp32) of a weight or table as floats.
template <typename XT>
__device__ __forceinline__ f32x4 load_side4(const void* p, int64_t i, int fp32) {
  if (fp32) return *(const f32x4*)((const float*)p + i);
  const u32x2 w = *(const u32x2*)((const uint16_t*)p + i);
  const uint32_t raw[2] = {w[0], w[1]};
  float out[4];
  Unpack<XT, 4>::run(raw, out);
  return f32x4{out[0], out[1], out[2], out[3]};
}

// Reductions over the 8, 16 or 32 neighbouring lanes of a row on the data-parallel-primitive path: lanes one and two apart, then
// (groups of four being equal) the mirrored half row and the mirrored row, then the neighbouring row of sixteen.
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ __forceinline__ float dpp(float x) { return __uint_as_float(dpp<CTRL>(__float_as_uint(x))); }
template <int CTRL> __device__ __forceinline__ double dpp(double x) {
  const u32x2 w = __builtin_bit_cast(u32x2, x);
  return __builtin_bit_cast(double, u32x2{dpp<CTRL>(w[0]), dpp<CTRL>(w[1])});
}
__device__ __forceinline__ uint32_t other_row(uint32_t x) {  // the same lane of the other row of sixteen in a pair of rows
  const u32x2 r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return (threadIdx.x & 16) ? r[0] : r[1];
}
__device__ __forceinline__ float other_row(float x) { return __uint_as_float(other_row(__float_as_uint(x))); }
__device__ __forceinline__ double other_row(double x) {
  const u32x2 w = __builtin_bit_cast(u32x2, x);
  return __builtin_bit_cast(double, u32x2{other_row(w[0]), other_row(w[1])});
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
template <typename T, typename F>
__device__ __forceinline__ T over_row(T x, int lanes, F f) {
  x = f(x, dpp<kXor1>(x));
  x = f(x, dpp<kXor2>(x));
  x = f(x, dpp<kHalfMirror>(x));
  if (lanes > 8) x = f(x, dpp<kMirror>(x));
  if (lanes > 16) x = f(x, other_row(x));
  return x;
}

__device__ __forceinline__ float inverse_root(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double inverse_root(double x) {  // the hardware's estimate and two Newton steps
  double r = __builtin_amdgcn_rsq(x);
  if (!(r > 0.0 && r < __builtin_inf())) return r;
  r = r * (1.5 - 0.5 * x * r * r);
  return r * (1.5 - 0.5 * x * r * r);
}

enum { kNoTurn = 0, kHalves = 1, kPairs = 2 };  // rotation: none, of the two halves, of neighbouring pairs

// Where a lane's eight elements stand in the rotation.
struct Turn {
  bool on, upper;  // they are rotated; they are the second half of their pairs
  int mate;        // lane of the row that holds the other half (its own for neighbouring pairs, or if they are not rotated)
};

// Coefficients of elements 4k .. 4k + 3 of the lane: y[e] = own[e] * c[e] + other[e] * s[e] with own, other normed rows.  Lanes that are not
// rotated read the first coefficients and take 1 and -0 (with other = +0 the sum leaves every value as it is, zeros and infinities too).
template <typename XT, int TURN>
__device__ __forceinline__ void side4(const AppendParams& p, const Turn& t, int64_t tpos, int j, int k, f32x4* c, f32x4* s) {
  const int half = p.rotary_dim >> 1;
  if constexpr (TURN == kNoTurn) {
    *c = f32x4{1.f, 1.f, 1.f, 1.f};
    *s = f32x4{0.f, 0.f, 0.f, 0.f};
  } else if constexpr (TURN == kPairs) {
    const int64_t at = tpos * half + (t.on ? 4 * j + 2 * k : 0);
    float c0, c1, s0, s1;
    if (p.table_fp32) {
      const f32x2 a = *(const f32x2*)((const float*)p.cos_table + at), b = *(const f32x2*)((const float*)p.sin_table + at);
      c0 = a[0], c1 = a[1], s0 = b[0], s1 = b[1];
    } else {
      const uint32_t ra[1] = {*(const uint32_t*)((const uint16_t*)p.cos_table + at)}, rb[1] = {*(const uint32_t*)((const uint16_t*)p.sin_table + at)};
      float a[2], b[2];
      Unpack<XT, 2>::run(ra, a);
      Unpack<XT, 2>::run(rb, b);
      c0 = a[0], c1 = a[1], s0 = b[0], s1 = b[1];
    }
    *c = f32x4{c0, c0, c1, c1};
    *s = f32x4{-s0, s0, -s1, s1};
  } else {
    const int64_t at = tpos * half + (t.on ? 8 * j - (t.upper ? half : 0) + 4 * k : 0);
    *c = load_side4<XT>(p.cos_table, at, p.table_fp32);
    *s = load_side4<XT>(p.sin_table, at, p.table_fp32);
#pragma unroll
    for (int e = 0; e < 4; e++) (*s)[e] = t.upper ? (*s)[e] : -(*s)[e];
  }
  if constexpr (TURN != kNoTurn) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      (*c)[e] = t.on ? (*c)[e] : 1.f;
      (*s)[e] = t.on ? (*s)[e] : -0.f;
    }
  }
}

// x / s for many values and one s in [2^-23, 2^120], |x| <= 448 s: the quotient corrected once by its remainder (Markstein), with one
// reciprocal for all of them instead of one division each.
struct Quotient {
  float s, r;
  __device__ __forceinline__ explicit Quotient(float d) : s(d) {
    const float r0 = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r0, 1.0f), r0, r0);
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * r;
    return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-s, q, x), r, q), x);  // (a zero keeps its sign)
  }
};

template <typename XT>
__device__ __forceinline__ u32x4 pack_row8(const float* y) {
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; e++) o[e] = (uint32_t)f32_to_elem_bits<XT>(y[2 * e]) | ((uint32_t)f32_to_elem_bits<XT>(y[2 * e + 1]) << 16);
  return o;
}

// Eight finished elements of row (token, head h) of a kind into the cache.
template <typename XT, int CACHE>
__device__ __forceinline__ void store_cached(const AppendParams& p, void* cache, void* scale, const float* y, int64_t slot, int h, int lanes, int j, bool store) {
  const int64_t token_row = slot * p.heads_kv + h;  // row of a token-major pool
  if constexpr (CACHE == kCache16) {
    if (store) *(u32x4*)((uint16_t*)cache + token_row * p.dim + 8 * j) = pack_row8<XT>(y);
  } else if constexpr (CACHE == kCacheFp8) {
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = max(amax, abs_bits(y[e]));
    amax = over_row(amax, lanes, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float sc = fp8_scale(amax);
    const Quotient over(sc);
    const bool plain = sc < 0x1p100f;  // (else NaN, an infinity or close to one: the division itself)
    u32x2 o;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float z[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float v = y[4 * e + k];
        z[k] = fp8_clamp(plain ? over(v) : v / sc, sc);
      }
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
      o[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], lo, true);
    }
    if (store) {
      *(u32x2*)((uint8_t*)cache + token_row * p.dim + 8 * j) = o;
      if (j == 0) ((float*)scale)[token_row] = sc;
    }
  } else {
    // four lanes hold a block
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = max(amax, abs_bits(y[e]));
    amax = max(amax, dpp<kXor1>(amax));
    amax = max(amax, dpp<kXor2>(amax));
    const uint32_t byte = fp4_scale_byte(amax);
    const uint32_t o = fp4_pack<4>(y, byte);
    if (store) {
      const uint32_t page = p.page_shift >= 0 ? (uint32_t)slot >> p.page_shift : (uint32_t)slot / (uint32_t)p.page_size;
      const uint32_t off = (uint32_t)slot - page * (uint32_t)p.page_size;
      const int64_t row = ((int64_t)page * p.heads_kv + h) * p.page_size + off;
      *(uint32_t*)((uint8_t*)cache + row * (p.dim >> 1) + 4 * j) = o;
      if ((j & 3) == 0) ((uint8_t*)scale)[row * (p.dim >> 5) + (j >> 2)] = (uint8_t)byte;
    }
  }
}

enum { kQuery, kKey, kValue };

// Rows of large calls stream past the caches (8192 tokens: 71 -> 65 us); the few of a decode step stay there for the attention that follows.
template <int PASSES> __device__ __forceinline__ u32x4 load_once(const u32x4* p) { return PASSES > 1 ? __builtin_nontemporal_load(p) : *p; }
template <int PASSES> __device__ __forceinline__ void store_once(u32x4* p, u32x4 v) {
  if constexpr (PASSES > 1) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// Rows of one kind.  R: the type that norm and rotation are formed in (see the general form).
template <typename XT, int CACHE, int KIND, typename R, int PASSES, int TURN>
__device__ __forceinline__ void append_rows(const AppendParams& p, int wave) {
  const int lane = threadIdx.x & 63;
  const int lanes = p.dim >> 3, j = lane & (lanes - 1), per_wave = 64 / lanes;  // lanes per row, the lane's place, rows per pass
  const int heads = KIND == kQuery ? p.heads : p.heads_kv, rows = p.tokens * heads;  // (below 2^26: the launcher checks)
  const int row0 = wave * PASSES * per_wave;
  if (row0 >= rows) return;
  const uint16_t* base = KIND == kQuery ? p.q : KIND == kKey ? p.k : p.v;
  const int64_t stride = KIND == kQuery ? p.q_stride : KIND == kKey ? p.k_stride : p.v_stride;
  const void* weight = KIND == kQuery ? p.q_weight : KIND == kKey ? p.k_weight : nullptr;
  constexpr bool rotates = KIND != kValue && TURN != kNoTurn;
  const int apart = p.rotary_dim >> 4;  // lanes between the halves of a pair
  Turn turn;
  turn.on = rotates && 8 * j < p.rotary_dim;
  turn.upper = j >= apart;
  turn.mate = turn.on && TURN == kHalves ? (turn.upper ? j - apart : j + apart) : j;
  const int mate_lane = lane - j + turn.mate;

  // the lane's rows, all requested at once: token and head, stepped instead of divided
  const int dt = per_wave / heads, dh = per_wave - dt * heads;
  const R inv_dim = (R)1 / (R)p.dim;  // (a power of two)
  int tokens[PASSES], head_of[PASSES];
  u32x4 raw[PASSES];
  {
    int token = (row0 + lane / lanes) / heads, head = row0 + lane / lanes - token * heads;
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
      tokens[i] = min(token, p.tokens - 1);  // (past the end: a row of the last token again, which is not stored)
      head_of[i] = head;
      raw[i] = load_once<PASSES>((const u32x4*)(base + tokens[i] * stride + head * p.dim + 8 * j));
      token += dt;
      head += dh;
      if (head >= heads) {
        head -= heads;
        token++;
      }
    }
  }
  // What depends on the token is requested here too, ahead of all stores (which the compiler keeps loads behind).
  int64_t slots[PASSES], tpos[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; i++) {
    slots[i] = KIND != kQuery ? p.slots[tokens[i]] : 0;
    tpos[i] = rotates ? min(max(p.positions[tokens[i]], 0), p.max_position - 1) : 0;  // never outside the tables
  }
  // 64-bit rows: tables and weights as they are; 32-bit rows: weight times cosine, the other half's weight times sine
  constexpr bool WIDE = sizeof(R) == 8;
  f32x4 c[WIDE ? PASSES : 1][2], s[WIDE ? PASSES : 1][2], w[2], wo[2];
  if constexpr (KIND != kValue) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      w[k] = wo[k] = f32x4{1.f, 1.f, 1.f, 1.f};
      if (weight) {
        w[k] = load_side4<XT>(weight, 8 * j + 4 * k, p.weight_fp32);
        wo[k] = TURN == kPairs ? f32x4{w[k][1], w[k][0], w[k][3], w[k][2]} : load_side4<XT>(weight, 8 * turn.mate + 4 * k, p.weight_fp32);
#pragma unroll
        for (int e = 0; e < 4; e++) wo[k][e] = turn.on ? wo[k][e] : 1.f;
      }
#pragma unroll
      for (int i = 0; i < (WIDE ? PASSES : 1); i++) side4<XT, TURN>(p, turn, tpos[i], j, k, &c[i][k], &s[i][k]);
      if constexpr (!WIDE) {
        c[0][k] *= w[k];
        s[0][k] *= wo[k];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; i++) {
    if (row0 + i * per_wave >= rows) break;
    const int r = row0 + i * per_wave + lane / lanes, t = tokens[i], h = head_of[i];
    const uint32_t x[4] = {raw[i][0], raw[i][1], raw[i][2], raw[i][3]};
    const int64_t slot = slots[i];
    float y[8];
    if constexpr (KIND == kValue) {
      Unpack<XT, 8>::run(x, y);
    } else {
      uint32_t other[4];
      if constexpr (rotates) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          other[e] = TURN == kPairs ? __builtin_amdgcn_alignbit(x[e], x[e], 16) : (uint32_t)__shfl((int)x[e], mate_lane, 64);
          other[e] = turn.on ? other[e] : 0u;
        }
      }
      float xf[8];
      Unpack<XT, 8>::run(x, xf);
      R sum = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) sum += (R)xf[e] * (R)xf[e];
      sum = over_row(sum, lanes, [](R a, R b) { return a + b; });
      const R root = inverse_root(sum * inv_dim + (R)p.eps), rstd = weight ? root : (R)1;
      float of[8];
      if constexpr (rotates) Unpack<XT, 8>::run(other, of);
      if constexpr (!WIDE) {
        if (rotates && i > 0 && __ballot(t != tokens[i > 0 ? i - 1 : 0])) {  // another token's tables
#pragma unroll
          for (int k = 0; k < 2; k++) {
            side4<XT, TURN>(p, turn, tpos[i], j, k, &c[0][k], &s[0][k]);
            c[0][k] *= w[k];
            s[0][k] *= wo[k];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float z = xf[e] * c[0][e >> 2][e & 3];
          if constexpr (rotates) z = __builtin_fmaf(of[e], s[0][e >> 2][e & 3], z);
          y[e] = z * rstd;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int k = e >> 2, l = e & 3;
          R z = (R)xf[e] * (R)w[k][l] * (R)c[WIDE ? i : 0][k][l];
          if constexpr (rotates) z += (R)of[e] * (R)wo[k][l] * (R)s[WIDE ? i : 0][k][l];
          y[e] = (float)(z * rstd);
        }
      }
    }
    const bool store = r < rows && (KIND == kQuery || (slot >= 0 && slot < p.n_tokens));
    if constexpr (KIND == kQuery) {
      if (store) store_once<PASSES>((u32x4*)(p.q_out + (int64_t)r * p.dim + 8 * j), pack_row8<XT>(y));
    } else {
      store_cached<XT, CACHE>(p, KIND == kKey ? p.k_cache : p.v_cache, KIND == kKey ? p.k_scale : p.v_scale, y, slot, h, lanes, j, store);
    }
  }
}

// PASSES of a wave over query rows; key and value rows, whose token changes more often, take half as many.
template <typename XT, int CACHE, int PASSES, int TURN>
__global__ __launch_bounds__(256, 4) void qk_norm_rope_append_rows_kernel(const AppendParams p, int q_waves, int k_waves) {
  constexpr int KP = (PASSES + 1) / 2;
  int wave = blockIdx.x * 4 + uni(threadIdx.x >> 6);
  if (wave < k_waves) {  // (the longest rows first)
    if constexpr (CACHE == kCache16) append_rows<XT, CACHE, kKey, float, KP, TURN>(p, wave);
    else append_rows<XT, CACHE, kKey, double, KP, TURN>(p, wave);
  } else if ((wave -= k_waves) < q_waves) {
    append_rows<XT, CACHE, kQuery, float, PASSES, TURN>(p, wave);
  } else {
    append_rows<XT, CACHE, kValue, float, KP, TURN>(p, wave - q_waves);
  }
}

template <typename XT, int PASSES, int TURN>
void launch_append_rows(const AppendParams& p, int cache, hipStream_t s) {
  auto waves = [&](int heads, int rows) { return (int)(((int64_t)p.tokens * heads + rows - 1) / rows); };
  const int q_waves = waves(p.heads, 512 / p.dim * PASSES), k_waves = waves(p.heads_kv, 512 / p.dim * ((PASSES + 1) / 2));
  const dim3 grid((q_waves + 2 * k_waves + 3) / 4), block(256);
  auto kern = cache == kCacheFp4 ? qk_norm_rope_append_rows_kernel<XT, kCacheFp4, PASSES, TURN>
              : cache == kCacheFp8 ? qk_norm_rope_append_rows_kernel<XT, kCacheFp8, PASSES, TURN> : qk_norm_rope_append_rows_kernel<XT, kCache16, PASSES, TURN>;
  hipLaunchKernelGGL(kern, grid, block, 0, s, p, q_waves, k_waves);
}

// --------------------------------------------------------------------------------------------- rows of the 4-bit cache
// Eight elements of a key row and of its value row per thread (four bytes of codes in, sixteen out).  Slots outside the pool give zeros.
// Bound: memory (8192 tokens of 8 heads, dim 128, 42 MB in 9.0 us, 4.7 TB/s, what a copy reaches; 64 tokens 2.9 us, the launch).
struct GatherParams {
  const uint8_t *codes[2], *scales[2];
  const int64_t* slots;
  u32x4* out[2];
  uint32_t items, heads_kv;  // (items: threads, below 2^32 as in any grid)
  int row_shift;             // log2 of the threads of a row, dim / 8
  int page_size, page_shift; // log2 of page_size, -1 if it is no power of two
  int64_t n_tokens;
};
template <typename XT>
__global__ __launch_bounds__(256) void kv_gather_fp4_kernel(const GatherParams p) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= p.items) return;
  const uint32_t row_of = i >> p.row_shift, c = i - (row_of << p.row_shift), t = row_of / p.heads_kv, h = row_of - t * p.heads_kv;
  const int64_t slot = p.slots[t];
  u32x4 r[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
  if (slot >= 0 && slot < p.n_tokens) {
    const int64_t page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    const int64_t row = (page * p.heads_kv + h) * p.page_size + (slot - page * p.page_size);
    uint32_t w[2], b[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      w[k] = *(const uint32_t*)(p.codes[k] + (row << (p.row_shift + 2)) + 4 * c);
      b[k] = p.scales[k][(row << (p.row_shift - 2)) + (c >> 2)];
    }
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const float sc = __uint_as_float(b[k] << 23);
      if constexpr (__is_same(XT, bf16_tag)) {
        r[k][0] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[k], sc, 0));
        r[k][1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[k], sc, 1));
        r[k][2] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[k], sc, 2));
        r[k][3] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[k], sc, 3));
      } else {
        r[k][0] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[k], sc, 0));
        r[k][1] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[k], sc, 1));
        r[k][2] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[k], sc, 2));
        r[k][3] = __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[k], sc, 3));
      }
    }
  }
  p.out[0][i] = r[0];
  p.out[1][i] = r[1];
}

const char* launched() {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? nullptr : hipGetErrorString(e);
}

}  // namespace

const char* launch_kv_alloc(const int32_t* cached, const int32_t* cu_q, int32_t* block_table, int64_t bt_row_stride, const int32_t* free_pages,
                            const int32_t* free_count, int64_t* slots, int32_t* positions, int32_t* seqlens_out, uint8_t* refused,
                            int32_t* free_count_out, int batch, int total_q, int page_size, int max_pages, int n_pages, hipStream_t s) {
  const dim3 grid(total_q > 0 ? (total_q + kAllocThreads - 1) / kAllocThreads : 1), block(kAllocThreads);
  if (cu_q)
    hipLaunchKernelGGL(kv_alloc_kernel<true>, grid, block, 0, s, cached, cu_q, block_table, bt_row_stride, free_pages, free_count, slots,
                       positions, seqlens_out, refused, free_count_out, batch, total_q, page_size, max_pages, n_pages);
  else
    hipLaunchKernelGGL(kv_alloc_kernel<false>, grid, block, 0, s, cached, cu_q, block_table, bt_row_stride, free_pages, free_count, slots,
                       positions, seqlens_out, refused, free_count_out, batch, total_q, page_size, max_pages, n_pages);
  return launched();
}

const char* launch_kv_release(const uint8_t* finished, const int32_t* seqlens, const int32_t* block_table, int64_t bt_row_stride,
                              int32_t* free_pages, const int32_t* free_count, int32_t* seqlens_out, int32_t* free_count_out, int batch,
                              int page_size, int max_pages, int n_pages, hipStream_t s) {
  hipLaunchKernelGGL(kv_release_kernel, dim3((batch + kReleaseWaves - 1) / kReleaseWaves), dim3(64 * kReleaseWaves), 0, s, finished, seqlens,
                     block_table, bt_row_stride, free_pages, free_count, seqlens_out, free_count_out, batch, page_size, max_pages, n_pages);
  return launched();
}

namespace {
// Passes of a wave: one while that leaves a few waves per SIMD, then four, six in the largest calls (all rows of a wave are requested ahead).
// 32 query heads on 8, dim 128, 4-bit cache, one / four / six passes: 256 tokens 4.3 / 4.8 us, 512 5.5 / 5.6, 1024 8.9 / 7.6 / 8.1, 2048
// 15.6 / 12.9 / 13.0, 4096 27.7 / 23.8 / 23.1, 8192 51.5 / 48.5 / 44.1 (FP8 and 16-bit caches alike; 2050 tokens of 20 heads, dim 256, 10.5 / 11.4).
int append_passes(int tokens, int heads, int heads_kv, int per_wave) {
  const int64_t passes = (int64_t)tokens * (heads + 2 * heads_kv) / per_wave;
  return passes < 8192 ? 1 : passes < 40960 ? 4 : 6;
}
}  // namespace

const char* launch_qk_norm_rope_append(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                       const void* q_weight, const void* k_weight, int weight_dtype, const void* cos_table,
                                       const void* sin_table, int table_dtype, int64_t max_position, const int32_t* positions,
                                       const int64_t* slots, void* q_out, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                       int tokens, int heads, int heads_kv, int dim, int rotary_dim, int interleaved, double eps,
                                       int page_size, int64_t n_phys_tokens, int x_dtype, int cache_dtype, hipStream_t s) {
  AppendParams p;
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.cos_table = cos_table;
  p.sin_table = sin_table;
  p.positions = positions;
  p.slots = slots;
  p.q_out = (uint16_t*)q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.n_tokens = n_phys_tokens;
  p.tokens = tokens;
  p.heads = heads;
  p.heads_kv = heads_kv;
  p.dim = dim;
  p.rotary_dim = rotary_dim;
  p.max_position = (int)(max_position < INT_MAX ? max_position : INT_MAX);
  p.page_size = page_size;
  p.eps = eps;
  p.weight_fp32 = weight_dtype == MI355_DT_FP32;
  p.table_fp32 = table_dtype == MI355_DT_FP32;
  p.interleaved = interleaved;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  const int cache = cache_dtype == MI355_DT_FP4_E2M1 ? kCacheFp4 : cache_dtype == MI355_DT_FP8_E4M3FN ? kCacheFp8 : kCache16;
  const bool bf16 = x_dtype == MI355_DT_BF16;
  const uintptr_t bases = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)cos_table | (uintptr_t)sin_table;
  const int64_t most_rows = (int64_t)tokens * (heads > heads_kv ? heads : heads_kv);
  if (rotary_dim % (interleaved ? 8 : 16) == 0 && (bases & 15) == 0 && ((q_stride | k_stride | v_stride) & 7) == 0 && most_rows < (1 << 26)) {
    const int passes = append_passes(tokens, heads, heads_kv, 512 / dim);
    auto launch = [&](auto x_tag, auto turn) {
      using XT = decltype(x_tag);
      constexpr int TURN = decltype(turn)::value;
      if (passes == 6) launch_append_rows<XT, 6, TURN>(p, cache, s);
      else if (passes == 4) launch_append_rows<XT, 4, TURN>(p, cache, s);
      else launch_append_rows<XT, 1, TURN>(p, cache, s);
    };
    auto launch_turn = [&](auto x_tag) {
      if (rotary_dim == 0) launch(x_tag, std::integral_constant<int, kNoTurn>{});
      else if (interleaved) launch(x_tag, std::integral_constant<int, kPairs>{});
      else launch(x_tag, std::integral_constant<int, kHalves>{});
    };
    if (bf16) launch_turn(bf16_tag{});
    else launch_turn(fp16_tag{});
    return launched();
  }
  if (tokens >= (1 << 24)) return "too many tokens for a grid";
  const dim3 grid(tokens, (heads + 2 * heads_kv + 3) / 4), block(256);
  auto kern = bf16 ? (cache == kCacheFp4 ? qk_norm_rope_append_kernel<bf16_tag, kCacheFp4>
                      : cache == kCacheFp8 ? qk_norm_rope_append_kernel<bf16_tag, kCacheFp8> : qk_norm_rope_append_kernel<bf16_tag, kCache16>)
                   : (cache == kCacheFp4 ? qk_norm_rope_append_kernel<fp16_tag, kCacheFp4>
                      : cache == kCacheFp8 ? qk_norm_rope_append_kernel<fp16_tag, kCacheFp8> : qk_norm_rope_append_kernel<fp16_tag, kCache16>);
  hipLaunchKernelGGL(kern, grid, block, 0, s, p);
  return launched();
}

const char* launch_kv_gather_fp4(const void* k, const void* v, const void* k_scale, const void* v_scale, const int64_t* slots, void* k_out,
                                 void* v_out, int tokens, int heads_kv, int dim, int page_size, int64_t n_phys_tokens, int out_dtype,
                                 hipStream_t s) {
  const int64_t items = (int64_t)tokens * heads_kv * (dim / 8);
  GatherParams p;
  p.codes[0] = (const uint8_t*)k;
  p.codes[1] = (const uint8_t*)v;
  p.scales[0] = (const uint8_t*)k_scale;
  p.scales[1] = (const uint8_t*)v_scale;
  p.slots = slots;
  p.out[0] = (u32x4*)k_out;
  p.out[1] = (u32x4*)v_out;
  p.items = (uint32_t)items;
  p.heads_kv = (uint32_t)heads_kv;
  p.row_shift = __builtin_ctz(dim / 8);  // (head dims 64, 128 and 256)
  p.page_size = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.n_tokens = n_phys_tokens;
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  auto kern = out_dtype == MI355_DT_BF16 ? kv_gather_fp4_kernel<bf16_tag> : kv_gather_fp4_kernel<fp16_tag>;
  hipLaunchKernelGGL(kern, grid, block, 0, s, p);
  return launched();
}

}  // namespace mi355
