// Paged GQA decode over a 4-bit KV cache for gfx950 (MI355X): e2m1 codes with one power-of-two scale byte per 32 head elements
// (layout: paged_cache_step.hip), head dims 64, 128 and 256, bf16 or fp16 queries.
//
//   o[r] = sum_t p[r, t] v[t] / sum_t p[r, t],  p[r, t] = exp2(logit2(q[r] . k[t]) - m[r]),  over the tokens that row r sees,
// one pass over the tokens with a running maximum m (moved only when it grows by more than 8 in the log2 domain) and sum.
//
//  * A workgroup of four waves owns (range of the token stream, kv head, block of query rows).  The stream -- every
//    128-token unit of every sequence, in batch order -- is cut into n_parts equal ranges on the device, so that compute
//    units get the same number of units whatever the lengths are and nothing is read back.  The waves take the 32-token
//    tiles of a unit in turn and meet once per sequence, in LDS.  A sequence that lies in one range is written out there;
//    the others leave normalised fp32 rows with log-sum-exps for the merge kernel.  Where the block tables address few tokens
//    a range is a sequence: nothing is left to merge.
//  * Q.K^T: v_mfma_scale_f32_16x16x128_f8f6f4 with the K codes as they lie in memory -- lane (c, g) supplies block g of token
//    c, sixteen bytes, and its scale byte -- against the query row as a sum of two (bf16) or three (fp16) e4m3 rows with scales of their own.
//    Tokens sit on the M axis, so every softmax quantity of a query row is local to a lane column.
//  * PV: O^T += V^T.P^T on v_mfma_f32_16x16x32_bf16.  Lane (c, g) loads the head elements [c * D/16, (c + 1) * D/16) of its eight
//    tokens -- those whose probabilities it holds already -- widens them with their scale (v_cvt_scalef32_pk_bf16_fp4) and pairs the
//    tokens with byte permutes: V needs no LDS, P does not move.
//  * K, V and scales go from memory to registers, a tile ahead of their use, across the borders of sequences.
//
// Roundings: the query's e4m3 rows add up to its elements down to 2^-14 (fp16: 2^-16) of the row's largest, smaller ones are off by 2^-22 (2^-27)
// of that one at most; a probability becomes two bf16 (2^-17 of it), because PV then runs at the rate of 16-bit products.  Waves with two blocks of
// rows and bf16 queries make do with one bf16 (2^-9; the output's own rounding is that large): they are bound by the vector unit, where
// the second part takes 40 instructions and 18 products a tile (32 x 1024 .. 16384 tokens with eight query tokens: 115 to 123 us, with both 142 to 154; calls with
// one block, one part / two: 8 x 131072 tokens 181 / 184 us, 64 ragged 59 / 61, 16 ragged at head dim 256 52 / 53, 4 x 3000 of 64 rows 17.1 / 18.0).  The row's sum is formed of the rounded ones, so that a
// common error cancels.  All else is fp32.
//
// Bound and measured (8 kv heads, dim 128): 64 query heads, 8 x 131072 tokens, 1.14 GB in 179 us, 6.4 TB/s: memory.  32 query heads, 64
// sequences of 512 .. 8192 tokens, 304 MB in 48 to 52 us, 5.8 to 6.3 TB/s: memory.  64 query heads, 32 sequences of 1024 .. 16384 tokens with
// eight query tokens and capped scores: 311 MB in 116 to 130 us, bound by the vector unit -- per tile of 32 tokens and two row blocks about
// 250 vector instructions, 48 of them exponentials and reciprocals at half rate, beside 26 matrix instructions.  One sequence of 300
// tokens: 7.2 to 8 us, the chain of loads length, table entry, tile.
#include <climits>
#include <type_traits>

#include "common.h"
#include "device_utils.h"

namespace mi355 {

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) int i32x8;

constexpr int kTile = 32;             // tokens per step of a wave
constexpr int kWaves = 4;             // waves of a workgroup
constexpr int kUnit = kTile * kWaves; // tokens per unit of the token stream
constexpr float kRescaleGap4 = 8.0f;
constexpr float kLargeCap = 4096.0f;  // of a cap in the log2 domain, see its use

struct Fp4Params {
  const uint16_t* q;
  const uint8_t *k, *v, *k_scale, *v_scale;
  const int32_t *seqlens, *block_table;
  int64_t bt_row_stride;
  uint16_t* out;
  float *part_o, *part_lse;
  int batch, q_len, heads, heads_kv, page_size, group, rows, row_groups, n_parts, max_len, causal, negate_q;
  int n_pages;
  int range_units;  // that a range has at least, where there are as many
  int by_sequence;  // part i is sequence i (tables of few tokens), with nothing to merge
  float score_scale, cap_log2e;  // scale of a score to its logit2, with a cap to 2 log2(e) times the tanh's argument
};

__device__ __forceinline__ int len_of(const Fp4Params& p, int b) { return min(max(p.seqlens[b], 0), p.max_len); }
__device__ __forceinline__ int units_of_len(int len) { return (int)(((uint32_t)len + kUnit - 1) / kUnit); }

// The T > 0 units cut into NP = min(n_parts, ceil(T / range_units)) ranges, none of them empty, with bounds floor(p * T / NP) = p * (T / NP) +
// floor(p * (T % NP) / NP); NP <= 4096 keeps the second product below 2^24.
struct Ranges {
  uint32_t np, tq, tr;
  __device__ __forceinline__ Ranges(int t, const Fp4Params& p) {
    np = (uint32_t)min(p.n_parts, 1 + (t - 1) / p.range_units);  // (t > 0)
    tq = (uint32_t)t / np;
    tr = (uint32_t)t % np;
  }
  __device__ __forceinline__ int begin(int p) const { return (int)((uint32_t)p * tq + ((uint32_t)p * tr) / np); }
  // the last range that begins at or before unit u
  __device__ __forceinline__ int owner(int u) const {
    // a float estimate, put right by the bounds (u and np / T carry 24 bits: off by a few at most, whatever their sizes)
    int p = min(max((int)((float)u * ((float)np / (float)(tq * np + tr))), 0), (int)np - 1);
    while (p > 0 && begin(p) > u) --p;
    while (p + 1 < (int)np && begin(p + 1) <= u) ++p;
    return p;
  }
};

// Units of all sequences, and of those before sequence `b` (whole wave).
__device__ __forceinline__ int total_units(const Fp4Params& p, int b, int* before) {
  const int lane = threadIdx.x & 63;
  int sum = 0, pre = 0;
  for (int base = 0; base < p.batch; base += 64) {
    const int n = base + lane < p.batch ? units_of_len(len_of(p, base + lane)) : 0, incl = wave_incl_scan(n);
    if (b >= base && b < base + 64) pre = sum + __builtin_amdgcn_readlane(incl - n, b - base);
    sum += __builtin_amdgcn_readlane(incl, 63);
  }
  *before = uni(pre);
  return uni(sum);
}

__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
template <typename QT> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<bf16_tag>(float lo, float hi) { return pack_bf16(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack16<fp16_tag>(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
}
__device__ __forceinline__ f32x4 mma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int SEL> __device__ __forceinline__ uint32_t widen2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}

// Sixteen tokens' K codes against sixteen query rows; SEL: byte of b_scales that is the scale byte of the lane's block of the query operand.
template <int SEL> __device__ __forceinline__ f32x4 mma_codes(u32x4 k, u32x4 b0, u32x4 b1, f32x4 c, uint32_t k_scale, uint32_t b_scales) {
  const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  const i32x8 b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, (int)k_scale, SEL, (int)b_scales);
}

// (a constant-address-space load of a wave-uniform address is a scalar load: the block table does not pass through the
// vector-memory counter, whose order the tile pipeline relies on)
typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
__device__ __forceinline__ int scalar_load(const int32_t* p, int i) { return ((scalar_ptr)(uintptr_t)p)[i]; }

// Stream reads: a tile is read once per row group, and never again (8 x 131072 tokens: 207 us through the caches, 191 past them).
typedef const __attribute__((address_space(1))) uint8_t* global_ptr;
template <typename T> __device__ __forceinline__ T stream_load(global_ptr p) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) T*)p);
}

// PT: a page holds whole tiles (its size is a multiple of kTile), else it holds whole blocks of sixteen tokens, each with a table entry
// and addresses of its own (pages of 64, whole tiles / blocks: 32 x 4096 tokens at dim 64 26.4 / 27.1 us, 8 x 4096 with eight query tokens
// at dim 128 28.9 / 29.6, else within 1%).  Caps far above any score are served by the latter only, so that the code for them is not in the way
// of the others (which it cost 3%).
template <typename QT, int D, int NRB, bool PT>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_decode_fp4_kernel(const Fp4Params p) {
  constexpr bool F16 = __is_same(QT, fp16_tag);
  constexpr int KD = D <= 128 ? 1 : 2;          // 128-deep steps of Q.K^T = 32-element blocks of a K row per lane
  constexpr int NQ = F16 ? 3 : 2;               // e4m3 rows that add up to the query row
  constexpr int NQM = D == 64 ? (NQ + 1) / 2 : NQ;  // matrix operands of them (head dim 64: two rows side by side in the depth)
  constexpr int NP = F16 || NRB == 1 ? 2 : 1;   // bf16 parts of a probability (see above)
  constexpr int DPL = D / 16;                   // head elements per lane of the PV operand
  constexpr int VW = D <= 128 ? 1 : 2;          // dwords of them per token (head dim 64: half a dword)
  constexpr int NB = kTile / 16;                // blocks of sixteen tokens in a tile
  constexpr int NS = D / 32;                    // dwords that hold the scale bytes of four tokens
  constexpr int ROW = D / 2;                    // bytes of a row of codes; its scale bytes are a sixteenth of that
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][D + 4];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];

  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = uni(threadIdx.x >> 6);
  // Row groups of one (range, kv head) read the same tiles: workgroup i runs on XCD i % 8, so they are eight apart.
  const int x = blockIdx.x & 7, y = blockIdx.x >> 3;
  const int pair = uni(x + 8 * (y / p.row_groups)), rg = uni(y % p.row_groups);
  const int part = uni(pair / p.heads_kv), kvh = uni(pair - part * p.heads_kv);
  if (part >= p.n_parts) return;

  // Units of all sequences, this range of them, and its first sequence.  lens holds the lengths of sequences lens_base + lane:
  // going on to the next sequence is a register read.
  int T = 0, n0 = 0, incl0 = 0, lens = 0, lens_base = 0;
  // (no branch over lanes: where one meets the uniform ones around it, the state behind them would be kept per lane)
  auto read_lens = [&](int base) __attribute__((always_inline)) -> int {
    const int len = len_of(p, min(base + lane, p.batch - 1));
    return base + lane < p.batch ? len : 0;
  };
  const int row0 = rg * 16 * NRB;
  int u_begin, u_end, b_first = -1, pre_first = 0;
  if (p.by_sequence) {
    lens = read_lens(part);
    lens_base = part;
    u_begin = 0;
    u_end = units_of_len(uni(__builtin_amdgcn_readlane(lens, 0)));
    b_first = part;
    if (u_end == 0) {
      for (int i = threadIdx.x; i < min(16 * NRB, p.rows - row0) * (D / 8); i += 64 * kWaves) {
        const int r = row0 + i / (D / 8), s = r / p.group, gi = r - s * p.group;
        *(u32x4*)(p.out + (((int64_t)part * p.q_len + s) * p.heads + kvh * p.group + gi) * D + 8 * (i % (D / 8))) = u32x4{0, 0, 0, 0};
      }
      return;
    }
  } else {
    for (int base = 0; base < p.batch; base += 64) {
      const int len = read_lens(base), n = units_of_len(len), incl = wave_incl_scan(n);
      if (base == 0) {
        lens = len;
        n0 = n;
        incl0 = incl;
      }
      T += __builtin_amdgcn_readlane(incl, 63);
    }
    T = uni(T);
    if (T == 0) return;
    const Ranges ranges(T, p);
    if (part >= (int)ranges.np) return;
    u_begin = uni(ranges.begin(part));
    u_end = uni(ranges.begin(part + 1));
    for (int base = 0, carry = 0; base < p.batch && b_first < 0; base += 64) {
      int n = n0, incl = incl0;
      if (base > 0) {
        lens = read_lens(base);
        lens_base = base;
        n = units_of_len(lens);
        incl = wave_incl_scan(n);
      }
      const uint64_t hit = __ballot(carry + incl > u_begin);
      if (hit) {
        const int at = uni(__ffsll((unsigned long long)hit) - 1);
        b_first = base + at;
        pre_first = carry + __builtin_amdgcn_readlane(incl - n, at);
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
  }

  // Of the two waves on a SIMD the one that was started first goes first: its workgroup is done after 93 us of 130, and the other goes on alone
  // with a unit half used.  So the second half of the workgroups go first until three quarters of their range (32 x 1024 .. 16384 tokens
  // with eight query tokens, whole call: 129 us without, 126 / 124 / 123 / 125 with 4 / 5 / 6 / 7 eighths; calls that wait for memory: 1%).
  // (That workgroups half a grid apart share a compute unit is how these grids of two per unit are dealt out, not a promise: where they do not,
  // the priority costs or gains a little time and nothing else.)
  const int first_until = !p.by_sequence && blockIdx.x >= gridDim.x / 2 ? u_begin + (int)((int64_t)(u_end - u_begin) * 3 / 4) : 0;
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  const bool causal = p.causal && p.q_len > 1, softcap = p.cap_log2e > 0.f, large_cap = p.cap_log2e > kLargeCap;
  const uint32_t q_sign = p.negate_q ? 0x80808080u : 0u;
  // byte of the lane's block in a word of V scales (head dim 64: of the first of the word's two tokens), turned right by this
  // many bits, sits in a float's exponent
  const uint32_t v_turn = (8 * (D == 64 ? c >> 3 : D == 128 ? c >> 2 : (c >> 1) & 3) + 9) & 31;
  // scale bytes of the query operands, one for each row n of its taking apart: 2^(-5n) (head dim 64: two rows side by side, in blocks 0, 1 and 2, 3)
  const uint32_t q_bytes = D == 64 ? (g < 2 ? 0x757fu : 0x707au) : 0x757a7fu;
  // what the lane reads of a block of sixteen tokens: K row c, block g (head dim 64: g % 2); V rows 4g .. 4g + 3, elements c * DPL ..
  const uint32_t k_lane = c * ROW + 16 * (D == 64 ? g & 1 : g), ks_lane = (D == 64 ? c & ~1 : c) * (ROW / 16);
  const uint32_t k_shift = D == 64 ? 16 * (c & 1) + 8 * (g & 1) : 8 * g;  // of the lane's scale byte in the word it reads
  const uint32_t v_lane = 4 * g * ROW + c * (DPL / 2), vs_lane = 4 * g * (ROW / 16);
  const uint32_t page_bytes = (uint32_t)p.heads_kv * p.page_size * ROW;  // (below 2^32: the launcher checks)
  const int64_t head_bytes = (int64_t)kvh * p.page_size * ROW;

  // One sequence of the range: units [u0, u1) of its nu; the wave's tiles are tok, tok + kUnit, .. below tok_end.
  struct Segment {
    int b, len, pre, nu, u0, u1, limit_min, tok, tok_end, last_page;
  };
  // The segment that begins at unit u, whose sequence is b0 or the first one behind it with tokens; pre: units before that.
  auto segment_at = [&](int b0, int pre, int u) __attribute__((always_inline)) -> Segment {
    Segment s;
    s.b = b0;
    while (true) {  // (u is below the number of units: there is such a sequence)
      if (s.b < lens_base || s.b - lens_base >= 64) {  // (requests run ahead of the products)
        lens_base = s.b;
        lens = read_lens(s.b);
      }
      s.len = __builtin_amdgcn_readlane(lens, s.b - lens_base);
      if (s.len > 0) break;
      s.b++;
    }
    s.last_page = (s.len - 1) / p.page_size;
    s.pre = pre;
    s.nu = units_of_len(s.len);
    s.u0 = u - pre;
    s.u1 = min(s.nu, u_end - pre);
    // tokens that the first and the last row of the group see; no row sees one past the latter
    const int r_last = min(row0 + 16 * NRB, p.rows) - 1;
    s.limit_min = causal ? s.len - p.q_len + row0 / p.group + 1 : s.len;
    s.tok = s.u0 * kUnit + wave * kTile;
    s.tok_end = min(s.u1 * kUnit, causal ? s.len - p.q_len + r_last / p.group + 1 : s.len);
    return s;
  };
  Segment cur = segment_at(uni(b_first), uni(pre_first), u_begin);

  // ---- requests: the wave's tiles of all segments as one stream, one tile ahead of the products, table entries one further ----
  // (Behind the last tile the stream goes on in the last sequence's last page: every place stays inside the pool, nothing of it is used,
  // and the number of loads in flight is the same in every step.)
  constexpr int NPG = PT ? 1 : NB;  // table entries of a tile
  const int step_lp = kUnit / p.page_size, step_off = kUnit - step_lp * p.page_size;
  int rq_b, rq_next_unit, rq_last_page;  // sequence of the tile that is requested next, first unit behind it, its last page,
  int rq_tok, rq_end, rq_lp, rq_off;     // the tile's first token, the end of the range's, and the token's logical page and offset
  const int32_t* rq_row;                 // the sequence's table row
  auto rq_enter = [&](const Segment& s) __attribute__((always_inline)) {
    rq_b = s.b;
    rq_next_unit = s.pre + s.nu;
    rq_last_page = s.last_page;
    rq_tok = s.tok;
    rq_end = s.tok_end;
    rq_lp = rq_tok / p.page_size;
    rq_off = rq_tok - rq_lp * p.page_size;
    rq_row = p.block_table + (int64_t)s.b * p.bt_row_stride;
  };
  auto rq_settle = [&]() __attribute__((always_inline)) {  // on to a segment that has a tile for this wave
    while (rq_tok >= rq_end) {
      if (rq_next_unit >= u_end) {
        rq_end = INT_MAX;
        return;
      }
      rq_enter(segment_at(rq_b + 1, rq_next_unit, rq_next_unit));
    }
  };
  int id[NPG], id_off[NPG];  // table entries of a tile and the offsets of its blocks in their pages
  auto rq_entries = [&]() __attribute__((always_inline)) {
    int lp = rq_lp, off = rq_off;
#pragma unroll
    for (int i = 0; i < NPG; i++) {
      id[i] = scalar_load(rq_row, min(lp, rq_last_page));  // (past the sequence's end: its last page again)
      id_off[i] = off;
      off += 16;
      if (off == p.page_size) {
        off = 0;
        lp++;
      }
    }
  };
  int64_t at[NPG];  // byte offset of each block of the requested tile in the codes
  auto rq_place = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NPG; i++) {
      const uint32_t page = (uint32_t)min(max(id[i], 0), p.n_pages - 1);
      at[i] = (int64_t)((uint64_t)page * page_bytes) + head_bytes + id_off[i] * ROW;
    }
  };
  auto rq_step = [&]() __attribute__((always_inline)) {
    rq_tok += kUnit;
    rq_lp += step_lp;
    rq_off += step_off;
    const bool turn = rq_off >= p.page_size;
    rq_off -= turn ? p.page_size : 0;
    rq_lp += turn ? 1 : 0;
    if (rq_tok >= rq_end) rq_settle();
    rq_entries();
  };
  // (a base kept in scalar registers: the loads add the lane's 32-bit offset themselves)
  auto base_of = [](const uint8_t* p, int64_t o) __attribute__((always_inline)) -> global_ptr {
    global_ptr at = (global_ptr)(uintptr_t)(p + o);
    asm("" : "+s"(at));
    return at;
  };
  u32x4 kr[NB][KD];
  uint32_t ksr[NB][KD], vr[NB][4][VW], vsr[NB][NS];
  auto load_k = [&]() __attribute__((always_inline)) {
    global_ptr kp, ksp;
#pragma unroll
    for (int i = 0; i < NB; i++) {
      constexpr uint32_t kStep = 16 * ROW;
      if (!PT || i == 0) {
        kp = base_of(p.k, at[PT ? 0 : i]);
        ksp = base_of(p.k_scale, at[PT ? 0 : i] >> 4);
      }
      const uint32_t o = PT ? i * kStep : 0;
#pragma unroll
      for (int kd = 0; kd < KD; kd++) {
        kr[i][kd] = stream_load<u32x4>(kp + k_lane + (o + 64 * kd));
        ksr[i][kd] = stream_load<uint32_t>(ksp + ks_lane + ((o >> 4) + 4 * kd));  // (shifted down at its use: nothing may touch it here)
      }
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
    global_ptr vp, vsp;
#pragma unroll
    for (int i = 0; i < NB; i++) {
      constexpr uint32_t kStep = 16 * ROW;
      if (!PT || i == 0) {
        vp = base_of(p.v, at[PT ? 0 : i]);
        vsp = base_of(p.v_scale, at[PT ? 0 : i] >> 4);
      }
      const uint32_t o = PT ? i * kStep : 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (D == 64) vr[i][j][0] = stream_load<uint16_t>(vp + v_lane + (o + j * ROW));
        else if constexpr (D == 128) vr[i][j][0] = stream_load<uint32_t>(vp + v_lane + (o + j * ROW));
        else {
          const u32x2 w = stream_load<u32x2>(vp + v_lane + (o + j * ROW));
          vr[i][j][0] = w[0];
          vr[i][j][1] = w[1];
        }
      }
      if constexpr (NS == 2) {
        const u32x2 w = stream_load<u32x2>(vsp + vs_lane + (o >> 4));
        vsr[i][0] = w[0];
        vsr[i][1] = w[1];
      } else {
#pragma unroll
        for (int h = 0; h < NS / 4; h++) {
          const u32x4 w = stream_load<u32x4>(vsp + vs_lane + ((o >> 4) + 16 * h));
#pragma unroll
          for (int e = 0; e < 4; e++) vsr[i][4 * h + e] = w[e];
        }
      }
    }
  };
  rq_enter(cur);
  rq_settle();
  rq_entries();
  rq_place();
  load_k();
  load_v();
  rq_step();

  // query rows of a sequence, as they are; the next sequence's are requested before this one's results are joined
  // (lanes behind the last row carry it once more; like all of this without a branch over lanes)
  u32x4 q_raw[NRB][D / 64][2];
  auto load_q = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      const int r = min(row0 + 16 * rb + c, p.rows - 1), s = r / p.group, gi = r - s * p.group;
      const uint16_t* qp = p.q + (((int64_t)b * p.q_len + s) * p.heads + kvh * p.group + gi) * D;
      // depth positions of the lane's sixteen-byte halves h: [64h + 16g, 64h + 16g + 16) of each 128-deep step
#pragma unroll
      for (int h = 0; h < D / 64; h++)
#pragma unroll
        for (int e = 0; e < 2; e++) q_raw[rb][h][e] = *(const u32x4*)(qp + 64 * h + 16 * g + 8 * e);
    }
  };
  load_q(cur.b);

  for (int seg = 0;; seg++) {
    // ---- one sequence of the range --------------------------------------------------------------------------------
    const int b = cur.b, len = cur.len, limit_min = cur.limit_min, tok_end = cur.tok_end;
    const bool whole = cur.u0 == 0 && cur.u1 == cur.nu;
    int tok = cur.tok;

    // query rows: scaled by a power of two that puts the row's largest magnitude in [128, 256), then taken apart into e4m3 rows, each 32 times
    // the remainder of the one before (8 at most; the operand's scale byte takes the factor back), so that small elements lose nothing
    u32x4 qf[NRB][KD][NQM][2];
    float q_scale[NRB];
    int limit[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      const int r = row0 + 16 * rb + c;
      constexpr int NH = D / 64;
      float f[16 * NH];
#pragma unroll
      for (int h = 0; h < NH; h++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t w[4] = {q_raw[rb][h][e][0], q_raw[rb][h][e][1], q_raw[rb][h][e][2], q_raw[rb][h][e][3]};
          Unpack<QT, 8>::run(w, f + 16 * h + 8 * e);
        }
      float am = 0.f;
#pragma unroll
      for (int e = 0; e < 16 * NH; e++) am = fmaxf(am, fabsf(f[e]));
      am = fmaxf(group_max(am), 1e-30f);
      const uint32_t be = (__float_as_uint(am) >> 23) & 0xffu;
      float inv = __uint_as_float((261u - be) << 23);  // 2^(7 - e)
      q_scale[rb] = __uint_as_float((be - 7u) << 23);
      if (be == 255u) inv = q_scale[rb] = __builtin_nanf("");  // an infinity in the row: its scores are not numbers
      q_scale[rb] *= p.score_scale;
      u32x4 parts[NH][NQ];
#pragma unroll
      for (int h = 0; h < NH; h++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
          float a[4];
#pragma unroll
          for (int e = 0; e < 4; e++) a[e] = f[16 * h + 4 * w + e] * inv;
#pragma unroll
          for (int n = 0; n < NQ; n++) {
            const uint32_t word = pack_fp8x4(a[0], a[1], a[2], a[3]);
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
            a[0] = (a[0] - lo[0]) * 32.f;
            a[1] = (a[1] - lo[1]) * 32.f;
            a[2] = (a[2] - hi[0]) * 32.f;
            a[3] = (a[3] - hi[1]) * 32.f;
            parts[h][n][w] = word ^ q_sign;
          }
        }
      if constexpr (D == 64) {
        // the depth holds the K row twice: two parts of the query side by side
#pragma unroll
        for (int n = 0; n < NQM; n++) {
          qf[rb][0][n][0] = parts[0][2 * n];
          qf[rb][0][n][1] = 2 * n + 1 < NQ ? parts[0][2 * n + 1 < NQ ? 2 * n + 1 : 0] : u32x4{0, 0, 0, 0};
        }
      } else {
#pragma unroll
        for (int kd = 0; kd < KD; kd++)
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) qf[rb][kd][n][h] = parts[2 * kd + h][n];
      }
      limit[rb] = r < p.rows ? (causal ? len - p.q_len + r / p.group + 1 : len) : 0;
    }

    f32x4 o[NRB][DPL], lsum[NRB];  // (lsum: four equal copies of the row's sum)
    float m_run[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      m_run[rb] = kNegFloor;
      lsum[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < DPL; n++) o[rb][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr uint32_t kOnes = 0x3f803f80u;  // two bf16 ones

    // scale of token 4g + j of block i for the lane's head elements: its byte turned to a float's exponent, all that the conversion
    // reads of it (255 is NaN); the bits beside it are other scales
    auto v_scale = [&](int i, int j) __attribute__((always_inline)) -> uint32_t {
      const uint32_t w = D == 64 ? vsr[i][j >> 1] : D == 128 ? vsr[i][j] : c & 8 ? vsr[i][NS > 4 ? 2 * j + 1 : 0] : vsr[i][NS > 4 ? 2 * j : 0];
      return __builtin_amdgcn_alignbit(w, w, D == 64 && (j & 1) ? (v_turn + 16) & 31 : v_turn);
    };
    // A operands of the PV product for two head elements at a time: word_of(j, w) is the pair w of token j (0..7) as two bf16
    auto value_operands = [&](auto word_of, auto use) __attribute__((always_inline)) {
#pragma unroll
      for (int w = 0; w < DPL / 2; w++) {
        uint32_t e8[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e8[j] = word_of(j, w);
        u32x4 lo, hi;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          lo[k] = __builtin_amdgcn_perm(e8[2 * k + 1], e8[2 * k], 0x05040100u);
          hi[k] = __builtin_amdgcn_perm(e8[2 * k + 1], e8[2 * k], 0x07060302u);
        }
        use(2 * w, lo);
        use(2 * w + 1, hi);
      }
    };

    // One tile.  The registers of K are free once its products are issued, those of V once it is widened: the next tile is
    // requested there, so a tile's reads have the rest of the step and the head of the next one to arrive.
    auto step = [&](auto masked_tag) __attribute__((always_inline)) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      if (cur.pre + (int)((uint32_t)tok / kUnit) < first_until) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      // (products into the same accumulator are kept NRB * NB products apart: back to back each would wait for the one before)
      f32x4 s[NRB][NB];
#pragma unroll
      for (int kd = 0; kd < KD; kd++)
#pragma unroll
        for (int n = 0; n < NQM; n++) {
#pragma unroll
          for (int i = 0; i < NB; i++)
#pragma unroll
            for (int rb = 0; rb < NRB; rb++) {
              const f32x4 sum = kd + n == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[rb][i];
              const u32x4 b0 = qf[rb][kd][n][0], b1 = qf[rb][kd][n][1];
              const uint32_t k_byte = ksr[i][kd] >> k_shift;
              s[rb][i] = n == 0 ? mma_codes<0>(kr[i][kd], b0, b1, sum, k_byte, q_bytes)
                         : n == 1 ? mma_codes<1>(kr[i][kd], b0, b1, sum, k_byte, q_bytes) : mma_codes<2>(kr[i][kd], b0, b1, sum, k_byte, q_bytes);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      rq_place();
      load_k();
      __builtin_amdgcn_sched_barrier(0);
      uint32_t pw[NRB][NB / 2][NP][4], seen_bits[NRB][NB / 2];
      float slope[NRB], offset[NRB], top[NRB];  // logit = slope * s + offset, slope >= 0 (the sign of the softmax scale is in the query)
      bool grown = false;
      bool capped = false;
      if constexpr (MASKED && !PT) {
        if (large_cap) {
          // the form below loses a large cap's 24th bit, which is too much of a score far below it: s becomes tanh(x), by its series for small
          // x (x^9 / 46 left out: 4e-7 of it)
          capped = true;
#pragma unroll
          for (int rb = 0; rb < NRB; rb++)
#pragma unroll
            for (int e = 0; e < 4 * NB; e++) {
              const float a = s[rb][e >> 2][e & 3] * q_scale[rb], x = a * (0.5f / kLog2e), xx = x * x;
              const float series = __builtin_fmaf(xx, __builtin_fmaf(xx, __builtin_fmaf(xx, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f) * x;
              const float whole = __builtin_fmaf(2.f, __builtin_amdgcn_rcpf(-1.0f - fast_exp2(a)), 1.f);
              s[rb][e >> 2][e & 3] = fabsf(x) < 0.25f ? series : whole;
            }
        }
      }
      if (softcap && !capped) {
        // cap * tanh(x) = cap - 2 cap / (exp(2x) + 1): s becomes -1 / (exp(2x) + 1)
#pragma unroll
        for (int rb = 0; rb < NRB; rb++)
#pragma unroll
          for (int e = 0; e < 4 * NB; e++) s[rb][e >> 2][e & 3] = fast_exp2(s[rb][e >> 2][e & 3] * q_scale[rb]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rb = 0; rb < NRB; rb++)
#pragma unroll
          for (int e = 0; e < 4 * NB; e++) s[rb][e >> 2][e & 3] = __builtin_amdgcn_rcpf(-1.0f - s[rb][e >> 2][e & 3]);
      }
#pragma unroll
      for (int rb = 0; rb < NRB; rb++) {
        slope[rb] = capped ? p.cap_log2e : softcap ? 2.f * p.cap_log2e : q_scale[rb];
        offset[rb] = softcap && !capped ? p.cap_log2e : 0.f;
        if constexpr (MASKED) {
#pragma unroll
          for (int h = 0; h < NB / 2; h++) seen_bits[rb][h] = 0;
#pragma unroll
          for (int e = 0; e < 4 * NB; e++) {
            const bool seen = tok + 16 * (e >> 2) + 4 * g + (e & 3) < limit[rb];
            s[rb][e >> 2][e & 3] = seen ? __builtin_fmaf(s[rb][e >> 2][e & 3], slope[rb], offset[rb]) : -INFINITY;
            seen_bits[rb][e >> 3] |= seen ? 1u << (e & 7) : 0u;
          }
          slope[rb] = 1.f;
          offset[rb] = 0.f;
        }
        // (med3 with +inf is a maximum that the compiler schedules behind the matrix results, without quieting its operands first)
        top[rb] = __builtin_amdgcn_fmed3f(s[rb][0][0], s[rb][0][1], INFINITY);
#pragma unroll
        for (int e = 2; e < 4 * NB; e++) top[rb] = __builtin_amdgcn_fmed3f(top[rb], s[rb][e >> 2][e & 3], INFINITY);
        top[rb] = __builtin_fmaf(group_max(top[rb]), slope[rb], offset[rb]);
        grown |= top[rb] > m_run[rb] + kRescaleGap4;
      }
      if (__ballot(grown)) {  // (the first tile with a visible token always comes here)
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) {
          const float m_new = top[rb] > m_run[rb] + kRescaleGap4 ? top[rb] : m_run[rb];
          const float shrink = fast_exp2(m_run[rb] - m_new);
          m_run[rb] = m_new;
          lsum[rb] *= shrink;
#pragma unroll
          for (int n = 0; n < DPL; n++) o[rb][n] *= shrink;
        }
      }
#pragma unroll
      for (int rb = 0; rb < NRB; rb++) {
        const float shift = offset[rb] - m_run[rb];
#pragma unroll
        for (int h = 0; h < NB / 2; h++) {
          float pr[8];
#pragma unroll
          for (int e = 0; e < 8; e++) pr[e] = fast_exp2(__builtin_fmaf(s[rb][2 * h + (e >> 2)][e & 3], slope[rb], shift));
#pragma unroll
          for (int e = 0; e < 4; e++) {
            pw[rb][h][0][e] = pack_bf16(pr[2 * e], pr[2 * e + 1]);
            if constexpr (NP == 2)
              pw[rb][h][1][e] = pack_bf16(pr[2 * e] - __uint_as_float(pw[rb][h][0][e] << 16), pr[2 * e + 1] - __uint_as_float(pw[rb][h][0][e] & 0xffff0000u));
          }
          // the row's sum of the probabilities as rounded, on the matrix unit: every row of ones . P^T
#pragma unroll
          for (int q = 0; q < NP; q++)
            lsum[rb] = mma_bf16(u32x4{kOnes, kOnes, kOnes, kOnes}, u32x4{pw[rb][h][q][0], pw[rb][h][q][1], pw[rb][h][q][2], pw[rb][h][q][3]}, lsum[rb]);
        }
      }
#pragma unroll
      for (int h = 0; h < NB / 2; h++) {
        float vsc[8];
        uint32_t bad = 0;       // tokens (bits) whose block is NaN
        bool infinite = false;  // a block's larger codes are infinities (2^128 and more: scale bytes 253 and 254)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const uint32_t word = v_scale(2 * h + (j >> 2), j & 3);
          vsc[j] = __uint_as_float(word);
          if constexpr (MASKED) {
            // a NaN block stays out of the product, where a weight of zero would not keep it from the rows that do not see it
            const bool is_nan = (word & 0x7f800000u) == 0x7f800000u;
            bad |= is_nan ? 1u << j : 0u;
            infinite |= !is_nan && (word & 0x7f800000u) >= 253u << 23;
            vsc[j] = is_nan ? 0.f : vsc[j];
          }
        }
        // Infinities would reach them likewise: such a tile enters at a sixteenth, as the numbers that its codes are.  (A scale below 2^-123 stays
        // what it is or loses less than a sixteenth leaves of it: 2^-120 beside values of 2^126.)
        bool sixteenth = false;
        if constexpr (MASKED) {
          sixteenth = __ballot(infinite) != 0;
          if (sixteenth) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const uint32_t word = __float_as_uint(vsc[j]);
              vsc[j] = __uint_as_float(word - min(word & 0x7f800000u, 4u << 23));
            }
#pragma unroll
            for (int rb = 0; rb < NRB; rb++)
#pragma unroll
              for (int n = 0; n < DPL; n++) o[rb][n] *= 0.0625f;
          }
        }
        value_operands(
            [&](int j, int w) __attribute__((always_inline)) -> uint32_t {
              const uint32_t word = vr[2 * h + (j >> 2)][j & 3][w >> 2];
              switch (w & 3) {
                case 0: return widen2<0>(word, vsc[j]);
                case 1: return widen2<1>(word, vsc[j]);
                case 2: return widen2<2>(word, vsc[j]);
                default: return widen2<3>(word, vsc[j]);
              }
            },
            [&](int n, u32x4 a) __attribute__((always_inline)) {
#pragma unroll
              for (int rb = 0; rb < NRB; rb++)
#pragma unroll
                for (int q = 0; q < NP; q++)
                  o[rb][n] = mma_bf16(a, u32x4{pw[rb][h][q][0], pw[rb][h][q][1], pw[rb][h][q][2], pw[rb][h][q][3]}, o[rb][n]);
            });
        if constexpr (MASKED) {
          if (sixteenth) {
#pragma unroll
            for (int rb = 0; rb < NRB; rb++)
#pragma unroll
              for (int n = 0; n < DPL; n++) o[rb][n] *= 16.f;
          }
          if (__ballot(bad != 0u)) {
            // rows that see a token with a NaN block get NaN there: count such tokens with the same product, 1 for every
            // NaN block against 1 for every visible token
#pragma unroll
            for (int rb = 0; rb < NRB; rb++) {
              u32x4 vis;
#pragma unroll
              for (int k = 0; k < 4; k++)
                vis[k] = ((seen_bits[rb][h] >> (2 * k)) & 1u ? 0x3f80u : 0u) | ((seen_bits[rb][h] >> (2 * k + 1)) & 1u ? 0x3f800000u : 0u);
              value_operands([&](int j, int) __attribute__((always_inline)) -> uint32_t { return (bad >> j) & 1u ? kOnes : 0u; },
                             [&](int n, u32x4 a) __attribute__((always_inline)) {
                               const f32x4 count = mma_bf16(a, vis, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                               for (int i = 0; i < 4; i++) o[rb][n][i] = count[i] > 0.f ? __builtin_nanf("") : o[rb][n][i];
                             });
            }
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_v();
      __builtin_amdgcn_sched_barrier(0);
      rq_step();
    };
    if (PT || !large_cap)
      for (; tok + kTile <= limit_min && tok < tok_end; tok += kUnit) step(std::false_type{});
    for (; tok < tok_end; tok += kUnit) step(std::true_type{});

    const int u_next = cur.pre + cur.nu;
    const bool last = u_next >= u_end;
    Segment next = cur;
    if (!last) {
      next = segment_at(b + 1, u_next, u_next);
      load_q(next.b);
    }

    // ---- the four waves' results of each block of rows meet in LDS ---------------------------------------------------
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      if (g == 0) {
        s_m[wave][c] = m_run[rb];
        s_l[wave][c] = lsum[rb][0];
      }
      // lane (c, g) holds head elements (D / 4) * g + DPL * i + n of row c
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int n = 0; n < DPL; n += 4)
          *(f32x4*)&s_o[wave][c][(D / 4) * g + DPL * i + n] = f32x4{o[rb][n][i], o[rb][n + 1][i], o[rb][n + 2][i], o[rb][n + 3][i]};
      __syncthreads();
      {
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * DPL, r = row0 + 16 * rb + row;
        if (r < p.rows) {
          float M = s_m[0][row];
#pragma unroll
          for (int w = 1; w < kWaves; w++) M = fmaxf(M, s_m[w][row]);
          float L = 0.f, acc[DPL];
#pragma unroll
          for (int n = 0; n < DPL; n++) acc[n] = 0.f;
#pragma unroll
          for (int w = 0; w < kWaves; w++) {
            const float f = fast_exp2(s_m[w][row] - M);
            L += s_l[w][row] * f;
#pragma unroll
            for (int n = 0; n < DPL; n += 4) {
              const f32x4 a = *(const f32x4*)&s_o[w][row][d0 + n];
#pragma unroll
              for (int e = 0; e < 4; e++) acc[n + e] += a[e] * f;
            }
          }
          const float inv = L == 0.f ? 0.f : 1.0f / L;  // (a row that sees nothing: zeros)
          if (whole) {
            const int s = r / p.group, gi = r - s * p.group;
            uint32_t* dst = (uint32_t*)(p.out + (((int64_t)b * p.q_len + s) * p.heads + kvh * p.group + gi) * D + d0);
#pragma unroll
            for (int n = 0; n < DPL; n += 2) dst[n >> 1] = pack16<QT>(acc[n] * inv, acc[n + 1] * inv);
          } else {
            const int64_t slot = (int64_t)(2 * part + (seg > 0 ? 1 : 0)) * rows_all + (int64_t)kvh * p.rows + r;
            f32x4* dst = (f32x4*)(p.part_o + slot * D + d0);
#pragma unroll
            for (int n = 0; n < DPL; n += 4) dst[n >> 2] = f32x4{acc[n] * inv, acc[n + 1] * inv, acc[n + 2] * inv, acc[n + 3] * inv};
            if (d0 == 0) p.part_lse[slot] = L == 0.f ? -INFINITY : M + log2f(L);
          }
        }
      }
      __syncthreads();
    }
    if (last) return;
    cur = next;
  }
}

// Rows of a sequence that several ranges share: weights exp2(lse - max) over the ranges' normalised rows.  A lane has four head elements, so the 64 / (D / 4)
// lane groups of a wave take different ranges.  All rows' first loads are in flight before the first weight is known.  Sequences
// without tokens get zeros here.
// SHARED: the four waves of a workgroup take a quarter of a row's ranges each and join in LDS.
// Bound: latency (a few MB in 3 to 7 us).
template <int D> struct MergeShared {
  float o[kWaves][D], m[kWaves], w[kWaves];
};
template <typename QT, int D, int R, int PRE, bool SHARED>
__device__ __forceinline__ void merge_rows(const Fp4Params& p, int b, int64_t row0, int64_t rows_all, int first, int n, bool second, MergeShared<D>* sh) {
  constexpr int LPR = D / 4, GROUPS = 64 / LPR;  // lanes per row, ranges side by side; PRE: loads of a row in flight
  static_assert(!SHARED || R == 1, "a shared row");
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), grp = lane / LPR, d0 = 4 * (lane % LPR);
  const int share = SHARED ? (n + kWaves - 1) / kWaves : n, begin = SHARED ? min(wave * share, n) : 0, end = SHARED ? min(begin + share, n) : n;
  auto slot_of = [&](int i, int64_t row) __attribute__((always_inline)) -> int64_t {
    const int k = min(i, n - 1);
    return (int64_t)(2 * (first + k) + (k == 0 && second ? 1 : 0)) * rows_all + row;
  };
  f32x4 acc[R];
  float M[R], W[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    M[r] = -INFINITY;
    W[r] = 0.f;
  }
  for (int base = begin; base < end; base += PRE * GROUPS) {
    f32x4 x[R][PRE];
    float lse[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int64_t row = row0 + r < rows_all ? row0 + r : rows_all - 1;
#pragma unroll
      for (int i = 0; i < PRE; i++) x[r][i] = *(const f32x4*)(p.part_o + slot_of(base + i * GROUPS + grp, row) * D + d0);
      lse[r] = lane < PRE * GROUPS && base + lane < end ? p.part_lse[slot_of(base + lane, row)] : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      float top = lse[r];
#pragma unroll
      for (int m = 1; m < PRE * GROUPS; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      top = fmaxf(M[r], __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, top), 0)));
      const float ref = top == -INFINITY ? 0.f : top;
      const float shrink = fast_exp2(M[r] - ref), wl = fast_exp2(lse[r] - ref);  // (NaN stays NaN)
      M[r] = top;
      W[r] *= shrink;
      acc[r] *= shrink;
#pragma unroll
      for (int i = 0; i < PRE; i++) {
        const float w = __shfl(wl, i * GROUPS + grp, 64);
        W[r] += w;
        if (w != 0.f) acc[r] += w * x[r][i];  // (a place past the last has no weight)
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
#pragma unroll
    for (int m = LPR; m < 64; m <<= 1) {
      W[r] += __shfl_xor(W[r], m, 64);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[r][e] += __shfl_xor(acc[r][e], m, 64);
    }
    const int64_t row = row0 + r;
    if constexpr (SHARED) {
      if (grp == 0) *(f32x4*)&sh->o[wave][d0] = acc[0];
      if (lane == 0) {
        sh->m[wave] = M[0];
        sh->w[wave] = W[0];
      }
      __syncthreads();
      if (wave > 0) return;
      float top = M[0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) top = fmaxf(top, sh->m[w]);
      const float ref = top == -INFINITY ? 0.f : top;
      acc[0] = f32x4{0.f, 0.f, 0.f, 0.f};
      W[0] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float f = fast_exp2(sh->m[w] - ref), sum = sh->w[w];
        if (f != 0.f || sum != sum) {  // (else no range, or none with a weight; ranges of NaN have no maximum)
          W[0] += f * sum;
          acc[0] += f * *(const f32x4*)&sh->o[w][d0];
        }
      }
    }
    if (grp > 0 || row >= rows_all) continue;
    const float inv = W[r] == 0.f ? 0.f : 1.0f / W[r];
    const int kvh = (int)(row / p.rows), qr = (int)(row - (int64_t)kvh * p.rows), s = qr / p.group, gi = qr - s * p.group;
    *(u32x2*)(p.out + (((int64_t)b * p.q_len + s) * p.heads + kvh * p.group + gi) * D + d0) =
        u32x2{pack16<QT>(acc[r][0] * inv, acc[r][1] * inv), pack16<QT>(acc[r][2] * inv, acc[r][3] * inv)};
  }
}

// R rows of a wave; R = 0: a row of a workgroup.
template <typename QT, int D, int R>
__global__ __launch_bounds__(64 * kWaves) void paged_decode_fp4_merge_kernel(const Fp4Params p) {
  __shared__ __attribute__((aligned(16))) MergeShared<D> sh[1];
  const int b = blockIdx.y;
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  const int64_t row0 = R == 0 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * kWaves + uni(threadIdx.x >> 6)) * R;
  int pre;
  const int T = total_units(p, b, &pre);
  const int nu = uni(units_of_len(len_of(p, b)));
  int first = 0, last = -1;
  bool second = false;
  if (nu > 0) {
    const Ranges ranges(T, p);
    first = uni(ranges.owner(pre));
    last = uni(ranges.owner(pre + nu - 1));
    if (first == last) return;  // written by the range that holds it
    second = ranges.begin(first) != pre;
  }
  const int n = last - first + 1;
  constexpr int GROUPS = 256 / D;
  if constexpr (R == 0) {
    if (n <= 2 * GROUPS * kWaves) merge_rows<QT, D, 1, 2, true>(p, b, row0, rows_all, first, n, second, sh);
    else merge_rows<QT, D, 1, 8, true>(p, b, row0, rows_all, first, n, second, sh);
  } else {
    if (row0 >= rows_all) return;
    if (n <= 2 * GROUPS) {
      merge_rows<QT, D, R, 2, false>(p, b, row0, rows_all, first, n, second, nullptr);
    } else {
      for (int r = 0; r < R && row0 + r < rows_all; r++) merge_rows<QT, D, 1, 8, false>(p, b, row0 + r, rows_all, first, n, second, nullptr);
    }
  }
}

constexpr int kMaxParts4 = 4096;
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Blocks of sixteen query rows per wave, for calls with much to read (two at head dim 256 do not fit the register file).
int row_blocks(int rows, int dim) { return rows <= 16 || dim == 256 ? 1 : 2; }
int row_groups_of(int rows, int blocks) { return (rows + 16 * blocks - 1) / (16 * blocks); }

template <typename QT, int D, int NRB>
const char* launch_fp4(const Fp4Params& p, hipStream_t s) {
  const int64_t pairs = (int64_t)p.n_parts * p.heads_kv;
  const int64_t grid = 8 * (int64_t)p.row_groups * ((pairs + 7) / 8);
  if (grid > INT_MAX) return "too many workgroups";
  if (p.page_size % kTile == 0 && p.cap_log2e <= kLargeCap)
    hipLaunchKernelGGL((paged_decode_fp4_kernel<QT, D, NRB, true>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, p);
  else
    hipLaunchKernelGGL((paged_decode_fp4_kernel<QT, D, NRB, false>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hipGetErrorString(e);
  if (p.by_sequence) return nullptr;
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  // Few rows have many ranges each: a workgroup per row; many rows are one round of waves with four rows each.  Whole call, wave per row / workgroup
  // per row: 64 rows of 16384 tokens 14.3 / 11.9 us, 256 rows 19.3 / 19.3, 512 rows 22.7 / 24.0; one row / four rows of a wave: 512 rows 31.3 / 35.2,
  // 4096 rows 52.1 / 52.8, 8192 rows 98.5 / 97.7, 32768 rows 117.7 / 111.5.
  if (rows_all * p.batch <= 256)
    hipLaunchKernelGGL((paged_decode_fp4_merge_kernel<QT, D, 0>), dim3((unsigned)rows_all, p.batch), dim3(256), 0, s, p);
  else if (rows_all * p.batch < 8192)
    hipLaunchKernelGGL((paged_decode_fp4_merge_kernel<QT, D, 1>), dim3((unsigned)((rows_all + 3) / 4), p.batch), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((paged_decode_fp4_merge_kernel<QT, D, 4>), dim3((unsigned)((rows_all + 15) / 16), p.batch), dim3(256), 0, s, p);
  e = hipGetLastError();
  return e == hipSuccess ? nullptr : hipGetErrorString(e);
}

template <typename QT>
const char* launch_fp4_dim(const Fp4Params& p, int dim, int blocks, hipStream_t s) {
  const bool one = blocks == 1;
  if (dim == 64) return one ? launch_fp4<QT, 64, 1>(p, s) : launch_fp4<QT, 64, 2>(p, s);
  if (dim == 128) return one ? launch_fp4<QT, 128, 1>(p, s) : launch_fp4<QT, 128, 2>(p, s);
  return launch_fp4<QT, 256, 1>(p, s);
}

}  // namespace

// Ranges of the token stream: two workgroups (eight waves) per compute unit, over all (kv head, row group) pairs (8 x 131072 tokens: two 191 us,
// three 218).
int fp4_num_parts(int heads_kv, int rows, int dim, int compute_units) {
  const int64_t parts = 2 * (int64_t)compute_units / ((int64_t)heads_kv * row_groups_of(rows, row_blocks(rows, dim)));
  return parts < 1 ? 1 : parts > kMaxParts4 ? kMaxParts4 : (int)parts;
}

// [part_o: 2 * n_parts slots x heads_kv * rows x dim fp32][part_lse: 2 * n_parts x heads_kv * rows fp32]
size_t fp4_workspace_bytes(int n_parts, int heads_kv, int rows, int dim) {
  const size_t slots = (size_t)2 * n_parts * heads_kv * rows;
  return align256(slots * dim * sizeof(float)) + align256(slots * sizeof(float));
}

// Units of the token stream that a call can have at most (the kernels count them in 32 bits).
int64_t fp4_max_units(int64_t batch, int64_t max_len) { return batch * ((max_len + kUnit - 1) / kUnit); }

const char* launch_decode_fp4(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, const int32_t* seqlens,
                              const int32_t* block_table, int64_t bt_row_stride, int max_len, void* out, void* workspace, int batch,
                              int q_len, int heads, int heads_kv, int dim, int page_size, int64_t n_pages, int q_dtype, float sm_scale, float softcap, int causal,
                              int n_parts, hipStream_t s) {
  Fp4Params p;
  p.q = (const uint16_t*)q;
  p.k = (const uint8_t*)k;
  p.v = (const uint8_t*)v;
  p.k_scale = (const uint8_t*)k_scale;
  p.v_scale = (const uint8_t*)v_scale;
  p.seqlens = seqlens;
  p.block_table = block_table;
  p.bt_row_stride = bt_row_stride;
  p.out = (uint16_t*)out;
  p.batch = batch;
  p.q_len = q_len;
  p.heads = heads;
  p.heads_kv = heads_kv;
  p.page_size = page_size;
  p.group = heads / heads_kv;
  p.rows = q_len * p.group;
  // What a range adds to the merge grows with the rows.  2 x 3000 tokens of 8 rows on 8 kv heads, ranges of 1 / 2 / 4 units: 10.7 / 9.6 /
  // 10.4 us, 1 x 4096 9.4 / 9.3 / 10.3; 4 x 4096 of 64 rows on 4: 20.2 / 20.8 / 17.7, 1 x 8192 of 64 rows on 8: 21.4 / 21.3 / 16.6.
  p.range_units = p.rows < 32 ? 2 : 4;
  p.max_len = max_len < INT_MAX - kUnit ? max_len : INT_MAX - kUnit;
  p.causal = causal;
  p.n_pages = (int)n_pages;
  // Two row blocks share what a wave does for K and V; one makes twice the workgroups, which calls with little to read need more.  64 rows on 8
  // kv heads, one / two blocks: 1 x 4096 tokens 11.6 / 14.3 us, 4 x 3000 16.3 / 20.9, 4 x 8192 26.0 / 28.0, 4 x 16384 40.7 / 39.4, 32 x 16384
  // 290 / 192; 24 rows on 4 kv heads: 4 x 4096 13.5 / 13.8, 32 x 4096 29.6 / 28.5.
  const int most_blocks = row_blocks(p.rows, dim);
  const int blocks = fp4_max_units(batch, p.max_len) * heads_kv <= 2048 ? 1 : most_blocks;
  p.row_groups = row_groups_of(p.rows, blocks);
  const int fewest_groups = row_groups_of(p.rows, most_blocks);
  if (p.row_groups > fewest_groups) n_parts = n_parts * fewest_groups / p.row_groups > 1 ? n_parts * fewest_groups / p.row_groups : 1;
  p.n_parts = n_parts;
  const size_t slots = (size_t)2 * n_parts * heads_kv * p.rows;
  // Tables of few tokens: a workgroup per (sequence, kv head, row group) and no merge.  64 query heads on 8, dim 128, ranges / whole: 1 x 384
  // tokens 8.2 / 5.7 us, 1 x 1024 8.6 / 8.3, 1 x 2048 8.9 / 12.4; 32 x 2048 19.3 / 16.6, 32 x 4096 30.1 / 29.9; 128 of 1 .. 512 24 / 15,
  // 128 of 1 .. 4096 62 / 68: up to eight units whatever the batch is, up to sixteen where it has work for half of the ranges' workgroups.
  p.by_sequence = p.max_len <= (2 * (int64_t)batch >= n_parts ? 16 : 8) * kUnit;
  if (p.by_sequence) p.n_parts = batch;
  p.part_o = (float*)workspace;
  p.part_lse = (float*)((char*)workspace + align256(slots * dim * sizeof(float)));
  // the kernel takes maxima before it scales: the sign of the scale goes into the query
  p.negate_q = sm_scale < 0.f;
  sm_scale = fabsf(sm_scale);
  p.score_scale = softcap > 0.f ? 2.f * kLog2e * (sm_scale / softcap) : sm_scale * kLog2e;
  p.cap_log2e = softcap * kLog2e;
  return q_dtype == MI355_DT_BF16 ? launch_fp4_dim<bf16_tag>(p, dim, blocks, s) : launch_fp4_dim<fp16_tag>(p, dim, blocks, s);
}

}  // namespace mi355
