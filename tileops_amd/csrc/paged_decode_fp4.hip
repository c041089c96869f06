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
//    the others leave normalised fp32 rows with log-sum-exps for the merge kernel.
//  * Q.K^T: v_mfma_scale_f32_16x16x128_f8f6f4 with the K codes as they lie in memory -- lane (c, g) supplies block g of token
//    c, sixteen bytes, and its scale byte -- against the query row as a sum of two (bf16: exact) or three (fp16: exact) e4m3 rows.
//    Tokens sit on the M axis, so every softmax quantity of a query row is local to a lane column.
//  * PV: O^T += V^T.P^T on v_mfma_f32_16x16x32_bf16.  Lane (c, g) loads the head elements [c * D/16, (c + 1) * D/16) of its eight
//    tokens -- those whose probabilities it holds already -- widens them with their scale (v_cvt_scalef32_pk_bf16_fp4) and pairs the
//    tokens with byte permutes: V needs no LDS, P does not move.
//  * K, V and scales go from memory to registers a tile ahead of their use.
#include <climits>

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

struct Fp4Params {
  const uint16_t* q;
  const uint8_t *k, *v, *k_scale, *v_scale;
  const int32_t *seqlens, *block_table;
  int64_t bt_row_stride;
  uint16_t* out;
  float *part_o, *part_lse;
  int batch, q_len, heads, heads_kv, page_size, group, rows, row_groups, n_parts, max_len, causal;
  int n_pages;
  float score_scale, cap_log2e, inv_cap_scale;
};

__device__ __forceinline__ int len_of(const Fp4Params& p, int b) { return min(max(p.seqlens[b], 0), p.max_len); }
__device__ __forceinline__ int units_of_len(int len) { return (int)(((uint32_t)len + kUnit - 1) / kUnit); }

// Range bounds floor(p * T / NP) = p * (T / NP) + floor(p * (T % NP) / NP); NP <= 4096 keeps the second product below 2^24.
struct Ranges {
  uint32_t np, tq, tr;
  __device__ __forceinline__ Ranges(int t, int n) : np(n), tq((uint32_t)t / (uint32_t)n), tr((uint32_t)t % (uint32_t)n) {}
  __device__ __forceinline__ int begin(int p) const { return (int)((uint32_t)p * tq + ((uint32_t)p * tr) / np); }
  // the last range that begins at or before unit u
  __device__ __forceinline__ int owner(int u) const {
    const uint32_t t = tq * np + tr;
    int p = (int)min((uint64_t)(np - 1), (uint64_t)u * np / t);
    while (p + 1 < (int)np && begin(p + 1) <= u) ++p;
    return p;
  }
};

// Units of all sequences, and of those before sequence `b` if it is not negative (whole wave).
__device__ __forceinline__ int total_units(const Fp4Params& p, int b, int* before) {
  const int lane = threadIdx.x & 63;
  int sum = 0, pre = 0;
  for (int base = 0; base < p.batch; base += 64) {
    const int i = base + lane, n = i < p.batch ? units_of_len(len_of(p, i)) : 0;
    sum += n;
    pre += i < b ? n : 0;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    sum += __shfl_xor(sum, m, 64);
    pre += __shfl_xor(pre, m, 64);
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

// What a lane holds of one tile: K blocks (16 bytes each) with scale bytes, V dwords and scale words of its eight tokens.
template <int D> struct TileRegs {
  static constexpr int KB = D <= 128 ? 1 : 2;   // 32-element blocks of a K row per lane
  static constexpr int VW = D <= 128 ? 1 : 2;   // dwords of a V row per lane (head dim 64: half a dword)
  static constexpr int SW = D / 64;             // dwords that hold the V scales of two (64), one (128) or half a (256) token
  u32x4 k[2][KB];
  uint32_t ks[2][KB];
  uint32_t v[8][VW];
  uint32_t vs[2][4 * SW / 2];  // four tokens of D / 32 bytes
};

template <typename QT, int D, int NRB, bool SOFTCAP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_decode_fp4_kernel(const Fp4Params p) {
  constexpr bool F16 = __is_same(QT, fp16_tag);
  constexpr int KD = D <= 128 ? 1 : 2;          // 128-deep steps of Q.K^T
  constexpr int NQ = F16 ? 3 : 2;               // e4m3 rows that add up to the query row
  constexpr int NQM = D == 64 ? (NQ + 1) / 2 : NQ;  // matrix operands of them (head dim 64: two rows side by side in the depth)
  constexpr int NP = F16 ? 2 : 1;               // bf16 parts of a probability
  constexpr int DPL = D / 16;                   // head elements per lane of the PV operand
  using Regs = TileRegs<D>;
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][D + 4];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];

  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = uni(threadIdx.x >> 6);
  // Row groups of one (range, kv head) read the same tiles: workgroup i runs on XCD i % 8, so they are eight apart.
  const int x = blockIdx.x & 7, y = blockIdx.x >> 3;
  const int pair = uni(x + 8 * (y / p.row_groups)), rg = uni(y % p.row_groups);
  const int part = uni(pair / p.heads_kv), kvh = uni(pair - part * p.heads_kv);
  if (part >= p.n_parts) return;

  int unused;
  const int T = total_units(p, -1, &unused);
  if (T == 0) return;
  const Ranges ranges(T, p.n_parts);
  int u = uni(ranges.begin(part));
  const int u_end = uni(ranges.begin(part + 1));
  if (u >= u_end) return;

  // first sequence of the range
  int b = -1, pre = 0;
  for (int base = 0, carry = 0; base < p.batch && b < 0; base += 64) {
    const int i = base + lane, n = i < p.batch ? units_of_len(len_of(p, i)) : 0;
    const int incl = wave_incl_scan(n);
    const uint64_t hit = __ballot(carry + incl > u);
    if (hit) {
      const int at = uni(__ffsll((unsigned long long)hit) - 1);
      b = base + at;
      pre = carry + __builtin_amdgcn_readlane(incl - n, at);
    }
    carry += __builtin_amdgcn_readlane(incl, 63);
  }
  b = uni(b);
  pre = uni(pre);

  const int row0 = rg * 16 * NRB;
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  const uint32_t page_rows = (uint32_t)p.page_size;
  const bool causal = p.causal && p.q_len > 1;
  const uint32_t v_shift = 8 * (D == 64 ? 0 : D == 128 ? c >> 2 : (c >> 1) & 3);

  for (int seg = 0; u < u_end; seg++) {
    // ---- one sequence of the range --------------------------------------------------------------------------------
    int len = uni(len_of(p, b));
    while (len == 0) len = uni(len_of(p, ++b));  // (u < T: a sequence with tokens follows)
    const int nu = units_of_len(len);
    const int seg_u0 = u - pre, seg_u1 = min(nu, u_end - pre);  // units of the sequence
    const bool whole = seg_u0 == 0 && seg_u1 == nu;

    // query rows: scaled by a power of two that puts the row's largest magnitude in [128, 256), then taken apart into e4m3 rows
    u32x4 qf[NRB][KD][NQM][2];
    float q_scale[NRB];
    int limit[NRB], limit_min = INT_MAX, limit_max = 0;
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      const int r = row0 + 16 * rb + c;
      const bool valid = r < p.rows;
      const int s = valid ? r / p.group : 0, gi = valid ? r - s * p.group : 0;
      const uint16_t* qp = p.q + (((int64_t)b * p.q_len + s) * p.heads + kvh * p.group + gi) * D;
      // depth positions of the lane's sixteen-byte halves h: [64h + 16g, 64h + 16g + 16) of each 128-deep step
      constexpr int NH = D / 64;
      float f[16 * NH];
#pragma unroll
      for (int h = 0; h < NH; h++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          u32x4 raw = {0, 0, 0, 0};
          if (valid) raw = *(const u32x4*)(qp + 64 * h + 16 * g + 8 * e);
          const uint32_t w[4] = {raw[0], raw[1], raw[2], raw[3]};
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
            a[0] -= lo[0];
            a[1] -= lo[1];
            a[2] -= hi[0];
            a[3] -= hi[1];
            parts[h][n][w] = word;
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
      limit[rb] = valid ? (causal ? len - p.q_len + s + 1 : len) : 0;
    }
    {
      // tokens that the first and the last row of the group see (uniform)
      const int r_last = min(row0 + 16 * NRB, p.rows) - 1;
      limit_min = causal ? len - p.q_len + row0 / p.group + 1 : len;
      limit_max = causal ? len - p.q_len + r_last / p.group + 1 : len;
      limit_min = uni(limit_min);
      limit_max = uni(limit_max);
    }

    f32x4 o[NRB][DPL];
    float m_run[NRB], l_run[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      m_run[rb] = kNegFloor;
      l_run[rb] = 0.f;
#pragma unroll
      for (int n = 0; n < DPL; n++) o[rb][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the wave's tiles -------------------------------------------------------------------------------------------
    const int tok_end = min(seg_u1 * kUnit, limit_max);  // tokens past it no row of the group sees
    int tok = seg_u0 * kUnit + wave * kTile;
    const int32_t* bt_row = p.block_table + (int64_t)b * p.bt_row_stride;
    const int last_page = (len - 1) / p.page_size;
    // rows of the pool (of this kv head) that hold the two sixteen-token halves of a tile
    auto pool_row = [&](int t) __attribute__((always_inline)) -> int64_t {
      const int lp = min(t / p.page_size, last_page), off = t % p.page_size;
      const int page = min(max(bt_row[lp], 0), p.n_pages - 1);
      return ((int64_t)page * p.heads_kv + kvh) * page_rows + off;
    };
    auto load = [&](int t, Regs& r) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int64_t row = pool_row(t + 16 * i);
        const uint8_t* kp = p.k + row * (D / 2);
        const uint8_t* ksp = p.k_scale + row * (D / 32);
        const uint8_t* vp = p.v + row * (D / 2);
        const uint8_t* vsp = p.v_scale + row * (D / 32);
#pragma unroll
        for (int kb = 0; kb < Regs::KB; kb++) {
          const int block = D == 64 ? (g & 1) : 4 * kb + g;
          r.k[i][kb] = *(const u32x4*)(kp + c * (D / 2) + 16 * block);
          r.ks[i][kb] = ksp[c * (D / 32) + block];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint8_t* vr = vp + (4 * g + j) * (D / 2) + c * (DPL / 2);
          if constexpr (D == 64) r.v[4 * i + j][0] = *(const uint16_t*)vr;
          else if constexpr (D == 128) r.v[4 * i + j][0] = *(const uint32_t*)vr;
          else {
            const u32x2 w = *(const u32x2*)vr;
            r.v[4 * i + j][0] = w[0];
            r.v[4 * i + j][1] = w[1];
          }
        }
#pragma unroll
        for (int j = 0; j < 4 * Regs::SW / 2; j++) r.vs[i][j] = ((const uint32_t*)(vsp + 4 * g * (D / 32)))[j];
      }
    };
    // scale of token j (0..7) for the lane's head elements: its byte in place of a float's exponent (255 reads as NaN)
    auto v_byte = [&](const Regs& r, int j) __attribute__((always_inline)) -> uint32_t {
      const int i = j >> 2, jj = j & 3;
      uint32_t w;
      if constexpr (D == 64) w = r.vs[i][jj >> 1] >> (16 * (jj & 1) + 8 * (c >> 3));
      else if constexpr (D == 128) w = r.vs[i][jj] >> v_shift;
      else w = (c & 8 ? r.vs[i][2 * jj + 1] : r.vs[i][2 * jj]) >> v_shift;
      return w & 0xffu;
    };

    auto step = [&](const Regs& r, int t) __attribute__((always_inline)) {
      const bool masked = t + kTile > limit_min;
      uint32_t pw[NRB][NP][4];
      uint32_t seen_bits[NRB];
#pragma unroll
      for (int rb = 0; rb < NRB; rb++) {
        f32x4 s[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kd = 0; kd < KD; kd++) {
            const u32x4 kk = r.k[i][kd];
            const i32x8 a = {(int)kk[0], (int)kk[1], (int)kk[2], (int)kk[3], 0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NQM; n++) {
              const u32x4 b0 = qf[rb][kd][n][0], b1 = qf[rb][kd][n][1];
              const i32x8 bq = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
              acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bq, acc, 4, 0, 0, (int)r.ks[i][kd], 0, 127);
            }
          }
          s[i] = acc;
        }
        float z[8];
        seen_bits[rb] = 0xffu;
#pragma unroll
        for (int e = 0; e < 8; e++)
          z[e] = to_logit2<SOFTCAP>(s[e >> 2][e & 3] * q_scale[rb], p.score_scale, p.cap_log2e, p.inv_cap_scale);
        if (masked) {
          seen_bits[rb] = 0;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const bool seen = t + 16 * (e >> 2) + 4 * g + (e & 3) < limit[rb];
            z[e] = seen ? z[e] : -INFINITY;
            seen_bits[rb] |= seen ? 1u << e : 0u;
          }
        }
        float top = max3(max3(z[0], z[1], z[2]), max3(z[3], z[4], z[5]), max2(z[6], z[7]));
        top = group_max(top);
        if (__ballot(top > m_run[rb] + kRescaleGap4)) {  // (the first tile with a visible token always comes here)
          const float m_new = top > m_run[rb] + kRescaleGap4 ? top : m_run[rb];
          const float f = fast_exp2(m_run[rb] - m_new);
          m_run[rb] = m_new;
          l_run[rb] *= f;
#pragma unroll
          for (int n = 0; n < DPL; n++) o[rb][n] *= f;
        }
        float pr[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          pr[e] = fast_exp2(z[e] - m_run[rb]);
          sum += pr[e];
        }
        l_run[rb] += sum;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pw[rb][0][e] = pack_bf16(pr[2 * e], pr[2 * e + 1]);
          if constexpr (NP == 2)
            pw[rb][1][e] = pack_bf16(pr[2 * e] - __uint_as_float(pw[rb][0][e] << 16), pr[2 * e + 1] - __uint_as_float(pw[rb][0][e] & 0xffff0000u));
        }
      }
      float vsc[8];
      uint32_t bad = 0;  // tokens (bits) whose block is NaN
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const uint32_t byte = v_byte(r, j);
        vsc[j] = __uint_as_float(byte << 23);
        if (masked) {
          // a NaN block stays out of the product, where a weight of zero would not keep it from the rows that do not see it
          bad |= byte == 255u ? 1u << j : 0u;
          vsc[j] = byte == 255u ? 0.f : vsc[j];
        }
      }
      auto value_step = [&](auto word_of, auto use) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < (DPL + 1) / 2; w++) {  // two head elements of the lane at a time
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
      value_step(
          [&](int j, int w) __attribute__((always_inline)) -> uint32_t {
            const uint32_t word = r.v[j][w >> 2];
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
              for (int q = 0; q < NP; q++) o[rb][n] = mma_bf16(a, u32x4{pw[rb][q][0], pw[rb][q][1], pw[rb][q][2], pw[rb][q][3]}, o[rb][n]);
          });
      if (masked && __ballot(bad != 0u)) {
        // rows that see a token with a NaN block get NaN there: count such tokens with the same product, 1 for every
        // NaN block against 1 for every visible token
#pragma unroll
        for (int rb = 0; rb < NRB; rb++) {
          u32x4 vis;
#pragma unroll
          for (int k = 0; k < 4; k++)
            vis[k] = ((seen_bits[rb] >> (2 * k)) & 1u ? 0x3f80u : 0u) | ((seen_bits[rb] >> (2 * k + 1)) & 1u ? 0x3f800000u : 0u);
          value_step([&](int j, int) __attribute__((always_inline)) -> uint32_t { return (bad >> j) & 1u ? 0x3f803f80u : 0u; },
                     [&](int n, u32x4 a) __attribute__((always_inline)) {
                       const f32x4 count = mma_bf16(a, vis, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                       for (int i = 0; i < 4; i++) o[rb][n][i] = count[i] > 0.f ? __builtin_nanf("") : o[rb][n][i];
                     });
        }
      }
    };

    if (tok < tok_end) {
      Regs cur;
      load(tok, cur);
      while (true) {
        const int next = tok + kUnit;
        Regs ahead;
        if (next < tok_end) load(next, ahead);
        step(cur, tok);
        if (next >= tok_end) break;
        cur = ahead;
        tok = next;
      }
    }

    // ---- the four waves' results of each block of rows meet in LDS ---------------------------------------------------
#pragma unroll
    for (int rb = 0; rb < NRB; rb++) {
      const float l_all = group_sum(l_run[rb]);
      if (g == 0) {
        s_m[wave][c] = m_run[rb];
        s_l[wave][c] = l_all;
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
    u = pre + seg_u1;
    pre += nu;
    if (u == pre) ++b;
    else pre -= nu;
  }
}

// Rows of a sequence that several ranges share: weights exp2(lse - max) over the ranges' normalised rows.  One wave per row.
// Sequences without tokens get zeros here.
template <typename QT, int D>
__global__ __launch_bounds__(256) void paged_decode_fp4_merge_kernel(const Fp4Params p) {
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  const int64_t row = (int64_t)blockIdx.x * 4 + uni(threadIdx.x >> 6);
  const int nu = uni(units_of_len(len_of(p, b)));
  int pre;
  const int T = total_units(p, b, &pre);
  int p_first = 0, p_last = -1;
  bool second = false;
  const Ranges ranges(T, p.n_parts);
  if (nu > 0) {
    p_first = uni(ranges.owner(pre));
    p_last = uni(ranges.owner(pre + nu - 1));
    if (p_first == p_last) return;  // written by the range that holds it
    second = ranges.begin(p_first) != pre;
  }
  if (row >= rows_all) return;
  const int kvh = (int)(row / p.rows), r = (int)(row - (int64_t)kvh * p.rows), s = r / p.group, gi = r - s * p.group;
  constexpr int E = D / 64;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.f;
  auto slot_of = [&](int part) { return (int64_t)(2 * part + (part == p_first && second ? 1 : 0)) * rows_all + row; };
  float M = -INFINITY, W = 0.f;
  for (int base = p_first; base <= p_last; base += 64) {
    const int part = base + lane;
    // (a range can be empty when there are fewer units than ranges: it wrote nothing)
    const bool there = part <= p_last && ranges.begin(part) < ranges.begin(part + 1);
    const float lse = there ? p.part_lse[slot_of(part)] : -INFINITY;
    float top = fmaxf(lse, __shfl_xor(lse, 1, 64));
#pragma unroll
    for (int m = 2; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
    const float M_new = fmaxf(M, top);
    if (__ballot(lse != lse)) W = __builtin_nanf("");
    if (M_new == -INFINITY) continue;
    const float f = fast_exp2(M - M_new), wl = there ? fast_exp2(lse - M_new) : 0.f;
    W *= f;
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] *= f;
    M = M_new;
    const int n = min(64, p_last - base + 1);
    for (int i = 0; i < n; i++) {
      const float w = __shfl(wl, i, 64);
      if (w == 0.f) continue;  // (a slot that nothing was written to may hold anything)
      const float* src = p.part_o + slot_of(base + i) * D + E * lane;
      W += w;
#pragma unroll
      for (int e = 0; e < E; e++) acc[e] += w * src[e];
    }
  }
  const float inv = W == 0.f ? 0.f : 1.0f / W;
  uint16_t* dst = p.out + (((int64_t)b * p.q_len + s) * p.heads + kvh * p.group + gi) * D + E * lane;
  if constexpr (E == 1) {
    dst[0] = (uint16_t)(pack16<QT>(acc[0] * inv, 0.f) & 0xffffu);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) *(uint32_t*)(dst + e) = pack16<QT>(acc[e] * inv, acc[e + 1] * inv);
  }
}

constexpr int kMaxParts4 = 4096;
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Blocks of sixteen query rows per wave (two at head dim 256 do not fit the register file).
int row_blocks(int rows, int dim) { return rows <= 16 || dim == 256 ? 1 : 2; }
int row_groups_of(int rows, int dim) { return (rows + 16 * row_blocks(rows, dim) - 1) / (16 * row_blocks(rows, dim)); }

template <typename QT, int D, int NRB>
const char* launch_fp4(const Fp4Params& p, bool softcap, hipStream_t s) {
  const int64_t pairs = (int64_t)p.n_parts * p.heads_kv;
  const int64_t grid = 8 * (int64_t)p.row_groups * ((pairs + 7) / 8);
  if (grid > INT_MAX) return "too many workgroups";
  if (softcap)
    hipLaunchKernelGGL((paged_decode_fp4_kernel<QT, D, NRB, true>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, p);
  else
    hipLaunchKernelGGL((paged_decode_fp4_kernel<QT, D, NRB, false>), dim3((unsigned)grid), dim3(64 * kWaves), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hipGetErrorString(e);
  const int64_t rows_all = (int64_t)p.heads_kv * p.rows;
  hipLaunchKernelGGL((paged_decode_fp4_merge_kernel<QT, D>), dim3((unsigned)((rows_all + 3) / 4), p.batch), dim3(256), 0, s, p);
  e = hipGetLastError();
  return e == hipSuccess ? nullptr : hipGetErrorString(e);
}

template <typename QT>
const char* launch_fp4_dim(const Fp4Params& p, int dim, bool softcap, hipStream_t s) {
  const bool one = row_blocks(p.rows, dim) == 1;
  if (dim == 64) return one ? launch_fp4<QT, 64, 1>(p, softcap, s) : launch_fp4<QT, 64, 2>(p, softcap, s);
  if (dim == 128) return one ? launch_fp4<QT, 128, 1>(p, softcap, s) : launch_fp4<QT, 128, 2>(p, softcap, s);
  return launch_fp4<QT, 256, 1>(p, softcap, s);
}

}  // namespace

// Ranges of the token stream: two workgroups (eight waves) per compute unit over all (kv head, row group) pairs.
int fp4_num_parts(int heads_kv, int rows, int dim, int compute_units) {
  const int64_t parts = 2 * (int64_t)compute_units / ((int64_t)heads_kv * row_groups_of(rows, dim));
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
  p.row_groups = row_groups_of(p.rows, dim);
  p.n_parts = n_parts;
  p.max_len = max_len < INT_MAX - kUnit ? max_len : INT_MAX - kUnit;
  p.causal = causal;
  p.n_pages = (int)n_pages;
  const size_t slots = (size_t)2 * n_parts * heads_kv * p.rows;
  p.part_o = (float*)workspace;
  p.part_lse = (float*)((char*)workspace + align256(slots * dim * sizeof(float)));
  const bool cap_on = softcap > 0.f;
  p.score_scale = sm_scale * kLog2e;
  p.cap_log2e = softcap * kLog2e;
  p.inv_cap_scale = cap_on ? sm_scale / softcap : 0.f;
  return q_dtype == MI355_DT_BF16 ? launch_fp4_dim<bf16_tag>(p, dim, cap_on, s) : launch_fp4_dim<fp16_tag>(p, dim, cap_on, s);
}

}  // namespace mi355
