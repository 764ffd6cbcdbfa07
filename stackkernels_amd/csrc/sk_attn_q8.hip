// Attention over a key/value cache held in 8-bit codes (int8 or float8 e4m3)
// with one scale per block of tokens and KV head, for one or a few query
// tokens per row.
//
// Mathematics.  With codes a_n, c_n and scales s_n, t_n >= 0 of key n,
//   O = sum_n softmax_n(sm_scale s_n (q . a_n)) t_n c_n.
// Every code is exact in fp16, so q . a_n is an fp16 matrix product with fp32 sums
// and the scales are applied in fp32: a cached element is never rounded again.
// * q (rotated in fp32 where the call rotates) is divided by a power of two that
//   brings its row's largest element into [1, 2), which its score's factor takes
//   back: bf16 queries are then exact in fp16 (down to 2^-24 of the row's
//   largest), rotated ones are rounded once to 11 bits.  fp32 queries are the sum
//   of two such numbers (22 bits).
// * Probabilities e = 2^(s - m) are summed in fp32 into l and enter the product
//   with V as fp16 numbers e t_n 2^(m - m2), where m2 is the running maximum of s
//   + log2 t_n as m is that of s: largest contributions are near 1 whatever the
//   scales are, and a rounding is off by 2^-12 of a contribution or 2^-25 of the
//   largest one.
// * m and m2 are raised only when a score exceeds them by 8 (probabilities up to
//   2^8), so the sums are rescaled a few times per row, not once per tile.
//
// Layout.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16 with 16 (query
// token, head) rows of one KV head as the 16 columns, NC such blocks per wave.  A
// wave takes 32 keys at a time straight from HBM into registers, no LDS:
// * K: lane (key r, group g) loads the 16 bytes 64 j + 16 g of its key's row,
//   two k-steps of eight consecutive head-dim columns; Q is laid out to match.
// * V: lane (m, group g) loads columns [VB m, VB m + VB) (VB = DP / 16) of the
//   eight keys whose probabilities group g holds; output block c is then the
//   columns VB m + c, so the transposition V^T needs is a byte selection.
// The four waves of a workgroup take tiles in turn and merge their sums in LDS.
#include <type_traits>

#include "sk_common.h"
#include "sk_q8.h"
#include "sk_rope.h"

namespace sk {

struct I8 {
  static constexpr int code = kCodeI8;
};
struct E4M3 {
  static constexpr int code = kCodeE4M3;
};

// u8 values in the low bytes of both halves (int8 codes with the sign bit still
// as it is) -> two fp16 numbers: 0x6400 | u is 1024 + u, and u = code + 128 with
// the sign bit flipped.
__device__ __forceinline__ uint32_t i8_halves(uint32_t w) {
  const f16x2 x = __builtin_bit_cast(f16x2, w ^ 0x64806480u);
  const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(uint32_t, x - bias);
}

// Codes 2 h and 2 h + 1 of one dword as two fp16 numbers.
template <class C, int H>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (C::code == kCodeE4M3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, H != 0));
  else
    return i8_halves(__builtin_amdgcn_perm(0u, w, H ? 0x0c030c02u : 0x0c010c00u));
}

// Codes 2 h and 2 h + 1 of two dwords a, b -> (a, b) pairs of fp16 numbers.
template <class C, int H>
__device__ __forceinline__ void widen_cols(uint32_t a, uint32_t b, uint32_t& c0, uint32_t& c1) {
  if constexpr (C::code == kCodeE4M3) {
    const uint32_t x = __builtin_amdgcn_perm(b, a, H ? 0x07030602u : 0x05010400u);
    c0 = widen2<C, 0>(x);
    c1 = widen2<C, 1>(x);
  } else {
    c0 = i8_halves(__builtin_amdgcn_perm(b, a, H ? 0x0c060c02u : 0x0c040c00u));
    c1 = i8_halves(__builtin_amdgcn_perm(b, a, H ? 0x0c070c03u : 0x0c050c01u));
  }
}

// (a, b) as a sum of TERMS pairs of fp16 numbers.
template <int TERMS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    w[t] = pack2<F16>(a, b);
    if (t + 1 < TERMS) {
      a -= to_f32<F16>((uint16_t)(w[t] & 0xffffu));
      b -= to_f32<F16>((uint16_t)(w[t] >> 16));
    }
  }
}

// Eight elements of a query at element offset at, as fp32.
__device__ __forceinline__ void load_q8x8(const void* q, int dtype, int64_t at, float (&x)[8]) {
  if (dtype == SK_F32) {
    const f32x4* p = reinterpret_cast<const f32x4*>((const float*)q + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    return;
  }
  const u32x4 a = ldg_b128_cached((const uint16_t*)q + at);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = a[i];
    const uint16_t lo = (uint16_t)(w & 0xffffu), hi = (uint16_t)(w >> 16);
    x[2 * i] = dtype == SK_F16 ? to_f32<F16>(lo) : to_f32<BF16>(lo);
    x[2 * i + 1] = dtype == SK_F16 ? to_f32<F16>(hi) : to_f32<BF16>(hi);
  }
}

// Four outputs of q's type at element offset at.
__device__ __forceinline__ void store_o4(void* o, int dtype, int64_t at, const float (&x)[4]) {
  if (dtype == SK_F32)
    *reinterpret_cast<f32x4*>((float*)o + at) = f32x4{x[0], x[1], x[2], x[3]};
  else
    *reinterpret_cast<u32x2*>((uint16_t*)o + at) =
        dtype == SK_F16 ? u32x2{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3])}
                        : u32x2{pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3])};
}

// Keys and queries of a row block (row = token * group + head of its KV head).
struct Q8Span {
  int len, ql;     // the batch row's keys and queries
  int hi;          // keys the block's last row sees
  int full;        // keys all of its rows see
};

__device__ __forceinline__ Q8Span q8_span(const Q8AttnParams& p, int b, int row0, int n_rows) {
  Q8Span s;
  s.len = p.seqlens ? min(max(__builtin_amdgcn_readfirstlane(p.seqlens[b]), 0), p.Sk) : p.Sk;
  s.ql = p.qlens ? min(max(__builtin_amdgcn_readfirstlane(p.qlens[b]), 0), p.Sq) : p.Sq;
  const int t_first = row0 / p.group;
  const int t_last = min((min(row0 + n_rows, p.rows) - 1) / p.group, s.ql - 1);
  s.hi = p.causal ? min(s.len, s.len - s.ql + t_last + 1) : s.len;
  if (t_first >= s.ql) s.hi = 0;
  s.hi = max(s.hi, 0);
  s.full = p.causal ? s.len - s.ql + t_first + 1 : s.len;
  return s;
}

constexpr int kQ8Waves = 4;
constexpr float kMinFactor = 1e-35f;  // of a score: keeps a masked -inf a -inf

// Column blocks whose queries are read from LDS each tile (the four waves share
// them): with more than 32 head-dim-128 columns the sums alone take 128
// registers, and the queries would take the second wave of a SIMD.
template <int DP, int NC>
constexpr bool q8_q_in_lds() {
  return NC * DP > 256;
}

template <class C, int TERMS, int DP, int NC, bool PAGED>
__global__ void __launch_bounds__(kQ8Waves * 64, 2) q8_attn_kernel(Q8AttnParams p) {
  constexpr int KC = DP / 64;   // 16-byte chunks of a K row per lane
  constexpr int KS = DP / 32;   // k-steps of S^T
  constexpr int VB = DP / 16;   // bytes of a V row per lane = output blocks
  constexpr int VW = VB / 4;
  constexpr int NW = kQ8Waves;
  constexpr bool kQLds = q8_q_in_lds<DP, NC>();

  __shared__ float red_m[NW][16 * NC];
  __shared__ float red_l[NW][16 * NC];
  __shared__ __attribute__((aligned(16))) float red_o[NW][16][DP + 4];
  __shared__ u32x4 qs[kQLds ? NC * KS * TERMS : 1][64];
  __shared__ float qmul_s[kQLds ? NC : 1][64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15;
  const int g = lane >> 4;

  int item = xcd_work_index(blockIdx.x, gridDim.x);
  const int rb = item % p.row_blocks;
  item /= p.row_blocks;
  const int split = item % p.num_splits;
  item /= p.num_splits;
  const int hkv = item % p.Hkv;
  const int b = item / p.Hkv;

  const int row0 = rb * 16 * NC;
  const Q8Span sp = q8_span(p, b, row0, 16 * NC);
  const int kps = ((sp.hi + p.num_splits - 1) / p.num_splits + 31) / 32 * 32;
  const int k_lo = split * kps;
  const int k_hi = min(sp.hi, k_lo + kps);

  int lim[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    lim[c] = min(p.causal ? sp.len - sp.ql + (row0 + 16 * c + c16) / p.group + 1 : sp.len, k_hi);

  // This lane's loads within a tile: constant offsets from the tile's base.
  const uint32_t k_off = (uint32_t)(c16 * (int)p.k.ss + 16 * g);
  const uint32_t v_off = (uint32_t)(4 * g * (int)p.v.ss + VB * c16);
  const bool v_in = VB * c16 < p.D;

  u32x4 kreg[2][KC];
  uint32_t vreg[8][VW];
  float ks_t = 0.f, vs_t = 0.f;  // scales of the tile in kreg / vreg
  bool ok_t = false;
  // The tile after it: its page (read a tile ahead) and where it lies.
  int page_n = 0;
  auto page_entry = [&](int n0) SK_INLINE {
    return PAGED && n0 < k_hi ? p.table[(int64_t)b * p.max_pages + p.page_div.quot(n0)] : 0;
  };
  int64_t k_at = 0, v_at = 0;
  int n_rows = 0;
  // A buffer resource that ends with the tile's last visible row returns zeros for
  // the rows past it (and for tiles whose page lies outside the pool).
  auto load_k = [&](int n0, int page_raw) SK_INLINE {
    int64_t unit = b;
    int row = n0;
    ok_t = true;
    if constexpr (PAGED) {
      const int page = __builtin_amdgcn_readfirstlane(page_raw);
      ok_t = page >= 0 && page < p.num_pages;
      unit = ok_t ? page : 0;
      row = n0 - p.page_div.quot(n0) * p.page_size;
    }
    n_rows = ok_t ? min(32, k_hi - n0) : 0;
    k_at = unit * p.k.sb + (int64_t)hkv * p.k.sh + (int64_t)row * p.k.ss;
    v_at = unit * p.v.sb + (int64_t)hkv * p.v.sh + (int64_t)row * p.v.ss;
    const int blk = p.block_div.quot(row);
    ks_t = ok_t ? p.k.scales[unit * p.k.cb + (int64_t)hkv * p.k.ch + (int64_t)blk * p.k.cs] : 0.f;
    vs_t = ok_t ? p.v.scales[unit * p.v.cb + (int64_t)hkv * p.v.ch + (int64_t)blk * p.v.cs] : 0.f;
    const buf_rsrc r =
        make_rsrc(p.k.codes + k_at, n_rows > 0 ? (int)((n_rows - 1) * p.k.ss) + p.D : 0);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < KC; ++j)
        kreg[kb][j] = buffer_load_b128(r, 64 * j + 16 * g < p.D
                                              ? k_off + (uint32_t)(16 * kb * (int)p.k.ss + 64 * j)
                                              : kBufferOob);
  };
  auto load_v = [&]() SK_INLINE {
    const buf_rsrc r =
        make_rsrc(p.v.codes + v_at, n_rows > 0 ? (int)((n_rows - 1) * p.v.ss) + p.D : 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t off =
          v_in ? v_off + (uint32_t)((e < 4 ? e : e + 12) * (int)p.v.ss) : kBufferOob;
      if constexpr (VW == 1) {
        vreg[e][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
      } else if constexpr (VW == 2) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
        vreg[e][0] = w[0], vreg[e][1] = w[1];
      } else {
        const u32x4 w = buffer_load_b128(r, off);
#pragma unroll
        for (int i = 0; i < 4; ++i) vreg[e][i] = w[i];
      }
    }
  };

  int n0 = k_lo + 32 * wave;
  if (n0 < k_hi) {
    load_k(n0, page_entry(n0));
    load_v();
    page_n = page_entry(n0 + 32 * NW);
  }

  // Q^T operand: k-step s = 2 j + h of lane group g is head-dim columns 64 j +
  // 16 g + 8 h .. + 7, divided by 2^(exponent of the row's largest element).
  u32x4 qreg[kQLds ? 1 : NC][KS][TERMS];
  float qmul[NC];
  if (k_lo < k_hi) {
    const int half = p.D >> 1;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (kQLds && c % NW != wave) continue;
      const int r = row0 + 16 * c + c16;
      const int t = r / p.group;
      const bool live = r < p.rows && t < sp.ql;
      const int64_t at = live ? (int64_t)b * p.q_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.q_sh +
                                    (int64_t)t * p.q_ss
                              : 0;
      const int rr = rope_row(p.rope, b, t);
      float x[KS][8];
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = 0.f;
        if (live && d0 < p.D) {
          load_q8x8(p.q, p.dtype, at + d0, x[s]);
          if (rr >= 0) {
            float y[8], cs[8], sn[8];
            load_q8x8(p.q, p.dtype, at + (d0 < half ? d0 + half : d0 - half), y);
            rope_coeffs<8>(p.rope, rr, d0, cs, sn);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = rope_mix(x[s][e], y[e], d0 < half, cs[e], sn[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[s][e]));
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = xhalf_max(top);
      int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
      if (ex > 127) ex = 0;  // an infinity: the row's scores are not finite anyway
      qmul[c] = __builtin_amdgcn_ldexpf(fabsf(p.scale_log2), ex);
      const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;
      if (kQLds) qmul_s[kQLds ? c : 0][lane] = qmul[c];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4 w[TERMS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t u[TERMS];
          split2<TERMS>(sign * __builtin_amdgcn_ldexpf(x[s][2 * i], -ex),
                        sign * __builtin_amdgcn_ldexpf(x[s][2 * i + 1], -ex), u);
#pragma unroll
          for (int k = 0; k < TERMS; ++k) w[k][i] = u[k];
        }
#pragma unroll
        for (int k = 0; k < TERMS; ++k) {
          if constexpr (kQLds)
            qs[(c * KS + s) * TERMS + k][lane] = w[k];
          else
            qreg[c][s][k] = w[k];
        }
      }
    }
    if constexpr (kQLds) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c) qmul[c] = qmul_s[c][lane];
    }
  }

  f32x4 oacc[NC][VB];
  // Per column: -m (0 while there is no key), m, m2, l, and 2^(m - m2).
  float m_neg[NC], m_run[NC], m2_run[NC], l_run[NC], w_run[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_run[c] = m2_run[c] = kNegInf, m_neg[c] = 0.f, l_run[c] = 0.f, w_run[c] = 0.f;
#pragma unroll
    for (int i = 0; i < VB; ++i) oacc[c][i] = f32x4{};
  }

  for (; n0 < k_hi; n0 += 32 * NW) {
    const float ks = ks_t, vs = vs_t;
    const bool ok = ok_t;
    f32x4 sacc[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) sacc[c][0] = sacc[c][1] = f32x4{};
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 a[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t w0 = kreg[kb][j][2 * h], w1 = kreg[kb][j][2 * h + 1];
          a[kb] = u32x4{widen2<C, 0>(w0), widen2<C, 1>(w0), widen2<C, 0>(w1), widen2<C, 1>(w1)};
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int u = TERMS - 1; u >= 0; --u) {
            u32x4 q;
            if constexpr (kQLds)
              q = qs[(c * KS + 2 * j + h) * TERMS + u][lane];
            else
              q = qreg[c][2 * j + h][u];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) sacc[c][kb] = mfma16<F16>(a[kb], q, sacc[c][kb]);
          }
      }
    const int n1 = n0 + 32 * NW;
    if (n1 < k_hi) {
      load_k(n1, page_n);
      page_n = page_entry(n1 + 32 * NW);
    }

    const bool masked = !ok || n0 + 32 > k_hi || n0 + 32 > sp.full;
    const float lv = __builtin_amdgcn_logf(vs);  // log2
    uint32_t pk[NC][4][TERMS];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float mul = fmaxf(ks * qmul[c], kMinFactor);
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = sacc[c][i >> 2][i & 3];
      if (masked) {
        const int end = ok ? lim[c] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n0 + 16 * (i >> 2) + 4 * g + (i & 3) >= end) e[i] = kNegInf;
      }
      float mt = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])),
                       fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = xhalf_max(mt) * mul;
      const float mt2 = mt + lv;
      if (__any(mt > m_run[c] + kRescaleLog2 || mt2 > m2_run[c] + kRescaleLog2)) {
        const float m_new = fmaxf(m_run[c], mt), m2_new = fmaxf(m2_run[c], mt2);
        const float al = m_new == kNegInf ? 1.f : fast_exp2(m_run[c] - m_new);
        const float ao = m2_new == kNegInf ? 1.f : fast_exp2(m2_run[c] - m2_new);
        m_run[c] = m_new, m2_run[c] = m2_new;
        m_neg[c] = m_new == kNegInf ? 0.f : -m_new;
        w_run[c] = m2_new == kNegInf ? 0.f : fast_exp2(m_new - m2_new);
        l_run[c] *= al;
#pragma unroll
        for (int i = 0; i < VB; ++i) oacc[c][i] *= ao;
      }
      const float wv = vs * w_run[c];
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = fast_exp2(fmaf(e[i], mul, m_neg[c]));
        ps += e[i];
        e[i] *= wv;
      }
      l_run[c] += ps;
#pragma unroll
      for (int i = 0; i < 4; ++i) split2<TERMS>(e[2 * i], e[2 * i + 1], pk[c][i]);
    }
    auto product = [&](int w, auto hc) SK_INLINE {
      constexpr int H = decltype(hc)::value;
      u32x4 a0, a1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x, y;
        widen_cols<C, H>(vreg[2 * i][w], vreg[2 * i + 1][w], x, y);
        a0[i] = x, a1[i] = y;
      }
      const int blk = 4 * w + 2 * H;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = TERMS - 1; u >= 0; --u) {
          const u32x4 pb = {pk[c][0][u], pk[c][1][u], pk[c][2][u], pk[c][3][u]};
          oacc[c][blk] = mfma16<F16>(a0, pb, oacc[c][blk]);
          oacc[c][blk + 1] = mfma16<F16>(a1, pb, oacc[c][blk + 1]);
        }
    };
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      product(w, std::integral_constant<int, 0>{});
      product(w, std::integral_constant<int, 1>{});
    }
    if (n1 < k_hi) load_v();
  }

  // Merge the four waves' sums: a row's common maximum M, then O scaled by 2^(m2 -
  // M) and l by 2^(m - M), added in wave order.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float l = l_run[c] + __shfl_xor(l_run[c], 16);
    l = xhalf_sum(l);
    if (g == 0) {
      red_m[wave][16 * c + c16] = m_run[c];
      red_l[wave][16 * c + c16] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float mm = red_m[0][16 * c + c16];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, red_m[w][16 * c + c16]);
    const float f = mm == kNegInf || m2_run[c] == kNegInf ? 1.f : fast_exp2(m2_run[c] - mm);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < VB; i += 4)
        *reinterpret_cast<f32x4*>(&red_o[wave][c16][VB * (4 * g + r) + i]) =
            f32x4{oacc[c][i][r], oacc[c][i + 1][r], oacc[c][i + 2][r], oacc[c][i + 3][r]} * f;
    __syncthreads();
    // 16 threads per row, DP / 16 columns each.
    {
      const int rr = tid >> 4;
      const int d0 = (tid & 15) * VB;
      const int r = row0 + 16 * c + rr;
      float mrow = kNegInf, lrow = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) mrow = fmaxf(mrow, red_m[w][16 * c + rr]);
#pragma unroll
      for (int w = 0; w < NW; ++w)
        lrow += red_l[w][16 * c + rr] * (mrow == kNegInf ? 1.f : fast_exp2(red_m[w][16 * c + rr] - mrow));
      const int t = r / p.group;
      const bool live = r < p.rows && t < sp.ql;
      const float inv = lrow == 0.f ? 0.f : 1.f / lrow;  // (NaN stays NaN)
      if (r < p.rows) {
        const int64_t row = (((int64_t)b * p.Hkv + hkv) * p.rows + r) * p.num_splits + split;
        const int64_t at = (int64_t)b * p.o_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.o_sh +
                           (int64_t)t * p.o_ss + d0;
#pragma unroll
        for (int i = 0; i < VB; i += 4) {
          f32x4 s = *reinterpret_cast<const f32x4*>(&red_o[0][rr][d0 + i]);
#pragma unroll
          for (int w = 1; w < NW; ++w) s += *reinterpret_cast<const f32x4*>(&red_o[w][rr][d0 + i]);
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = live ? s[e] * inv : 0.f;
          if (p.num_splits > 1)
            *reinterpret_cast<f32x4*>(p.part_o + row * p.dpad + d0 + i) = f32x4{x[0], x[1], x[2], x[3]};
          else if (d0 + i < p.D)
            store_o4(p.o, p.dtype, at + i, x);
        }
        if (p.num_splits > 1 && (tid & 15) == 0)
          p.part_lse[row] = !live || lrow == 0.f ? kNegInf
                            : mrow == kNegInf    ? lrow
                                                 : mrow + __log2f(lrow);
      }
    }
    __syncthreads();
  }
}

// Merge the splits of a row (query token, head), one wave a row: weights 2^(lse -
// max) of the splits that saw a key, sums over lanes of 16 bytes of columns and, up
// to 128 columns, over groups of lanes that take splits in turn.
template <int DP>
__global__ void __launch_bounds__(256) q8_combine_kernel(Q8AttnParams p) {
  constexpr int LPG = DP / 4;    // lanes per split
  constexpr int G = 64 / LPG;    // splits at a time
  __shared__ float w[4][kQ8MaxSplits];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  const int64_t bh = row / p.rows;
  if (bh >= (int64_t)p.B * p.Hkv) return;
  const int ns = p.num_splits;
  const float* lse = p.part_lse + row * ns;
  const float* po = p.part_o + row * ns * DP + (lane % LPG) * 4;
  float mx = kNegInf;
  for (int s = lane; s < ns; s += 64) mx = fmaxf(mx, lse[s]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  float den = 0.f;
  for (int s = lane; s < ns; s += 64) {
    const float l = lse[s];
    const float x = l == kNegInf ? 0.f : fast_exp2(l - (mx == kNegInf ? 0.f : mx));
    w[wave][s] = x;
    den += x;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
  // (The wave's own LDS writes: ordered before its reads.)
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = lane / LPG; s < ns; s += G) {
    const float x = w[wave][s];
    if (x != 0.f) acc += x * *reinterpret_cast<const f32x4*>(po + (int64_t)s * DP);
  }
#pragma unroll
  for (int o = LPG; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o);
  const int d = (lane % LPG) * 4;
  if (lane >= LPG || d >= p.D) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int r = (int)(row - bh * p.rows);
  const int hkv = (int)(bh % p.Hkv);
  const int64_t b = bh / p.Hkv;
  const int t = r / p.group;
  const float x[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
  store_o4(p.o, p.dtype,
           b * p.o_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.o_sh + (int64_t)t * p.o_ss + d, x);
}

int q8_dpad(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Column blocks of 16 rows that a workgroup takes: as many as leave two waves a SIMD
// without spills.  At D = 128 two blocks against one and four: 64 MQA heads, 8 x
// 131,072 keys 114, 144 and 358 us (four spill); 512 queries against 16,000 keys
// 252, 443 and 744; 2 x 4,096 against 16,384 1.84, 2.67 and 6.48 ms.
static int q8_cols(int dtype, int D, int rows) {
  const int most = D > 128 ? 1 : D > 64 || dtype == SK_F32 ? 2 : 4;
  const int want = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return want < most ? want : most;
}

int q8_rows_per_block(int dtype, int D, int rows) { return 16 * q8_cols(dtype, D, rows); }

int q8_splits(int dtype, int B, int Hkv, int rows, int keys, int D) {
  const int per = q8_rows_per_block(dtype, D, rows);
  const int64_t units = (int64_t)B * Hkv * ((rows + per - 1) / per);
  if (units <= 0) return 1;
  int64_t s = 1024 / units;
  const int64_t most = keys / 256;
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s > kQ8MaxSplits ? kQ8MaxSplits : s);
}

template <class C, int TERMS, int DP, int NC>
static hipError_t launch_nc(const Q8AttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * p.num_splits * p.row_blocks));
  if (p.table)
    hipLaunchKernelGGL((q8_attn_kernel<C, TERMS, DP, NC, true>), grid, dim3(kQ8Waves * 64), 0, s, p);
  else
    hipLaunchKernelGGL((q8_attn_kernel<C, TERMS, DP, NC, false>), grid, dim3(kQ8Waves * 64), 0, s, p);
  return hipGetLastError();
}

template <class C, int TERMS, int DP>
static hipError_t launch_dp(const Q8AttnParams& p, hipStream_t s) {
  const int nc = q8_cols(p.dtype, p.D, p.rows);
  if (nc == 1) return launch_nc<C, TERMS, DP, 1>(p, s);
  if constexpr (DP <= 128)
    if (nc == 2) return launch_nc<C, TERMS, DP, 2>(p, s);
  if constexpr (DP <= 64 && TERMS == 1)
    if (nc == 4) return launch_nc<C, TERMS, DP, 4>(p, s);
  return hipErrorInvalidValue;
}

template <class C, int TERMS>
static hipError_t launch_ct(const Q8AttnParams& p, hipStream_t s) {
  if (p.D <= 64) return launch_dp<C, TERMS, 64>(p, s);
  if (p.D <= 128) return launch_dp<C, TERMS, 128>(p, s);
  return launch_dp<C, TERMS, 256>(p, s);
}

hipError_t launch_q8_attn(int code, const Q8AttnParams& p, hipStream_t s) {
  const bool wide = p.dtype == SK_F32;
  const hipError_t e =
      code == kCodeI8 ? (wide ? launch_ct<I8, 2>(p, s) : launch_ct<I8, 1>(p, s))
                      : (wide ? launch_ct<E4M3, 2>(p, s) : launch_ct<E4M3, 1>(p, s));
  if (e != hipSuccess || p.num_splits == 1) return e;
  const dim3 grid((unsigned)(((int64_t)p.B * p.Hkv * p.rows + 3) / 4));
  if (p.dpad == 64)
    hipLaunchKernelGGL(q8_combine_kernel<64>, grid, dim3(256), 0, s, p);
  else if (p.dpad == 128)
    hipLaunchKernelGGL(q8_combine_kernel<128>, grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL(q8_combine_kernel<256>, grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace sk
