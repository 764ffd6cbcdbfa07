// Attention over a key/value cache held in 8-bit codes (int8 or float8 e4m3)
// with one scale per block of tokens and KV head, for one or a few query
// tokens per row.
//
// Mathematics.  With codes a_n, c_n and scales s_n, t_n of key n,
//   O = sum_n softmax_n(sm_scale s_n (q . a_n)) t_n c_n.
// Every code is exact in bf16 and fp16, so q . a_n is a 16-bit matrix product
// with fp32 sums and the scales are applied in fp32, s_n to the score and t_n
// to the probability: a cached element is never rounded a second time.  fp32
// queries and probabilities are written as the sum of three bf16 numbers (8 + 8
// + 8 significant bits), whose three products with exact codes give the fp32
// product.
//
// Layout.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32 with 16 (query
// token, head) rows of one KV head as the 16 columns.  A wave takes 32 keys at a
// time straight from HBM into registers, no LDS:
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

// Matrix element type of a query type: fp32 queries run as bf16 terms.
template <class T>
struct Q8Elem {
  using M = T;
  static constexpr int kTerms = 1;
};
template <>
struct Q8Elem<float> {
  using M = BF16;
  static constexpr int kTerms = 3;
};

__device__ __forceinline__ float byte_f32(uint32_t w, int i) {
  return (float)(int8_t)((w >> (8 * i)) & 0xffu);
}

// Two codes of one dword (bytes 2 h, 2 h + 1) as two 16-bit values, exactly.
template <class M, class C>
__device__ __forceinline__ uint32_t widen2(uint32_t w, int h) {
  if constexpr (C::code == kCodeE4M3) {
    if constexpr (M::code == BF16::code)
      return h ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
    else
      return h ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  } else {
    return pack2<M>(byte_f32(w, 2 * h), byte_f32(w, 2 * h + 1));
  }
}

// Byte i (0..3) of two dwords as two 16-bit values.
template <class M, class C>
__device__ __forceinline__ void widen_col2(uint32_t a, uint32_t b, int h, uint32_t& c0,
                                           uint32_t& c1) {
  if constexpr (C::code == kCodeE4M3) {
    const uint32_t x = widen2<M, C>(a, h), y = widen2<M, C>(b, h);
    c0 = __builtin_amdgcn_perm(y, x, 0x05040100u);  // low halves
    c1 = __builtin_amdgcn_perm(y, x, 0x07060302u);  // high halves
  } else {
    c0 = pack2<M>(byte_f32(a, 2 * h), byte_f32(b, 2 * h));
    c1 = pack2<M>(byte_f32(a, 2 * h + 1), byte_f32(b, 2 * h + 1));
  }
}

// x as a sum of kTerms 16-bit values, two at a time.
template <class M, int TERMS>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&w)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    w[t] = pack2<M>(a, b);
    if (t + 1 < TERMS) {
      a -= to_f32<M>((uint16_t)(w[t] & 0xffffu));
      b -= to_f32<M>((uint16_t)(w[t] >> 16));
    }
  }
}

template <int VB>
struct VWords;
template <>
struct VWords<4> {
  static constexpr int N = 1;
};
template <>
struct VWords<8> {
  static constexpr int N = 2;
};
template <>
struct VWords<16> {
  static constexpr int N = 4;
};

constexpr int kQ8Waves = 4;

template <class T, class C, int DP, int NC, bool PAGED>
__global__ void __launch_bounds__(kQ8Waves * 64) q8_attn_kernel(Q8AttnParams p) {
  using M = typename Q8Elem<T>::M;
  constexpr int TERMS = Q8Elem<T>::kTerms;
  constexpr int KC = DP / 64;   // 16-byte chunks of a K row per lane
  constexpr int KS = DP / 32;   // k-steps of S^T
  constexpr int VB = DP / 16;   // bytes of a V row per lane = output blocks
  constexpr int VW = VWords<VB>::N;
  constexpr int NW = kQ8Waves;
  // The probability carries the V scale where its 16-bit type has fp32's
  // range; fp16 would lose small products, so there the scale goes on the sums.
  constexpr bool kFold = M::code == BF16::code;

  __shared__ float red_m[NW][16 * NC];
  __shared__ float red_l[NW][16 * NC];
  __shared__ __attribute__((aligned(16))) float red_o[NW][16][DP + 4];

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

  const int len = p.seqlens ? min(max(__builtin_amdgcn_readfirstlane(p.seqlens[b]), 0), p.Sk) : p.Sk;
  const int ql = p.qlens ? min(max(__builtin_amdgcn_readfirstlane(p.qlens[b]), 0), p.Sq) : p.Sq;
  const int row0 = rb * 16 * NC;
  const int t_first = row0 / p.group;
  const int t_last = min((min(row0 + 16 * NC, p.rows) - 1) / p.group, ql - 1);
  // Keys the block's last row sees, and those that all of its rows see.
  int hi = p.causal ? min(len, len - ql + t_last + 1) : len;
  const int full = p.causal ? len - ql + t_first + 1 : len;
  if (t_first >= ql) hi = 0;
  hi = max(hi, 0);
  const int kps = ((hi + p.num_splits - 1) / p.num_splits + 31) / 32 * 32;
  const int k_lo = split * kps;
  const int k_hi = min(hi, k_lo + kps);

  int lim[NC];
  bool col_ok[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = row0 + 16 * c + c16;
    const int t = r / p.group;
    col_ok[c] = r < p.rows && t < ql;
    lim[c] = p.causal ? len - ql + t + 1 : len;
  }

  // Q^T operand: k-step s = 2 j + h of lane group g is head-dim columns 64 j +
  // 16 g + 8 h .. + 7.
  u32x4 qreg[NC][KS][TERMS];
  if (k_lo < k_hi) {
    const int half = p.D >> 1;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int r = row0 + 16 * c + c16;
      const int t = col_ok[c] ? r / p.group : 0;
      const int hq = hkv * p.group + (col_ok[c] ? r - t * p.group : 0);
      const int64_t base = (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh + (int64_t)t * p.q_ss;
      const int rr = rope_row(p.rope, b, t);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
        const bool ok = col_ok[c] && d0 < p.D;
        if constexpr (TERMS == 1) {
          const uint16_t* qp = (const uint16_t*)p.q + base;
          u32x4 x = {0u, 0u, 0u, 0u};
          if (ok) {
            x = ldg_b128_cached(qp + d0);
            if (rr >= 0)
              x = rope8_at<T>(x, ldg_b128_cached(qp + (d0 < half ? d0 + half : d0 - half)), d0,
                              half, p.rope, rr);
          }
          qreg[c][s][0] = x;
        } else {
          const float* qp = (const float*)p.q + base;
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = !ok ? 0.f : rr >= 0 ? rope1(qp, d0 + e, half, p.rope, rr) : qp[d0 + e];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[TERMS];
            split2<M, TERMS>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) qreg[c][s][u][i] = w[u];
          }
        }
      }
    }
  }

  f32x4 oacc[NC][VB];
  float m_run[NC], l_run[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_run[c] = kNegInf, l_run[c] = 0.f;
#pragma unroll
    for (int i = 0; i < VB; ++i) oacc[c][i] = f32x4{};
  }

  // Offsets of this lane's loads within a tile: constant, the tile's base moves.
  const uint32_t k_off0 = (uint32_t)(c16 * p.k.ss + 16 * g);
  const uint32_t v_off0 = (uint32_t)(4 * g * p.v.ss + VB * c16);
  const bool v_in = VB * c16 < p.D;

  u32x4 kreg[2][KC];
  uint32_t vreg[8][VW];
  float ks_n = 0.f, vs_n = 0.f;
  bool ok_n = false;

  // Base addresses of the tile at n0 and its loads.  A buffer resource that ends
  // with the tile's last visible row returns zeros for the rows past it.
  auto load_tile = [&](int n0) {
    int64_t unit = b;
    int row = n0;
    bool ok = true;
    if constexpr (PAGED) {
      const int pi = n0 / p.page_size;
      const int page = __builtin_amdgcn_readfirstlane(p.table[(int64_t)b * p.max_pages + pi]);
      ok = page >= 0 && page < p.num_pages;
      unit = ok ? page : 0;
      row = n0 - pi * p.page_size;
    }
    const int n_rows = ok ? min(32, k_hi - n0) : 0;
    const uint8_t* kp = p.k.codes + unit * p.k.sb + (int64_t)hkv * p.k.sh + (int64_t)row * p.k.ss;
    const uint8_t* vp = p.v.codes + unit * p.v.sb + (int64_t)hkv * p.v.sh + (int64_t)row * p.v.ss;
    const int blk = row / p.block;
    ks_n = ok ? p.k.scales[unit * p.k.cb + (int64_t)hkv * p.k.ch + (int64_t)blk * p.k.cs] : 0.f;
    vs_n = ok ? p.v.scales[unit * p.v.cb + (int64_t)hkv * p.v.ch + (int64_t)blk * p.v.cs] : 0.f;
    ok_n = ok;
    const buf_rsrc kr = make_rsrc(kp, n_rows > 0 ? (int)((n_rows - 1) * p.k.ss + p.D) : 0);
    const buf_rsrc vr = make_rsrc(vp, n_rows > 0 ? (int)((n_rows - 1) * p.v.ss + p.D) : 0);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const bool in = 64 * j + 16 * g < p.D;
        kreg[kb][j] = buffer_load_b128(
            kr, in ? k_off0 + (uint32_t)(16 * kb * (int)p.k.ss + 64 * j) : kBufferOob);
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t off =
          v_in ? v_off0 + (uint32_t)((e < 4 ? e : e + 12) * (int)p.v.ss) : kBufferOob;
      if constexpr (VW == 1) {
        vreg[e][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(vr, off, 0, 0);
      } else if constexpr (VW == 2) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vr, off, 0, 0));
        vreg[e][0] = w[0], vreg[e][1] = w[1];
      } else {
        const u32x4 w = buffer_load_b128(vr, off);
#pragma unroll
        for (int i = 0; i < 4; ++i) vreg[e][i] = w[i];
      }
    }
  };

  for (int n0 = k_lo + 32 * wave; n0 < k_hi; n0 += 32 * NW) {
    load_tile(n0);
    const float kscale = ks_n * p.scale_log2, vscale = vs_n;
    f32x4 sacc[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) sacc[c][0] = sacc[c][1] = f32x4{};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = kreg[kb][j][2 * h], w1 = kreg[kb][j][2 * h + 1];
          const u32x4 a = {widen2<M, C>(w0, 0), widen2<M, C>(w0, 1), widen2<M, C>(w1, 0),
                           widen2<M, C>(w1, 1)};
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int u = TERMS - 1; u >= 0; --u)
              sacc[c][kb] = mfma16<M>(a, qreg[c][2 * j + h][u], sacc[c][kb]);
        }
    uint32_t pk[NC][4][TERMS];
    float alpha[NC];
    const bool masked = !ok_n || n0 + 32 > k_hi || n0 + 32 > full;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = sacc[c][i >> 2][i & 3] * kscale;
      if (masked) {
        const int end = ok_n ? min(lim[c], k_hi) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n0 + 16 * (i >> 2) + 4 * g + (i & 3) >= end) e[i] = kNegInf;
      }
      float mt = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])),
                       fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = xhalf_max(mt);
      const float m_new = fmaxf(m_run[c], mt);
      const float m_sub = m_new == kNegInf ? 0.f : m_new;
      alpha[c] = fast_exp2(m_run[c] - m_sub);
      m_run[c] = m_new;
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = fast_exp2(e[i] - m_sub);
        ps += e[i];
        if constexpr (kFold) e[i] *= vscale;
      }
      l_run[c] = l_run[c] * alpha[c] + ps;
#pragma unroll
      for (int i = 0; i < 4; ++i) split2<M, TERMS>(e[2 * i], e[2 * i + 1], pk[c][i]);
#pragma unroll
      for (int i = 0; i < VB; ++i) oacc[c][i] *= alpha[c];
    }
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 a0, a1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x, y;
          widen_col2<M, C>(vreg[2 * i][w], vreg[2 * i + 1][w], h, x, y);
          a0[i] = x, a1[i] = y;
        }
        const int blk = 4 * w + 2 * h;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
          for (int u = TERMS - 1; u >= 0; --u) {
            const u32x4 pb = {pk[c][0][u], pk[c][1][u], pk[c][2][u], pk[c][3][u]};
            if constexpr (kFold) {
              oacc[c][blk] = mfma16<M>(a0, pb, oacc[c][blk]);
              oacc[c][blk + 1] = mfma16<M>(a1, pb, oacc[c][blk + 1]);
            } else {
              oacc[c][blk] += vscale * mfma16<M>(a0, pb, f32x4{});
              oacc[c][blk + 1] += vscale * mfma16<M>(a1, pb, f32x4{});
            }
          }
        }
      }
  }

  // Merge the four waves' sums: a row's common maximum M, then O and l scaled by
  // 2^(m - M) and added in wave order.
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
    const float fw = mm == kNegInf ? 1.f : fast_exp2(m_run[c] - mm);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < VB; i += 4)
        *reinterpret_cast<f32x4*>(&red_o[wave][c16][VB * (4 * g + r) + i]) =
            f32x4{oacc[c][i][r], oacc[c][i + 1][r], oacc[c][i + 2][r], oacc[c][i + 3][r]} * fw;
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
      const bool live = r < p.rows && t < ql;
      const float inv = lrow > 0.f ? 1.f / lrow : (lrow == 0.f ? 0.f : lrow);
      if (r < p.rows) {
        float x[VB];
#pragma unroll
        for (int i = 0; i < VB; i += 4) {
          f32x4 s = *reinterpret_cast<const f32x4*>(&red_o[0][rr][d0 + i]);
#pragma unroll
          for (int w = 1; w < NW; ++w) s += *reinterpret_cast<const f32x4*>(&red_o[w][rr][d0 + i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i + e] = live ? s[e] * inv : 0.f;
        }
        if (p.num_splits == 1) {
          if (d0 < p.D) {
            const int hq = hkv * p.group + (r - t * p.group);
            const int64_t at = (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh + (int64_t)t * p.o_ss + d0;
            if constexpr (std::is_same<T, float>::value) {
#pragma unroll
              for (int i = 0; i < VB; i += 4)
                *reinterpret_cast<f32x4*>((float*)p.o + at + i) =
                    f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            } else {
#pragma unroll
              for (int i = 0; i < VB; i += 4)
                *reinterpret_cast<u32x2*>((uint16_t*)p.o + at + i) =
                    u32x2{pack2<T>(x[i], x[i + 1]), pack2<T>(x[i + 2], x[i + 3])};
            }
          }
        } else {
          const int64_t row = (((int64_t)b * p.Hkv + hkv) * p.rows + r) * p.num_splits + split;
          float* po = p.part_o + row * p.dpad + d0;
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            *reinterpret_cast<f32x4*>(po + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
          if ((tid & 15) == 0)
            p.part_lse[row] = !live || lrow == 0.f ? kNegInf
                              : mrow == kNegInf    ? lrow
                                                   : mrow + __log2f(lrow);
        }
      }
    }
    __syncthreads();
  }
}

// Merge the splits of one row (query token, head): weights 2^(lse - max) over
// the splits that saw a key, summed in split order.
template <class T>
__global__ void __launch_bounds__(256) q8_combine_kernel(Q8AttnParams p) {
  const int64_t row = blockIdx.x;
  const int r = (int)(row % p.rows);
  const int64_t bh = row / p.rows;
  const int hkv = (int)(bh % p.Hkv);
  const int b = (int)(bh / p.Hkv);
  const int t = r / p.group;
  const int hq = hkv * p.group + (r - t * p.group);
  const float* lse = p.part_lse + row * p.num_splits;
  const float* po = p.part_o + row * p.num_splits * p.dpad;
  float mx = kNegInf;
  for (int s = 0; s < p.num_splits; ++s) mx = fmaxf(mx, lse[s]);
  const int d = threadIdx.x;
  if (d >= p.D) return;
  float acc = 0.f, den = 0.f;
  for (int s = 0; s < p.num_splits; ++s) {
    const float l = lse[s];
    if (l == kNegInf) continue;
    const float w = fast_exp2(l - (mx == kNegInf ? 0.f : mx));
    den += w;
    acc += w * po[(int64_t)s * p.dpad + d];
  }
  const float x = den == 0.f ? 0.f : acc / den;
  const int64_t at = (int64_t)b * p.o_sb + (int64_t)hq * p.o_sh + (int64_t)t * p.o_ss + d;
  if constexpr (std::is_same<T, float>::value)
    ((float*)p.o)[at] = x;
  else
    ((uint16_t*)p.o)[at] = (uint16_t)(pack2<T>(x, x) & 0xffffu);
}

int q8_dpad(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

static int q8_cols(int dtype, int D, int rows) {
  const int most = dtype == SK_F32 || D > 128 ? 1 : 4;
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
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

template <class T, class C, int DP, int NC>
static hipError_t launch_nc(const Q8AttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * p.num_splits * p.row_blocks));
  if (p.table)
    hipLaunchKernelGGL((q8_attn_kernel<T, C, DP, NC, true>), grid, dim3(kQ8Waves * 64), 0, s, p);
  else
    hipLaunchKernelGGL((q8_attn_kernel<T, C, DP, NC, false>), grid, dim3(kQ8Waves * 64), 0, s, p);
  return hipGetLastError();
}

template <class T, class C>
static hipError_t launch_tc(int dtype, const Q8AttnParams& p, hipStream_t s) {
  const int nc = q8_cols(dtype, p.D, p.rows);
  if constexpr (std::is_same<T, float>::value) {
    if (p.D <= 64) return launch_nc<T, C, 64, 1>(p, s);
    if (p.D <= 128) return launch_nc<T, C, 128, 1>(p, s);
    return launch_nc<T, C, 256, 1>(p, s);
  } else {
    if (p.D <= 64)
      return nc == 1   ? launch_nc<T, C, 64, 1>(p, s)
             : nc == 2 ? launch_nc<T, C, 64, 2>(p, s)
                       : launch_nc<T, C, 64, 4>(p, s);
    if (p.D <= 128)
      return nc == 1   ? launch_nc<T, C, 128, 1>(p, s)
             : nc == 2 ? launch_nc<T, C, 128, 2>(p, s)
                       : launch_nc<T, C, 128, 4>(p, s);
    return launch_nc<T, C, 256, 1>(p, s);
  }
}

template <class T>
static hipError_t launch_t(int dtype, int code, const Q8AttnParams& p, hipStream_t s) {
  hipError_t e = code == kCodeI8 ? launch_tc<T, I8>(dtype, p, s) : launch_tc<T, E4M3>(dtype, p, s);
  if (e != hipSuccess || p.num_splits == 1) return e;
  hipLaunchKernelGGL(q8_combine_kernel<T>, dim3((unsigned)((int64_t)p.B * p.Hkv * p.rows)),
                     dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_q8_attn(int dtype, int code, const Q8AttnParams& p, hipStream_t s) {
  if (dtype == SK_F32) return launch_t<float>(dtype, code, p, s);
  if (dtype == SK_F16) return launch_t<F16>(dtype, code, p, s);
  return launch_t<BF16>(dtype, code, p, s);
}

}  // namespace sk
