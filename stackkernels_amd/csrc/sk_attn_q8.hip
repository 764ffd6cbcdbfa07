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
//   largest), rotated ones are rounded once to 11 bits.  fp32 queries and rotated
//   fp16 ones are the sum of two such numbers (22 bits).
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
// wave takes 32 keys at a time through LDS of its own, which loads fill that pass no
// register: the next tile is on its way while one is worked on, and no wave waits for
// another before the end.  (Loads into registers instead: 804 us for 655 at 64 x 8 heads
// x 32,768 keys, D = 128, where the second wave of a SIMD did not fit.)
// * Row 4 a + b of a 16-row operand block of K is key 4 b + a, so that group g's four
//   results are keys 4 b + g and each load of V below covers whole rows.
// * K: lane (key r, group g) brings the 16 bytes 64 j + 16 g of its key's row and
//   reads them back itself, two k-steps of eight consecutive head-dim columns; Q is
//   laid out to match.
// * V: rows as they are; lane (m, group g) reads columns [VB m, VB m + VB) (VB = DP /
//   16) of the eight keys whose probabilities group g holds; output block c is then
//   the columns VB m + c, so the transposition V^T needs is a byte selection.
// The waves of a workgroup take tiles in turn and merge their sums in LDS.
//
// What bounds it: long caches of many rows HBM (64 x 8 KV heads x 32,768 keys, D = 128:
// 4.3 GB of codes in 673 us, 6.4 TB/s); few or short ones the chain of one tile, loads,
// scores, maximum, probabilities, sums, about 1 us an iteration at D = 128.
#include <type_traits>
#include <utility>

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
  const int t_first = p.group_div.quot(row0);
  const int t_last = min(p.group_div.quot(min(row0 + n_rows, p.rows) - 1), s.ql - 1);
  s.hi = p.causal ? min(s.len, s.len - s.ql + t_last + 1) : s.len;
  if (t_first >= s.ql) s.hi = 0;
  s.hi = max(s.hi, 0);
  s.full = p.causal ? s.len - s.ql + t_first + 1 : s.len;
  return s;
}

// f(0), f(1), ..., f(N - 1) with compile-time arguments.
template <class F, int... I>
__device__ __forceinline__ void static_for_impl(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

constexpr float kMinFactor = 1e-35f;  // of a score: keeps a masked -inf a -inf

// How a tile's scores x (log2 units) become probabilities of one row: e = 2^(x +
// offset) are the fp16 operands, in units of 2^m2; to_l takes their sum to the units
// of l.  lost: the tile's V scale is so small (or 0) next to others that its operands
// are all 0 in fp16; offset is then -inf, and l takes the sum of 2^(x + l_offset).
struct Q8Weight {
  float offset, to_l, l_offset;
  bool lost;
};

// Running references of one row: m of the scores x, m2 of x + log2 t (t: the V
// scale), l = sum of 2^(x - m).  -inf while no key was seen.
struct Q8Ref {
  float m = kNegInf, m2 = kNegInf, l = 0.f;
  // mt, mt2: the tile's maxima.  True for a wave where some row's references rise,
  // by more than kRescaleLog2 (smaller excesses only make e larger than 1): ao is
  // then the factor of the row's sums.
  __device__ __forceinline__ bool raise(float mt, float mt2, float& ao) {
    if (!__any(exceeded(mt, mt2))) return false;
    ao = raised(mt, mt2);
    return true;
  }
  __device__ __forceinline__ bool exceeded(float mt, float mt2) const {
    return mt > m + kRescaleLog2 || mt2 > m2 + kRescaleLog2;
  }
  __device__ __forceinline__ float raised(float mt, float mt2) {
    const float m_new = fmaxf(m, mt), m2_new = fmaxf(m2, mt2);
    l *= m_new == kNegInf ? 1.f : fast_exp2(m - m_new);
    const float ao = m2_new == kNegInf ? 1.f : fast_exp2(m2 - m2_new);
    m = m_new, m2 = m2_new;
    return ao;
  }
  // lv: log2 of the tile's V scale.  (A row that has seen no key has only -inf
  // scores, whose e is 0 for any finite offset.)
  __device__ __forceinline__ Q8Weight weight(float lv) const {
    const float ms = m == kNegInf ? 0.f : m, m2s = m2 == kNegInf ? 0.f : m2;
    Q8Weight w;
    const float lw = lv + ms - m2s;  // log2 of an operand of a score m
    w.lost = lw < -90.f;
    w.offset = w.lost ? kNegInf : lv - m2s;
    w.to_l = w.lost ? 1.f : fast_exp2(-lw);
    w.l_offset = -ms;
    return w;
  }
};

// The query row of a lane as matrix operands: k-step s takes the eight columns from
// col(s), divided by 2^(exponent of the row's largest element), which is spread
// over the lanes that reduce() joins.  Returns the row's score factor.
template <int KS, int TERMS, class Col, class Reduce>
__device__ __forceinline__ float q8_query(const Q8AttnParams& p, int b, int hkv, int r, int ql,
                                          Col col, Reduce reduce, u32x4 (&out)[KS][TERMS]) {
  const int half = p.D >> 1;
  const int t = p.group_div.quot(r);
  const bool live = r < p.rows && t < ql;
  const int64_t at = live ? (int64_t)b * p.q_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.q_sh +
                                (int64_t)t * p.q_ss
                          : 0;
  const int rr = rope_row(p.rope, b, t);
  float x[KS][8];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d0 = col(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[s][e] = 0.f;
    if (live && d0 < p.D) load_q8x8(p.q, p.dtype, at + d0, x[s]);
  }
  if (rr >= 0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = col(s);
      if (live && d0 < p.D) {
        float y[8], cs[8], sn[8];
        load_q8x8(p.q, p.dtype, at + (d0 < half ? d0 + half : d0 - half), y);
        rope_coeffs<8>(p.rope, rr, d0, cs, sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = rope_mix(x[s][e], y[e], d0 < half, cs[e], sn[e]);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[s][e]));
  top = reduce(top);
  int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
  if (ex > 127) ex = 0;  // an infinity: the row's scores are not finite anyway
  const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[TERMS];
      split2<TERMS>(sign * __builtin_amdgcn_ldexpf(x[s][2 * i], -ex),
                    sign * __builtin_amdgcn_ldexpf(x[s][2 * i + 1], -ex), u);
#pragma unroll
      for (int k = 0; k < TERMS; ++k) out[s][k][i] = u[k];
    }
  return __builtin_amdgcn_ldexpf(fabsf(p.scale_log2), ex);
}

// max / sum of a value across the lanes l and l ^ 16 (as xhalf_max: v_permlane16_swap
// leaves a row of 16 lanes' own value in one result and the next row's in the other).
__device__ __forceinline__ float xrow_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x),
                                                  __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float xrow_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x),
                                                  __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// What a workgroup does: row block rb of piece split of the keys of (b, hkv), the
// blocks that share keys next to one another on one XCD.
struct Q8Item {
  int rb, split, hkv, b;
};
__device__ __forceinline__ Q8Item q8_item(const Q8AttnParams& p) {
  Q8Item w;
  const int i = xcd_work_index(blockIdx.x, gridDim.x);
  const int j = p.block_rows_div.quot(i);
  w.rb = i - j * p.row_blocks;
  const int k = p.split_div.quot(j);
  w.split = j - k * p.num_splits;
  w.b = p.hkv_div.quot(k);
  w.hkv = k - w.b * p.Hkv;
  return w;
}

// Until at most N loads are in flight.  (Also a fence to the compiler: what the wave
// reads from LDS behind it stays behind it.)
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Waves of a workgroup: eight, sharing the queries in LDS, where the sums take half
// the registers.
template <int DP, int NC>
constexpr int q8_waves() {
  return NC * DP > 256 ? 8 : 4;
}
// Tiles in flight per wave: two of 4 KB, one of 8 KB or more, where a CU's other
// workgroups keep it loading.  (Two of 8 KB: 64 query heads of one KV head, 8 x 100,000
// keys 65 us for 60; 300 x 8 heads x 300 keys 57 for 42; 32 x 8 heads, up to 4,096 keys
// each, 43 for 41; only 64 x 8 heads x 32,768 keys gain, 655 for 673.  One of 4 KB: 16 x
// 8 heads x 3,000 keys, 40 rows 43 us for 38.)
template <int DP>
constexpr int q8_stages() {
  return DP > 64 ? 1 : 2;
}

// Column blocks whose queries are read from LDS each tile (the waves share them): with
// more than 32 head-dim-128 columns the sums alone take 128 registers, and the queries
// would take the second wave of a SIMD.
template <int DP, int NC>
constexpr bool q8_q_in_lds() {
  return NC * DP > 256;
}

// QT, PT: fp16 terms of a query element, of a probability.
template <class C, int QT, int PT, int DP, int NC, int NW, bool PAGED>
__global__ void __launch_bounds__(NW * 64, 2) q8_attn_kernel(Q8AttnParams p) {
  constexpr int KC = DP / 64;   // 16-byte chunks of a K row per lane
  constexpr int KS = DP / 32;   // k-steps of S^T
  constexpr int VB = DP / 16;   // bytes of a V row per lane = output blocks
  constexpr int VW = VB / 4;
  constexpr bool kQLds = q8_q_in_lds<DP, NC>();
  // Where registers allow: V is taken from LDS before the softmax, and a score's
  // products run in two chains.
  constexpr bool kEarly = NC * DP * QT <= 256;
  constexpr int CH = NC == 1 ? 2 : 1;

  constexpr int ST = q8_stages<DP>();
  constexpr int KBYTES = 32 * DP;            // codes of K (and of V) of a tile
  constexpr int LK = KBYTES / 1024;          // loads of them, 16 bytes a lane each
  constexpr int STAGE = 2 * KBYTES;
  constexpr int RING = NW * ST * STAGE;
  constexpr int OUT = NW * 16 * (DP + 4) * 4;  // (the merge reuses the ring)
  __shared__ float red_m[NW][16 * NC];
  __shared__ float red_l[NW][16 * NC];
  __shared__ __attribute__((aligned(1024))) uint8_t ring[RING > OUT ? RING : OUT];
  __shared__ float meta[NW][ST][4];  // of a stage: k's and v's scale, a page
  __shared__ u32x4 qs[kQLds ? NC * KS * QT : 1][64];
  __shared__ float qmul_s[kQLds ? NC : 1][64];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15;
  const int g = lane >> 4;

  const Q8Item item = q8_item(p);
  const int rb = item.rb, split = item.split, hkv = item.hkv, b = item.b;

  const int row0 = rb * 16 * NC;
  const Q8Span sp = q8_span(p, b, row0, 16 * NC);
  const int kps = (p.split_div.quot(sp.hi + p.num_splits - 1) + 31) / 32 * 32;
  const int k_lo = split * kps;
  const int k_hi = min(sp.hi, k_lo + kps);

  int lim[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    lim[c] = min(p.causal ? sp.len - sp.ql + p.group_div.quot(row0 + 16 * c + c16) + 1 : sp.len, k_hi);

  // This lane's pieces of a tile.  K: load (kb, j) brings the 16 bytes the lane itself
  // multiplies, which it finds at its own place again.  V: row by row.
  const uint32_t k_off = (uint32_t)((4 * (c16 & 3) + (c16 >> 2)) * (int)p.k.ss + 16 * g);
  constexpr int LPR = DP / 16;  // lanes per row of V
  const uint32_t v_off = 16 * (lane % LPR) < p.D
                             ? (uint32_t)(lane / LPR * (int)p.v.ss + 16 * (lane % LPR))
                             : kBufferOob;
  uint8_t* const my = ring + wave * ST * STAGE;
  const uint32_t my_lds = __builtin_amdgcn_readfirstlane((int)lds_addr(my));
  const uint32_t meta_lds = __builtin_amdgcn_readfirstlane((int)lds_addr(&meta[wave][0][0]));
  const bool once = p.row_blocks == 1;  // read by this workgroup alone: past the caches

  // Of tile it: its place in k, v and their scales, from its page.  With K of a tile
  // come its two scales and the page of the tile that takes its stage next, 4 bytes
  // each, so that the loop has no load whose wait could hold up another's.
  struct Tile {
    int64_t k, v;      // first elements
    int64_t ks, vs;
    int rows;          // visible keys, 0 past the last one and in a page outside the pool
  };
  const int64_t unit0 = PAGED ? 0 : b;
  const int64_t k_base = unit0 * p.k.sb + (int64_t)hkv * p.k.sh;
  const int64_t v_base = unit0 * p.v.sb + (int64_t)hkv * p.v.sh;
  const int64_t ks_base = unit0 * p.k.cb + (int64_t)hkv * p.k.ch;
  const int64_t vs_base = unit0 * p.v.cb + (int64_t)hkv * p.v.ch;
  const int* const table = PAGED ? p.table + (int64_t)b * p.max_pages : nullptr;
  const int k_end = max(k_hi - 1, 0);
  auto key_of = [&](int it) SK_INLINE { return k_lo + 32 * (wave + NW * it); };
  auto page_at = [&](int it) SK_INLINE { return p.page_div.quot(min(key_of(it), k_end)); };
  auto tile_of = [&](int it, int page) SK_INLINE {
    const int n = key_of(it);
    const bool ok = n < k_hi && (!PAGED || (page >= 0 && page < p.num_pages));
    const uint32_t unit = PAGED && ok ? (uint32_t)page : 0u;
    const uint32_t row = (uint32_t)(PAGED ? n - p.page_div.quot(n) * p.page_size : n);
    const uint32_t blk = (uint32_t)p.block_div.quot((int)row);
    Tile t;
    t.k = k_base + (int64_t)((uint64_t)unit * (uint32_t)p.k.sb + (uint64_t)row * (uint32_t)p.k.ss);
    t.v = v_base + (int64_t)((uint64_t)unit * (uint32_t)p.v.sb + (uint64_t)row * (uint32_t)p.v.ss);
    t.ks = ks_base + (int64_t)((uint64_t)unit * (uint32_t)p.k.cb + (uint64_t)blk * (uint32_t)p.k.cs);
    t.vs = vs_base + (int64_t)((uint64_t)unit * (uint32_t)p.v.cb + (uint64_t)blk * (uint32_t)p.v.cs);
    t.rows = ok ? min(32, k_hi - n) : 0;
    return t;
  };
  // Loads of a tile into stage st: every tile the same number, so the waits below
  // count them.  A range that ends with the last visible row gives zeros for the rows
  // past it.  reused: the wave's own reads of the stage come first.
  constexpr int GK = LK + 2 + (PAGED ? 1 : 0), GV = LK;
  auto load_k = [&](int it, const Tile& t, int st, auto reused) SK_INLINE {
    const i32x4 r = uniform_words(
        make_rsrc_words(p.k.codes + t.k, t.rows > 0 ? (t.rows - 1) * (int)p.k.ss + p.D : 0));
    const i32x4 rk = uniform_words(make_rsrc_words(p.k.scales + t.ks, t.rows > 0 ? 4 : 0));
    const i32x4 rv = uniform_words(make_rsrc_words(p.v.scales + t.vs, t.rows > 0 ? 4 : 0));
    const uint32_t to = my_lds + st * STAGE;
    if constexpr (decltype(reused)::value) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < LK; ++i) {
      const int j = i % KC, kb = i / KC;
      const uint32_t off = 64 * j + 16 * g < p.D ? k_off + (uint32_t)(16 * kb * (int)p.k.ss + 64 * j)
                                                 : kBufferOob;
      if (once)
        buffer_load_lds_b128_nt(r, to + i * 1024, off);
      else
        buffer_load_lds_b128(r, to + i * 1024, off);
    }
    if (lane == 0) {
      const uint32_t mt = meta_lds + st * 16;
      buffer_load_lds_b32(rk, mt, 0);
      buffer_load_lds_b32(rv, mt + 4, 0);
      if constexpr (PAGED)
        buffer_load_lds_b32(uniform_words(make_rsrc_words(table + page_at(it + ST), 4)), mt + 8, 0);
    }
  };
  auto load_v = [&](const Tile& t, int st, auto reused) SK_INLINE {
    const i32x4 r = uniform_words(
        make_rsrc_words(p.v.codes + t.v, t.rows > 0 ? (t.rows - 1) * (int)p.v.ss + p.D : 0));
    const uint32_t to = my_lds + st * STAGE + KBYTES;
    if constexpr (decltype(reused)::value) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < LK; ++i) {
      const uint32_t off = v_off == kBufferOob ? v_off : v_off + (uint32_t)(i * (64 / LPR) * (int)p.v.ss);
      if (once)
        buffer_load_lds_b128_nt(r, to + i * 1024, off);
      else
        buffer_load_lds_b128(r, to + i * 1024, off);
    }
  };

  const int n_it = k_hi > k_lo + 32 * wave ? (k_hi - k_lo - 32 * wave + 32 * NW - 1) / (32 * NW) : 0;
  int rows_t[ST] = {};  // of the tiles in the ring, oldest first
  if (n_it > 0) {
    int page[ST];
#pragma unroll
    for (int i = 0; i < ST; ++i)
      page[i] = PAGED ? __builtin_amdgcn_readfirstlane(table[page_at(i)]) : 0;
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const Tile t = tile_of(i, page[i]);
      rows_t[i] = t.rows;
      load_k(i, t, i, std::false_type{});
      load_v(t, i, std::false_type{});
    }
  }

  // Q^T operand: k-step s = 2 j + h of lane group g is head-dim columns 64 j +
  // 16 g + 8 h .. + 7, divided by 2^(exponent of the row's largest element).
  u32x4 qreg[kQLds ? 1 : NC][KS][QT];
  float qmul[NC];
  if (k_lo < k_hi) {
    auto col = [&](int s) SK_INLINE { return 64 * (s >> 1) + 16 * g + 8 * (s & 1); };
    auto reduce = [](float x) SK_INLINE { return xhalf_max(xrow_max(x)); };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int r = row0 + 16 * c + c16;
      if constexpr (kQLds) {
        if (c % NW != wave) continue;
        qmul_s[c][lane] = q8_query<KS, QT>(p, b, hkv, r, sp.ql, col, reduce, qreg[0]);
#pragma unroll
        for (int i = 0; i < KS * QT; ++i)
          qs[c * KS * QT + i][lane] = qreg[0][i / QT][i % QT];
      } else {
        qmul[c] = q8_query<KS, QT>(p, b, hkv, r, sp.ql, col, reduce, qreg[c]);
      }
    }
    if constexpr (kQLds) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c) qmul[c] = qmul_s[c][lane];
    }
  }

  f32x4 oacc[NC][VB];
  Q8Ref ref[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < VB; ++i) oacc[c][i] = f32x4{};

  int st = 0;
  for (int it = 0; it < n_it; ++it) {
    const int n0 = key_of(it);
    const uint8_t* const kt = my + st * STAGE;
    const uint8_t* const vt = kt + KBYTES;
    // K(it) has landed: behind it at most V(it) and the other stages' loads.
    wait_loads<GV + (ST - 1) * (GK + GV)>();
    const float* const mt_at = &meta[wave][st][0];
    const float ks = mt_at[0], vs = mt_at[1];
    const int page = PAGED ? __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mt_at[2])) : 0;
    const bool ok = !PAGED || rows_t[0] > 0;
    const Tile next = tile_of(it + ST, page);
#pragma unroll
    for (int i = 0; i + 1 < ST; ++i) rows_t[i] = rows_t[i + 1];
    rows_t[ST - 1] = next.rows;
    f32x4 sacc[NC][2], chain[NC][2][CH];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 2 * CH; ++i) chain[c][i & 1][i >> 1] = f32x4{};
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      u32x4 raw[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        raw[kb] = *reinterpret_cast<const u32x4*>(kt + (kb * KC + j) * 1024 + lane * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 a[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t w0 = raw[kb][2 * h], w1 = raw[kb][2 * h + 1];
          a[kb] = u32x4{widen2<C, 0>(w0), widen2<C, 1>(w0), widen2<C, 0>(w1), widen2<C, 1>(w1)};
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int u = QT - 1; u >= 0; --u) {
            u32x4 q;
            if constexpr (kQLds)
              q = qs[(c * KS + 2 * j + h) * QT + u][lane];
            else
              q = qreg[c][2 * j + h][u];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
              chain[c][kb][h % CH] = mfma16<F16>(a[kb], q, chain[c][kb][h % CH]);
          }
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        sacc[c][kb] = CH == 1 ? chain[c][kb][0] : chain[c][kb][0] + chain[c][kb][CH - 1];
    load_k(it + ST, next, st, std::true_type{});

    uint32_t vreg[8][VW];
    auto read_v = [&]() SK_INLINE {
      // V(it) has landed: behind it the other stages' loads and K(it + ST).
      wait_loads<(ST - 1) * (GK + GV) + GK>();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint8_t* const at = vt + (4 * e + g) * DP + VB * c16;
        if constexpr (VW == 1) {
          vreg[e][0] = *reinterpret_cast<const uint32_t*>(at);
        } else if constexpr (VW == 2) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(at);
          vreg[e][0] = w[0], vreg[e][1] = w[1];
        } else {
          const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
          for (int i = 0; i < 4; ++i) vreg[e][i] = w[i];
        }
      }
      load_v(next, st, std::true_type{});
    };
    if constexpr (kEarly) read_v();

    const bool masked = !ok || n0 + 32 > k_hi || n0 + 32 > sp.full;
    const float lv = __builtin_amdgcn_logf(vs);  // log2
    uint32_t pk[NC][4][PT];
    // All blocks' maxima first and one test for all of them: their chains then run
    // side by side.
    float mul[NC], mt[NC];
    bool above = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      mul[c] = fmaxf(ks * qmul[c], kMinFactor);
      if (masked) {
        const int end = ok ? lim[c] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n0 + 4 * i + g >= end) sacc[c][i >> 2][i & 3] = kNegInf;
      }
      const f32x4 &a = sacc[c][0], &b = sacc[c][1];
      mt[c] = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])));
      mt[c] = xhalf_max(xrow_max(mt[c])) * mul[c];
      above |= ref[c].exceeded(mt[c], mt[c] + lv);
    }
    if (__any(above)) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float ao = ref[c].raised(mt[c], mt[c] + lv);
#pragma unroll
        for (int i = 0; i < VB; ++i) oacc[c][i] *= ao;
      }
    }
    Q8Weight w[NC];
    bool lost = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      w[c] = ref[c].weight(lv);
      lost |= w[c].lost;
    }
    if (__any(lost)) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float ps = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ps += fast_exp2(fmaf(sacc[c][i >> 2][i & 3], mul[c], w[c].l_offset));
        ref[c].l += w[c].lost ? ps : 0.f;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = fast_exp2(fmaf(sacc[c][i >> 2][i & 3], mul[c], w[c].offset));
      ref[c].l += (((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]))) * w[c].to_l;
#pragma unroll
      for (int i = 0; i < 4; ++i) split2<PT>(e[2 * i], e[2 * i + 1], pk[c][i]);
    }
    if constexpr (!kEarly) read_v();
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
        for (int u = PT - 1; u >= 0; --u) {
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
    st = st + 1 == ST ? 0 : st + 1;
  }
  wait_loads<0>();  // the loads past the last tile write zeros to the ring

  float(*const red_o)[DP + 4] = reinterpret_cast<float(*)[DP + 4]>(ring);
  // Merge the four waves' sums: a row's common maximum M, then O scaled by 2^(m2 -
  // M) and l by 2^(m - M), added in wave order.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float l = xhalf_sum(xrow_sum(ref[c].l));
    if (g == 0) {
      red_m[wave][16 * c + c16] = ref[c].m;
      red_l[wave][16 * c + c16] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float mm = red_m[0][16 * c + c16];
#pragma unroll
    for (int w = 1; w < NW; ++w) mm = fmaxf(mm, red_m[w][16 * c + c16]);
    const float f = mm == kNegInf || ref[c].m2 == kNegInf ? 1.f : fast_exp2(ref[c].m2 - mm);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < VB; i += 4)
        *reinterpret_cast<f32x4*>(&red_o[wave * 16 + c16][VB * (4 * g + r) + i]) =
            f32x4{oacc[c][i][r], oacc[c][i + 1][r], oacc[c][i + 2][r], oacc[c][i + 3][r]} * f;
    __syncthreads();
    // 16 threads per row, DP / 16 columns each.
    if (tid < 256) {
      const int rr = tid >> 4;
      const int d0 = (tid & 15) * VB;
      const int r = row0 + 16 * c + rr;
      float mrow = kNegInf, lrow = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) mrow = fmaxf(mrow, red_m[w][16 * c + rr]);
#pragma unroll
      for (int w = 0; w < NW; ++w)
        lrow += red_l[w][16 * c + rr] * (mrow == kNegInf ? 1.f : fast_exp2(red_m[w][16 * c + rr] - mrow));
      const int t = p.group_div.quot(r);
      const bool live = r < p.rows && t < sp.ql;
      const float inv = lrow == 0.f ? 0.f : 1.f / lrow;  // (NaN stays NaN)
      if (r < p.rows) {
        const int64_t row = (((int64_t)b * p.Hkv + hkv) * p.rows + r) * p.num_splits + split;
        const int64_t at = (int64_t)b * p.o_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.o_sh +
                           (int64_t)t * p.o_ss + d0;
#pragma unroll
        for (int i = 0; i < VB; i += 4) {
          f32x4 s = *reinterpret_cast<const f32x4*>(&red_o[rr][d0 + i]);
#pragma unroll
          for (int w = 1; w < NW; ++w) s += *reinterpret_cast<const f32x4*>(&red_o[w * 16 + rr][d0 + i]);
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = live ? s[e] * inv : 0.f;
          if (p.num_splits > 1)
            *reinterpret_cast<f32x4*>(p.part_o + row * DP + d0 + i) = f32x4{x[0], x[1], x[2], x[3]};
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

// Many rows: a workgroup of eight waves takes 256 rows of a KV head, 32 per wave,
// and shares each tile of 8192 / DP keys, whose codes it widens to fp16 once, in
// LDS.  S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16.
// * Pipeline: the body of a 32-key part u multiplies S(u + 1) and O += V(u) P(u), one
//   MFMA a slot, and spreads over those slots the softmax of part u and a share of
//   the widening: during tile t, K(t + 2) and then V(t + 1) go from registers into
//   the LDS buffer that the tile before has read (three for K, two for V, one barrier
//   a tile); the codes after those are loaded as the registers fall free.  Each slot
//   is fenced, so the matrix unit waits for no long stretch of other work.
// * V is widened in columns: a thread takes four columns of four keys and writes
//   four rows of V^T, the keys in the order in which a lane of S^T's result holds
//   them (0-3, 8-11 | 4-7, 12-15 of each 16).
// * Rows of K and V^T are padded by 16 bytes: the 16 rows of an operand read lie in
//   distinct banks.  A wave writes V^T in 16 rows four apart, 16 bytes each; chunk c
//   of row d stands at c ^ (d / 16 % 4), which spreads those too, is the same for the
//   16 rows of a read and, for a lane, one register and constants.  (Without it the
//   writes made 45% of the LDS cycles conflicts.)
// * Page ids and scales come through vector loads a tile or more ahead: scalar ones
//   would make every LDS wait wait for them.
// Against the kernel above a code is widened once per 256 rows, not per 64.  Bound by
// power: 2 x up to 4,096 tokens of 32 heads against up to 16,384 keys, D = 128, paged
// (876 GFLOP): 1.2 to 1.4 ms, 610 to 730 TFLOP/s, the matrix unit 47% and the vector
// unit 57% busy at about 1.7 GHz; 512 tokens against 16,000 keys 0.15 ms.
template <int DP>
struct Q8Big {
  static constexpr int BN = 8192 / DP;   // keys per tile
  static constexpr int NH = BN / 32;     // 32-key parts, each with its own scales
  static constexpr int KSTR = DP + 8;    // fp16 per K row
  static constexpr int VSTR = BN + 8;    // fp16 per V^T row
};

constexpr int kQ8BigWaves = 8;
constexpr int kQ8BigRows = 32 * kQ8BigWaves;

// PARTS: pages a tile may lie in (1: contiguous caches, pages of whole tiles).
template <class C, int QT, int DP, bool PAGED, int PARTS>
__global__ void __launch_bounds__(kQ8BigWaves * 64) q8_big_kernel(Q8AttnParams p) {
  using L = Q8Big<DP>;
  constexpr int NT = kQ8BigWaves * 64;
  constexpr int BN = L::BN, NH = L::NH, KSTR = L::KSTR, VSTR = L::VSTR;
  constexpr int PK = BN / PARTS;  // keys per part with an address of its own
  constexpr int KS = DP / 16;     // k-steps of S^T
  constexpr int DB = DP / 32;     // output blocks
  constexpr int CPK = DP / 16;    // 16-byte pieces of a K row's codes: one per thread
  constexpr int DC = DP / 4;      // 4-byte pieces of a V row's codes
  static_assert(BN * CPK == NT && BN / 4 * DC == NT, "one piece of K and four of V per thread");
  __shared__ __attribute__((aligned(16))) uint16_t ksm[3][BN * KSTR];
  __shared__ __attribute__((aligned(16))) uint16_t vsm[2][DP * VSTR];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31;
  const int hi2 = lane >> 5;

  const Q8Item item = q8_item(p);
  const int rb = p.row_blocks - 1 - item.rb;  // (causal: longest first)
  const int split = item.split, hkv = item.hkv, b = item.b;

  const int row0 = rb * kQ8BigRows;
  const Q8Span sp = q8_span(p, b, row0, kQ8BigRows);
  const int kps = (p.split_div.quot(sp.hi + p.num_splits - 1) + BN - 1) / BN * BN;
  const int k_lo = split * kps;
  const int k_hi = min(sp.hi, k_lo + kps);
  const int n_tiles = k_hi > k_lo ? (k_hi - k_lo + BN - 1) / BN : 0;
  const int r = row0 + 32 * wave + c32;
  const int t = p.group_div.quot(r);
  const int lim = min(p.causal ? sp.len - sp.ql + t + 1 : sp.len, k_hi);
  // Tiles this wave's rows see, and keys that all of them see.
  const int w0 = row0 + 32 * wave;
  int w_tiles = 0, w_full = sp.len;
  if (w0 < p.rows && p.group_div.quot(w0) < sp.ql) {
    const int last = min(p.group_div.quot(min(w0 + 32, p.rows) - 1), sp.ql - 1);
    const int w_hi = p.causal ? min(sp.len - sp.ql + last + 1, k_hi) : k_hi;
    w_tiles = w_hi > k_lo ? (w_hi - k_lo + BN - 1) / BN : 0;
    if (p.causal) w_full = sp.len - sp.ql + p.group_div.quot(w0) + 1;
  }

  // Where the codes of this KV head start (contiguous caches: of this row's too).
  const int64_t unit0 = PAGED ? 0 : b;
  const uint8_t* const kbase = p.k.codes + unit0 * p.k.sb + (int64_t)hkv * p.k.sh;
  const uint8_t* const vbase = p.v.codes + unit0 * p.v.sb + (int64_t)hkv * p.v.sh;
  const uint32_t ksb = (uint32_t)p.k.sb, vsb = (uint32_t)p.v.sb;  // (paged: below 2^32)
  const uint32_t kss = (uint32_t)p.k.ss, vss = (uint32_t)p.v.ss;

  // Lane j < 2 NH reads the scale of part j % NH: k's below NH, v's from there.
  const int spart = lane % NH;
  // Page of the lane's part of tile it (any page past the last key's).
  const buf_rsrc table = make_rsrc(PAGED ? p.table + (int64_t)b * p.max_pages : nullptr,
                                   PAGED ? p.max_pages * 4 : 0);
  auto lane_key = [&](int it) SK_INLINE { return min(k_lo + it * BN + 32 * spart, k_hi - 1); };
  auto load_page = [&](int it) SK_INLINE {
    if constexpr (!PAGED) return 0;
    return (int)__builtin_amdgcn_raw_buffer_load_b32(table, (uint32_t)p.page_div.quot(lane_key(it)) * 4, 0, 0);
  };
  auto settled_page = [&](int page) SK_INLINE {
    return PARTS == 1 ? __builtin_amdgcn_readfirstlane(page) : page;
  };
  auto in_pool = [&](int page) SK_INLINE { return !PAGED || (page >= 0 && page < p.num_pages); };
  auto load_scale = [&](int it, int page) SK_INLINE {
    const int n = lane_key(it);
    const int row = PAGED ? n - p.page_div.quot(n) * p.page_size : n;
    const uint32_t unit = PAGED ? (in_pool(page) ? (uint32_t)page : 0u) : (uint32_t)b;
    const uint32_t blk = (uint32_t)p.block_div.quot(row);
    const bool is_v = lane / NH % 2;
    const float* const base = is_v ? p.v.scales + (int64_t)hkv * p.v.ch : p.k.scales + (int64_t)hkv * p.k.ch;
    return base[(uint64_t)unit * (uint32_t)(is_v ? p.v.cb : p.k.cb) +
                (uint64_t)blk * (uint32_t)(is_v ? p.v.cs : p.k.cs)];
  };
  // Resource of part h of tile it: its keys below k_hi, none past the last tile or
  // in a page outside the pool.
  auto part_rsrc = [&](const uint8_t* base, uint32_t sb, uint32_t ss, int it, int h, int page) SK_INLINE {
    const int n = k_lo + it * BN + h * PK;
    int rows = max(min(PK, k_hi - n), 0);
    uint64_t at = (uint64_t)(uint32_t)n * ss;
    if constexpr (PAGED) {
      const int pg = PARTS == 1 ? page : __builtin_amdgcn_readlane(page, h * (NH / PARTS));
      rows = in_pool(pg) ? rows : 0;
      at = (uint64_t)(in_pool(pg) ? (uint32_t)pg : 0u) * sb +
           (uint64_t)(uint32_t)(n - p.page_div.quot(n) * p.page_size) * ss;
    }
    return make_rsrc(base + at, rows > 0 ? (rows - 1) * (int)ss + p.D : 0);
  };

  u32x4 kraw;
  uint32_t vraw[4];
  const int krow = tid / CPK, kcol = 16 * (tid % CPK);
  const int kpart = PARTS == 1 ? 0 : __builtin_amdgcn_readfirstlane(krow / PK);
  const uint32_t koff = kcol < p.D ? (uint32_t)((krow & (PK - 1)) * (int)kss + kcol) : kBufferOob;
  // The thread's V: positions 4 vq .. 4 vq + 3, keys vkey .. vkey + 3 of the tile.
  const int vq = 4 * (wave / (DC / 16)) + lane / 16, vcol = 64 * (wave % (DC / 16)) + 4 * (lane % 16);
  const int vkey = 16 * (vq >> 2) + 8 * (vq & 1) + 4 * (vq >> 1 & 1);
  const int vpart = PARTS == 1 ? 0 : __builtin_amdgcn_readfirstlane(vkey / PK);
  const uint32_t voff = vcol < p.D ? (uint32_t)((vkey & (PK - 1)) * (int)vss + vcol) : kBufferOob;
  auto load_k = [&](int it, int page) SK_INLINE {
    kraw = buffer_load_b128(part_rsrc(kbase, ksb, kss, it, kpart, page), koff);
  };
  auto load_v = [&](int it, int page) SK_INLINE {
    const buf_rsrc rs = part_rsrc(vbase, vsb, vss, it, vpart, page);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      vraw[e] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, voff, e * (int)vss, 0);
  };
  // Widening in steps, into buffer offsets kb and vb (fp16): K in eight (two codes
  // each), V in four (two keys' two columns).
  u32x4 kw;
  u32x2 vw[2];
  uint16_t* const kto = &ksm[0][krow * KSTR + kcol];
  uint16_t* const vto = &vsm[0][vcol * VSTR + 8 * ((vq >> 1) ^ (vcol / 16 % 4)) + 4 * (vq & 1)];
  auto widen_k = [&](int kb, auto step) SK_INLINE {
    constexpr int st = decltype(step)::value;
    kw[st & 3] = widen2<C, (st & 1)>(kraw[st >> 1]);
    if constexpr ((st & 3) == 3) *reinterpret_cast<u32x4*>(kto + kb + 2 * (st - 3)) = kw;
  };
  auto widen_v = [&](int vb, auto step) SK_INLINE {
    constexpr int st = decltype(step)::value, hf = st >> 1, i = st & 1;
    uint32_t c0, c1;
    widen_cols<C, hf>(vraw[2 * i], vraw[2 * i + 1], c0, c1);
    vw[0][i] = c0, vw[1][i] = c1;
    if constexpr (i == 1) {
#pragma unroll
      for (int c = 0; c < 2; ++c) *reinterpret_cast<u32x2*>(vto + vb + (2 * hf + c) * VSTR) = vw[c];
    }
  };

  u32x4 q[KS][QT];
  f32x16 oacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) oacc[i] = f32x16{};
  Q8Ref ref;
  float qmul = 0.f;
  // Scales of tile t's parts, settled when t is next: k's, and log2 of v's (0 and
  // -inf: no such page); ok: parts whose page lies in the pool.
  float ks_t[NH], lv_t[NH];
  uint32_t ok_t = 0;
  auto settle_scales = [&](float sv, int page) SK_INLINE {
    sv = in_pool(page) ? sv : 0.f;
    const float lv = __builtin_amdgcn_logf(sv);  // log2
    ok_t = (1u << NH) - 1;
    if constexpr (PAGED) {
      if constexpr (PARTS == 1)
        ok_t = in_pool(page) ? ok_t : 0u;
      else
        ok_t &= (uint32_t)__ballot(in_pool(page));
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      ks_t[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sv), h));
      lv_t[h] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lv), NH + h));
    }
  };

  // Of the part whose scores are next: factor, operand offset, factor of the sum.
  float mul = 0.f, off = 0.f, to_l = 0.f;
  // Mask the scores of part h of the tile at n0 where some are hidden (mx: their raw
  // maximum), raise the references.
  auto settle = [&](int n0, auto part, f32x16& sc, float mx) SK_INLINE {
    constexpr int h = decltype(part)::value;
    const bool ok = ok_t >> h & 1;
    if (!ok || n0 + 32 * h + 32 > w_full || n0 + 32 * h + 32 > k_hi) {
      const int end = (ok ? lim : 0) - n0 - 32 * h - 4 * hi2;
      mx = kNegInf;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (8 * (i >> 2) + (i & 3) >= end) sc[i] = kNegInf;
        mx = fmaxf(mx, sc[i]);
      }
    }
    mul = fmaxf(ks_t[h] * qmul, kMinFactor);
    mx = xhalf_max(mx) * mul;
    float ao;
    if (ref.raise(mx, mx + lv_t[h], ao)) {
#pragma unroll
      for (int i = 0; i < DB; ++i) oacc[i] *= ao;
    }
    const Q8Weight w = ref.weight(lv_t[h]);
    off = w.offset, to_l = w.to_l;
    if (__any(w.lost)) {
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ps += fast_exp2(fmaf(sc[i], mul, w.l_offset));
      ref.l += w.lost ? ps : 0.f;
    }
  };

  constexpr int NS = KS;        // score MFMAs of a part
  constexpr int NO = 2 * DB;    // output MFMAs
  constexpr int NM = NS + NO;
  constexpr int NG = 8;         // pairs of scores a lane holds
  // MFMAs an operand is read ahead of its own.
  constexpr int KLEAD = 4, OLEAD = NS < 6 ? NS : 6;
  constexpr int FL = NS + DB - 4;  // first slot of the last pair
  constexpr int KST = 16 / NH, VST = 8 / NH;  // widening steps of a body that has some
  static_assert(FL > 0 && NM >= KST && NM >= VST && KLEAD <= NS && OLEAD <= NS, "slots");

  const uint16_t* const kfrom = &ksm[0][c32 * KSTR + 8 * hi2];
  const uint16_t* const vfrom = &vsm[0][c32 * VSTR + 8 * (hi2 ^ (c32 / 16))];

  // Body of part h (scores sc) of a tile: kr, vr: buffer offsets of the next part's
  // tile in K and of this tile in V; kb, vb: of the tiles being widened.  nx: the
  // next part's scores, mx their raw maximum.  kNow, kNext: this wave sees this
  // part's tile, the next part's.
  auto body = [&](auto part, auto now, auto next, int kr, int vr, int kb, int vb, const f32x16& sc,
                  f32x16& nx, float& mx) SK_INLINE {
    constexpr bool kNow = decltype(now)::value, kNext = decltype(next)::value;
    constexpr int h = decltype(part)::value, hn = (h + 1) % NH;
    u32x4 a[NS], vt[NO], pk[2];
    float y[2 * NG], e[2 * NG], ps = 0.f;
    auto read_k = [&](int i) SK_INLINE { return lds_read_b128(kfrom + kr + hn * 32 * KSTR + 16 * i); };
    auto read_v = [&](int j) SK_INLINE {
      const int blk = j % DB;  // (rows 32 blk + c32: chunk 4 h + 2 (j / DB) + hi2)
      return lds_read_b128(vfrom + vr + blk * 32 * VSTR + 32 * h + 16 * (j / DB ^ blk % 2));
    };
    mx = kNegInf;
    if constexpr (kNext) {
#pragma unroll
      for (int i = 0; i < KLEAD; ++i) a[i] = read_k(i);
      nx = f32x16{};
    }
    static_for<NM>([&](auto ic) SK_INLINE {
      constexpr int i = decltype(ic)::value;
      if constexpr (kNext && i + KLEAD < NS) a[i + KLEAD] = read_k(i + KLEAD);
      if constexpr (kNow && i + OLEAD >= NS && i + OLEAD - NS < NO)
        vt[i + OLEAD - NS] = read_v(i + OLEAD - NS);
      if constexpr (i < NS) {
        if constexpr (kNext) {
#pragma unroll
          for (int k = QT - 1; k >= 0; --k) nx = mfma32<F16>(a[i], q[i][k], nx);
        }
      } else if constexpr (kNow) {
        constexpr int j = i - NS;
        oacc[j % DB] = mfma32<F16>(vt[j], pk[j / DB], oacc[j % DB]);
      }
      if constexpr (kNow)
        static_for<NG>([&](auto gc) SK_INLINE {
          constexpr int g = decltype(gc)::value, f = g * FL / (NG - 1);
          if constexpr (f == i) {
            y[2 * g] = fmaf(sc[2 * g], mul, off);
            y[2 * g + 1] = fmaf(sc[2 * g + 1], mul, off);
          }
          if constexpr (f + 1 == i) {
            e[2 * g] = fast_exp2(y[2 * g]);
            e[2 * g + 1] = fast_exp2(y[2 * g + 1]);
          }
          if constexpr (f + 2 == i) {
            ps += e[2 * g] + e[2 * g + 1];
            pk[g >> 2][g & 3] = pack2<F16>(e[2 * g], e[2 * g + 1]);
            asm volatile("" : "+v"(ps));
          }
        });
      // K in the first half of a tile's parts, V in the second.
      if constexpr (h < NH / 2)
        static_for<KST>([&](auto st) SK_INLINE {
          if constexpr (decltype(st)::value * NM / KST == i)
            widen_k(kb, std::integral_constant<int, h * KST + decltype(st)::value>{});
        });
      else
        static_for<VST>([&](auto st) SK_INLINE {
          if constexpr (decltype(st)::value * NM / VST == i)
            widen_v(vb, std::integral_constant<int, (h - NH / 2) * VST + decltype(st)::value>{});
        });
      // The maximum of the new scores, from two slots behind their last MFMA.
      if constexpr (kNext && i >= NS)
        static_for<NG>([&](auto uc) SK_INLINE {
          constexpr int u = decltype(uc)::value, at = NS + 2 + u * (NO - 2) / NG;
          if constexpr (at == i) {
            mx = fmaxf(mx, fmaxf(nx[2 * u], nx[2 * u + 1]));
            asm volatile("" : "+v"(mx));
          }
        });
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (kNow) ref.l += ps * to_l;
  };

  if (n_tiles > 0) {
    constexpr int KB = BN * KSTR, VB = DP * VSTR;  // fp16 per buffer
    // Pages of tiles 0 .. 3, then K(0), V(0), scales 0 and 1, K(1).
    int pg0 = load_page(0), pg1 = load_page(1), pg2 = load_page(2), pg3 = load_page(3);
    pg0 = settled_page(pg0), pg1 = settled_page(pg1), pg2 = settled_page(pg2), pg3 = settled_page(pg3);
    load_k(0, pg0);
    load_v(0, pg0);
    const float sv0 = load_scale(0, pg0);
    float sv = load_scale(1, pg1);
    qmul = q8_query<KS, QT>(
        p, b, hkv, r, sp.ql, [&](int s) SK_INLINE { return 16 * s + 8 * hi2; },
        [](float x) SK_INLINE { return xhalf_max(x); }, q);
    static_for<8>([&](auto st) SK_INLINE { widen_k(0, st); });
    load_k(1, pg1);
    static_for<4>([&](auto st) SK_INLINE { widen_v(0, st); });
    load_v(1, pg1);
    static_for<8>([&](auto st) SK_INLINE { widen_k(KB, st); });
    load_k(2, pg2);
    __syncthreads();
    f32x16 sa = {}, sb;
    float mx = kNegInf;
    settle_scales(sv0, pg0);
    if (w_tiles > 0) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 a = lds_read_b128(kfrom + 16 * s);
#pragma unroll
        for (int k = QT - 1; k >= 0; --k) sa = mfma32<F16>(a, q[s][k], sa);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sa[i]);
      settle(k_lo, std::integral_constant<int, 0>{}, sa, mx);
    }
    // At tile t: k0, k1, k2: K buffers of t, t + 1 and of t + 2, being written; v0, v1:
    // V's of t and t + 1, being written; sv: scales of t + 1, pg1 .. pg3: pages of t +
    // 1 .. t + 3.
    int k0 = 0, k1 = KB, k2 = 2 * KB, v0 = 0, v1 = VB;
    auto tile = [&](int it, auto now, auto next) SK_INLINE {
      constexpr bool kNow = decltype(now)::value;
      const int n0 = k_lo + it * BN;
      const int pg4 = load_page(it + 4);
      const float sv2 = load_scale(it + 2, pg2);
      static_for<NH>([&](auto part) SK_INLINE {
        constexpr int h = decltype(part)::value;
        if constexpr (h + 1 < NH) {
          // The next part lies in this tile.
          if constexpr (h % 2 == 0)
            body(part, now, now, k0, v0, k2, v1, sa, sb, mx);
          else
            body(part, now, now, k0, v0, k2, v1, sb, sa, mx);
          if constexpr (kNow) {
            std::integral_constant<int, h + 1> after;
            if constexpr (h % 2 == 0)
              settle(n0, after, sb, mx);
            else
              settle(n0, after, sa, mx);
          }
        } else {
          static_assert(NH % 2 == 0, "a tile starts with its scores in sa");
          body(part, now, next, k1, v0, k2, v1, sb, sa, mx);
          settle_scales(sv, pg1);
          if constexpr (decltype(next)::value)
            settle(n0 + BN, std::integral_constant<int, 0>{}, sa, mx);
        }
        if constexpr (h == NH / 2 - 1) load_k(it + 3, pg3);
        if constexpr (h == NH - 1) load_v(it + 2, pg2);
      });
      sv = sv2;
      pg1 = pg2, pg2 = pg3, pg3 = settled_page(pg4);
      const int kx = k0;
      k0 = k1, k1 = k2, k2 = kx;
      const int vx = v0;
      v0 = v1, v1 = vx;
      __syncthreads();
    };
    // Tiles with another behind them, the wave's last one, and those that only other
    // waves see (past the last tile nothing is loaded; zeros are widened).
    int it = 0;
    for (; it + 1 < w_tiles; ++it) tile(it, std::true_type{}, std::true_type{});
    if (it < w_tiles) tile(it++, std::true_type{}, std::false_type{});
    for (; it < n_tiles; ++it) tile(it, std::false_type{}, std::false_type{});
  }

  const float l = xhalf_sum(ref.l);
  if (r >= p.rows) return;
  const bool live = t < sp.ql;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // (NaN stays NaN)
  const float f = !live ? 0.f : ref.m2 == kNegInf ? inv : fast_exp2(ref.m2 - ref.m) * inv;
  const int64_t row = (((int64_t)b * p.Hkv + hkv) * p.rows + r) * p.num_splits + split;
  const int64_t at = (int64_t)b * p.o_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.o_sh + (int64_t)t * p.o_ss;
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * i + 8 * j + 4 * hi2;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = live ? oacc[i][4 * j + e] * f : 0.f;
      if (p.num_splits > 1)
        *reinterpret_cast<f32x4*>(p.part_o + row * DP + d) = f32x4{x[0], x[1], x[2], x[3]};
      else if (d < p.D)
        store_o4(p.o, p.dtype, at + d, x);
    }
  if (p.num_splits > 1 && hi2 == 0)
    p.part_lse[row] = !live || l == 0.f ? kNegInf : ref.m == kNegInf ? l : ref.m + __log2f(l);
}

// Merge the splits of a row (query token, head): weights 2^(lse - max) of the splits
// that saw a key, sums over lanes of 16 bytes of columns.  WPR waves take a row, DP /
// 4 lanes a split; the first eight partials of each lane are on their way while the
// weights are made.  Few splits: one wave a row; from 17 on: four.
template <int DP, int WPR>
__global__ void __launch_bounds__(256) q8_combine_kernel(Q8AttnParams p) {
  constexpr int LPG = DP / 4;            // lanes per split
  constexpr int G = 64 / LPG * WPR;      // splits at a time
  constexpr int PRE = 8;
  __shared__ float w[4][kQ8MaxSplits];
  __shared__ f32x4 part[WPR > 1 ? 4 : 1][LPG];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int row = blockIdx.x * (4 / WPR) + (WPR > 1 ? 0 : wave);  // (below 2^31: host check)
  const int bh = p.rows_div.quot(row);
  if (bh >= p.B * p.Hkv) return;
  const int ns = p.num_splits;
  const float* lse = p.part_lse + (int64_t)row * ns;
  const float* po = p.part_o + (int64_t)row * ns * DP + (lane % LPG) * 4;
  const int first = lane / LPG + (WPR > 1 ? wave * (64 / LPG) : 0);
  f32x4 pre[PRE];
#pragma unroll
  for (int k = 0; k < PRE; ++k) {
    const int s = first + k * G;
    pre[k] = s < ns ? *reinterpret_cast<const f32x4*>(po + (int64_t)s * DP) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
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
  // (Each wave reads the weights it wrote itself: in order.  A split that saw no key
  // has written no sums: whatever stands there is left out, not multiplied by 0.)
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < PRE; ++k) {
    const int s = first + k * G;
    const float x = s < ns ? w[wave][s] : 0.f;
    if (x != 0.f) acc += x * pre[k];
  }
  for (int s = first + PRE * G; s < ns; s += G) {
    const float x = w[wave][s];
    if (x != 0.f) acc += x * *reinterpret_cast<const f32x4*>(po + (int64_t)s * DP);
  }
#pragma unroll
  for (int o = LPG; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o);
  if constexpr (WPR > 1) {
    if (lane < LPG) part[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    if (lane < LPG) acc = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
  }
  const int d = (lane % LPG) * 4;
  if (lane >= LPG || d >= p.D) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int r = row - bh * p.rows;
  const int64_t b = p.hkv_div.quot(bh);
  const int hkv = bh - (int)b * p.Hkv;
  const int t = p.group_div.quot(r);
  const float x[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
  store_o4(p.o, p.dtype,
           b * p.o_sb + (int64_t)(hkv * p.group + r - t * p.group) * p.o_sh + (int64_t)t * p.o_ss + d, x);
}

template <int DP>
static hipError_t launch_combine(const Q8AttnParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.B * p.Hkv * p.rows;
  if (p.num_splits > 16)
    hipLaunchKernelGGL((q8_combine_kernel<DP, 4>), dim3((unsigned)rows), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((q8_combine_kernel<DP, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
  return hipGetLastError();
}

int q8_dpad(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Whether a query element takes two fp16 terms: fp32 queries, and fp16 ones that are
// rotated (which one term would round a second time, to the precision of the result:
// twice its error over long rows).  bf16 results are coarser than one term.
static bool q8_two_terms(int dtype, bool rotated) {
  return dtype == SK_F32 || (dtype == SK_F16 && rotated);
}

// Column blocks of 16 rows that a workgroup takes: as many as the registers of a lane
// hold the sums of.  One block against two and four, each with its best split count:
// 64 rows, D = 128, 8 x 100,000 keys of one KV head 129, 91 and 64 us; 64 rows, D = 64,
// 64 x 8,000 keys 98, 66 and 40; 40 rows, D = 64, 16 x 8 heads x about 3,000 keys: 39 in
// three blocks, 45 in four.  (With more, fp32 queries and D > 128 would spill.)
static int q8_cols(int dtype, int D, int rows) {
  const int most = D > 128 ? 1 : dtype == SK_F32 ? 2 : 4;
  const int want = rows <= 16 ? 1 : (rows + 15) / 16;
  return want < most ? want : most;
}

// Whether the kernel of many rows runs (16-bit queries): from 65 rows of a KV head
// on.  8 KV heads of D = 128, each with its best split count, first kernel and this
// one: 16 x 8,000 keys 61 and 94 us at 32 rows, 81 and 110 at 64, 117 and 118 at 96, 121
// and 131 at 128, 222 and 187 at 256; 1 x 16,000 keys 20 and 23, 28 and 24, 30 and 27,
// 31 and 29, 42 and 41.
static bool q8_big(int dtype, int D, int rows) {
  return dtype != SK_F32 && D <= 128 && rows > 64;
}

int q8_rows_per_block(int dtype, int D, int rows) {
  return q8_big(dtype, D, rows) ? kQ8BigRows : 16 * q8_cols(dtype, D, rows);
}

int q8_splits(int dtype, int B, int Hkv, int rows, int keys, int D) {
  const int per = q8_rows_per_block(dtype, D, rows);
  const int64_t units = (int64_t)B * Hkv * ((rows + per - 1) / per);
  if (units <= 0) return 1;
  if (q8_big(dtype, D, rows)) {
    // Rounds of the 256 CUs (one workgroup each) times a piece's tiles and the fixed
    // cost of a workgroup and of a row's partials, in tiles.
    const int tiles = (int)(((int64_t)keys * (D <= 64 ? 64 : 128) + 8191) / 8192);
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && (s == 1 || 2 * s <= tiles); ++s) {
      const double rounds = (double)((units * s + 255) / 256);
      const double cost = rounds * ((double)((tiles + s - 1) / s) + 6) + (s > 1 ? 4 + units * s / 64.0 : 0);
      if (cost < least) least = cost, best = s;
    }
    return best;
  }
  // Microseconds, from times of 40 shapes over 1 to 128 splits: a workgroup's iteration
  // (32 keys a wave) takes `step`; a CU gets through its workgroups one after the other,
  // or in three quarters of that where registers and LDS let it hold several; 1.5 + nc is
  // a workgroup's own cost; a quarter of its time is lost at the end, where CUs finish
  // unevenly; splits cost the second kernel and the partials' traffic.  The count it
  // takes came within 10% of the best one's time.
  const int nc = per / 16, dp = q8_dpad(D), waves = nc * dp > 256 ? 8 : 4;
  const bool shares = dp == 64 || (dp == 128 && nc <= 2);
  const double step = (dp == 64 ? 0.76 : dp == 256 ? 1.84 : nc == 1 ? 1.3 : 1.12) *
                      (1 + 0.3 * (nc - 1)) * (waves == 8 ? 1.4 : 1.0);
  const int tiles = (keys + 31) / 32;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 128 && (s == 1 || s <= tiles / 2); ++s) {
    const double run = ((tiles + s - 1) / s + waves - 1) / waves * step;
    const double held = (double)((units * s + 255) / 256);
    const double cost = (shares ? 0.25 + 0.75 * held : held) * (run + 1.5 + nc) + 0.25 * run +
                        (s > 1 ? 3 + (double)B * Hkv * rows * s * dp * 2.5e-6 : 0);
    if (cost < 0.99 * least) least = cost, best = s;
  }
  return best;
}

template <class C, int QT, int PT, int DP, int NC>
static hipError_t launch_nc(const Q8AttnParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * p.num_splits * p.row_blocks));
  constexpr int NW = q8_waves<DP, NC>();
  if (p.table)
    hipLaunchKernelGGL((q8_attn_kernel<C, QT, PT, DP, NC, NW, true>), grid, dim3(NW * 64), 0, s, p);
  else
    hipLaunchKernelGGL((q8_attn_kernel<C, QT, PT, DP, NC, NW, false>), grid, dim3(NW * 64), 0, s, p);
  return hipGetLastError();
}

template <class C, int QT, int PT, int DP>
static hipError_t launch_dp(const Q8AttnParams& p, hipStream_t s) {
  const int nc = q8_cols(p.dtype, p.D, p.rows);
  if (nc == 1) return launch_nc<C, QT, PT, DP, 1>(p, s);
  if constexpr (DP <= 128)
    if (nc == 2) return launch_nc<C, QT, PT, DP, 2>(p, s);
  if constexpr (DP <= 128 && PT == 1)
    if (nc == 3) return launch_nc<C, QT, PT, DP, 3>(p, s);
  if constexpr (DP <= 128 && PT == 1)
    if (nc == 4) return launch_nc<C, QT, PT, DP, 4>(p, s);
  return hipErrorInvalidValue;
}

template <class C, int QT, int DP>
static hipError_t launch_big(const Q8AttnParams& p, hipStream_t s) {
  using L = Q8Big<DP>;
  const dim3 block(kQ8BigWaves * 64);
  const dim3 grid((unsigned)((int64_t)p.B * p.Hkv * p.num_splits * p.row_blocks));
  if (!p.table) {
    hipLaunchKernelGGL((q8_big_kernel<C, QT, DP, false, 1>), grid, block, 0, s, p);
    return hipGetLastError();
  }
  if (p.page_size % L::BN != 0)
    hipLaunchKernelGGL((q8_big_kernel<C, QT, DP, true, L::NH>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((q8_big_kernel<C, QT, DP, true, 1>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <class C, int QT, int PT>
static hipError_t launch_ct(const Q8AttnParams& p, hipStream_t s) {
  if constexpr (PT == 1)
    if (q8_big(p.dtype, p.D, p.rows))
      return p.D <= 64 ? launch_big<C, QT, 64>(p, s) : launch_big<C, QT, 128>(p, s);
  if (p.D <= 64) return launch_dp<C, QT, PT, 64>(p, s);
  if (p.D <= 128) return launch_dp<C, QT, PT, 128>(p, s);
  return launch_dp<C, QT, PT, 256>(p, s);
}

hipError_t launch_q8_attn(int code, const Q8AttnParams& p0, hipStream_t s) {
  Q8AttnParams p = p0;
  p.group_div = FastDiv(p.group);
  p.rows_div = FastDiv(p.rows);
  p.hkv_div = FastDiv(p.Hkv);
  p.split_div = FastDiv(p.num_splits);
  p.block_rows_div = FastDiv(p.row_blocks);
  const bool two = q8_two_terms(p.dtype, p.rope.cos != nullptr);
  auto launch = [&](auto c) {
    using C = decltype(c);
    return p.dtype == SK_F32 ? launch_ct<C, 2, 2>(p, s) : two ? launch_ct<C, 2, 1>(p, s) : launch_ct<C, 1, 1>(p, s);
  };
  const hipError_t e = code == kCodeI8 ? launch(I8{}) : launch(E4M3{});
  if (e != hipSuccess || p.num_splits == 1) return e;
  return p.dpad == 64 ? launch_combine<64>(p, s) : p.dpad == 128 ? launch_combine<128>(p, s) : launch_combine<256>(p, s);
}

}  // namespace sk
