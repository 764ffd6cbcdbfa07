// Writing a cache held in 8-bit codes, and the page plan of a serving step.
//
// Append.  A block of block_size tokens of a KV head has one scale s; the value
// of a code c is s c.  New values x of a block ask for
//   int8: amax / 127;  e4m3: the smallest power of two 2^e with amax 2^-e <= 448
// (amax over the finite ones; at least 2^-126), and the block takes s' = that,
// or the larger of that and s where the block already holds tokens.  New codes
// are round(x * (1 / s')), saturated; where s' > s the older codes become
// round(c * (s / s')).  In e4m3 that factor is a power of two, so older codes
// keep their value exactly down to the subnormal range: moving a block's scale
// several times costs no more than moving it once.  In int8 each move rounds
// once more, by at most half a step of the new scale.
//
// One workgroup owns a (batch row, block, KV head, k or v): amax, scale and codes
// need no atomics and results do not depend on order.  Bound by the new tokens'
// bytes (2 or 4 in, 1 out per element) and by the rotation's entries, 8 bytes per
// element of K, from the caches; the older codes of a block are read only when its
// scale grows.  8 x 2,048 tokens, 8 heads, D = 128, fp16, ragged lengths (59 MB, 11.4
// us as a copy): 20.4 us, 15.4 unrotated (31.2 and 23.5 with each element of K read
// twice and every element's infinity and NaN looked for one by one; 21.7 with a
// block's heads on all XCDs).  One token: 5.3 us, a launch and two dependent loads.
#include <type_traits>

#include "sk_common.h"
#include "sk_q8.h"
#include "sk_rope.h"

namespace sk {

constexpr float kTinyScale = 1.17549435e-38f;  // 2^-126

template <int CODE>
__device__ __forceinline__ float needed_scale(float amax) {
  if constexpr (CODE == kCodeI8) {
    return fmaxf(amax * (1.f / 127.f), kTinyScale);
  } else {
    // amax = 1.m x 2^(e - 127): 448 = 1.75 x 2^8, so the exponent to divide by
    // is e - 127 - 8, one more where 1.m > 1.75.
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, 1);
    return __builtin_bit_cast(float, (uint32_t)e << 23);
  }
}

// Four scaled values as four codes, nearest (ties to even), saturated.  NaN: code
// 0 in int8 (which has none), NaN in e4m3.  FINITE: none is infinite or NaN, and
// none exceeds the largest code by more than its scale's rounding, so that nothing
// needs saturating: in int8 the sum with 1.5 2^23 leaves the rounded number's low
// byte in place.
template <int CODE, bool FINITE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (CODE == kCodeI8) {
    float x[4] = {a, b, c, d};
    if constexpr (FINITE) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        asm("" : "+v"(x[i]));  // (a rounded product, never fused into the sum)
        u[i] = __builtin_bit_cast(uint32_t, x[i] + 12582912.f);
      }
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u),
                                   __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = x[i] == x[i] ? fminf(fmaxf(x[i], -127.f), 127.f) : 0.f;
      w |= ((uint32_t)(int)__builtin_rintf(y) & 0xffu) << (8 * i);
    }
    return w;
  } else {
    auto sat = [](float y) SK_INLINE {
      return FINITE ? y : y == y ? fminf(fmaxf(y, -448.f), 448.f) : y;
    };
    uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), w, true);
  }
}

template <int CODE>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (CODE == kCodeI8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)((w >> (8 * i)) & 0xffu);
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  }
}

// Eight elements at p as fp32.
template <class T>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    const f32x4* p = reinterpret_cast<const f32x4*>((const float*)base + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const u32x4 a = ldg_b128_cached((const uint16_t*)base + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = a[i];
      x[2 * i] = to_f32<T>((uint16_t)(w & 0xffffu));
      x[2 * i + 1] = to_f32<T>((uint16_t)(w >> 16));
    }
  }
}

// A thread takes pairs of eight columns, d .. d + 7 and D / 2 + d .. + 7 of a token:
// what a rotation mixes, each element read once.  The first KEEP pairs of a thread
// stay in registers between the pass for amax and the pass that writes codes; a
// larger block re-reads the rest.  (Five waves a SIMD cost two spilled registers and
// gain 3% over four.)
template <class T, int CODE, int NT, int KEEP>
__global__ void __launch_bounds__(NT, KEEP == 2 ? 5 : 3) q8_append_kernel(Q8AppendParams p) {
  __shared__ float red[2][NT / 64];
  const int tid = threadIdx.x;
  // The 2 Hkv workgroups of a block follow one another on one XCD (workgroups go to
  // the eight round robin), which then reads the rotation's entries once.
  const int turn = blockIdx.x >> 3;
  const int kv = turn & 1;
  const int group = p.hkv_div.quot(turn >> 1);
  const int h = (turn >> 1) - group * p.Hkv;
  const int bj = group * 8 + (blockIdx.x & 7);
  if (bj >= p.B * p.blocks) return;
  const int b = p.blocks_div.quot(bj);
  const int j = bj - b * p.blocks;
  const int start = max(__builtin_amdgcn_readfirstlane(p.lens[b]), 0);
  const int n_new = p.news ? min(max(__builtin_amdgcn_readfirstlane(p.news[b]), 0), p.T) : p.T;
  if (n_new == 0 || start >= p.cap) return;
  // Tokens [lo, lo + block) of the row; the new ones among them [a, z).
  const int64_t lo64 = ((int64_t)p.block_div.quot(start) + j) * p.block;
  const int64_t end = min((int64_t)start + n_new, (int64_t)p.cap);
  if (lo64 >= end) return;
  const int lo = (int)lo64;  // (below cap)
  const int a = max(lo, start);
  const int z = (int)min(end, lo64 + p.block);
  int64_t unit = b;
  int row = lo;
  if (p.table) {
    const int at = p.page_div.quot(lo);
    const int page = __builtin_amdgcn_readfirstlane(p.table[(int64_t)b * p.max_pages + at]);
    if (page < 0 || page >= p.num_pages) return;
    unit = page;
    row = lo - at * p.page_size;
  }
  const Q8Cache& c = p.c[kv];
  uint8_t* codes = c.codes + unit * c.sb + (int64_t)h * c.sh + (int64_t)row * c.ss;
  float* scale = c.scales + unit * c.cb + (int64_t)h * c.ch + (int64_t)p.block_div.quot(row) * c.cs;
  const int older = a - lo;
  const int half = p.D >> 1;
  const int ppr = p.D >> 4;  // pairs per token
  const int n = (z - a) * ppr;
  const int t0 = a - start;
  const float had = older > 0 ? *scale : 0.f;
  const int64_t x0 = (int64_t)b * p.x_sb[kv] + (int64_t)h * p.x_sh[kv] + (int64_t)t0 * p.x_ss[kv];
  const int64_t x_ss = p.x_ss[kv];

  auto fetch = [&](int i, float (&x)[2][8]) SK_INLINE {
    const int r = p.pairs_div.quot(i);
    const int d0 = (i - r * ppr) * 8;
    const int64_t at = x0 + r * x_ss + d0;
    load8<T>(p.x[kv], at, x[0]);
    load8<T>(p.x[kv], at + half, x[1]);
    if (kv == 0) {
      const int rr = rope_row(p.rope, b, t0 + r);
      if (rr >= 0) {
        float cs[2][8], sn[2][8];
        rope_coeffs<8>(p.rope, rr, d0, cs[0], sn[0]);
        rope_coeffs<8>(p.rope, rr, d0 + half, cs[1], sn[1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x[0][e], v = x[1][e];
          x[0][e] = rope_mix(u, v, true, cs[0][e], sn[0][e]);
          x[1][e] = rope_mix(v, u, false, cs[1][e], sn[1][e]);
        }
      }
    }
  };
  // amax: of the elements that are numbers.  zero becomes NaN at an infinity or NaN.
  float amax = 0.f, zero = 0.f;
  auto widest = [&](const float (&x)[2][8]) SK_INLINE {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      amax = fmaxf(fmaxf(amax, fabsf(x[0][e])), fabsf(x[1][e]));
      zero = __builtin_fmaf(x[0][e], 0.f, zero);
      zero = __builtin_fmaf(x[1][e], 0.f, zero);
    }
  };
  float keep[KEEP][2][8];
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (tid + i * NT < n) fetch(tid + i * NT, keep[i]);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (tid + i * NT < n) widest(keep[i]);
  for (int i = tid + KEEP * NT; i < n; i += NT) {
    float x[2][8];
    fetch(i, x);
    widest(x);
  }
  // Over the workgroup.
  auto joined = [&](float x, float (&out)[NT / 64]) SK_INLINE {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    if constexpr (NT > 64) {
      if ((tid & 63) == 0) out[tid >> 6] = x;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) x = fmaxf(x, out[w]);
    }
    return x;
  };
  amax = joined(zero == 0.f ? amax : __builtin_inff(), red[0]);
  const bool finite = amax < __builtin_inff();
  if (!finite) {
    // Some elements are not: the largest of those that are.
    amax = 0.f;
    auto widest_finite = [&](const float (&x)[2][8]) SK_INLINE {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float y = fabsf(x[e >> 3][e & 7]);
        amax = y < __builtin_inff() ? fmaxf(amax, y) : amax;
      }
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (tid + i * NT < n) widest_finite(keep[i]);
    for (int i = tid + KEEP * NT; i < n; i += NT) {
      float x[2][8];
      fetch(i, x);
      widest_finite(x);
    }
    amax = joined(amax, red[1]);
  }
  const float need = needed_scale<CODE>(amax);
  const float now = older > 0 && had > need ? had : need;
  const float inv = 1.f / now;
  auto put = [&](int i, const float (&x)[2][8], auto fin) SK_INLINE {
    const int r = p.pairs_div.quot(i);
    uint8_t* at = codes + (int64_t)(older + r) * c.ss + (i - r * ppr) * 8;
    constexpr bool F = decltype(fin)::value;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float (&v)[8] = x[q];
      *reinterpret_cast<u32x2*>(at + q * half) =
          u32x2{encode4<CODE, F>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                encode4<CODE, F>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
    }
  };
  auto write = [&](auto fin) SK_INLINE {
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (tid + i * NT < n) put(tid + i * NT, keep[i], fin);
    for (int i = tid + KEEP * NT; i < n; i += NT) {
      float x[2][8];
      fetch(i, x);
      put(i, x, fin);
    }
  };
  if (finite)
    write(std::true_type{});
  else
    write(std::false_type{});
  if (older > 0 && had < now) {
    const float f = had / now;
    for (int i = tid; i < older * 2 * ppr; i += NT) {
      const int r = p.pairs_div.quot(i >> 1);
      u32x2* at = reinterpret_cast<u32x2*>(codes + (int64_t)r * c.ss + (i - 2 * r * ppr) * 8);
      u32x2 w = *at;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float x[4];
        decode4<CODE>(w[q], x);
        w[q] = encode4<CODE, false>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
      }
      *at = w;
    }
  }
  if constexpr (NT > 64) __syncthreads();  // every thread has read the old scale
  if (tid == 0) *scale = now;
}

template <class T, int CODE>
static hipError_t append_tc(const Q8AppendParams& p0, hipStream_t s) {
  Q8AppendParams p = p0;
  if ((int64_t)p.B * p.blocks * p.Hkv == 0) return hipSuccess;
  p.block_div = FastDiv(p.block);
  p.hkv_div = FastDiv(p.Hkv);
  p.blocks_div = FastDiv(p.blocks);
  p.pairs_div = FastDiv(p.D / 16);
  if (p.table) p.page_div = FastDiv(p.page_size);
  const int64_t pairs = (int64_t)(p.T < p.block ? p.T : p.block) * (p.D / 16);
  const dim3 grid((unsigned)(((int64_t)p.B * p.blocks + 7) / 8 * 16 * p.Hkv));
  // Two pairs a thread (of one wave, or of four), four in the largest blocks: one and
  // four pairs a thread of as many as make up a block took 25.3 and 24.5 us above.
  if (pairs <= 64 * 2)
    hipLaunchKernelGGL((q8_append_kernel<T, CODE, 64, 2>), grid, dim3(64), 0, s, p);
  else if (pairs <= 256 * 2)
    hipLaunchKernelGGL((q8_append_kernel<T, CODE, 256, 2>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((q8_append_kernel<T, CODE, 256, 4>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

template <int CODE>
static hipError_t append_c(int dtype, const Q8AppendParams& p, hipStream_t s) {
  if (dtype == SK_F32) return append_tc<float, CODE>(p, s);
  if (dtype == SK_F16) return append_tc<F16, CODE>(p, s);
  return append_tc<BF16, CODE>(p, s);
}

hipError_t launch_q8_append(int dtype, int code, const Q8AppendParams& p, hipStream_t s) {
  return code == kCodeI8 ? append_c<kCodeI8>(dtype, p, s) : append_c<kCodeE4M3>(dtype, p, s);
}

// ---------------------------------------------------------------- page plan
//
// Rows that grow take pages from the front of the ring of free pages in row
// order, rows that shrink put theirs behind its end in row order: two exclusive
// prefix sums over the batch.  A workgroup sums the rows in front of its own by
// itself (8 bytes a row, from the L2), so one launch needs no order among
// workgroups.  The entries a call reads (table entries that rows hold, ring
// entries in front of the old end) are not the ones it writes (entries past those
// held, ring entries behind the end), and lengths and ring state go to buffers of
// their own: a call with the same inputs gives the same outputs again.
// Bound by a chain of three dependent loads and two scans: 256 rows of a token 6.9 us,
// 48 rows of 8,192 tokens (3.1 MB of slots) 8.1.

constexpr int kPlanThreads = 256;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PlanRow {
  int old_len, grow, po, pn, need, back;
};

__device__ __forceinline__ int pages_of(const PagePlanParams& p, int n) {
  const int q = p.page_div.quot(n);
  return q + (q * p.page_size != n);
}

__device__ __forceinline__ PlanRow plan_row(const PagePlanParams& p, int b) {
  PlanRow r;
  const int cap = p.max_pages * p.page_size;  // (below 2^31: checked on the host)
  const int o = min(max(p.lens[b], 0), cap);
  int64_t want = (int64_t)o + min(p.news[b], p.T);
  want = want < 0 ? 0 : want > cap ? o : want;
  r.old_len = o;
  r.grow = (int)want - o;
  r.po = pages_of(p, o);
  r.pn = pages_of(p, (int)want);
  r.need = max(r.pn - r.po, 0);
  r.back = max(r.po - r.pn, 0);
  return r;
}

// Inclusive prefix sums of x and y over the workgroup's threads; totals in tx, ty.
__device__ __forceinline__ void block_scan2(int& x, int& y, int& tx, int& ty,
                                            int (&red)[2][kPlanWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(x, o), v = __shfl_up(y, o);
    if (lane >= o) x += u, y += v;
  }
  if (lane == 63) red[0][wave] = x, red[1][wave] = y;
  __syncthreads();
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w == wave) x += tx, y += ty;
    tx += red[0][w], ty += red[1][w];
  }
  __syncthreads();
}

// Last of n ascending numbers that is at most i (the first one is).
__device__ __forceinline__ int last_at_most(const int* v, int n, int i) {
  int lo = 0;
  while (n > 1) {
    const int h = n >> 1;
    if (v[lo + h] <= i) lo += h, n -= h;
    else n = h;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PagePlanParams p) {
  __shared__ int red[2][kPlanWaves];
  __shared__ int s_old[kPlanThreads], s_grow[kPlanThreads], s_po[kPlanThreads], s_pn[kPlanThreads];
  __shared__ int s_front[kPlanThreads], s_end[kPlanThreads];
  const int tid = threadIdx.x;
  const int b0 = blockIdx.x * p.rows_per_wg;
  const int nb = min(p.rows_per_wg, p.B - b0);
  int head = p.state[0] % p.N;
  if (head < 0) head += p.N;
  const int count = min(max(p.state[1], 0), p.N);
  PlanRow r{};
  if (tid < nb) r = plan_row(p, b0 + tid);

  // Pages that the rows in front take and give back.
  int need = 0, back = 0;
  if (b0 > 0) {
    for (int b = tid; b < b0; b += kPlanThreads) {
      const PlanRow f = plan_row(p, b);
      need += f.need, back += f.back;
    }
    int tx, ty;
    block_scan2(need, back, tx, ty, red);
    need = tx, back = ty;
  }
  int cum = r.need, end = r.back, all_need, all_back;
  block_scan2(cum, end, all_need, all_back, red);
  const bool granted = r.need == 0 || need + cum <= count;
  if (!granted) r.grow = 0, r.pn = r.po;
  s_old[tid] = r.old_len, s_grow[tid] = r.grow, s_po[tid] = r.po, s_pn[tid] = r.pn;
  s_front[tid] = cum - r.need;
  s_end[tid] = end - r.back;
  __syncthreads();

  // Ring place i behind the front (0 <= i < N).
  auto ring_at = [&](int i) SK_INLINE {
    const uint32_t at = (uint32_t)head + (uint32_t)i;
    return at >= (uint32_t)p.N ? at - (uint32_t)p.N : at;
  };

  if (blockIdx.y == 0) {
    if (tid < nb) p.lens_out[b0 + tid] = r.old_len + r.grow;
    // Pages taken by rows that grow, page by page over the workgroup's rows.
    for (int i = tid; i < all_need && need + i < count; i += kPlanThreads) {
      const int q = last_at_most(s_front, kPlanThreads, i);
      const int j = s_po[q] + i - s_front[q];
      if (j < s_pn[q])  // (a refused row has no new pages)
        p.table[(int64_t)(b0 + q) * p.table_stride + j] = p.ring[ring_at(need + i)];
    }
    // Pages given back by rows that shrink.
    for (int i = tid; i < all_back; i += kPlanThreads) {
      const int q = last_at_most(s_end, kPlanThreads, i);
      const int64_t at = (int64_t)count + back + i;
      if (at < p.N)
        p.ring[ring_at((int)at)] = p.table[(int64_t)(b0 + q) * p.table_stride + s_pn[q] + i - s_end[q]];
    }
    if (b0 + nb == p.B) {
      // Pages taken in all: those up to the last row that was granted some, which
      // is in front of this workgroup's where their sum exceeds the ring's.
      int taken = granted && r.need > 0 ? need + cum : need <= count ? need : 0;
      if (need > count) {
        int carry = 0;
        for (int c0 = 0; c0 < b0; c0 += kPlanThreads) {
          const int b = c0 + tid;
          int x = b < b0 ? plan_row(p, b).need : 0, y = 0, tx, ty;
          block_scan2(x, y, tx, ty, red);
          if (carry + x <= count) taken = max(taken, carry + x);
          carry += tx;
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) taken = max(taken, __shfl_xor(taken, o));
      if ((tid & 63) == 0) red[0][tid >> 6] = taken;
      __syncthreads();
      if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kPlanWaves; ++w) taken = max(taken, red[0][w]);
        p.state_out[0] = (int)ring_at(taken < p.N ? taken : 0);
        p.state_out[1] = (int)min((int64_t)p.N, (int64_t)count - taken + back + all_back);
      }
    }
  }

  // Slots of this workgroup's rows and tokens.
  const int c0 = blockIdx.y * p.toks_per_wg;
  const int nc = min(p.toks_per_wg, p.T - c0);
  for (int i = tid; i < nb * nc; i += kPlanThreads) {
    const int q = p.rows_per_wg == 1 ? 0 : p.tok_div.quot(i);  // (several rows: all T tokens)
    const int t = c0 + i - q * nc;
    int64_t slot = -1;
    if (t < s_grow[q]) {
      const int pos = s_old[q] + t;
      const int j = p.page_div.quot(pos);
      const int page = j < s_po[q] ? p.table[(int64_t)(b0 + q) * p.table_stride + j]
                                   : p.ring[ring_at(need + s_front[q] + j - s_po[q])];
      if (page >= 0) slot = (int64_t)page * p.page_size + (pos - j * p.page_size);
    }
    p.slots[(int64_t)(b0 + q) * p.T + t] = slot;
  }
}

hipError_t launch_page_plan(const PagePlanParams& p0, hipStream_t s) {
  PagePlanParams p = p0;
  if (p.B == 0) return hipSuccess;
  // About 2,048 slots a workgroup: whole rows while several fit, else parts of one.
  const int64_t most = 2048;
  p.rows_per_wg = (int)(p.T >= most ? 1 : p.T <= most / kPlanThreads ? kPlanThreads : most / p.T);
  p.toks_per_wg = p.T < most ? (p.T > 0 ? p.T : 1) : (int)most;
  p.page_div = FastDiv(p.page_size);
  p.tok_div = FastDiv(p.T > 0 ? p.T : 1);
  const int64_t gx = (p.B + p.rows_per_wg - 1) / p.rows_per_wg;
  const int64_t gy = p.T > 0 ? (p.T + p.toks_per_wg - 1) / p.toks_per_wg : 1;
  if (gy > 65535) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(page_plan_kernel, dim3((unsigned)gx, (unsigned)gy), dim3(kPlanThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace sk
