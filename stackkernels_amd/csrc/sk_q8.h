// Parameter blocks and launchers of the 8-bit cache: page plans, the quantising
// append, and attention over cached codes.
//
// Format.  A cache holds 8-bit codes c (int8, or float8 e4m3 in the OCP
// encoding) and one fp32 scale s for each block of block_size consecutive
// tokens of a KV head; the value of an element is s * c.  Contiguous caches
// are (B, Hkv, S, D) with scales (B, Hkv, ceil(S / block_size)), paged ones
// (num_pages, Hkv, page_size, D) with scales (num_pages, Hkv, page_size /
// block_size); block_size is a multiple of 32 and divides page_size.
#pragma once

#include "sk_kernels.h"

namespace sk {

// Code types (SK_I8 and SK_E4M3 of sk_attn.h).
constexpr int kCodeI8 = 3;
constexpr int kCodeE4M3 = 4;

// Quotients by a fixed positive number of 0 <= n < 2^31: floor(n / d) = high word of
// n * mul, shifted, with mul = floor(2^(32 + shift) / d) + 1 and 2^shift the
// largest power of two below d (d > 1): the error n (mul d - 2^(32 + shift)) <= n d
// stays below 2^(32 + shift).
struct FastDiv {
  uint32_t mul;
  int shift;
  FastDiv() = default;
  explicit FastDiv(int d) {
    shift = 0;
    while ((2LL << shift) < d) ++shift;
    mul = d <= 1 ? 0 : (uint32_t)((1ULL << (32 + shift)) / (uint64_t)d + 1);
  }
  __device__ __forceinline__ int quot(int n) const {
    return mul ? (int)(__umulhi((uint32_t)n, mul) >> shift) : n;
  }
};

constexpr int kQ8MaxSplits = 256;

// One cache (k or v) as the kernels address it: strides in elements.
struct Q8Cache {
  uint8_t* codes;
  float* scales;
  int64_t sb, sh, ss;     // codes: unit (batch row or page), head, token
  int64_t cb, ch, cs;     // scales: unit, head, block
};

// Page plan (see sk_kv_page_plan in sk_attn.h).
struct PagePlanParams {
  int* table;
  int64_t table_stride;
  const int* lens;
  const int* news;
  int* ring;
  const int* state;   // {head, count}
  int64_t* slots;     // (B, T)
  int* lens_out;
  int* state_out;
  int B, max_pages, page_size, T, N;
  int rows_per_wg, toks_per_wg;  // whole rows (toks_per_wg = T), or parts of one
  FastDiv page_div, tok_div;
};

// Quantising append: token t < news[b] of batch row b becomes token
// lens[b] + t of its cache.
struct Q8AppendParams {
  const void* x[2];      // new keys, new values
  int64_t x_sb[2], x_sh[2], x_ss[2];
  Q8Cache c[2];
  const int* lens;
  const int* news;       // null: T each
  const int* table;      // null: contiguous
  int B, Hkv, T, D;
  int cap;               // tokens a batch row can hold
  int page_size, max_pages, num_pages;
  int block;
  int blocks;            // blocks a row's new tokens can touch
  FastDiv block_div, hkv_div, blocks_div, pairs_div, page_div;  // (set by the launcher)
  RopeParams rope;       // keys only
};

// Attention of Sq query tokens per row over the cache.  Row r of a KV head is
// (token r / group, head r % group).
struct Q8AttnParams {
  const void* q;
  void* o;
  Q8Cache k, v;
  float* part_o;         // [B*Hkv*rows][splits][dpad], normalised per split
  float* part_lse;       // [B*Hkv*rows][splits], log2 units; -inf: no key
  int64_t q_sb, q_sh, q_ss;
  int64_t o_sb, o_sh, o_ss;
  int B, Hq, Hkv, Sq, Sk, D, group;
  int rows, row_blocks;
  int num_splits, dpad;
  int causal;
  int dtype;             // of q and o
  float scale_log2;      // sm_scale * log2(e), signed
  const int* seqlens;    // null: Sk
  const int* qlens;      // null: Sq
  const int* table;      // null: contiguous
  int page_size, max_pages, num_pages;
  FastDiv block_div, page_div;
  FastDiv group_div, rows_div, hkv_div, split_div, block_rows_div;  // (set by the launcher)
  RopeParams rope;
};

hipError_t launch_page_plan(const PagePlanParams& p, hipStream_t s);
hipError_t launch_q8_append(int dtype, int code, const Q8AppendParams& p, hipStream_t s);
hipError_t launch_q8_attn(int code, const Q8AttnParams& p, hipStream_t s);
// Rows of a KV head (query tokens x group) that one workgroup takes, and the
// split count for a shape (keys: the most keys a row can see).
int q8_rows_per_block(int dtype, int D, int rows);
int q8_splits(int dtype, int B, int Hkv, int rows, int keys, int D);
int q8_dpad(int D);

}  // namespace sk
