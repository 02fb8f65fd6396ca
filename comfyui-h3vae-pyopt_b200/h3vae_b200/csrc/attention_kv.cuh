// Attention over the paged INT8 key/value cache.
//
// For a query row q at position p and the keys j it sees, with K codes kc, V
// codes vc and their page's scales ks, vs:
//   x_j = (q . kc_j) * (ks * scale * log2 e) + log2(vs),   m = max_j x_j,
//   w_j = 2^(x_j - m) <= 1   (= the softmax weight times vs, up to a factor),
//   out = sum_j w_j vc_j / sum_j (w_j / vs).
// Folding vs into the exponent lets both products run on the codes themselves:
// they are whole numbers, exact in fp16, so the only rounding of the inputs is
// that of w to fp16, and scales that differ by any factor between pages stay
// relative to the largest weighted one.
//
// The sum of w_j / vs = 2^(q.k - m) has to hold keys whose w_j is below fp32's
// range, those of a page of zeros (vs = 1e-30) beside one of large values first of
// all.  So pages with vs < kKvLowScale are summed from the scores, without w_j, where
// any are met; and where m moves from such pages to others the sum is rescaled in two
// steps of half the way, since 2^(m - m') alone may be below the range.  Keys from
// 2^-26 of the largest weight up then count for values up to 2^77; smaller values
// leave more.  In place of 1 / vs such a page has log2 vs < -30: what the usual sum
// adds with that, at most 100 w_j, is 1e-7 of the w_j / vs > 2^30 w_j that belongs there.
#pragma once

#include "kv_common.cuh"

namespace h3b {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kKvLowScale = 0x1p-30f;   // a page of |v| < 1.2e-7

struct KvAttnParams {
  KvView c;
  const void* q;
  void* out;
  float* lse;
  const int32_t* lengths;
  const int32_t* counts;
  const int32_t* selected;
  int64_t qs[3], os[3];
  int q_heads, group, tokens, n_selected, window;
  bool causal, vec_q, vec_out;
  float scale_log2;
  // split plan (see attention_kv_split_kernel)
  int row_tiles, slots, chunk;
  int share, fit;  // runs of keys per (kv head, row tile): as many as that many equal ones, at most so many in all
  int join_warps;  // warps that join a row's parts: 1 or 4
  int cluster;     // > 0: the slots of a row tile are one cluster, which joins them itself
  float* part;     // [slot, kv head, row tile, row] x (dim + 2): weighted codes, m, l
  int2* plan;      // per sequence: first slot, number of slots
};

// Tokens of sequence b, clamped to its table, and its number of query tokens.
__device__ __forceinline__ int kv_length(const KvView& c, const int32_t* lengths, int b) {
  const int len = max(lengths[b], 0);
  if (len > c.width * c.page) {
    record_error(kErrKvPage);
    return c.width * c.page;
  }
  return len;
}
__device__ __forceinline__ int kv_count(const int32_t* counts, int tokens, int b) {
  return counts ? max(0, min(counts[b], tokens)) : tokens;
}

// The keys [first, last) that query token t of n sees in a sequence of len
// tokens, before any page selection; empty for padding rows.
__device__ __forceinline__ void kv_range(const KvAttnParams& p, int len, int n, int t, int& first, int& last) {
  const int pos = len - n + t;
  first = last = 0;
  if (t >= n || pos < 0) return;
  last = p.causal ? pos + 1 : len;
  if (p.window > 0) first = max(0, pos + 1 - p.window);
}

// Two codes as fp16: the bytes (sign bit flipped) become the low mantissa bits
// of 1024.
__device__ __forceinline__ uint32_t codes_to_h2(uint32_t biased, uint32_t selector) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, selector);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), __floats2half2_rn(1152.0f, 1152.0f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// l 2^d, for d down to -inf: a sum of weights that is rescaled (the product may be in range where 2^d is not).
__device__ __forceinline__ float rescale_sum(float l, float d) {
  const float h = ex2_approx(0.5f * d);
  return __fmul_rn(__fmul_rn(l, h), h);
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// Copies `bytes` (a multiple of 16, both addresses 16-byte aligned) to shared
// memory; their arrival counts on the barrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A query row as fp16.  bf16 rows are scaled by a power of two so that their
// largest value lies in [1, 2).  Values down to 2^-17 of it (8 bits each) are then
// exact in fp16, and smaller ones are off by 2^-25 of it at most, half an fp32 ulp
// of the largest; `back` undoes the scaling.
__device__ __forceinline__ float row_scaling(__half, float, float& back) {
  back = 1.0f;
  return 1.0f;
}
__device__ __forceinline__ float row_scaling(__nv_bfloat16, float top, float& back) {
  int e = static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127;
  e = top == 0.0f ? 0 : max(-126, min(126, e));
  back = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}

}  // namespace h3b
