// Attention over the paged INT8 key/value cache.
//
// For a query row q at position p and the keys j it sees, with K codes kc, V
// codes vc and their page's scales ks, vs:
//   x_j = (q . kc_j) * (ks * scale * log2 e),   m = max_j x_j,
//   out = sum_j 2^(x_j - m) vs vc_j / sum_j 2^(x_j - m).
// One block per query row, lanes over keys for the scores and over dimensions
// for the values, with a running maximum and sum per warp.
#include "kv_common.cuh"

namespace h3b {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
  bool causal;
  float scale_log2;
};

// The keys [first, last) a query token sees (before any page selection), and
// its position; an empty range for a padding row.
__device__ __forceinline__ int kv_range(const KvAttnParams& p, int b, int t, int& first, int& last) {
  int len = max(p.lengths[b], 0);
  if (len > p.c.width * p.c.page) {
    record_error(kErrKvPage);
    len = p.c.width * p.c.page;
  }
  const int n = p.counts ? min(p.counts[b], p.tokens) : p.tokens;
  const int pos = len - n + t;
  first = 0;
  last = 0;
  if (t >= n || pos < 0) return -1;
  last = p.causal ? pos + 1 : len;
  if (p.window > 0) first = max(0, pos + 1 - p.window);
  return pos;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) attention_kv_row_kernel(const KvAttnParams p) {
  __shared__ float s_q[D];
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int first, last;
  kv_range(p, b, t, first, last);
  const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
  for (int d = threadIdx.x; d < D; d += 128) s_q[d] = to_f32(q[d]);
  __syncthreads();
  const int32_t* sel =
      p.selected ? p.selected + ((static_cast<int64_t>(b) * p.c.heads + hk) * p.tokens + t) * p.n_selected : nullptr;
  // keys in the order walked: positions, or slots of the selected pages
  const int64_t walk0 = sel ? 0 : first;
  const int64_t walk1 = sel ? (last > first ? static_cast<int64_t>(p.n_selected) * p.c.page : 0) : last;
  float m = -INFINITY, l = 0.0f, o[D / 32] = {};
  for (int64_t base = walk0 + warp * 32; base < walk1; base += 128) {
    const int64_t i = base + lane;
    float x = -INFINITY, vs = 0.0f;
    int64_t off = -1;
    if (i < walk1) {
      int slot = sel ? sel[i >> p.c.page_shift] : static_cast<int>(i >> p.c.page_shift);
      const int64_t pos = (static_cast<int64_t>(slot) << p.c.page_shift) + (i & (p.c.page - 1));
      if (slot >= 0 && pos >= first && pos < last) {
        const int page = kv_page(p.c, b, slot);
        if (page >= 0) {
          const int64_t ph = static_cast<int64_t>(page) * p.c.heads + hk;
          off = (ph * p.c.page + (i & (p.c.page - 1))) * D;
          vs = p.c.scale[1][ph];
          float acc = 0.0f;
          for (int d = 0; d < D; d += 16) {
            const uint4 w = *reinterpret_cast<const uint4*>(p.c.code[0] + off + d);
            float k[16];
            codes_to_f32(w.x, k);
            codes_to_f32(w.y, k + 4);
            codes_to_f32(w.z, k + 8);
            codes_to_f32(w.w, k + 12);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc = __fmaf_rn(s_q[d + e], k[e], acc);
          }
          x = acc * (p.c.scale[0][ph] * p.scale_log2);
        }
      }
    }
    const bool seen = off >= 0;
    if (!__any_sync(0xffffffffu, seen)) continue;
    const float m_new = fmaxf(m, warp_max(seen ? x : -INFINITY));
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = exp2f(m - ref);
    const float e = seen ? exp2f(x - ref) : 0.0f;
    l = l * alpha + warp_sum(e);
    m = m_new;
    const float w = seen ? e * vs : 0.0f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] *= alpha;
    for (int j = 0; j < 32; ++j) {
      const int64_t at = __shfl_sync(0xffffffffu, off, j);
      const float wj = __shfl_sync(0xffffffffu, w, j);
      if (at < 0) continue;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) o[k] = __fmaf_rn(wj, static_cast<float>(p.c.code[1][at + lane + 32 * k]), o[k]);
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int k = 0; k < D / 32; ++k) s_o[warp][lane + 32 * k] = o[k];
  __syncthreads();
  float mm = -INFINITY;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w]);
  const float ref = mm == -INFINITY ? 0.0f : mm;
  float ll = 0.0f;
  for (int w = 0; w < 4; ++w) ll += s_l[w] * exp2f(s_m[w] - ref);
  T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2];
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.0f;
    for (int w = 0; w < 4; ++w) v += s_o[w][d] * exp2f(s_m[w] - ref);
    from_f32(ll == 0.0f ? 0.0f : v / ll, out[d]);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[(static_cast<int64_t>(b) * p.q_heads + h) * p.tokens + t] = ll == 0.0f ? -INFINITY : (ref + log2f(ll)) * kLn2;
}

}  // namespace h3b

extern "C" size_t h3b_attention_kv_i8_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens,
                                                     int64_t head_dim, int64_t table_width, int64_t page_size,
                                                     int64_t n_selected) {
  return 16;
}

extern "C" int h3b_attention_kv_i8(const void* q, const int64_t* q_strides, const h3b_kv_cache* cache,
                                   const int32_t* page_table, int64_t batch, int64_t table_width,
                                   const int32_t* lengths, const int32_t* counts, int64_t q_heads, int64_t tokens,
                                   float scale, int causal, int64_t window, const int32_t* selected,
                                   int64_t n_selected, int dtype, void* out, const int64_t* out_strides, float* lse,
                                   void* workspace, size_t workspace_bytes, h3b_stream_t stream) {
  const char* name = "h3b_attention_kv_i8";
  h3b::KvAttnParams p{};
  int rc = h3b_host::kv_view(name, cache, page_table, batch, table_width, &p.c);
  if (rc) return rc;
  if (!q || !out || !q_strides || !out_strides || !lengths) return h3b_host::set_error(H3B_EINVAL, "%s: NULL argument", name);
  if (dtype != H3B_TYPE_F16 && dtype != H3B_TYPE_BF16)
    return h3b_host::set_error(H3B_EINVAL, "%s: q must be fp16 or bf16", name);
  if (q_heads <= 0 || q_heads % cache->kv_heads || q_heads > 65535)
    return h3b_host::set_error(H3B_EINVAL, "%s: q_heads must be a positive multiple of kv_heads", name);
  if (tokens < 0 || tokens > (int64_t(1) << 26)) return h3b_host::set_error(H3B_EINVAL, "%s: bad token count", name);
  if (window < 0 || (window > 0 && !causal)) return h3b_host::set_error(H3B_EINVAL, "%s: a window needs causal", name);
  if (selected && (n_selected <= 0 || n_selected > (int64_t(1) << 20) || !causal || window > 0))
    return h3b_host::set_error(H3B_EINVAL, "%s: selected pages need causal, no window and 1 to 2^20 pages", name);
  if (tokens == 0) return H3B_OK;
  p.q = q;
  p.out = out;
  p.lse = lse;
  p.lengths = lengths;
  p.counts = counts;
  p.selected = selected;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = out_strides[i];
  }
  p.q_heads = (int)q_heads;
  p.group = (int)(q_heads / cache->kv_heads);
  p.tokens = (int)tokens;
  p.n_selected = (int)n_selected;
  p.window = (int)(window > (int64_t(1) << 30) ? int64_t(1) << 30 : window);
  p.causal = causal != 0;
  p.scale_log2 = scale * h3b::kLog2e;
  dim3 grid((unsigned)tokens, (unsigned)q_heads, (unsigned)batch);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = cache->head_dim == 128;
  if (dtype == H3B_TYPE_F16) {
    if (wide) h3b::attention_kv_row_kernel<__half, 128><<<grid, 128, 0, st>>>(p);
    else h3b::attention_kv_row_kernel<__half, 64><<<grid, 128, 0, st>>>(p);
  } else {
    if (wide) h3b::attention_kv_row_kernel<__nv_bfloat16, 128><<<grid, 128, 0, st>>>(p);
    else h3b::attention_kv_row_kernel<__nv_bfloat16, 64><<<grid, 128, 0, st>>>(p);
  }
  return h3b_host::check_launch(name);
}
