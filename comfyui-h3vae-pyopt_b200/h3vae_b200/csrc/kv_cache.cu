// Writing and reading the paged INT8 key/value cache.
//
// Write.  For the new tokens x of one (page, head) and K or V:
//   a = max|x|;  s = max(a * fp32(1/127), 1e-30), and max(s, old scale) when the
//   page keeps earlier tokens, whose codes become rint(code * (old / s)) if s
//   grew;  code = rint(x * (1/s)).
// One CTA per (page slot, head, K or V): the page's new values (at most 32 KB
// of fp16) stay in registers between the maximum and the quantisation, so every
// input is read once and every code written once.  They stay as they came, in 16
// bits (as fp32 a 128 x 128 page took 128 registers a thread and 250 us where it
// now takes 52), and are asked for before the page number is known.  Bound: HBM,
// 2 B read and 1 B written per element, and the ~6 instructions an element takes:
// 4 x 16 heads x 5120 tokens of dim 64, fp16, 126 MB in 26.7 us = 4.7 TB/s; bf16
// prompts of up to 16001 tokens, 8 heads of dim 128, 52 us.  A single token per
// sequence is a launch: 3.4 us.
#include <cstring>

#include "kv_common.cuh"

namespace h3b {

struct KvWriteParams {
  KvView c;
  const int32_t* start;
  const int32_t* counts;
  const void* x[2];        // K, V
  int64_t stride[2][3];    // elements: batch, head, token
  int tokens, dim;
  bool vec[2];             // rows can be read 16 bytes at a time
};

// Eight elements as they are in memory, and the largest magnitude among them:
// for the 16-bit types on the bits (sign cleared, the order of the floats is the
// order of the integers, infinities and NaN above all finite values).
template <typename T> struct KvRaw {
  uint32_t w[KvVec8<T>::kWords];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < KvVec8<T>::kWords / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
      memcpy(w, e, sizeof(w));
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < KvVec8<T>::kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    T e[8];
    memcpy(e, w, sizeof(w));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  }
  __device__ __forceinline__ uint32_t top(uint32_t most) const {
    if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < KvVec8<T>::kWords; ++i) most = max(most, w[i] & 0x7fffffffu);
    } else {
#pragma unroll
      for (int i = 0; i < KvVec8<T>::kWords; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
    }
    return most;
  }
  // The magnitude as fp32 bits; anything above 0x7f7fffff stands for an infinity or a NaN.
  static __device__ __forceinline__ uint32_t top_f32(uint32_t most) {
    if (sizeof(T) == 4) return most;
    const uint16_t m = static_cast<uint16_t>(max(most & 0xffffu, most >> 16));
    T v;
    memcpy(&v, &m, 2);
    return __float_as_uint(to_f32(v));
  }
};

// VPT: vectors of 8 elements per thread = page * dim / 8 / threads.
template <typename T, int VPT, int kThreads>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvWriteParams p) {
  constexpr int kWarps = kThreads / 32;
  __shared__ uint32_t s_max[kWarps];
  __shared__ __align__(16) uint32_t s_sum[kWarps][64];
  const int kv = blockIdx.x & 1, head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int count = p.counts ? min(p.counts[b], p.tokens) : p.tokens;
  const int start = p.start[b];
  if (start < 0) {
    if (tid == 0 && count > 0) record_error(kErrKvPage);
    return;
  }
  const int slot = (start >> p.c.page_shift) + (blockIdx.x >> 1);
  const int64_t page_begin = static_cast<int64_t>(slot) << p.c.page_shift;
  const int64_t end = static_cast<int64_t>(start) + count;
  const int lo = static_cast<int>(max(static_cast<int64_t>(start), page_begin) - page_begin);   // first new row
  const int hi = static_cast<int>(min(end - page_begin, static_cast<int64_t>(p.c.page)));       // past the last one
  if (hi <= lo) return;

  // the new rows are asked for before the page is looked up; a thread's vectors lie kThreads apart, in one column
  const int chunk_shift = p.dim == 64 ? 3 : 4, row_step = kThreads >> chunk_shift;
  const int row0 = tid >> chunk_shift;
  const T* src = static_cast<const T*>(p.x[kv]) + b * p.stride[kv][0] + head * p.stride[kv][1] +
                 (page_begin - start + row0) * p.stride[kv][2] + (tid & ((1 << chunk_shift) - 1)) * 8;
  const int64_t src_step = row_step * p.stride[kv][2];
  KvRaw<T> x[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j, src += src_step) {
    const int row = row0 + j * row_step;
    if (row >= lo && row < hi) x[j].load(src, p.vec[kv]);
    else x[j].zero();
  }
  const int page = kv_page(p.c, b, slot);
  if (page < 0) return;
  const int64_t ph = static_cast<int64_t>(page) * p.c.heads + head;
  int8_t* codes = p.c.code[kv] + ph * p.c.page * p.dim;
  float* scale_at = p.c.scale[kv] + ph;
  const float old_scale = lo > 0 ? *scale_at : 0.0f;

  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < VPT; ++j) most = x[j].top(most);
  most = __reduce_max_sync(0xffffffffu, KvRaw<T>::top_f32(most));
  if ((tid & 31) == 0) s_max[tid >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) most = max(most, s_max[w]);

  const bool lost = most > 0x7f7fffffu || isnan(old_scale);    // a NaN or an infinity, now or before
  float s = fmaxf(__fmul_rn(__uint_as_float(most), kKvInv127), kKvMinScale);
  s = old_scale > s ? old_scale : s;
  const bool grown = lo > 0 && s > old_scale;
  const bool complete = kv == 0 && hi == p.c.page;
  const float inv = __frcp_rn(s), ratio = __fdiv_rn(old_scale, s);
  // Column sums of codes + 128, two to a word: at most 128 rows of 255 fit 16 bits.
  uint32_t sum[4] = {};      // codes 0 and 2, 1 and 3, 4 and 6, 5 and 7 of the column's eight
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int row = row0 + j * row_step;
    uint2* at = reinterpret_cast<uint2*>(codes) + tid + j * kThreads;
    uint2 w = make_uint2(0u, 0u);
    bool store = false;
    if (row >= lo && row < hi) {
      store = true;
      if (!lost) {   // |x * inv| <= 127 * (1 + 2^-22): no clamp is needed after rounding
        float f[8];
        x[j].values(f);
        w = quantise8(f, inv);
      }
    } else if (row < lo && (grown || complete)) {
      w = *at;
      if (grown && !lost) {
        store = true;
        float f[8];
        codes_to_f32(w.x, f);
        codes_to_f32(w.y, f + 4);
        w = quantise8(f, ratio);
      }
    }
    if (store) *at = w;
    if (complete) {
      const uint32_t a = w.x ^ 0x80808080u, c = w.y ^ 0x80808080u;
      sum[0] += a & 0x00ff00ffu;
      sum[1] += (a >> 8) & 0x00ff00ffu;
      sum[2] += c & 0x00ff00ffu;
      sum[3] += (c >> 8) & 0x00ff00ffu;
    }
  }
  if (tid == 0) *scale_at = lost ? __int_as_float(0x7fffffff) : s;
  if (complete) {
    const int chunks = 1 << chunk_shift;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      for (int o = chunks; o < 32; o <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
    if ((tid & 31) < chunks)
      *reinterpret_cast<uint4*>(&s_sum[tid >> 5][(tid & 31) * 4]) = make_uint4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (tid < p.dim) {
      // dim tid: word (tid / 8) * 4 + its place in the order above, low or high half
      const int in = tid & 7, word = (tid >> 3) * 4 + (in >> 2) * 2 + (in & 1), shift = (in & 2) * 8;
      int t = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += static_cast<int>((s_sum[w][word] >> shift) & 0xffffu);
      p.c.k_sum[ph * p.dim + tid] = static_cast<int16_t>(t - 128 * p.c.page);
    }
  }
}

// Read: a thread takes 8 codes of K and of V (8 B in, 16 B out of fp16 each) of
// kKvReadRows rows, so that several loads are on their way.  Bound: HBM.  8 x up
// to 32768 tokens, 8 heads of dim 128, bf16: 222 us = 6.4 TB/s (250 with one
// product at a time, 241 with four rows, 225 with one).
struct KvReadParams {
  KvView c;
  const int32_t* start;
  const int32_t* lengths;
  void* out[2];
  int tokens, chunk_shift;   // dim = 8 << chunk_shift
};

constexpr int kKvReadThreads = 256;
constexpr int kKvReadRows = 2;

template <typename T>
__global__ void __launch_bounds__(kKvReadThreads) kv_read_kernel(const KvReadParams p) {
  const int head = blockIdx.y, b = blockIdx.z;
  const int dim = 8 << p.chunk_shift, step = kKvReadThreads >> p.chunk_shift;
  const int row0 = blockIdx.x * step * kKvReadRows + (threadIdx.x >> p.chunk_shift);
  const int col = (threadIdx.x & ((1 << p.chunk_shift) - 1)) * 8;
  const int64_t first = p.start ? p.start[b] : 0, len = p.lengths[b];
  uint2 w[kKvReadRows][2];
  float s[kKvReadRows][2];
#pragma unroll
  for (int r = 0; r < kKvReadRows; ++r) {
    const int row = row0 + r * step;
    const int64_t pos = first + row;
    const int page = row < p.tokens && pos >= 0 && pos < len ? kv_page(p.c, b, static_cast<int>(pos >> p.c.page_shift)) : -1;
    const int64_t ph = static_cast<int64_t>(page) * p.c.heads + head;
    const int64_t from = (ph * p.c.page + (pos & (p.c.page - 1))) * dim + col;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      w[r][kv] = make_uint2(0u, 0u);
      s[r][kv] = 0.0f;
      if (page >= 0) {
        w[r][kv] = *reinterpret_cast<const uint2*>(p.c.code[kv] + from);
        s[r][kv] = p.c.scale[kv][ph];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kKvReadRows; ++r) {
    const int row = row0 + r * step;
    if (row >= p.tokens) return;
    const int64_t to = ((static_cast<int64_t>(b) * p.c.heads + head) * p.tokens + row) * dim + col;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[8];
      codes_to_f32(w[r][kv].x, x);
      codes_to_f32(w[r][kv].y, x + 4);
      scale8(x, s[r][kv]);
      __align__(16) T y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) from_f32(x[e], y[e]);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out[kv]) + to);
#pragma unroll
      for (int k = 0; k < KvVec8<T>::kWords / 4; ++k) dst[k] = reinterpret_cast<const uint4*>(y)[k];
    }
  }
}

}  // namespace h3b

namespace {

template <typename T>
void launch_kv_write(const h3b::KvWriteParams& p, dim3 grid, cudaStream_t st) {
  switch (p.c.page * p.dim / 1024) {
    case 1: h3b::kv_write_kernel<T, 1, 128><<<grid, 128, 0, st>>>(p); break;
    case 2: h3b::kv_write_kernel<T, 2, 128><<<grid, 128, 0, st>>>(p); break;
    case 4: h3b::kv_write_kernel<T, 4, 128><<<grid, 128, 0, st>>>(p); break;
    case 8: h3b::kv_write_kernel<T, 4, 256><<<grid, 256, 0, st>>>(p); break;
    default: h3b::kv_write_kernel<T, 8, 256><<<grid, 256, 0, st>>>(p); break;
  }
}

}  // namespace

extern "C" int h3b_kv_write_i8(const h3b_kv_cache* cache, const int32_t* page_table, int64_t batch,
                               int64_t table_width, const int32_t* start, const int32_t* counts, const void* k,
                               const int64_t* k_strides, const void* v, const int64_t* v_strides, int64_t tokens,
                               int dtype, h3b_stream_t stream) {
  const char* name = "h3b_kv_write_i8";
  h3b::KvWriteParams p{};
  int rc = h3b_host::kv_view(name, cache, page_table, batch, table_width, &p.c);
  if (rc) return rc;
  if (!start || !k || !v || !k_strides || !v_strides) return h3b_host::set_error(H3B_EINVAL, "%s: NULL argument", name);
  if (dtype != H3B_TYPE_F16 && dtype != H3B_TYPE_BF16 && dtype != H3B_TYPE_F32)
    return h3b_host::set_error(H3B_EINVAL, "%s: unknown dtype %d", name, dtype);
  if (tokens < 0 || tokens > (int64_t(1) << 30)) return h3b_host::set_error(H3B_EINVAL, "%s: bad token count", name);
  if (tokens == 0) return H3B_OK;
  p.start = start;
  p.counts = counts;
  p.x[0] = k;
  p.x[1] = v;
  p.tokens = (int)tokens;
  p.dim = (int)cache->head_dim;
  const int size = dtype == H3B_TYPE_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? v_strides : k_strides;
    p.vec[i] = h3b_host::aligned16(p.x[i]);
    for (int j = 0; j < 3; ++j) {
      p.stride[i][j] = s[j];
      p.vec[i] = p.vec[i] && s[j] * size % 16 == 0;
    }
  }
  const int64_t slots = (tokens + p.c.page - 2) / p.c.page + 1;
  if (slots > (int64_t(1) << 30) || cache->kv_heads > 65535)
    return h3b_host::set_error(H3B_EUNSUPPORTED, "%s: problem too large", name);
  dim3 grid((unsigned)(2 * slots), (unsigned)cache->kv_heads, (unsigned)batch);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == H3B_TYPE_F16) launch_kv_write<__half>(p, grid, st);
  else if (dtype == H3B_TYPE_BF16) launch_kv_write<__nv_bfloat16>(p, grid, st);
  else launch_kv_write<float>(p, grid, st);
  return h3b_host::check_launch(name);
}

extern "C" int h3b_kv_read_i8(const h3b_kv_cache* cache, const int32_t* page_table, int64_t batch,
                              int64_t table_width, const int32_t* start, const int32_t* lengths, void* k, void* v,
                              int64_t tokens, int dtype, h3b_stream_t stream) {
  const char* name = "h3b_kv_read_i8";
  h3b::KvReadParams p{};
  int rc = h3b_host::kv_view(name, cache, page_table, batch, table_width, &p.c);
  if (rc) return rc;
  if (!lengths || !k || !v) return h3b_host::set_error(H3B_EINVAL, "%s: NULL argument", name);
  if (!h3b_host::aligned16(k) || !h3b_host::aligned16(v))
    return h3b_host::set_error(H3B_EINVAL, "%s: outputs must be 16-byte aligned", name);
  if (tokens < 0 || tokens > (int64_t(1) << 26)) return h3b_host::set_error(H3B_EINVAL, "%s: bad token count", name);
  if (tokens == 0) return H3B_OK;
  p.start = start;
  p.lengths = lengths;
  p.out[0] = k;
  p.out[1] = v;
  p.tokens = (int)tokens;
  p.chunk_shift = cache->head_dim == 64 ? 3 : 4;
  const int64_t rows = (int64_t)(h3b::kKvReadThreads >> p.chunk_shift) * h3b::kKvReadRows;
  dim3 grid((unsigned)((tokens + rows - 1) / rows), (unsigned)cache->kv_heads, (unsigned)batch);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == H3B_TYPE_F16) h3b::kv_read_kernel<__half><<<grid, h3b::kKvReadThreads, 0, st>>>(p);
  else if (dtype == H3B_TYPE_BF16) h3b::kv_read_kernel<__nv_bfloat16><<<grid, h3b::kKvReadThreads, 0, st>>>(p);
  else if (dtype == H3B_TYPE_F32) h3b::kv_read_kernel<float><<<grid, h3b::kKvReadThreads, 0, st>>>(p);
  else return h3b_host::set_error(H3B_EINVAL, "%s: unknown dtype %d", name, dtype);
  return h3b_host::check_launch(name);
}
