// Shared pieces of the paged INT8 key/value cache kernels: the device view of
// the cache, bounds-checked page lookups, element loads and stores of the
// supported types, argument checks.
#pragma once

#include <cuda_bf16.h>

#include "../../../include/h3vae_b200_kv.h"
#include "common.cuh"

namespace h3b {

constexpr unsigned int kErrKvPage = 1u << 3;   // page number or position outside its table
constexpr float kKvInv127 = 1.0f / 127.0f;
constexpr float kKvMinScale = 1e-30f;

struct KvView {
  int8_t* code[2];      // K, V
  float* scale[2];
  int16_t* k_sum;
  const int32_t* table;
  int num_pages, heads, page, page_shift, width, batch;
};

// The page number of slot `slot` of sequence b, or -1 (and the error bit) when
// the slot lies outside the table or the number outside the pool.
__device__ __forceinline__ int kv_page(const KvView& c, int b, int slot) {
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(c.width)) {
    record_error(kErrKvPage);
    return -1;
  }
  const int p = c.table[static_cast<int64_t>(b) * c.width + slot];
  if (static_cast<unsigned>(p) >= static_cast<unsigned>(c.num_pages)) {
    record_error(kErrKvPage);
    return -1;
  }
  return p;
}

// The barrier of a cluster's blocks, in its two halves.  The .aligned forms want all
// lanes of a warp at once, and what comes before (a loop that some lanes leave
// earlier, a branch) may have split them: the warp is joined first.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}

template <typename T> struct KvVec8;   // eight elements as 32-bit words
template <> struct KvVec8<__half> { static constexpr int kWords = 4; };
template <> struct KvVec8<__nv_bfloat16> { static constexpr int kWords = 4; };
template <> struct KvVec8<float> { static constexpr int kWords = 8; };

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(float x, float& y) { y = x; }

// Eight consecutive elements; `vec` = the address is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  __align__(16) T e[8];
  if (vec) {
#pragma unroll
    for (int i = 0; i < KvVec8<T>::kWords / 4; ++i)
      reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}

// fp32 of each of four signed bytes, exactly: the byte with its sign bit
// flipped goes into the low mantissa bits of 2^23.
__device__ __forceinline__ void codes_to_f32(uint32_t w, float* x) {
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = __fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)), 8388736.0f);
}

// Eight products with `f`, each rounded to nearest: packed fp32 pairs round each
// lane like the scalar operation.
__device__ __forceinline__ void scale8(float (&x)[8], float f) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 y = f2x_mul(make_float2(x[e], x[e + 1]), make_float2(f, f));
    x[e] = y.x;
    x[e + 1] = y.y;
  }
}

// The low byte of rint(x) for |x| < 2^21 sits in the low mantissa byte of
// x + 1.5 * 2^23 (two's complement, ties to even).
__device__ __forceinline__ uint32_t rint_bits(float x) { return __float_as_uint(__fadd_rn(x, 12582912.0f)); }

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// rint(x * f) of eight values as bytes, |x * f| < 2^21: the product rounded to
// nearest, then to an integer by the addition of rint_bits.
__device__ __forceinline__ uint2 quantise8(float (&x)[8], float f) {
  scale8(x, f);
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = rint_bits(x[e]);   // scalar: with the packed addition, codes differed (the pair was fused)
  return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

}  // namespace h3b

namespace h3b_host {

// Largest sizes of a call: grid dimensions, and positions that fit 32 bits.
constexpr int64_t kKvMostBatch = 65535, kKvMostHeads = 65535, kKvMostKeys = int64_t(1) << 30;
constexpr int64_t kKvMostSelected = int64_t(1) << 20;

// The product of sizes, or SIZE_MAX where that does not fit.
inline size_t kv_bytes(std::initializer_list<int64_t> sizes) {
  size_t n = 1;
  for (const int64_t s : sizes)
    if (__builtin_mul_overflow(n, static_cast<size_t>(s), &n)) return SIZE_MAX;
  return n;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks the cache and table arguments every entry point shares and fills the device view.
inline int kv_view(const char* name, const h3b_kv_cache* c, const int32_t* table, int64_t batch, int64_t width,
                   h3b::KvView* view) {
  if (c == nullptr || table == nullptr || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_sum)
    return set_error(H3B_EINVAL, "%s: NULL cache or page table", name);
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_sum))
    return set_error(H3B_EINVAL, "%s: cache codes and k_sum must be 16-byte aligned", name);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(H3B_EUNSUPPORTED, "%s: head_dim must be 64 or 128, got %lld", name, (long long)c->head_dim);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return set_error(H3B_EUNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128, got %lld", name,
                     (long long)c->page_size);
  if (batch <= 0 || width <= 0 || c->num_pages <= 0 || c->kv_heads <= 0)
    return set_error(H3B_EINVAL, "%s: batch, table width, pages and heads must be positive", name);
  if (batch > kKvMostBatch || c->kv_heads > kKvMostHeads || c->num_pages > (int64_t(1) << 30) ||
      width > kKvMostKeys / c->page_size)
    return set_error(H3B_EUNSUPPORTED, "%s: problem too large", name);
  view->code[0] = c->k;
  view->code[1] = c->v;
  view->scale[0] = c->k_scale;
  view->scale[1] = c->v_scale;
  view->k_sum = c->k_sum;
  view->table = table;
  view->num_pages = (int)c->num_pages;
  view->heads = (int)c->kv_heads;
  view->page = (int)c->page_size;
  view->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  view->width = (int)width;
  view->batch = (int)batch;
  return H3B_OK;
}

}  // namespace h3b_host
