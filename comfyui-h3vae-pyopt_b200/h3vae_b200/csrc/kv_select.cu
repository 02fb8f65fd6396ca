// Page selection for sparse attention over the paged INT8 cache.
//
// A row (query token, kv head) scores every complete page before its own with
//   max over the group's heads of float(q8 . k_sum[page]) * s_q, times k_scale[page]
// (q8, s_q: the row quantisation of the query; k_sum: the sum of the page's K
// codes, so the score is the query's mean product with the page's keys up to a
// common factor) and keeps the best n - 1 and its own page.  The products are
// whole numbers below 2^31, so scores do not depend on the summation order and
// ties (lower page first) are exact.
//
// Two steps: scores (a thread per page, all rows of the sequence and head
// from shared memory) and the selection (a block per row: the (n-1)-th largest
// key by bisection, then an ordered compaction); a kernel each, or one for few tokens.
// Both are latency: 2048 pages of 16 heads, 4 MB of sums, take 11 us together (3.6 for the scores alone).
// Tokens are not spread over blocks: a block of the score kernel takes them one after the other, which is made for few
// (1024 tokens x 4 x 16 heads: 480 us over 80 pages, 784 us over 640).
#include <algorithm>

#include "kv_common.cuh"

namespace h3b {

struct KvSelectParams {
  KvView c;
  const void* q;
  const int32_t* lengths;
  const int32_t* counts;
  uint32_t* keys;        // [batch, heads, tokens, row_keys]
  int32_t* selected;
  int64_t qs[3];
  int group, tokens, n, row_keys;
};

// Query tokens of sequence b.
__device__ __forceinline__ int kv_queries(const KvSelectParams& p, int b) {
  return p.counts ? max(0, min(p.counts[b], p.tokens)) : p.tokens;
}

// Last page ordinal row t of sequence b sees, -1 if none (t = -1, a sequence without queries, among them).
__device__ __forceinline__ int kv_last_page(const KvSelectParams& p, int b, int t) {
  int len = max(p.lengths[b], 0);
  if (len > p.c.width * p.c.page) {
    record_error(kErrKvPage);
    len = p.c.width * p.c.page;
  }
  const int n = kv_queries(p, b);
  const int pos = len - n + t;
  return t < 0 || t >= n || pos < 0 ? -1 : pos >> p.c.page_shift;
}

constexpr int kSelThreads = 128;
constexpr int kSelRows = 64;     // query rows held in shared memory at once

// The scale and the sums of a page's K codes.
template <int D>
__device__ __forceinline__ void load_sums(const KvSelectParams& p, int page, int head, uint32_t (&k)[D / 2], float& k_scale) {
  const int64_t ph = static_cast<int64_t>(page) * p.c.heads + head;
  k_scale = p.c.scale[0][ph];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(p.c.k_sum + ph * D + 8 * i);
    k[4 * i] = w.x, k[4 * i + 1] = w.y, k[4 * i + 2] = w.z, k[4 * i + 3] = w.w;
  }
}

// One query row to codes and their scale, by a warp.  A row with a NaN or an infinity
// has no codes: its scale becomes NaN and with it all its scores, which fmaxf over
// the group then leaves out.
template <typename T, int D>
__device__ __forceinline__ void quantise_row(const T* q, uint32_t* codes, float* scale) {
  const int lane = threadIdx.x & 31;
  float x[D / 32];
  uint32_t top = 0;      // magnitudes as bits: their order is the floats', infinities and NaN above all
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    x[e] = to_f32(q[lane * (D / 32) + e]);
    top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const float s = fmaxf(__fmul_rn(__uint_as_float(top), kKvInv127), kKvMinScale), inv = __frcp_rn(s);
#pragma unroll
  for (int e = 0; e < D / 32; ++e)
    reinterpret_cast<uint8_t*>(codes)[lane * (D / 32) + e] = static_cast<uint8_t>(rint_bits(__fmul_rn(x[e], inv)));
  if (lane == 0) *scale = top > 0x7f7fffffu ? __int_as_float(0x7fffffff) : s;
}

// A row's product with a page's sums.
template <int D>
__device__ __forceinline__ float row_score(const uint32_t (&k)[D / 2], const uint32_t* codes, float scale) {
  int dots[4] = {0, 0, 0, 0};       // four chains, so that they run into one another's latency
#pragma unroll
  for (int i = 0; i < D / 4; i += 4) {
    const uint4 q4 = *reinterpret_cast<const uint4*>(codes + i);
    const uint32_t w[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dots[e] = __dp2a_lo(static_cast<int>(k[2 * (i + e)]), static_cast<int>(w[e]), dots[e]);
      dots[e] = __dp2a_hi(static_cast<int>(k[2 * (i + e) + 1]), static_cast<int>(w[e]), dots[e]);
    }
  }
  return __fmul_rn(static_cast<float>((dots[0] + dots[1]) + (dots[2] + dots[3])), scale);
}

// The key by which pages are ordered: 0 stays below every score.
__device__ __forceinline__ uint32_t score_key(float best, float k_scale) {
  const float y = __fadd_rn(__fmul_rn(best, k_scale), 0.0f);   // -0 becomes +0
  return isnan(y) ? 0xffffffffu : float_to_ordered(y);
}

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads) kv_score_kernel(const KvSelectParams p) {
  __shared__ __align__(16) uint32_t s_q[kSelRows][D / 4];   // four codes a word
  __shared__ float s_s[kSelRows];
  const int head = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5;
  const int slot = blockIdx.x * kSelThreads + threadIdx.x;
  const int tokens = kv_queries(p, b);
  const int last = kv_last_page(p, b, tokens - 1);
  if (static_cast<int>(blockIdx.x) * kSelThreads >= last) return;   // no complete page here (uniform)
  uint32_t k[D / 2];
  float k_scale = 0.0f;
  const int page = slot < last ? kv_page(p.c, b, slot) : -1;
  if (page >= 0) load_sums<D>(p, page, head, k, k_scale);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per = max(1, kSelRows / p.group);      // query tokens per round
  float best = 0.0f;
  for (int t0 = 0; t0 < tokens; t0 += per) {      // padding rows have no keys, and none are looked for
    const int t1 = min(t0 + per, tokens);
    for (int g0 = 0; g0 < p.group; g0 += kSelRows) {   // groups wider than the buffer take several rounds
      const int g1 = min(g0 + kSelRows, p.group), gn = g1 - g0, rows = (t1 - t0) * gn;
      __syncthreads();
      for (int r = warp; r < rows; r += kSelThreads / 32) {
        const int t = t0 + r / gn, h = head * p.group + g0 + r % gn;
        const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
        quantise_row<T, D>(q, s_q[r], &s_s[r]);
      }
      __syncthreads();
      if (page >= 0) {
        for (int r = 0; r < rows; ++r) {
          const float x = row_score<D>(k, s_q[r], s_s[r]);
          const int g = r % gn;
          best = g0 + g == 0 ? x : fmaxf(best, x);
          if (g0 + g + 1 == p.group) {
            const int64_t row = (static_cast<int64_t>(b) * p.c.heads + head) * p.tokens + t0 + r / gn;
            p.keys[row * p.row_keys + slot] = score_key(best, k_scale);
          }
        }
      } else if (slot < last && g1 == p.group) {   // a bad page number: never worth choosing
        for (int t = t0; t < t1; ++t)
          p.keys[((static_cast<int64_t>(b) * p.c.heads + head) * p.tokens + t) * p.row_keys + slot] = 0u;
      }
    }
  }
}

// The n - 1 best of a row's `last` keys, by bisection on the key's bits: the
// threshold is built from the top down, two bits a round, counting the keys at or
// above it, and found as soon as that count is right.  Each thread holds kPer consecutive
// keys in registers; more pages than the block holds are read again each round.
// Four warps a row: a round is 3 kPer comparisons and one barrier, and the
// barrier's latency is what a wider block pays for (2048 pages: 10 us with 16
// warps, 22 us with a histogram of 8-bit digits that most keys share).
constexpr int kPickThreads = 128;

template <int kPer, int kThreads, bool kShared>
__device__ __forceinline__ void pick_pages(const KvSelectParams& p, const uint32_t* keys, int last, int32_t* out) {
  constexpr int kWarps = kThreads / 32;
  static_assert(kWarps % 4 == 0, "a round's counts are read as vectors");
  __shared__ __align__(16) int s_count[2][3][kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (last < p.n) {   // every page fits
    for (int i = tid; i < p.n; i += kThreads) out[i] = i <= last ? i : -1;
    return;
  }
  const int want = p.n - 1;
  if (tid == 0) out[want] = last;
  if (want == 0) return;
  const int rounds = (last + kThreads * kPer - 1) / (kThreads * kPer);
  uint32_t k[kPer];
  auto load = [&](int round) {
    const int i0 = (round * kThreads + tid) * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e += 4) {   // rows are 16-byte aligned and whole vectors long
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      const uint4* at = reinterpret_cast<const uint4*>(keys + i0 + e);
      if (i0 + e < last) v = kShared ? *at : __ldcg(at);
      k[e] = v.x;
      k[e + 1] = i0 + e + 1 < last ? v.y : 0u;
      k[e + 2] = i0 + e + 2 < last ? v.z : 0u;
      k[e + 3] = i0 + e + 3 < last ? v.w : 0u;
    }
  };
  if (rounds == 1) load(0);
  // largest threshold with at least `want` keys at or above it, two bits a round (keys are never 0 but on bad pages)
  uint32_t thr = 0;
  int at_least = last;
  for (int bit = 30; bit >= 0 && at_least != want; bit -= 2) {
    int n[3] = {0, 0, 0};
    for (int r = 0; r < rounds; ++r) {
      if (rounds > 1) load(r);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
#pragma unroll
        for (int c = 0; c < 3; ++c) n[c] += k[e] >= (thr | static_cast<uint32_t>(c + 1) << bit) ? 1 : 0;
    }
    const int buf = (bit >> 1) & 1;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      n[c] = __reduce_add_sync(0xffffffffu, n[c]);
      if (lane == 0) s_count[buf][c][warp] = n[c];
    }
    __syncthreads();
    int take = 0;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      n[c] = 0;
#pragma unroll
      for (int w = 0; w < kWarps; w += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&s_count[buf][c][w]);
        n[c] += (v.x + v.y) + (v.z + v.w);
      }
      if (n[c] >= want) {
        take = c + 1;
        at_least = n[c];
      }
    }
    thr |= static_cast<uint32_t>(take) << bit;
  }
  // keys above the threshold, and of those that equal it the first in page order
  int above = 0;
  if (at_least != want) {
    for (int r = 0; r < rounds; ++r) {
      if (rounds > 1) load(r);
#pragma unroll
      for (int e = 0; e < kPer; ++e) above += k[e] > thr ? 1 : 0;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    __syncthreads();
    if (lane == 0) s_count[0][0][warp] = above;
    __syncthreads();
    above = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) above += s_count[0][0][w];
  }
  const int ties = at_least != want ? want - above : last;    // that are taken
  int n_out = 0, n_tie = 0;
  for (int r = 0; r < rounds; ++r) {
    if (rounds > 1) load(r);
    const int i0 = (r * kThreads + tid) * kPer;
    int mine = 0;                                             // above << 16 | equal
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (i0 + e < last) mine += k[e] > thr ? 1 << 16 : k[e] == thr ? 1 : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) s_count[1][0][warp] = incl;
    __syncthreads();
    int before = incl - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before += w < warp ? s_count[1][0][w] : 0;
      all += s_count[1][0][w];
    }
    int tie = n_tie + (before & 0xffff);
    int at = n_out + (before >> 16) + min(tie, ties) - min(n_tie, ties);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (i0 + e >= last) continue;
      const bool equal = k[e] == thr;
      if (k[e] > thr || (equal && tie < ties)) out[at++] = i0 + e;
      tie += equal ? 1 : 0;
    }
    n_out += (all >> 16) + min(n_tie + (all & 0xffff), ties) - min(n_tie, ties);
    n_tie += all & 0xffff;
  }
}

template <int kPer>
__global__ void __launch_bounds__(kPickThreads) kv_pick_kernel(const KvSelectParams p) {
  const int t = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int64_t row = (static_cast<int64_t>(b) * p.c.heads + head) * p.tokens + t;
  const int last = kv_last_page(p, b, t);
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the scores; every block waits, so that none outlive this call
  pick_pages<kPer, kPickThreads, false>(p, p.keys + row * p.row_keys, last, p.selected + row * p.n);
}

// Both in one launch for few tokens: the blocks of a cluster score a share of
// the pages each and put token t's keys into the shared memory of block t, which
// then picks.  A launch less is 2.3 us less of a call (14 to 11.7), and on the device
// it is the same (2048 pages of 16 heads: 10.6 us, 10.2 with two; 1 head: 8.1, 8.5)
// as long as every block has an SM to itself and a page a thread: 128-thread blocks
// that take two pages each need 11.4 us, and 64 x 8 heads of 257 pages 22 us against 17.
constexpr int kFusedBlocks = 8;
constexpr int kFusedPages = 4096;
__host__ __device__ constexpr int fused_threads(int64_t width) { return width <= 128 * kFusedBlocks ? 128 : 256; }

template <typename T, int D, int kPer, int kThreads>
__global__ void __launch_bounds__(kThreads) kv_select_kernel(const KvSelectParams p) {
  __shared__ __align__(16) uint32_t s_q[kSelRows][D / 4];
  __shared__ float s_s[kSelRows];
  extern __shared__ __align__(16) uint32_t s_keys[];     // row_keys of this block's token
  const int rank = blockIdx.x, blocks = gridDim.x, head = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5;
  cluster_arrive();   // waited for below: all blocks run
  const int tokens = kv_queries(p, b);
  const int end = kv_last_page(p, b, tokens - 1);   // complete pages
  int slot = rank * kThreads + tid, page = slot < end ? kv_page(p.c, b, slot) : -1;
  uint32_t k[D / 2];
  float k_scale = 0.0f;
  if (page >= 0) load_sums<D>(p, page, head, k, k_scale);
  const int rows = tokens * p.group;
  for (int r = warp; r < rows; r += kThreads / 32) {
    const int t = r / p.group, h = head * p.group + r % p.group;
    quantise_row<T, D>(static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2], s_q[r], &s_s[r]);
  }
  __syncthreads();
  cluster_wait();
  const uint32_t base = smem_u32(s_keys);
  while (slot < end) {
    for (int t = 0; t < tokens; ++t) {
      uint32_t key = 0;                                  // a bad page number: never worth choosing
      if (page >= 0) {
        float best = row_score<D>(k, s_q[t * p.group], s_s[t * p.group]);
        for (int g = 1; g < p.group; ++g) best = fmaxf(best, row_score<D>(k, s_q[t * p.group + g], s_s[t * p.group + g]));
        key = score_key(best, k_scale);
      }
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(base + slot * 4), "r"(t));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(key) : "memory");
    }
    slot += blocks * kThreads;
    page = slot < end ? kv_page(p.c, b, slot) : -1;
    if (page >= 0) load_sums<D>(p, page, head, k, k_scale);
  }
  cluster_sync();
  if (rank >= p.tokens) return;
  const int64_t row = (static_cast<int64_t>(b) * p.c.heads + head) * p.tokens + rank;
  pick_pages<kPer, kThreads, true>(p, s_keys, kv_last_page(p, b, rank), p.selected + row * p.n);
}

}  // namespace h3b

namespace {

template <typename T, int D>
int launch_kv_select(const char* name, const h3b::KvSelectParams& p, int blocks, int64_t batch, cudaStream_t st) {
  using namespace h3b;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)p.c.heads, (unsigned)batch);
  cfg.blockDim = dim3(fused_threads(p.c.width));
  cfg.dynamicSmemBytes = (size_t)p.row_keys * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const int keys = p.c.width - 1;    // at most: a row's own page is not scored
  cudaError_t e = fused_threads(p.c.width) == 128
                      ? keys <= 4 * 128 ? cudaLaunchKernelEx(&cfg, kv_select_kernel<T, D, 4, 128>, p)
                                        : cudaLaunchKernelEx(&cfg, kv_select_kernel<T, D, 8, 128>, p)
                  : keys <= 8 * 256 ? cudaLaunchKernelEx(&cfg, kv_select_kernel<T, D, 8, 256>, p)
                                    : cudaLaunchKernelEx(&cfg, kv_select_kernel<T, D, 16, 256>, p);
  if (e != cudaSuccess) return h3b_host::set_error(H3B_ECUDA, "%s: launch: %s", name, cudaGetErrorString(e));
  return h3b_host::check_launch(name);
}

}  // namespace

extern "C" size_t h3b_kv_select_i8_workspace_size(int64_t batch, int64_t kv_heads, int64_t tokens,
                                                  int64_t table_width) {
  if (batch <= 0 || kv_heads <= 0 || tokens <= 0 || table_width <= 0) return 16;
  if (table_width > h3b_host::kKvMostKeys) return SIZE_MAX;
  return h3b_host::kv_bytes({batch, kv_heads, tokens, (table_width + 3) & ~int64_t(3), 4});
}

extern "C" int h3b_kv_select_i8(const void* q, const int64_t* q_strides, const h3b_kv_cache* cache,
                                const int32_t* page_table, int64_t batch, int64_t table_width, const int32_t* lengths,
                                const int32_t* counts, int64_t q_heads, int64_t tokens, int64_t n_selected, int dtype,
                                int32_t* selected, void* workspace, size_t workspace_bytes, h3b_stream_t stream) {
  const char* name = "h3b_kv_select_i8";
  h3b::KvSelectParams p{};
  int rc = h3b_host::kv_view(name, cache, page_table, batch, table_width, &p.c);
  if (rc) return rc;
  if (!q || !q_strides || !lengths || !selected) return h3b_host::set_error(H3B_EINVAL, "%s: NULL argument", name);
  if (dtype != H3B_TYPE_F16 && dtype != H3B_TYPE_BF16)
    return h3b_host::set_error(H3B_EINVAL, "%s: q must be fp16 or bf16", name);
  if (q_heads <= 0 || q_heads % cache->kv_heads || q_heads > h3b_host::kKvMostHeads)
    return h3b_host::set_error(H3B_EINVAL, "%s: q_heads must be a positive multiple of kv_heads", name);
  if (tokens < 0 || tokens > (int64_t(1) << 20) || n_selected <= 0 || n_selected > h3b_host::kKvMostSelected)
    return h3b_host::set_error(H3B_EINVAL, "%s: bad token count or page count", name);
  if (tokens == 0) return H3B_OK;
  if (!workspace || !h3b_host::aligned16(workspace) ||
      workspace_bytes < h3b_kv_select_i8_workspace_size(batch, cache->kv_heads, tokens, table_width))
    return h3b_host::set_error(H3B_EINVAL, "%s: workspace missing, misaligned or too small", name);
  p.q = q;
  p.lengths = lengths;
  p.counts = counts;
  p.keys = static_cast<uint32_t*>(workspace);
  p.selected = selected;
  for (int i = 0; i < 3; ++i) p.qs[i] = q_strides[i];
  p.group = (int)(q_heads / cache->kv_heads);
  p.tokens = (int)tokens;
  p.n = (int)n_selected;
  p.row_keys = (int)((table_width + 3) & ~int64_t(3));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = cache->head_dim == 128;
  const int threads = h3b::fused_threads(table_width);
  const int blocks = (int)std::min<int64_t>(h3b::kFusedBlocks, (table_width + threads - 1) / threads);
  if (table_width <= h3b::kFusedPages && tokens <= blocks && tokens * p.group <= h3b::kSelRows &&
      batch * cache->kv_heads * blocks <= h3b_host::num_sms()) {
    if (dtype == H3B_TYPE_F16) return wide ? launch_kv_select<__half, 128>(name, p, blocks, batch, st) : launch_kv_select<__half, 64>(name, p, blocks, batch, st);
    return wide ? launch_kv_select<__nv_bfloat16, 128>(name, p, blocks, batch, st)
                : launch_kv_select<__nv_bfloat16, 64>(name, p, blocks, batch, st);
  }
  dim3 g1((unsigned)((table_width + h3b::kSelThreads - 1) / h3b::kSelThreads), (unsigned)cache->kv_heads, (unsigned)batch);
  dim3 g2((unsigned)tokens, (unsigned)cache->kv_heads, (unsigned)batch);
  if (dtype == H3B_TYPE_F16) {
    if (wide) h3b::kv_score_kernel<__half, 128><<<g1, h3b::kSelThreads, 0, st>>>(p);
    else h3b::kv_score_kernel<__half, 64><<<g1, h3b::kSelThreads, 0, st>>>(p);
  } else {
    if (wide) h3b::kv_score_kernel<__nv_bfloat16, 128><<<g1, h3b::kSelThreads, 0, st>>>(p);
    else h3b::kv_score_kernel<__nv_bfloat16, 64><<<g1, h3b::kSelThreads, 0, st>>>(p);
  }
  rc = h3b_host::check_launch(name);
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = g2;
  cfg.blockDim = dim3(h3b::kPickThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};   // its blocks may be resident before the scores are done; they wait for them
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = table_width <= 4 * h3b::kPickThreads    ? cudaLaunchKernelEx(&cfg, h3b::kv_pick_kernel<4>, p)
                  : table_width <= 8 * h3b::kPickThreads  ? cudaLaunchKernelEx(&cfg, h3b::kv_pick_kernel<8>, p)
                  : table_width <= 20 * h3b::kPickThreads ? cudaLaunchKernelEx(&cfg, h3b::kv_pick_kernel<20>, p)
                                                          : cudaLaunchKernelEx(&cfg, h3b::kv_pick_kernel<64>, p);
  if (e != cudaSuccess) return h3b_host::set_error(H3B_ECUDA, "%s: selection launch: %s", name, cudaGetErrorString(e));
  return h3b_host::check_launch(name);
}
