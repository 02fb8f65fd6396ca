// Attention over the paged INT8 cache for few query rows: keys split over
// blocks, joined by a second kernel (the mathematics: attention_kv.cuh).
#include <type_traits>

#include "attention_kv.cuh"

namespace h3b {

// D += A B, m16n8k16, fp16 operands, fp32 accumulators.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A block takes 16 rows (query tokens x heads of one group) and a run of key
// tiles; its warps take the tiles in turn, each with its own ring of shared
// memory that bulk copies fill (a page's codes of one head are contiguous).
// Codes go from shared memory straight into the m16n8k16 operand layout: a
// dot product does not care in which order dims are taken, nor a weighted sum
// in which order keys are, so each thread reads 16 consecutive bytes of a key
// (four k-steps of K) or D/8 consecutive dims of four keys (a k-step of V).
// With at most 8 rows the rows 8..15 of the second product carry what fp16
// rounds off the weights, so that rounding costs nothing. With more, fp16 outputs
// take the product twice for it: 16 rows over 4 x 32768 keys take 92 us instead
// of 86 (dim 64) and 102 instead of 96 (dim 128), and the error over short runs
// of keys falls from 3.0e-4 to the 2.1e-4 that rounding the output alone leaves.
// bf16 outputs round eight times coarser and go without.
//
// The rows see nearly all keys of their sequence, so a call moves the cache's
// bytes once per 16-row tile (with selected pages, a token's pages once per token and
// tile) and is bound by HBM when it is long and by latency (table, scale
// and code loads in a row, then the join) when it is short.  One token each over
// 16 x 6553..32768 keys, 8 heads of dim 128, 32 query heads: 690 MB in 134 us =
// 5.2 TB/s, with the issue slots 51 % and the tensor pipe 33 % in use; 12 warps an
// SM hide each other's latency.  Before runs were fitted to waves, at 141 us: 8 warps
// 154 us, tiles of half the size 165 us, of twice the size 178 us.  One token over 1797 keys of 16 heads: 7.2 us.
// (Pages with a low scale of V cost their branch and the two-step joins: 131 and 7.0 us without;
// a second instance of the loop for them spills: 137 us.)
constexpr int kSplitWarps = 4;
constexpr int kSplitStages = 2;
constexpr int kSplitBlocks = 3;       // blocks an SM holds (two with three stages: 154 against 141 us on 16 x 6553..32768 keys)
constexpr int kSplitCluster = 8;      // most blocks that join through shared memory
constexpr int kSplitRows = 16;
constexpr int kSplitPages = 256;      // pages a block's run of tiles may span
constexpr int kSplitStageBytes = 8192;

template <int D>
struct KvSplit {
  static constexpr int kKeys = kSplitStageBytes / 2 / D;    // keys per tile: 64 or 32
  static constexpr int kRing = kSplitWarps * kSplitStages * kSplitStageBytes;
  static constexpr int kMeta = kSplitPages * 16 + kSplitPages * 4;
  static constexpr int kSmem = kRing + kMeta + kSplitWarps * kSplitStages * 8 + 128;
};

// Tiles a sequence's rows need, in tiles of `keys`: none without queries.
__device__ __forceinline__ int split_tiles(const KvAttnParams& p, int b, int keys, int& tile0) {
  const int len = kv_length(p.c, p.lengths, b), n = kv_count(p.counts, p.tokens, b);
  int first, last, unused;
  tile0 = 0;
  if (n == 0) return 0;
  const int t0 = max(0, n - len);             // the first row that has a position
  kv_range(p, len, n, t0, first, unused);
  kv_range(p, len, n, n - 1, unused, last);
  tile0 = first / keys;
  return last > first ? (last + keys - 1) / keys - tile0 : 0;
}

template <typename T, int D, bool kSparse, bool kSmall>
__global__ void __launch_bounds__(32 * kSplitWarps, kSplitBlocks) attention_kv_split_kernel(const KvAttnParams p) {
  using S = KvSplit<D>;
  constexpr int KT = S::kKeys, kTiles = KT / 8, kSteps = D / 16, kThreads = 32 * kSplitWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  float4* s_meta = reinterpret_cast<float4*>(smem + S::kRing);                 // per page: x scale, log2 vs, 1/vs or log2 vs
  int* s_page = reinterpret_cast<int*>(s_meta + kSplitPages);                  // pool page, -1: none
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(s_page + kSplitPages);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const int hk = blockIdx.y;

  // ---- which sequence, rows and tiles ----
  int b, t_sparse = 0, rt, slot, split, splits, tile0, tile1;
  if (kSparse) {
    b = blockIdx.z;
    int x = blockIdx.x;
    split = x % p.slots;
    x /= p.slots;
    rt = x % p.row_tiles;
    t_sparse = x / p.row_tiles;
    splits = p.slots;
    slot = (b * p.tokens + t_sparse) * p.slots + split;
    const int tiles = (p.n_selected * p.c.page + KT - 1) / KT;
    tile0 = min(split * p.chunk, tiles);
    tile1 = min(tile0 + p.chunk, tiles);
  } else if (p.cluster) {
    b = blockIdx.z;
    rt = blockIdx.x / p.slots;
    slot = split = blockIdx.x % p.slots;
    splits = p.slots;
    int t0;
    const int tiles = split_tiles(p, b, KT, t0), chunk = (tiles + splits - 1) / splits;
    tile0 = t0 + min(split * chunk, tiles);
    tile1 = t0 + min(split * chunk + chunk, tiles);
  } else {
    rt = blockIdx.x / p.slots;
    slot = blockIdx.x % p.slots;
    int t0, chunk, first_slot;
    // Runs of `chunk` tiles, equal for the whole batch, about p.share of them and at most p.fit
    auto clamp_chunk = [&](int64_t n) {
      return static_cast<int>(min(max(n, static_cast<int64_t>(kSplitWarps)), static_cast<int64_t>(p.chunk)));
    };
    if (p.c.batch == 1 || p.plan == nullptr) {       // one sequence, or none is split
      b = p.plan == nullptr ? slot : 0;
      const int tiles = split_tiles(p, b, KT, t0);
      chunk = p.plan == nullptr ? max(tiles, 1) : clamp_chunk((tiles + p.share - 1) / p.share);
      splits = max(1, (tiles + chunk - 1) / chunk);
      first_slot = b;
      if (slot >= first_slot + splits) return;
    } else {                                         // every warp scans the lengths
      int base, sum = 0, longest = 0;
      const bool wide = p.c.batch > 32;              // more than a warp's: the block's warps share them
      for (int i = wide ? tid : lane; i < p.c.batch; i += wide ? kThreads : 32) {
        const int tiles = split_tiles(p, i, KT, base);
        sum += tiles;
        longest = max(longest, tiles);
      }
      sum = __reduce_add_sync(0xffffffffu, sum);
      longest = __reduce_max_sync(0xffffffffu, longest);
      if (wide) {
        __shared__ int2 s_sum[kSplitWarps];
        if (lane == 0) s_sum[warp] = make_int2(sum, longest);
        __syncthreads();
        sum = longest = 0;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) sum += s_sum[w].x, longest = max(longest, s_sum[w].y);
      }
      chunk = clamp_chunk((sum + p.share - 1) / p.share);
      if (p.fit < p.c.batch + p.share) {
        // Sequences end inside runs, so more come out than that.  A length that does for p.fit in any case, and the
        // eighths down to the one above; each warp counts the runs of two of them.
        __shared__ int s_runs[2 * kSplitWarps];
        const int lo = chunk;
        const int hi = p.fit > p.c.batch ? clamp_chunk((sum + p.fit - p.c.batch - 1) / (p.fit - p.c.batch)) : p.chunk;
        auto eighth = [&](int i) { return lo + (hi - lo) * i / (2 * kSplitWarps); };
        const int c0 = eighth(2 * warp), c1 = eighth(2 * warp + 1);
        int runs0 = 0, runs1 = 0;
        for (int i = lane; i < p.c.batch; i += 32) {
          const int tiles = split_tiles(p, i, KT, base);
          runs0 += max(1, (tiles + c0 - 1) / c0);
          runs1 += max(1, (tiles + c1 - 1) / c1);
        }
        runs0 = __reduce_add_sync(0xffffffffu, runs0);
        runs1 = __reduce_add_sync(0xffffffffu, runs1);
        if (lane == 0) s_runs[2 * warp] = runs0, s_runs[2 * warp + 1] = runs1;
        __syncthreads();
        chunk = hi;
#pragma unroll
        for (int i = 2 * kSplitWarps - 1; i >= 0; --i)
          if (s_runs[i] <= p.fit) chunk = eighth(i);
      }
      if (longest <= chunk) {
        if (slot >= p.c.batch) return;
        b = first_slot = slot;
        splits = 1;
      } else {
        int mine = 0;                                // a lane has every 32nd sequence; runs go by lane, then sequence
        for (int i = lane; i < p.c.batch; i += 32) mine += max(1, (split_tiles(p, i, KT, base) + chunk - 1) / chunk);
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += up;
        }
        before -= mine;
        b = -1, first_slot = splits = 0;
        for (int i = lane; i < p.c.batch; i += 32) {
          const int n = max(1, (split_tiles(p, i, KT, base) + chunk - 1) / chunk);
          if (slot >= before && slot < before + n) b = i, first_slot = before, splits = n;
          before += n;
        }
        const unsigned found = __ballot_sync(0xffffffffu, b >= 0);
        if (!found) return;
        const int from = __ffs(found) - 1;
        b = __shfl_sync(0xffffffffu, b, from);
        first_slot = __shfl_sync(0xffffffffu, first_slot, from);
        splits = __shfl_sync(0xffffffffu, splits, from);
      }
    }
    split = slot - first_slot;
    const int tiles = split_tiles(p, b, KT, t0);
    tile0 = t0 + min(split * chunk, tiles);
    tile1 = t0 + min(split * chunk + chunk, tiles);
    if (split == 0 && tid == 0 && hk == 0 && rt == 0 && p.plan) p.plan[b] = make_int2(first_slot, splits);
  }
  const int len = kv_length(p.c, p.lengths, b), n_tok = kv_count(p.counts, p.tokens, b);
  if ((kSparse ? t_sparse : rt * kSplitRows / p.group) >= n_tok) tile1 = tile0;      // padding rows see nothing

  // ---- the pages of the run: numbers, then the first copies, then scales ----
  const int page0 = (tile0 * KT) >> p.c.page_shift;
  const int n_pages = tile1 > tile0 ? ((tile1 * KT - 1) >> p.c.page_shift) - page0 + 1 : 0;
  const int32_t* sel =
      kSparse ? p.selected + ((static_cast<int64_t>(b) * p.c.heads + hk) * p.tokens + t_sparse) * p.n_selected : nullptr;
  for (int i = tid; i < n_pages; i += kThreads) {
    int ord = page0 + i;
    if (kSparse) ord = ord < p.n_selected ? sel[ord] : -1;
    int page = -1;
    if (ord >= 0 && static_cast<int64_t>(ord) * p.c.page < len) page = kv_page(p.c, b, ord);
    s_page[i] = page;
  }
  if (tid < kSplitWarps * kSplitStages) {
    mbar_init(&s_bar[tid], 1);
    fence_barrier_init();     // of this thread's own barrier: a fence orders only what its thread did
  }
  __syncthreads();

  const uint32_t ring = smem_u32(smem) + warp * kSplitStages * kSplitStageBytes;
  const uint32_t bars = smem_u32(s_bar + warp * kSplitStages);
  const int seg_keys = min(p.c.page, KT);
  const uint32_t seg_bytes = seg_keys * D;
  auto issue = [&](int tile, int stage) {
    // lane j copies the j-th segment (a page or the part of it in this tile)
    const int key = tile * KT + lane * seg_keys;
    int page = -1;
    if (lane * seg_keys < KT) page = s_page[(key >> p.c.page_shift) - page0];
    const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
    const uint32_t bar = bars + stage * 8;
    if (lane == 0)
      asm volatile(
          "{\n\t.reg .b64 st;\n\t"
          "mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar),
          "r"(2 * seg_bytes * __popc(there))
          : "memory");
    __syncwarp();
    if (page >= 0) {
      const int64_t off = ((static_cast<int64_t>(page) * p.c.heads + hk) * p.c.page + (key & (p.c.page - 1))) * D;
      const uint32_t dst = ring + stage * kSplitStageBytes + lane * seg_bytes;
      bulk_load(dst, p.c.code[0] + off, seg_bytes, bar);
      bulk_load(dst + KT * D, p.c.code[1] + off, seg_bytes, bar);
    }
  };
  for (int s = 0; s < kSplitStages; ++s) {
    const int tile = tile0 + warp + s * kSplitWarps;
    if (tile < tile1) issue(tile, s);
  }
  bool low = false;
  for (int i = tid; i < n_pages; i += kThreads) {
    const int page = s_page[i];
    float4 f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);   // no page: weight 0
    if (page >= 0) {
      const int64_t ph = static_cast<int64_t>(page) * p.c.heads + hk;
      float vs = p.c.scale[1][ph];
      vs = vs < kKvMinScale ? kKvMinScale : vs;            // a page never written holds zeros; NaN stays
      // a NaN scale of V goes with the scores, which are masked, and not with the factor of the sums, which is not:
      // rows that do not see the page add 0 * (1 / vs)
      f = make_float4(p.c.scale[0][ph] * p.scale_log2, log2f(vs), isnan(vs) ? 0.0f : __frcp_rn(vs), 0.0f);
      if (vs < kKvLowScale) low = true, f.z = f.y;         // its keys are summed from their scores
    }
    if (kSparse && page >= 0) f.w = __int_as_float(sel[page0 + i] << p.c.page_shift);   // first position
    s_meta[i] = f;
  }

  // ---- the query rows ----
  const int g_rows = kSparse ? p.group : p.group * p.tokens;      // rows of this (sequence, kv head)
  uint32_t qa[kSteps][4];
  float back[2];
  int first[2], last[2];
  int first_max = 0, last_min = 0x7fffffff;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = rt * kSplitRows + r + 8 * u;
    const bool real = row < g_rows && !(kSmall && u == 1);
    const int t = kSparse ? t_sparse : row / p.group, h = hk * p.group + (kSparse ? row : row % p.group);
    first[u] = 0, last[u] = 0x7fffffff;      // padding rows never force masking
    if (real) kv_range(p, len, n_tok, t, first[u], last[u]);
    first_max = max(first_max, first[u]);
    last_min = min(last_min, last[u]);
    float x[D / 4];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
    if (real) {
      const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
#pragma unroll
      for (int v = 0; v < D / 64; ++v)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          load8(q + 64 * v + 16 * c + 8 * i, p.vec_q, *reinterpret_cast<float(*)[8]>(&x[16 * v + 8 * i]));
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float f = row_scaling(T(), top, back[u]);
    // k index 2c + e of step s is dim 64 (s / 4) + 16 c + 4 (s % 4) + e, and 2c + 8 + e the dim two further
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 16 * (s >> 2) + 4 * (s & 3) + 2 * e;
        qa[s][u + 2 * e] = h2_bits(__floats2half2_rn(x[i] * f, x[i + 1] * f));
      }
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    first_max = max(first_max, __shfl_xor_sync(0xffffffffu, first_max, o));
    last_min = min(last_min, __shfl_xor_sync(0xffffffffu, last_min, o));
  }
  low = __syncthreads_or(low);   // scales are in shared memory

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  constexpr int kU = kSmall ? 1 : 2;
  constexpr bool kLow = !kSmall && std::is_same<T, __half>::value;
  // column j of an S tile is key (j >> 1) + 4 (j & 1) of its eight, so that the
  // four keys a V load touches at once are neighbours
  const int k_row = (r >> 1) + 4 * (r & 1);
  bool ok = true;
  int stage = 0, tile = tile0 + warp;
  uint32_t phase = 0;
  for (; tile < tile1; tile += kSplitWarps) {
    ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(bars + stage * 8, phase, nullptr));
    if (!ok) break;
    const uint8_t* ks = smem + (warp * kSplitStages + stage) * kSplitStageBytes;
    const uint8_t* vs = ks + KT * D;
    // S = Q K^T
    float x[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0.0f;
#pragma unroll
      for (int v = 0; v < D / 64; ++v) {
        const uint4 w = *reinterpret_cast<const uint4*>(ks + (8 * t + k_row) * D + 64 * v + 16 * c);
        const uint32_t ww[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
        for (int s = 0; s < 4; ++s)
          mma_16816(x[t], qa[4 * v + s], codes_to_h2(ww[s], 0x4140), codes_to_h2(ww[s], 0x4342));
      }
    }
    // scores in base 2 with log2 of the V scale; masked where a row does not see the key
    float inv[kTiles / 2];
    float top[2] = {-INFINITY, -INFINITY};
    const int key0 = tile * KT;
    const bool clear = !kSparse && key0 >= first_max && key0 + KT <= last_min;
#pragma unroll
    for (int t2 = 0; t2 < kTiles / 2; ++t2) {
      const float4 f = s_meta[((key0 + 16 * t2) >> p.c.page_shift) - page0];
      inv[t2] = f.z;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float sc = f.x * back[u];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& y = x[2 * t2 + tt][2 * u + e];
            y = __fmaf_rn(y, sc, f.y);
            if (!clear) {
              const int in = 16 * t2 + 8 * tt + c + 4 * e;
              const int key = kSparse ? __float_as_int(f.w) + ((key0 + in) & (p.c.page - 1)) : key0 + in;
              if (key < first[u] || key >= last[u]) y = -INFINITY;
            }
            top[u] = fmaxf(top[u], y);
          }
      }
    }
    float ref[2];
    bool moved = low;      // (a run with low pages always goes there)
    float fall[2], alpha[2];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 1));
      top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 2));
      const float m_new = fmaxf(m[u], top[u]);
      ref[u] = m_new == -INFINITY ? 0.0f : m_new;
      moved |= m_new > m[u];
      fall[u] = m[u] - ref[u];
      alpha[u] = ex2_approx(fall[u]);
      m[u] = m_new;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int u = 0; u < kU; ++u) l[u] = fall[u] > -126.0f ? l[u] * alpha[u] : rescale_sum(l[u], fall[u]);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= alpha[0];
        o[i][1] *= alpha[0];
        o[i][2] *= alpha[kSmall ? 0 : 1];
        o[i][3] *= alpha[kSmall ? 0 : 1];
      }
      if (low) {
#pragma unroll
        for (int s = 0; s < kTiles / 2; ++s)
          if (inv[s] < 0.0f) {      // the same for the warp
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) l[u] += ex2_approx(x[2 * s + (e >> 1)][2 * u + (e & 1)] - (ref[u] + inv[s]));
          }
      }
    }
    // weights, their sums, and O += W V
#pragma unroll
    for (int s = 0; s < kTiles / 2; ++s) {
      uint32_t pa[4], pl[4];
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const float w0 = ex2_approx(x[2 * s + tt][2 * u] - ref[u]), w1 = ex2_approx(x[2 * s + tt][2 * u + 1] - ref[u]);
          l[u] = __fmaf_rn(w0 + w1, inv[s], l[u]);
          const __half2 hi = __floats2half2_rn(w0, w1);
          pa[2 * tt + u] = h2_bits(hi);
          if (kSmall || kLow) {
            const float2 f = __half22float2(hi);
            (kSmall ? pa[2 * tt + 1] : pl[2 * tt + u]) = h2_bits(__floats2half2_rn(w0 - f.x, w1 - f.y));
          }
        }
      }
      // keys 16 s + {c, c + 4, c + 8, c + 12}, dims D/8 r ..: words of four dims
      uint32_t w[4][D / 32];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* at = vs + (16 * s + c + 4 * k) * D + (D / 8) * r;
        if (D == 64) {
          const uint2 q2 = *reinterpret_cast<const uint2*>(at);
          w[k][0] = q2.x, w[k][1] = q2.y;
        } else {
          const uint4 q4 = *reinterpret_cast<const uint4*>(at);
          w[k][0] = q4.x, w[k][1] = q4.y, w[k][D / 32 - 2] = q4.z, w[k][D / 32 - 1] = q4.w;
        }
      }
#pragma unroll
      for (int d4 = 0; d4 < D / 32; ++d4) {
        uint32_t lo[2], hi[2];   // key pairs interleaved: bytes (k0, k1) of dims 0, 1 and of dims 2, 3
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          lo[k] = __byte_perm(w[2 * k][d4], w[2 * k + 1][d4], 0x5140) ^ 0x80808080u;
          hi[k] = __byte_perm(w[2 * k][d4], w[2 * k + 1][d4], 0x7362) ^ 0x80808080u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b0 = codes_to_h2(e < 2 ? lo[0] : hi[0], e & 1 ? 0x4342 : 0x4140);
          const uint32_t b1 = codes_to_h2(e < 2 ? lo[1] : hi[1], e & 1 ? 0x4342 : 0x4140);
          mma_16816(o[4 * d4 + e], pa, b0, b1);
          if (kLow) mma_16816(o[4 * d4 + e], pl, b0, b1);
        }
      }
    }
    __syncwarp();   // every lane has read the stage
    const int next = tile + kSplitStages * kSplitWarps;
    if (next < tile1) issue(next, stage);
    if (++stage == kSplitStages) stage = 0, phase ^= 1;
  }
  if (!ok) {   // a wait gave up (the error word says so): let the copies issued after it land
    for (int s = 1; s < kSplitStages; ++s) {
      if (++stage == kSplitStages) stage = 0, phase ^= 1;
      if (tile + s * kSplitWarps < tile1) mbar_wait_u32(bars + stage * 8, phase, nullptr);
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
    l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
  }

  // ---- join the warps: thread (r, c) holds dims D/4 c .. of rows r and r + 8 ----
  __syncthreads();   // all copies have landed and been read (every warp waited for each of its own)
  constexpr int kOut = kSmall ? 8 : 16;
  float* s_o = reinterpret_cast<float*>(smem);                       // [warp][row][D + 4]
  float* s_ml = s_o + kSplitWarps * kOut * (D + 4);                  // [warp][row][2]
  static_assert(kSplitWarps * kOut * (D + 6) * 4 <= S::kRing, "join buffer");
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    float* dst = s_o + (warp * kOut + r + 8 * u) * (D + 4) + (D / 4) * c;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      dst[i] = kSmall ? o[i][0] + o[i][2] : o[i][2 * u];
      dst[D / 8 + i] = kSmall ? o[i][1] + o[i][3] : o[i][2 * u + 1];
    }
    if (c == 0) {
      s_ml[(warp * kOut + r + 8 * u) * 2] = m[u];
      s_ml[(warp * kOut + r + 8 * u) * 2 + 1] = l[u];
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  const int rows = min(kOut, g_rows - rt * kSplitRows);
  auto finish = [&](int row, int d, float4 acc, float m_row, float l_row) {   // dims d .. d + 3 of a joined row
    const int full = rt * kSplitRows + row;
    const int t = kSparse ? t_sparse : full / p.group, h = hk * p.group + (kSparse ? full : full % p.group);
    const float f = l_row == 0.0f ? 0.0f : __frcp_rn(l_row);
    T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] + d;
    from_f32(acc.x * f, out[0]);
    from_f32(acc.y * f, out[1]);
    from_f32(acc.z * f, out[2]);
    from_f32(acc.w * f, out[3]);
    if (p.lse && d == 0)
      p.lse[(static_cast<int64_t>(b) * p.q_heads + h) * p.tokens + t] =
          l_row == 0.0f ? -INFINITY : ((m_row == -INFINITY ? 0.0f : m_row) + log2f(l_row)) * kLn2;
  };
  constexpr int kRow = D + 4;                                        // weighted codes, m, l of a row of this block
  float* s_c = s_ml + kSplitWarps * kOut * 2;
  static_assert((kSplitWarps * kOut * (D + 6) + kOut * kRow) * 4 <= S::kRing, "join buffer");
  for (int i = tid; i < rows * (D / 4); i += kThreads) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) mm = fmaxf(mm, s_ml[(w * kOut + row) * 2]);
    const float rf = mm == -INFINITY ? 0.0f : mm;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float f = ex2_approx(s_ml[(w * kOut + row) * 2] - rf);
      const float4 v = *reinterpret_cast<const float4*>(s_o + (w * kOut + row) * (D + 4) + d);
      acc.x = __fmaf_rn(f, v.x, acc.x);
      acc.y = __fmaf_rn(f, v.y, acc.y);
      acc.z = __fmaf_rn(f, v.z, acc.z);
      acc.w = __fmaf_rn(f, v.w, acc.w);
      ll += rescale_sum(s_ml[(w * kOut + row) * 2 + 1], s_ml[(w * kOut + row) * 2] - rf);
    }
    if (splits == 1) {
      finish(row, d, acc, mm, ll);
    } else {
      const int64_t at = ((static_cast<int64_t>(slot) * p.c.heads + hk) * p.row_tiles + rt) * kSplitRows + row;
      float* dst = p.cluster ? s_c + row * kRow : p.part + at * kRow;
      *reinterpret_cast<float4*>(dst + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mm, ll);
    }
  }
  if (p.cluster && splits > 1) {
    // the cluster's blocks join their rows through each other's shared memory, a share of the dims each
    cluster_sync();
    const uint32_t mine = smem_u32(s_c);
    for (int i = split * kThreads + tid; i < rows * (D / 4); i += splits * kThreads) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4;
      float mm = -INFINITY, ll = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float2 ml[kSplitCluster];
      float4 v[kSplitCluster];
#pragma unroll
      for (int w = 0; w < kSplitCluster; ++w) {
        if (w >= splits) break;
        uint32_t at;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine + row * kRow * 4), "r"(w));
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[w].x), "=f"(ml[w].y) : "r"(at + D * 4));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[w].x), "=f"(v[w].y), "=f"(v[w].z), "=f"(v[w].w)
                     : "r"(at + d * 4));
        mm = fmaxf(mm, ml[w].x);
      }
      const float rf = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
      for (int w = 0; w < kSplitCluster; ++w) {
        if (w >= splits) break;
        const float f = ex2_approx(ml[w].x - rf);
        acc.x = __fmaf_rn(f, v[w].x, acc.x);
        acc.y = __fmaf_rn(f, v[w].y, acc.y);
        acc.z = __fmaf_rn(f, v[w].z, acc.z);
        acc.w = __fmaf_rn(f, v[w].w, acc.w);
        ll += rescale_sum(ml[w].y, ml[w].x - rf);
      }
      finish(row, d, acc, mm, ll);
    }
    // no block leaves while another reads its shared memory
    cluster_sync();
  }
}

enum KvParts { kPartsPlan, kPartsSparse, kPartsTile };   // how the parts of a row are laid out

template <typename T, int D, KvParts kParts>
__global__ void __launch_bounds__(128) attention_kv_join_kernel(const KvAttnParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int per = p.join_warps, sub = warp % per;   // warps a row has
  const int full = blockIdx.x * (4 / per) + warp / per;   // row of the (sequence, kv head): token * group + head
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (full >= p.group * p.tokens) return;
  const int t = full / p.group, g = full % p.group, h = hk * p.group + g;
  int n;
  int64_t at, step;      // in rows of the parts
  if (kParts == kPartsTile) {
    n = p.slots;
    at = (static_cast<int64_t>(b) * p.c.heads + hk) * p.group * p.tokens + full;
    step = static_cast<int64_t>(p.c.batch) * p.c.heads * p.group * p.tokens;
  } else {
    int slot, in = full;
    if (kParts == kPartsSparse) {
      slot = (b * p.tokens + t) * p.slots;
      n = p.slots;
      in = g;
    } else {
      slot = p.plan[b].x;
      n = p.plan[b].y;
    }
    step = static_cast<int64_t>(p.c.heads) * p.row_tiles * kSplitRows;
    at = slot * step + static_cast<int64_t>(hk) * p.row_tiles * kSplitRows + in;
  }
  if (n <= 1) return;       // written by the block itself
  const float* src = p.part + at * (D + 4);
  step *= D + 4;
  // the parts' maxima and sums a lane each, then the parts four at a time
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, src[s * step + D]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, o[D / 32] = {};
  const int share = (n + per - 1) / per, mine1 = min(n, sub * share + share);
  for (int s0 = sub * share; s0 < mine1; s0 += 32) {
    float f = 0.0f;
    if (s0 + lane < mine1) {
      const float2 ml = *reinterpret_cast<const float2*>(src + (s0 + lane) * step + D);
      f = ex2_approx(ml.x - ref);
      l += rescale_sum(ml.y, ml.x - ref);
    }
    const int end = min(32, mine1 - s0);
#pragma unroll 8
    for (int s = 0; s < end; ++s) {
      const float fs = __shfl_sync(0xffffffffu, f, s);
      const float* v = src + (s0 + s) * step + lane * (D / 32);
#pragma unroll
      for (int k = 0; k < D / 32; k += 2) {
        const float2 x = *reinterpret_cast<const float2*>(v + k);
        o[k] = __fmaf_rn(x.x, fs, o[k]);
        o[k + 1] = __fmaf_rn(x.y, fs, o[k + 1]);
      }
    }
  }
  l = warp_sum(l);
  if (per > 1) {            // four warps, one row a block
    __shared__ float s_part[4][D + 1];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) s_part[warp][lane * (D / 32) + k] = o[k];
    if (lane == 0) s_part[warp][D] = l;
    __syncthreads();
    if (warp > 0) return;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) l += s_part[w][D];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      o[k] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) o[k] += s_part[w][lane * (D / 32) + k];
    }
  }
  const float f = l == 0.0f ? 0.0f : __frcp_rn(l);
  T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] + lane * (D / 32);
#pragma unroll
  for (int k = 0; k < D / 32; ++k) from_f32(o[k] * f, out[k]);
  if (p.lse && lane == 0)
    p.lse[(static_cast<int64_t>(b) * p.q_heads + h) * p.tokens + t] =
        l == 0.0f ? -INFINITY : (ref + log2f(l)) * kLn2;
}

}  // namespace h3b
