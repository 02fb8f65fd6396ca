// Host side of attention over the paged INT8 cache: the choice between the
// kernels of attention_kv_split.cu and attention_kv_tile.cu, workspaces, checks.
#include <atomic>

#include "attention_kv.cuh"

namespace {

// The tensor-core tiles are taken above kTileRows rows of a (sequence, kv head)
// if the 16-row tiles of the other kernel would read more than kTileBytes of
// codes.  Measured, tiles against 16-row tiles, us: 16 heads over 5120 keys, dim 64:
// 33 rows 20 / 16, 64 rows 20 / 19; 8 x 8 heads over 8192 keys, dim 128, fp16 and
// bf16: 17 rows 80 / 81 and 72, 33 rows 80 / 112 and 99, 64 rows 81 / 144 and 128; 32 x
// 16 heads over 2000 keys: 40 rows 127 / 103, 70 rows 128 / 163; 2 x 16 heads over 1024 keys:
// 64 rows (17 MB) 17 / 12, 128 rows (34 MB) 18 / 33.  One limit for both dims: at dim 128
// and 17 to 48 rows over long caches it takes the slower side, by up to 40 % (33 rows, fp16).
constexpr int64_t kTileRows = 48;
constexpr int64_t kTileBytes = int64_t(24) << 20;

// The plan of a call.  tile: attention_kv_tile_kernel, 256 rows a block, the
// keys in `slots` parts.  Otherwise attention_kv_split_kernel: rows in tiles of
// 16, `slots` runs of key tiles at most (dense: over the whole batch, sparse:
// per query token).
struct KvPlan {
  bool tile;
  int64_t row_tiles, slots, chunk, share, fit, cluster, join_warps;
  size_t plan_bytes, part_bytes;
};

KvPlan kv_plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens, int64_t dim, int64_t width,
               int64_t page, int64_t n_selected) {
  using namespace h3b;
  using h3b_host::kv_bytes;
  KvPlan k{};
  k.join_warps = 1;
  const int64_t group = q_heads / kv_heads;
  const int64_t keys = kSplitStageBytes / 2 / dim;
  const int64_t most = (kSplitPages - 1) * page / keys;    // tiles a run may have: it may start inside a page
  const int64_t rows = n_selected > 0 ? group : group * tokens;
  const int64_t row_tiles = (rows + kSplitRows - 1) / kSplitRows;
  k.tile = n_selected <= 0 && rows > kTileRows &&
           batch * kv_heads * row_tiles > kTileBytes / (2 * dim * width * page);
  if (k.tile) {
    k.row_tiles = (rows + 2 * kKtRows - 1) / (2 * kKtRows);
    const int64_t blocks = batch * kv_heads * k.row_tiles, most_blocks = (width * page + kKtKeys - 1) / kKtKeys;
    k.slots = std::max<int64_t>(1, std::min(h3b_host::num_sms() / blocks, most_blocks / 4));
    k.part_bytes = k.slots > 1 ? kv_bytes({k.slots, batch, kv_heads, rows, dim + 4, 4}) : 0;
    k.join_warps = k.slots >= 4 ? 4 : 1;
    return k;
  }
  k.row_tiles = row_tiles;
  const int64_t items = batch * kv_heads * k.row_tiles * (n_selected > 0 ? tokens : 1);
  const int64_t tiles = ((n_selected > 0 ? n_selected : width) * page + keys - 1) / keys;
  // Up to eight runs of a row tile's keys join inside a cluster: one launch and no trip through global memory
  // (one token over 1797 keys, 16 heads: 7.2 us, about 2 more with a second kernel).  For short runs, and for selected pages,
  // which are as many for every row; long sequences of different lengths are better cut into equal parts
  // (16 x 6553..32768 keys: 154 us in clusters of eight, 129 in parts; 134 with low scales looked for).
  const int64_t wave = kSplitBlocks * h3b_host::num_sms();
  const int64_t c = std::max<int64_t>(
      1, std::min({(int64_t)kSplitCluster, wave / items, (tiles + kSplitWarps - 1) / kSplitWarps}));
  if ((tiles + c - 1) / c <= most && (tiles <= c * kSplitWarps * 4 || (n_selected > 0 && c * items >= wave / 2))) {
    k.cluster = c;
    k.slots = c;
    k.chunk = (tiles + c - 1) / c;
    return k;
  }
  // Few rows over long runs: parts through the workspace, joined by a second kernel.
  if (n_selected > 0) {
    const int64_t want = std::max<int64_t>(1, std::min(wave / items, (tiles + kSplitWarps - 1) / kSplitWarps));
    k.chunk = std::min(most, (tiles + want - 1) / want);
    k.slots = (tiles + k.chunk - 1) / k.chunk;
    k.join_warps = k.slots >= 4 ? 4 : 1;
    k.part_bytes = k.slots > 1 ? kv_bytes({batch, tokens, k.slots, kv_heads, k.row_tiles, kSplitRows, dim + 4, 4}) : 0;
  } else {
    k.chunk = most;
    const int64_t per = kv_heads * k.row_tiles;
    const int64_t most_runs = batch * ((tiles + kSplitWarps - 1) / kSplitWarps);
    // Runs fill whole waves of blocks exactly, as few as leave every row tile a few runs: the last wave of a count that
    // fits none is nearly empty, and every run costs the join.  Measured, us for one, two, three waves (140, 50, 80, 217
    // with 2 x wave + batch runs), 8 heads, dim 128: 16 x 6553..32768 keys 135, 129, 133; 1 x 32768 25, 33, 38; 7 x .. 65,
    // 71, 80; 28 x .. 245, 215, 206.  More row tiles than blocks: equal runs of three waves' share, sequences not
    // fitted (64 x 8192: 134, fitted 138); than two waves': only what is longer than a block's share of one is cut
    // (200 x 4096: 195, cut to a third 213, nothing cut 190).
    const bool many = items > wave;
    const int64_t waves = many ? (items > 2 * wave ? 1 : 3) : items * 2 > wave ? 3 : items * 4 > wave ? 2 : 1;
    k.share = std::max<int64_t>(1, std::min(waves * wave / per, most_runs));
    k.fit = many ? batch + k.share : k.share;
    k.slots = std::max(k.fit, batch + batch * (tiles / most));
    k.plan_bytes = k.slots > batch ? ((size_t)batch * 8 + 15) & ~size_t(15) : 0;
    k.join_warps = k.slots >= 4 * batch ? 4 : 1;   // 56 parts of a row: the call takes 60 us with four, 75 with one
    k.part_bytes = k.slots > batch ? kv_bytes({k.slots, kv_heads, k.row_tiles, kSplitRows, dim + 4, 4}) : 0;
  }
  return k;
}

// Lets `kernel` use `bytes` of shared memory; asked of the driver once per kernel and device (`done`: a bit for each
// of the first 64 devices; a kernel's own word).  Nothing here throws: the C entries have no caller that could catch it.
int allow_smem(const char* name, const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
  if (e == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return H3B_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return h3b_host::set_error(H3B_ECUDA, "%s: smem attribute: %s", name, cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return H3B_OK;
}

template <typename T, int D, h3b::KvParts kParts>
int launch_kv_join(const char* name, const h3b::KvAttnParams& p, int64_t batch, cudaStream_t st) {
  using namespace h3b;
  cudaLaunchConfig_t cfg{};
  const int64_t a_block = 4 / p.join_warps;   // rows
  cfg.gridDim = dim3((unsigned)(((int64_t)p.group * p.tokens + a_block - 1) / a_block), (unsigned)p.c.heads, (unsigned)batch);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr{};   // the join's blocks may be resident before the parts are done; they wait for them
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attention_kv_join_kernel<T, D, kParts>, p);
  if (e != cudaSuccess) return h3b_host::set_error(H3B_ECUDA, "%s: join launch: %s", name, cudaGetErrorString(e));
  return h3b_host::check_launch(name);
}

template <typename T, int D, bool kSparse>
int launch_kv_split(const char* name, const h3b::KvAttnParams& p, int64_t batch, cudaStream_t st) {
  using namespace h3b;
  const int rows = kSparse ? p.group : p.group * p.tokens;
  auto kernel = rows <= 8 ? attention_kv_split_kernel<T, D, kSparse, true> : attention_kv_split_kernel<T, D, kSparse, false>;
  constexpr int smem = KvSplit<D>::kSmem;
  static std::atomic<uint64_t> allowed[2];
  int rc = allow_smem(name, reinterpret_cast<const void*>(kernel), smem, allowed[rows <= 8]);
  if (rc) return rc;
  const int64_t x = (int64_t)p.slots * p.row_tiles * (kSparse ? p.tokens : 1);
  if (x > 0x7fffffff) return h3b_host::set_error(H3B_EUNSUPPORTED, "%s: problem too large", name);
  const dim3 grid((unsigned)x, (unsigned)p.c.heads, kSparse || p.cluster ? (unsigned)batch : 1u);
  if (p.cluster > 1) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * kSplitWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return h3b_host::set_error(H3B_ECUDA, "%s: launch: %s", name, cudaGetErrorString(e));
    return h3b_host::check_launch(name);
  }
  kernel<<<grid, 32 * kSplitWarps, smem, st>>>(p);
  rc = h3b_host::check_launch(name);
  if (rc || p.part == nullptr) return rc;
  return launch_kv_join<T, D, kSparse ? kPartsSparse : kPartsPlan>(name, p, batch, st);
}

template <typename T, int D>
int launch_kv_tile(const char* name, const h3b::KvAttnParams& p, int64_t batch, cudaStream_t st) {
  using namespace h3b;
  auto kernel = attention_kv_tile_kernel<T, D>;
  constexpr int smem = KvTile<D>::kSmem;
  static_assert(smem <= 232448, "shared memory budget");
  static std::atomic<uint64_t> allowed;
  int rc = allow_smem(name, reinterpret_cast<const void*>(kernel), smem, allowed);
  if (rc) return rc;
  kernel<<<dim3((unsigned)(p.row_tiles * p.slots), (unsigned)p.c.heads, (unsigned)batch), kKtThreads, smem, st>>>(p);
  rc = h3b_host::check_launch(name);
  if (rc || p.part == nullptr) return rc;
  return launch_kv_join<T, D, kPartsTile>(name, p, batch, st);
}

template <typename T, int D>
int launch_kv_attention(const char* name, const h3b::KvAttnParams& p, bool tile, int64_t batch, cudaStream_t st) {
  if (tile) return launch_kv_tile<T, D>(name, p, batch, st);
  return p.selected ? launch_kv_split<T, D, true>(name, p, batch, st) : launch_kv_split<T, D, false>(name, p, batch, st);
}

}  // namespace

extern "C" size_t h3b_attention_kv_i8_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens,
                                                     int64_t head_dim, int64_t table_width, int64_t page_size,
                                                     int64_t n_selected) {
  using namespace h3b_host;
  if (batch <= 0 || batch > kKvMostBatch || kv_heads <= 0 || q_heads < kv_heads || q_heads > kKvMostHeads || tokens <= 0 ||
      tokens > kKvMostKeys / q_heads || page_size < 16 || page_size > 128 || table_width <= 0 ||
      table_width > kKvMostKeys / page_size || n_selected > kKvMostSelected || (head_dim != 64 && head_dim != 128))
    return 16;   // the call refuses these
  const KvPlan k = kv_plan(batch, q_heads, kv_heads, tokens, head_dim, table_width, page_size, n_selected);
  return k.part_bytes > SIZE_MAX - 16 - k.plan_bytes ? SIZE_MAX : 16 + k.plan_bytes + k.part_bytes;
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
  if (q_heads <= 0 || q_heads % cache->kv_heads || q_heads > h3b_host::kKvMostHeads)
    return h3b_host::set_error(H3B_EINVAL, "%s: q_heads must be a positive multiple of kv_heads", name);
  if (tokens < 0 || tokens > h3b_host::kKvMostKeys / q_heads)
    return h3b_host::set_error(H3B_EINVAL, "%s: bad token count", name);
  if (window < 0 || (window > 0 && !causal)) return h3b_host::set_error(H3B_EINVAL, "%s: a window needs causal", name);
  if (selected && (n_selected <= 0 || n_selected > h3b_host::kKvMostSelected || !causal || window > 0))
    return h3b_host::set_error(H3B_EINVAL, "%s: selected pages need causal, no window and 1 to 2^20 pages", name);
  if (tokens == 0) return H3B_OK;
  const KvPlan k = kv_plan(batch, q_heads, cache->kv_heads, tokens, cache->head_dim, table_width, cache->page_size,
                           selected ? n_selected : 0);
  if (k.part_bytes > SIZE_MAX / 2 || k.slots > INT32_MAX) return h3b_host::set_error(H3B_EUNSUPPORTED, "%s: problem too large", name);
  const size_t need = k.plan_bytes + k.part_bytes;
  if (need && (!workspace || !h3b_host::aligned16(workspace) || workspace_bytes < 16 + need))
    return h3b_host::set_error(H3B_EINVAL, "%s: workspace missing, misaligned or too small", name);
  p.q = q;
  p.out = out;
  p.lse = lse;
  p.lengths = lengths;
  p.counts = counts;
  p.selected = selected;
  p.vec_q = h3b_host::aligned16(q);
  p.vec_out = h3b_host::aligned16(out);
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = out_strides[i];
    p.vec_q = p.vec_q && q_strides[i] % 8 == 0;
    p.vec_out = p.vec_out && out_strides[i] % 8 == 0;
  }
  p.q_heads = (int)q_heads;
  p.group = (int)(q_heads / cache->kv_heads);
  p.tokens = (int)tokens;
  p.n_selected = (int)n_selected;
  p.window = (int)(window > (int64_t(1) << 30) ? int64_t(1) << 30 : window);
  p.causal = causal != 0;
  p.scale_log2 = scale * h3b::kLog2e;
  p.row_tiles = (int)k.row_tiles;
  p.slots = (int)k.slots;
  p.share = (int)k.share;
  p.fit = (int)k.fit;
  p.join_warps = (int)k.join_warps;
  p.chunk = (int)k.chunk;
  p.cluster = (int)k.cluster;
  p.plan = k.plan_bytes ? static_cast<int2*>(workspace) : nullptr;
  p.part = k.part_bytes ? reinterpret_cast<float*>(static_cast<char*>(workspace) + k.plan_bytes) : nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = cache->head_dim == 128;
  if (dtype == H3B_TYPE_F16)
    return wide ? launch_kv_attention<__half, 128>(name, p, k.tile, batch, st) : launch_kv_attention<__half, 64>(name, p, k.tile, batch, st);
  return wide ? launch_kv_attention<__nv_bfloat16, 128>(name, p, k.tile, batch, st)
              : launch_kv_attention<__nv_bfloat16, 64>(name, p, k.tile, batch, st);
}
