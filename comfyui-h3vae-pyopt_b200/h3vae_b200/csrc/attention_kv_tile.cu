// Attention over the paged INT8 cache for many query rows, on the tcgen05
// tensor cores (the mathematics: attention_kv.cuh).
//
// One CTA = one (sequence, kv head) and two tiles of 128 rows; a row is a
// (query token, head of the group), so grouped heads share the keys a CTA
// reads.  12 warps:
//   warps 0..2   codes to operands: half tiles of 64 keys of K or V are read from
//                their pages 16 codes at a time, converted to fp16 (exactly: codes are
//                whole numbers) and written to shared memory in the 128-byte
//                swizzle the tensor core reads; tiles go through one ring in the
//                order they are used: K0 K1 V0 K2 V1 K3 V2 ...  The block's scales,
//                per 16 keys, go with K.
//   warp 3       TMEM owner and MMA issuer: S(t) = Q(t) K^T, O(t) += W(t) V(t).
//   warps 4..11  softmax, four per row tile, one row per thread (its TMEM lane):
//                a row's 128 products come out of TMEM at once, which frees S for
//                the next block; x = S * (ks * scale * log2 e) + log2 vs against
//                the running maximum gives weights in fp16 for the second product
//                and, times 1 / vs in fp32, the denominator.
// The reference maximum moves only when a block's exceeds it by more than 8
// (weights stay <= 256); O is rescaled in TMEM then.  The two row tiles take
// turns on the SFU, so that one tile's exponentials overlap the other's products.
// Blocks that no row of the CTA sees are not visited, and only blocks on an edge
// of a row's range test each key.
#include "attention_kv.cuh"

namespace h3b {

constexpr int kKtRows = 128;                 // rows per tile
constexpr int kKtKeys = 128;                 // keys per block
constexpr int kKtConvWarps = 3;
constexpr int kKtThreads = 32 * (kKtConvWarps + 1 + 8);   // three warps a scheduler: 168 registers a thread
constexpr int kKtUnit = 64;                  // keys a converter warp takes at a time
constexpr int kKtMeta = 8;                   // blocks whose scales are kept

template <int D>
struct KvTile {
  static constexpr int kSlots = D == 64 ? 6 : 3;
  static constexpr uint32_t kTile = 128 * D * 2;           // Q, K or V tile in fp16
  static constexpr uint32_t kP = kKtRows * kKtKeys * 2;
  static constexpr uint32_t kSmem = 2 * kTile + kSlots * kTile + 2 * kP + kKtMeta * 8 * 16 + 256 + 1024;
};

// A row's 128 products out of TMEM.  One statement with its wait, so that no use
// of a register moves above it.
__device__ __forceinline__ void tmem_ld128_wait(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
      "}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
        "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
        "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr)
      : "memory");
}

// Scales of 16 keys.  Not volatile, so that the loads move ahead of the stores
// of earlier weights; the address carries the order after the barrier wait.
__device__ __forceinline__ float4 meta_load(uint32_t addr) {
  float4 f;
  asm("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(addr));
  return f;
}

// The rare parts of the softmax loop, out of line: inside it they cost the loop
// registers and its schedule (a causal prompt of 8101 tokens, dim 128: 1.90 ms
// with both inline).

// Sets a row's products outside lo <= k < hi to -inf, in TMEM.
__device__ __noinline__ void mask_products(uint32_t taddr, int lo, int hi) {
#pragma unroll 1
  for (int c = 0; c < kKtKeys; c += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (c + k < lo || c + k >= hi) r[k] = 0xff800000u;
    tmem_st32(taddr + c, r);
  }
  tmem_st_wait();
}

// Multiplies a row of O by alpha, in TMEM.
__device__ __noinline__ void rescale_row(uint32_t taddr, int dims, float alpha) {
#pragma unroll 1
  for (int c = 0; c < dims; c += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int d = 0; d < 32; ++d) r[d] = __float_as_uint(__fmul_rn(__uint_as_float(r[d]), alpha));
    tmem_st32(taddr + c, r);
  }
  tmem_st_wait();
}

// The factor of 16 keys' products: positive, so that a masked product stays
// -inf (a scale of zero or a tiny query row would make it a NaN).
__device__ __forceinline__ float score_scale(float x_scale, float back) { return fmaxf(x_scale * back, 1e-37f); }

// The largest score of a row's 128 products, in base 2 with log2 vs; scales are
// positive, so the largest product of 16 keys is found first.
__device__ __forceinline__ float row_max(const uint32_t (&x)[128], uint32_t meta, float back) {
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const uint32_t* v = x + 16 * u;
    auto at = [v](int k) { return __uint_as_float(v[k]); };
    float a = fmax3(at(0), at(1), at(2)), c = fmax3(at(3), at(4), at(5));
    a = fmax3(a, at(6), at(7));
    c = fmax3(c, at(8), at(9));
    a = fmax3(a, at(10), at(11));
    c = fmax3(c, at(12), at(13));
    a = fmax3(a, at(14), at(15));
    const float4 f = meta_load(meta + 16 * u);
    top = fmaxf(top, __fmaf_rn(fmaxf(a, c), score_scale(f.x, back), f.y));
  }
  return top;
}

// Weights of the products, rounded to fp16 into the row of P; returns the sum of
// weight / vs.
template <int D>
__device__ __forceinline__ float weights(const uint32_t (&x)[128], uint32_t meta, float back, float ref, uint32_t prow,
                                         int row) {
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float4 f = meta_load(meta + 16 * u);
    const float sc = score_scale(f.x, back), sh = f.y - ref;
    uint64_t acc = 0;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * u + 8 * v + 2 * e;
        float x0, x1;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), f2_pack(sc, sc), f2_pack(sh, sh)),
                  x0, x1);
        const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
        acc = f2_add(acc, f2_pack(w0, w1));
        w[e] = h2_bits(__floats2half2_rn(w0, w1));
      }
      const int q = 2 * u + v;
      st_shared_v4(prow + (q >> 3) * (KvTile<D>::kP / 2) + (((q & 7) ^ (row & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
    }
    float a0, a1;
    f2_unpack(acc, a0, a1);
    sum = __fmaf_rn(a0 + a1, f.z, sum);
  }
  return sum;
}

template <typename T, int D>
__global__ void __launch_bounds__(kKtThreads, 1) attention_kv_tile_kernel(const KvAttnParams p) {
  using L = KvTile<D>;
  constexpr int NS = L::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* ring = sq + 2 * L::kTile;
  uint8_t* sp = ring + NS * L::kTile;
  float4* s_meta = reinterpret_cast<float4*>(sp + 2 * L::kP);      // [block % 8][16 keys]: x scale, log2 vs, 1/vs
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_meta + kKtMeta * 8);
  uint64_t* q_full = bars;
  uint64_t* slot_full = bars + 1;
  uint64_t* slot_empty = slot_full + NS;
  uint64_t* s_full = slot_empty + NS;      // [tile]
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* meta_full = o_full + 2;        // [kKtMeta]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(meta_full + kKtMeta);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.slots;
  const int rt = p.row_tiles - 1 - blockIdx.x / p.slots;      // the longest causal ranges first
  const int g_rows = p.group * p.tokens;
  const int row0 = rt * 2 * kKtRows;
  const int tiles = g_rows - row0 > kKtRows ? 2 : 1;

  // the blocks of keys this CTA visits
  const int len = kv_length(p.c, p.lengths, b), n_tok = kv_count(p.counts, p.tokens, b);
  int blk0, n_blocks;
  {
    const int t0 = max(row0 / p.group, n_tok - len), t1 = min((min(row0 + 2 * kKtRows, g_rows) - 1) / p.group, n_tok - 1);
    int first = 0, last = 0, other;
    if (t0 <= t1) {
      kv_range(p, len, n_tok, t0, first, other);
      kv_range(p, len, n_tok, t1, other, last);
    }
    blk0 = first / kKtKeys;
    n_blocks = last > first ? (last + kKtKeys - 1) / kKtKeys - blk0 : 0;
    const int per = (n_blocks + p.slots - 1) / p.slots;
    const int from = min(split * per, n_blocks);
    n_blocks = min(per, n_blocks - from);
    blk0 += from;
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 32 * 4 * tiles);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&slot_full[s], kKtKeys / kKtUnit);
      mbar_init(&slot_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_empty[t], 128);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < kKtMeta; ++s) mbar_init(&meta_full[s], kKtKeys / kKtUnit);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 3) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // ring position of K_j and V_j: K0 K1 V0 K2 V1 ...
  auto seq_k = [](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto seq_v = [n_blocks](int j) { return min(2 * j + 2, 2 * n_blocks - 1); };

  if (warp < kKtConvWarps) {
    // ----------------------------- codes to fp16 -----------------------------
    // The warps take half tiles (64 keys) in turn: unit g is half g & 1 of the
    // tile with ring position g >> 1.  A lane's vectors of 16 codes lie 32 lanes
    // apart, so that vector i's keys are all in 16-key group i * 4 / kVecs of the
    // unit, whose place lane i * 4 / kVecs looked up.
    constexpr int kPerKey = D / 16;                        // vectors of a key
    constexpr int kVecs = kKtUnit * kPerKey / 32;
    constexpr int kKeyStep = 32 / kPerKey;
    const int key_in = lane / kPerKey, col = lane % kPerKey;
    const int units = 4 * n_blocks;
    auto tile_of = [n_blocks](int seq, bool& is_v) {   // the block whose K or V has ring position seq
      const bool end = seq == 2 * n_blocks - 1;
      is_v = end || (seq > 0 && !(seq & 1));
      return end ? n_blocks - 1 : is_v ? seq / 2 - 1 : (seq + 1) / 2;
    };
    // loads run ahead of their use: page numbers two of the warp's units, codes and scales one
    auto fetch_page = [&](int g) {       // lanes 0..3: the page of their 16 keys
      int page = -1;
      if (lane < 4 && g < units) {
        bool is_v;
        const int key = (blk0 + tile_of(g >> 1, is_v)) * kKtKeys + (g & 1) * kKtUnit + 16 * lane;
        if (key < len) page = kv_page(p.c, b, key >> p.c.page_shift);
      }
      return page;
    };
    uint4 codes[kVecs];
    float ks = 0.0f, vs = 0.0f;
    bool have = false;                   // lanes 0..3: their keys have a page
    auto fetch = [&](int g, int page) {  // zeros where no page holds the key
      bool is_v;
      const int key = (blk0 + tile_of(g >> 1, is_v)) * kKtKeys + (g & 1) * kKtUnit + 16 * lane;
      const int64_t ph = static_cast<int64_t>(page) * p.c.heads + hk;
      have = page >= 0;
      int64_t off = -1;
      if (have) {
        off = (ph * p.c.page + (key & (p.c.page - 1))) * D;
        if (!is_v) {
          ks = p.c.scale[0][ph];
          vs = p.c.scale[1][ph];
        }
      }
      const int8_t* base = p.c.code[is_v] + key_in * D + 16 * col;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int64_t at = __shfl_sync(0xffffffffu, off, w);
#pragma unroll
        for (int i = 0; i < kVecs / 4; ++i)
          codes[w * (kVecs / 4) + i] =
              at >= 0 ? __ldg(reinterpret_cast<const uint4*>(base + at + i * kKeyStep * D)) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    int page = fetch_page(warp);
    if (warp < units) fetch(warp, page);
    page = fetch_page(warp + kKtConvWarps);
    for (int g = warp; g < units; g += kKtConvWarps) {
      bool is_v;
      const int seq = g >> 1, j = tile_of(seq, is_v), s = seq % NS;
      // A page with a NaN scale gets NaN keys instead, so that it reaches the rows that see it and no other.
      unsigned poisoned = 0;
      if (!is_v) {
        poisoned = __ballot_sync(0xffffffffu, have && (isnan(ks) || isnan(vs)));
        if (lane < 4) {
          float4 f = make_float4(1.0f, -INFINITY, 0.0f, 0.0f);       // no page: weight 0
          if (have) {   // a scale of zero: a page never written holds zeros
            const float v = fmaxf(vs, kKvMinScale);
            f = make_float4(fmaxf(ks, kKvMinScale) * fabsf(p.scale_log2), log2f(v), __frcp_rn(v), 0.0f);
          }
          s_meta[(j % kKtMeta) * 8 + (g & 1) * 4 + lane] = f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&meta_full[j % kKtMeta]);
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&slot_empty[s], ((seq / NS) & 1) ^ 1, abort_flag))) break;
      // 16-byte chunks 2 (col % 4) and + 1 of the key's 128-byte row; the second half of the head's dims
      // writes them in the other order, which keeps the eight lanes of a store in different banks
      const int swap = col >> 2;
      const uint32_t dst = smem_u32(ring + s * L::kTile) + swap * (128 * 128) + ((g & 1) * kKtUnit + key_in) * 128;
      uint32_t at0[kVecs > 8 ? 2 : 1], at1[kVecs > 8 ? 2 : 1];   // the swizzle repeats every 8 keys
#pragma unroll
      for (int i = 0; i < (kVecs > 8 ? 2 : 1); ++i) {
        const int r = (key_in + i * kKeyStep) & 7;
        at0[i] = dst + (((2 * (col & 3) + swap) ^ r) << 4);
        at1[i] = dst + (((2 * (col & 3) + 1 - swap) ^ r) << 4);
      }
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const uint32_t w[4] = {codes[i].x ^ 0x80808080u, codes[i].y ^ 0x80808080u, codes[i].z ^ 0x80808080u,
                               codes[i].w ^ 0x80808080u};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[2 * e] = codes_to_h2(w[e], 0x4140);
          h[2 * e + 1] = codes_to_h2(w[e], 0x4342);
        }
        const int v = kVecs > 8 ? i & 1 : 0;
        st_shared_v4(at0[v] + i * kKeyStep * 128,
                     swap ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]));
        st_shared_v4(at1[v] + i * kKeyStep * 128,
                     swap ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]));
      }
      if (poisoned) {
        const uint4 nan = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u);
#pragma unroll 1
        for (int i = 0; i < kVecs; ++i)
          if (poisoned >> (i * 4 / kVecs) & 1u) {
            const int r = (key_in + i * kKeyStep) & 7;
            st_shared_v4(dst + i * kKeyStep * 128 + (((2 * (col & 3)) ^ r) << 4), nan);
            st_shared_v4(dst + i * kKeyStep * 128 + (((2 * (col & 3) + 1) ^ r) << 4), nan);
          }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&slot_full[s]);
      if (g + kKtConvWarps < units) fetch(g + kKtConvWarps, page);
      page = fetch_page(g + 2 * kKtConvWarps);
    }
  } else if (warp == 3) {
    // ------------------------------- MMA issuer -------------------------------
    if (elect_one_sync()) {
      constexpr uint32_t idesc_qk = make_idesc_f16(kKtRows, kKtKeys);
      constexpr uint32_t idesc_pv = make_idesc_f16(kKtRows, D) | (1u << 16);   // V is MN-major
      bool ok = n_blocks == 0 || mbar_poll(q_full, 0, abort_flag);
      auto issue_s = [&](int j, int t) -> bool {
        const int seq = seq_k(j), s = seq % NS;
        if (!mbar_poll(&slot_full[s], (seq / NS) & 1, abort_flag)) return false;
        if (!mbar_poll(&s_empty[t], (j & 1) ^ 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t qb = smem_u32(sq + t * L::kTile), kb = smem_u32(ring + s * L::kTile);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_f16(tmem + t * 256, make_sw128_desc(qb + (k >> 2) * 16384) + 2 * (k & 3),
                  make_sw128_desc(kb + (k >> 2) * 16384) + 2 * (k & 3), idesc_qk, k > 0 ? 1u : 0u);
        tc_commit(&s_full[t]);
        if (t == tiles - 1) tc_commit(&slot_empty[s]);
        return true;
      };
      for (int t = 0; t < tiles && ok && n_blocks > 0; ++t) ok = issue_s(0, t);
      for (int j = 0; j < n_blocks && ok; ++j) {
        for (int t = 0; t < tiles && ok && j + 1 < n_blocks; ++t) ok = issue_s(j + 1, t);
        const int seq = seq_v(j), s = seq % NS;
        for (int t = 0; t < tiles && ok; ++t) {
          if (t == 0 && !mbar_poll(&slot_full[s], (seq / NS) & 1, abort_flag)) { ok = false; break; }
          if (!mbar_poll(&p_full[t], j & 1, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t pb = smem_u32(sp + t * L::kP), vb = smem_u32(ring + s * L::kTile);
#pragma unroll
          for (int k = 0; k < kKtKeys / 16; ++k) {
            // 64 dims of 16 keys are one swizzle atom column; the next 64 dims lie 16 KB further
            uint64_t vd = make_sw128_desc(vb + k * 16 * 128);
            vd = (vd & ~(uint64_t(0x3FFFu) << 16)) | (uint64_t(16384 >> 4) << 16);
            mma_f16(tmem + t * 256 + 128, make_sw128_desc(pb + (k >> 2) * (L::kP / 2)) + 2 * (k & 3), vd, idesc_pv,
                    (j > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit(&o_full[t]);
        }
        if (ok) tc_commit(&slot_empty[s]);
      }
    }
  } else {
    // ------------------------------ softmax warps ------------------------------
    const int tile = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const int full = row0 + tile * kKtRows + row;            // row of this (sequence, kv head)
    if (tile < tiles) {
      const uint32_t t_s = tmem + tile * 256 + (static_cast<uint32_t>(quad * 32) << 16), t_o = t_s + 128;
      const bool real = full < g_rows;
      const int t = real ? full / p.group : 0, h = hk * p.group + (real ? full % p.group : 0);
      int first = 0, last = 0x7fffffff;                      // rows past the end never force masking
      if (real) kv_range(p, len, n_tok, t, first, last);
      const int first_max = __reduce_max_sync(0xffffffffu, first), last_min = __reduce_min_sync(0xffffffffu, last);
      // Q row to shared memory
      float back;
      {
        const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
        float top = 0.0f;
        if (sizeof(T) == 2 && real) {
#pragma unroll 1
          for (int i = 0; i < D / 8; ++i) {
            float x[8];
            load8(q + 8 * i, p.vec_q, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
          }
        }
        // a negative scale turns the row, so that larger products are larger scores
        const float f = row_scaling(T(), top, back) * (p.scale_log2 < 0.0f ? -1.0f : 1.0f);
        const uint32_t dst = smem_u32(sq + tile * L::kTile) + row * 128;
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) {
          float x[8] = {};
          if (real) load8(q + 8 * i, p.vec_q, x);
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = h2_bits(__floats2half2_rn(x[2 * e] * f, x[2 * e + 1] * f));
          st_shared_v4(dst + (i >> 3) * 16384 + (((i & 7) ^ (row & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      const uint32_t prow = smem_u32(sp + tile * L::kP + row * 128);
      const uint32_t bar_s_full = smem_u32(&s_full[tile]), bar_s_empty = smem_u32(&s_empty[tile]);
      const uint32_t bar_p_full = smem_u32(&p_full[tile]), bar_o_full = smem_u32(&o_full[tile]);
      const bool turns = tiles == 2;
      if (turns && tile == 1 && n_blocks > 0) asm volatile("bar.arrive 1, 256;" ::: "memory");
      for (int j = 0; j < n_blocks; ++j) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(smem_u32(&meta_full[j % kKtMeta]), (j / kKtMeta) & 1, abort_flag));
        ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(bar_s_full, j & 1, abort_flag));
        uint32_t meta = smem_u32(s_meta + (j % kKtMeta) * 8);
        asm volatile("" : "+r"(meta));     // its loads stay below the wait
        // (after a wait that gave up the values mean nothing, but every warp keeps in step)
        tc_fence_after();
        const int key0 = (blk0 + j) * kKtKeys;
        if (key0 < first_max || key0 + kKtKeys > last_min) mask_products(t_s, first - key0, last - key0);
        uint32_t x[128];
        tmem_ld128_wait(t_s, x);
        tc_fence_before();
        mbar_arrive_u32(bar_s_empty);
        const float top = row_max(x, meta, back);
        const bool move = top > m + 8.0f;
        const float m_new = move ? top : m;
        const float alpha = move ? ex2_approx(m - m_new) : 1.0f;
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        m = m_new;
        if (j > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(bar_o_full, (j - 1) & 1, abort_flag));
        if (turns) asm volatile("bar.sync %0, 256;" ::"r"(tile == 0 ? 1 : 2) : "memory");
        const float sum = weights<D>(x, meta, back, ref, prow, row);
        if (turns && (tile == 0 || j + 1 < n_blocks))
          asm volatile("bar.arrive %0, 256;" ::"r"(tile == 0 ? 2 : 1) : "memory");
        l = __fmaf_rn(l, alpha, sum);
        if (ok && j > 0) {
          tc_fence_after();
          if (__any_sync(0xffffffffu, move)) rescale_row(t_o, D, alpha);
        }
        if (ok) {
          tc_fence_before();
          fence_proxy_async_smem();
          mbar_arrive_u32(bar_p_full);
        }
      }
      if (n_blocks > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(bar_o_full, (n_blocks - 1) & 1, abort_flag));
      const bool have = ok && n_blocks > 0;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (have) tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (have) {
          tmem_ld32(t_o + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int d = 0; d < 32; ++d) r[d] = 0u;
        }
        if (!real) continue;
        if (p.part) {
          float* dst = p.part + ((((static_cast<int64_t>(split) * p.c.batch + b) * p.c.heads + hk) * g_rows) + full) * (D + 4);
#pragma unroll
          for (int d = 0; d < 32; d += 4)
            *reinterpret_cast<uint4*>(dst + c * 32 + d) = make_uint4(r[d], r[d + 1], r[d + 2], r[d + 3]);
          if (c == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m, l);
        } else {
          T* dst = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] + c * 32;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            __align__(16) T y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) from_f32(__uint_as_float(r[8 * v + e]) * inv, y[e]);
            if (p.vec_out) {
              *reinterpret_cast<uint4*>(dst + 8 * v) = *reinterpret_cast<const uint4*>(y);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[8 * v + e] = y[e];
            }
          }
        }
      }
      if (real && p.lse && !p.part)
        p.lse[(static_cast<int64_t>(b) * p.q_heads + h) * p.tokens + t] =
            l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) + log2f(l)) * kLn2;
    }
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) tmem_dealloc(tmem, 512);
}

}  // namespace h3b
