// Attention over the paged INT8 cache for many query rows, on the tcgen05
// tensor cores (the mathematics: attention_kv.cuh).
//
// One CTA = one (sequence, kv head) and two tiles of 128 rows; a row is a
// (query token, head of the group), so grouped heads share the keys a CTA
// reads.  13 warps:
//   warps 0..3   codes to operands: a tile of 128 keys of K or V is read from its
//                pages 16 codes at a time, converted to fp16 (exactly: codes are
//                whole numbers) and written to shared memory in the 128-byte
//                swizzle the tensor core reads; tiles go through one ring in the
//                order they are used: K0 K1 V0 K2 V1 K3 V2 ...  The first eight
//                threads also leave the block's scales, per 16 keys.
//   warps 4..11  softmax, four per row tile, one row per thread (its TMEM lane):
//                a row's 128 products come out of TMEM at once, which frees S for
//                the next block; x = S * (ks * scale * log2 e) + log2 vs against
//                the running maximum gives weights in fp16 for the second product
//                and, times 1 / vs in fp32, the denominator.
//   warp 12      TMEM owner and MMA issuer: S(t) = Q(t) K^T, O(t) += W(t) V(t).
// The reference maximum moves only when a block's exceeds it by more than 8
// (weights stay <= 256); O is rescaled in TMEM then.  The two row tiles take
// turns on the SFU, so that one tile's exponentials overlap the other's products.
// Blocks that no row of the CTA sees are not visited, and only blocks on an edge
// of a row's range test each key.
#include "attention_kv.cuh"

namespace h3b {

constexpr int kKtRows = 128;                 // rows per tile
constexpr int kKtKeys = 128;                 // keys per block
constexpr int kKtConvWarps = 4;
constexpr int kKtThreads = 32 * (kKtConvWarps + 8 + 4);   // whole warpgroups, for their register shares
constexpr int kKtMeta = 8;                   // blocks whose scales are kept

// Registers a thread of each warpgroup: converters, softmax (twice), MMA; they
// add up to the launch's 4 x 128.
constexpr int kKtConvRegs = 80, kKtSoftRegs = 184, kKtMmaRegs = 64;
static_assert(kKtConvRegs + 2 * kKtSoftRegs + kKtMmaRegs == 512, "register shares");

template <int D>
struct KvTile {
  static constexpr int kSlots = D == 64 ? 6 : 3;
  static constexpr uint32_t kTile = 128 * D * 2;           // Q, K or V tile in fp16
  static constexpr uint32_t kP = kKtRows * kKtKeys * 2;
  static constexpr uint32_t kSmem = 2 * kTile + kSlots * kTile + 2 * kP + kKtMeta * 8 * 16 + 256 + 1024;
};

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
      mbar_init(&slot_full[s], 32 * kKtConvWarps);
      mbar_init(&slot_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_empty[t], 128);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < kKtMeta; ++s) mbar_init(&meta_full[s], 8);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kKtConvRegs));
    // ----------------------------- codes to fp16 -----------------------------
    constexpr int kPerKey = D / 16;                       // 16-code vectors of a key
    constexpr int kVecs = kKtKeys * kPerKey / (32 * kKtConvWarps);
    constexpr int kKeyStep = 32 * kKtConvWarps / kPerKey;
    const int tid = threadIdx.x, key0 = tid / kPerKey, col = tid % kPerKey;
    uint4 codes[kVecs];
    int pages[kVecs];
    auto tile_of = [n_blocks](int seq, bool& is_v) {   // the block whose K or V has ring position seq
      const bool end = seq == 2 * n_blocks - 1;
      is_v = end || (seq > 0 && !(seq & 1));
      return end ? n_blocks - 1 : is_v ? seq / 2 - 1 : (seq + 1) / 2;
    };
    auto page_of = [&](int key) { return key < len ? kv_page(p.c, b, key >> p.c.page_shift) : -1; };
    // loads run ahead of their use: page numbers two tiles, codes one
    auto fetch_pages = [&](int seq) {
      bool is_v;
      const int first = (blk0 + tile_of(seq, is_v)) * kKtKeys + key0;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) pages[i] = page_of(first + i * kKeyStep);
    };
    auto fetch_codes = [&](int seq) {   // zeros where no page holds the key
      bool is_v;
      const int first = (blk0 + tile_of(seq, is_v)) * kKtKeys + key0;
      const int8_t* base = p.c.code[is_v] + 16 * col;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int in = (first + i * kKeyStep) & (p.c.page - 1);
        codes[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pages[i] >= 0)
          codes[i] = __ldg(reinterpret_cast<const uint4*>(
              base + ((static_cast<int64_t>(pages[i]) * p.c.heads + hk) * p.c.page + in) * D));
      }
    };
    // thread tid < 8 keeps the scales of keys 16 tid .. of the next block, and the page of the one after
    float next_ks = 0.0f, next_vs = 0.0f;
    int next_page = -1, page_after = -1;
    auto fetch_scales = [&](int j) {    // of block j, whose page is page_after
      next_page = page_after;
      if (next_page >= 0) {
        const int64_t ph = static_cast<int64_t>(next_page) * p.c.heads + hk;
        next_ks = p.c.scale[0][ph];
        next_vs = p.c.scale[1][ph];
      }
      page_after = page_of((blk0 + j + 1) * kKtKeys + 16 * tid);
    };
    const int total = 2 * n_blocks;
    if (total > 0) {
      fetch_pages(0);
      fetch_codes(0);
      fetch_pages(1);
      if (tid < 8) {
        page_after = page_of(blk0 * kKtKeys + 16 * tid);
        fetch_scales(0);
      }
    }
    for (int seq = 0; seq < total; ++seq) {
      bool is_v;
      const int j = tile_of(seq, is_v);
      if (!is_v && tid < 8) {
        float4 f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
        if (next_page >= 0) {
          const float vs = next_vs < kKvMinScale ? kKvMinScale : next_vs;
          f = make_float4(next_ks * fabsf(p.scale_log2), log2f(vs), __frcp_rn(vs), 0.0f);
        }
        s_meta[(j % kKtMeta) * 8 + tid] = f;
        mbar_arrive(&meta_full[j % kKtMeta]);
        fetch_scales(j + 1);
      }
      const int s = seq % NS;
      if (!mbar_wait(&slot_empty[s], ((seq / NS) & 1) ^ 1, abort_flag)) break;
      const uint32_t dst = smem_u32(ring + s * L::kTile) + (col >> 2) * (128 * 128);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int key = key0 + i * kKeyStep;
        const uint32_t w[4] = {codes[i].x ^ 0x80808080u, codes[i].y ^ 0x80808080u, codes[i].z ^ 0x80808080u,
                               codes[i].w ^ 0x80808080u};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[2 * e] = codes_to_h2(w[e], 0x4140);
          h[2 * e + 1] = codes_to_h2(w[e], 0x4342);
        }
        // 16-byte chunks 2 (col % 4) and + 1 of the key's 128-byte row; the second half of the head's
        // dims writes them in the other order, which keeps the eight lanes of a store in different banks
        const int c0 = 2 * (col & 3), swap = col >> 2;
        st_shared_v4(dst + key * 128 + (((c0 + swap) ^ (key & 7)) << 4),
                     swap ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]));
        st_shared_v4(dst + key * 128 + (((c0 + 1 - swap) ^ (key & 7)) << 4),
                     swap ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]));
      }
      fence_proxy_async_smem();
      mbar_arrive(&slot_full[s]);
      if (seq + 1 < total) fetch_codes(seq + 1);
      if (seq + 2 < total) fetch_pages(seq + 2);
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kKtMmaRegs));
    // ------------------------------- MMA issuer -------------------------------
    if (warp == 12 && elect_one_sync()) {
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kKtSoftRegs));
    // ------------------------------ softmax warps ------------------------------
    const int tile = (warp - kKtConvWarps) >> 2, quad = warp & 3, row = quad * 32 + lane;
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
        const float4* meta = s_meta + (j % kKtMeta) * 8;
        uint32_t x[128];
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[32 * c]));
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 128; ++k) asm volatile("" : "+r"(x[k]));   // no use moves above the wait
          tc_fence_before();
          mbar_arrive_u32(bar_s_empty);
        } else {
#pragma unroll
          for (int k = 0; k < 128; ++k) x[k] = 0xff800000u;
        }
        const int key0 = (blk0 + j) * kKtKeys;
        const bool edge = key0 < first_max || key0 + kKtKeys > last_min;
        if (edge) {
          const int lo = first - key0, hi = last - key0;
#pragma unroll
          for (int k = 0; k < 128; ++k)
            if (k < lo || k >= hi) x[k] = 0xff800000u;
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float a = fmax3(__uint_as_float(x[16 * u]), __uint_as_float(x[16 * u + 1]), __uint_as_float(x[16 * u + 2]));
          float c = fmax3(__uint_as_float(x[16 * u + 3]), __uint_as_float(x[16 * u + 4]), __uint_as_float(x[16 * u + 5]));
#pragma unroll
          for (int k = 6; k < 14; k += 4) {
            a = fmax3(a, __uint_as_float(x[16 * u + k]), __uint_as_float(x[16 * u + k + 1]));
            c = fmax3(c, __uint_as_float(x[16 * u + k + 2]), __uint_as_float(x[16 * u + k + 3]));
          }
          a = fmax3(a, __uint_as_float(x[16 * u + 14]), __uint_as_float(x[16 * u + 15]));
          const float4 f = meta[u];
          top = fmaxf(top, __fmaf_rn(fmaxf(a, c), f.x * back, f.y));   // a NaN (no key, or a NaN page) is passed over
        }
        const bool move = top > m + 8.0f;
        const float m_new = move ? top : m;
        const float alpha = move ? ex2_approx(m - m_new) : 1.0f;
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        m = m_new;
        if (j > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(bar_o_full, (j - 1) & 1, abort_flag));
        if (turns) asm volatile("bar.sync %0, 256;" ::"r"(tile == 0 ? 1 : 2) : "memory");
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float4 f = meta[u];
          const float sc = f.x * back, sh = f.y - ref;
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
              if (edge) {   // -inf times a zero or NaN scale
                if (x[k] == 0xff800000u) x0 = -INFINITY;
                if (x[k + 1] == 0xff800000u) x1 = -INFINITY;
              }
              const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
              acc = f2_add(acc, f2_pack(w0, w1));
              w[e] = h2_bits(__floats2half2_rn(w0, w1));
            }
            const int q = 2 * u + v;
            if (ok)
              st_shared_v4(prow + (q >> 3) * (L::kP / 2) + (((q & 7) ^ (row & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
          }
          float a0, a1;
          f2_unpack(acc, a0, a1);
          sum = __fmaf_rn(a0 + a1, f.z, sum);
        }
        if (turns && (tile == 0 || j + 1 < n_blocks))
          asm volatile("bar.arrive %0, 256;" ::"r"(tile == 0 ? 2 : 1) : "memory");
        l = __fmaf_rn(l, alpha, sum);
        if (ok && j > 0) {
          tc_fence_after();
          if (__any_sync(0xffffffffu, move)) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t r[32];
              tmem_ld32(t_o + c * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int d = 0; d < 32; ++d) r[d] = __float_as_uint(__fmul_rn(__uint_as_float(r[d]), alpha));
              tmem_st32(t_o + c * 32, r);
            }
            tmem_st_wait();
          }
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
  if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace h3b
