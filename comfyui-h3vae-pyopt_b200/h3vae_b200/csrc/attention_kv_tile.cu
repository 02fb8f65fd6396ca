// Attention over the paged INT8 cache for many query rows, on the tcgen05
// tensor cores (the mathematics: attention_kv.cuh).
//
// One CTA = one (sequence, kv head) and two tiles of 128 rows; a row is a
// (query token, head of the group), so grouped heads share the keys a CTA
// reads.  12 warps:
//   warps 0..2   codes to operands: half tiles of 64 keys of K or V come from their
//                pages by bulk copies, are converted to fp16 (exactly: codes are
//                whole numbers) and written to shared memory in the 128-byte
//                swizzle the tensor core reads; tiles of 128 keys go through one
//                ring, K0 V0 K1 V1 ...  The block's scales, per 16 keys, go with K.
//   warp 3       TMEM owner and MMA issuer: S(t) = Q(t) K^T, O(t) += W(t) V, the two
//                row tiles in turn, so that one's products run under the other's
//                exponentials.
//   warps 4..11  softmax, four per row tile, one row per thread (its TMEM lane):
//                x = S * (ks * scale * log2 e) + log2 vs against the row's maximum
//                gives weights and, times 1 / vs in fp32, the denominator.  The
//                weights go back in fp16 over the products, and the second product
//                takes them from there: shared memory, which both products and the
//                converters also read and write, is what runs out first.
// The maximum is that of the first block a row sees keys in; a later block is taken
// against it as it is, and only when 16 of its weights sum to more than 2^14 (fp16
// holds 65504, and keeps its 11 bits up to there) is its own maximum looked for,
// the block redone and O rescaled in TMEM.  Blocks that no row of the CTA sees are
// not visited, and only blocks on an edge of a row's range mask keys.
//
// Weights have 11 bits and no low part (the second operand of the few-row kernel): rows see hundreds of
// keys here, their roundings average out, and the product would be taken twice.  Error against 64 bits,
// with the weights in fp32 beside it: 1024 tokens over 5120 keys, fp16, 2.02e-4 and 1.97e-4; the causal
// prompt, bf16, 1.639e-3 and 1.638e-3.
//
// What bounds it: not the tensor pipe (27 % active at dim 64) nor the SFU (16
// exponentials a clock: 55 %), but the chain of a row tile -- products, wait, weights
// (2000 to 2200 cycles a block), wait, products -- which two row tiles only half cover,
// and at dim 128 the converters beside it.  1024 tokens over 5120 keys, 2 x 16 heads of
// dim 64: 81 us = 530 TFLOP/s (bf16 84); a causal prompt of 8101 tokens, 2 x 32 heads over 8 of
// dim 128: 1.20 ms = 897 TFLOP/s (1.17 without pages of a low scale; 81 and 82 at dim 64).  A call over 256 keys takes 12 us at dim 64 and 17 at dim
// 128, every further 128 keys 2.0 and 2.3.  Measured and left, against 85 us and 1.27 ms:
// 64-key steps with two buffers of products (99 us, 1.45 ms: twice the waits of the
// issuing warp), 16 warps with an issuer per row tile and six converters (91 us, 1.52 ms:
// 128 registers a thread), all 128 products of a row in registers (109 us, 1.65 ms).
#include <type_traits>

#include "attention_kv.cuh"

namespace h3b {

constexpr int kKtRows = 128;                 // rows per tile
constexpr int kKtKeys = 128;                 // keys per block
constexpr int kKtConvWarps = 3;
constexpr int kKtThreads = 32 * (kKtConvWarps + 1 + 8);   // three warps a scheduler: 168 registers a thread
constexpr int kKtUnit = 64;                  // keys a converter warp takes at a time
constexpr int kKtBatch = 4;                  // blocks whose pages and scales are looked up together, a lane per 16 keys
constexpr int kKtMeta = 16;                  // blocks whose pages and scales are kept
constexpr float kKtMostWeight = 16384.0f;    // sum of 16 weights above which their maximum moves

constexpr int kPoisoned = 1 << 30;           // beside a page number (below 2^30): its scale is NaN

template <int D>
struct KvTile {
  static constexpr int kSlots = D == 64 ? 6 : 3;
  static constexpr uint32_t kTile = 128 * D * 2;           // Q, K or V tile in fp16
  static constexpr int kStages = D == 64 ? 3 : 2;          // units of codes a converter warp has in flight
  static constexpr uint32_t kUnit = kKtUnit * D;           // their bytes
  static constexpr uint32_t kSmem = (2 + kSlots) * kTile + kKtConvWarps * kStages * kUnit + kKtMeta * 8 * 16 + 384 + 1024;
};

// Some of a row's products out of TMEM.  One statement with its wait, so that no
// use of a register moves above it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t taddr, float (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
        "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
        "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
        "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
        "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
      : "r"(taddr)
      : "memory");
}

// A row's 64 words into TMEM.
__device__ __forceinline__ void tmem_st64(uint32_t taddr, const uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x64.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,"
      "%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,"
      "%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,%64"
      "};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(r[32]), "r"(r[33]), "r"(r[34]), "r"(r[35]), "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]),
        "r"(r[40]), "r"(r[41]), "r"(r[42]), "r"(r[43]), "r"(r[44]), "r"(r[45]), "r"(r[46]), "r"(r[47]),
        "r"(r[48]), "r"(r[49]), "r"(r[50]), "r"(r[51]), "r"(r[52]), "r"(r[53]), "r"(r[54]), "r"(r[55]),
        "r"(r[56]), "r"(r[57]), "r"(r[58]), "r"(r[59]), "r"(r[60]), "r"(r[61]), "r"(r[62]), "r"(r[63])
      : "memory");
}

// D[tmem] (+)= A[tmem] * B, fp16 x fp16 -> fp32; A: row in the lane, two elements a column.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
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
__device__ __noinline__ float row_max(uint32_t taddr, uint32_t meta, float back) {
  float top = -INFINITY;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    float x[64];
    tmem_ld_wait(taddr + 64 * h, x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float a = x[16 * u];
#pragma unroll
      for (int k = 1; k < 16; ++k) a = fmaxf(a, x[16 * u + k]);
      const float4 f = meta_load(meta + 64 * h + 16 * u);
      top = fmaxf(top, __fmaf_rn(a, score_scale(f.x, back), f.y));
    }
  }
  return top;
}

// A row's maximum with this block's, what O and l are scaled by for it (1: it has not moved), and l: scaled by the rest
// where 2^(m - m') is below fp32's range.
__device__ __noinline__ float4 look_row(uint32_t taddr, uint32_t meta, float back, float m, float l) {
  const float m_new = fmaxf(m, row_max(taddr, meta, back));
  const bool moved = m_new > m;
  const float fall = moved ? fmaxf(m - m_new, -126.0f) : 0.0f;
  return make_float4(m_new, ex2_approx(fall), moved ? rescale_sum(l, m - m_new - fall) : l, 0.0f);
}

// Adds to l the weights of keys of pages with a low scale, from their scores; a row without a maximum takes this block's.
__device__ __noinline__ float2 low_sums(uint32_t taddr, uint32_t meta, float back, float m, float l) {
  const float top = row_max(taddr, meta, back);
  if (m == -INFINITY) m = top;
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    float x[64];
    tmem_ld_wait(taddr + 64 * h, x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 f = meta_load(meta + 64 * h + 16 * u);
      if (f.z < 0.0f) {       // the same for the warp
        const float sc = score_scale(f.x, back);
#pragma unroll
        for (int k = 0; k < 16; ++k) l += ex2_approx(__fmaf_rn(x[16 * u + k], sc, -ref));
      }
    }
  }
  return make_float2(m, l);
}

// Weights of half kHalf of a row's products, rounded to fp16 pairs; returns the
// sum of weight / vs, and keeps in `most` a bound of the largest weight.
template <int kHalf>
__device__ __forceinline__ float weights(uint32_t taddr, uint32_t meta, float back, float ref, uint32_t (&w)[64],
                                         float& most) {
  float x[64];
  tmem_ld_wait(taddr + 64 * kHalf, x);
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float4 f = meta_load(meta + 64 * kHalf + 16 * u);
    const float sc = score_scale(f.x, back), sh = f.y - ref;
    uint64_t acc = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 16 * u + 2 * e;
      float x0, x1;
      f2_unpack(f2_fma(f2_pack(x[k], x[k + 1]), f2_pack(sc, sc), f2_pack(sh, sh)), x0, x1);
      const float w0 = ex2_approx(x0), w1 = ex2_approx(x1);
      acc = f2_add(acc, f2_pack(w0, w1));
      w[32 * kHalf + 8 * u + e] = h2_bits(__floats2half2_rn(w0, w1));
    }
    float a0, a1;
    f2_unpack(acc, a0, a1);
    most = fmaxf(most, a0 + a1);
    sum = __fmaf_rn(a0 + a1, f.z, sum);
  }
  return sum;
}

// A warp's 32 rows move between global and shared memory with a row over D / 8
// lanes (a row a lane touches 32 lines an instruction: 4000 cycles each way at dim
// 128), 16-byte chunks in the tile's swizzle.  The way out is out of line for the
// registers of the softmax loop, the way in is not (256 rows of fp16, dim 128, over 4096
// keys: 87 us, both inside 91; a bf16 prompt: 1160 us, both out of line 1230).
__device__ __forceinline__ uint32_t chunk_at(uint32_t rows_at, int row, int chunk) {
  return rows_at + row * 128 + (chunk >> 3) * 16384 + (((chunk & 7) ^ (row & 7)) << 4);
}

// Q: `mine` is this lane's row (null: zeros); returns what its products are scaled back by.
template <typename T, int D>
__device__ __forceinline__ float load_rows(const T* mine, bool vec, float sign, uint32_t rows_at) {
  constexpr int kLanes = D / 8, kStepRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, in_row = lane / kLanes, chunk = lane % kLanes;
  uint4 raw[D / 8];      // all in flight
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const T* q = reinterpret_cast<const T*>(
        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), i * kStepRows + in_row));
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (q && vec) {
      raw[i] = *reinterpret_cast<const uint4*>(q + 8 * chunk);
    } else if (q) {
      const unsigned short* bits = reinterpret_cast<const unsigned short*>(q + 8 * chunk);
      raw[i] = make_uint4(bits[0] | static_cast<uint32_t>(bits[1]) << 16, bits[2] | static_cast<uint32_t>(bits[3]) << 16,
                          bits[4] | static_cast<uint32_t>(bits[5]) << 16, bits[6] | static_cast<uint32_t>(bits[7]) << 16);
    }
  }
  float back = 1.0f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float x[8], top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned short half = static_cast<unsigned short>(words[e >> 1] >> (16 * (e & 1)));
      x[e] = to_f32(reinterpret_cast<const T&>(half));
      top = fmaxf(top, fabsf(x[e]));
    }
    float row_back, f;
    if (std::is_same<T, __half>::value) {
      f = sign * row_scaling(T(), top, row_back);
    } else {
#pragma unroll
      for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      f = sign * row_scaling(T(), top, row_back);
      row_back = __shfl_sync(0xffffffffu, row_back, (lane % kStepRows) * kLanes);
      if (lane / kStepRows == i) back = row_back;
    }
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = h2_bits(__floats2half2_rn(x[2 * e] * f, x[2 * e + 1] * f));
    st_shared_v4(chunk_at(rows_at, i * kStepRows + in_row, chunk), make_uint4(w[0], w[1], w[2], w[3]));
  }
  return back;
}

// 32 columns of a row's O out of TMEM, zeros where there is none.
__device__ __forceinline__ void load_o(uint32_t taddr, bool have, uint32_t (&r)[32]) {
  if (have) {
    tmem_ld32(taddr, r);
    tmem_ld_wait();
  } else {
#pragma unroll
    for (int d = 0; d < 32; ++d) r[d] = 0u;
  }
}

// O: to `out` times inv, or as it is to `part`, D * 2 bytes of a row at a time (null rows are not written).
template <typename T, int D>
__device__ __noinline__ void store_rows(uint32_t t_o, bool have, float inv, T* out, float* part, bool parts, uint32_t rows_at) {
  constexpr int kLanes = D / 8, kStepRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, in_row = lane / kLanes, chunk = lane % kLanes;
  const unsigned long long mine =
      parts ? reinterpret_cast<unsigned long long>(part) : reinterpret_cast<unsigned long long>(out);
#pragma unroll 1
  for (int round = 0; round < (parts ? 2 : 1); ++round) {
    uint32_t r[32];
    if (parts) {
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        load_o(t_o + round * (D / 2) + c * 32, have, r);
#pragma unroll
        for (int v = 0; v < 8; ++v)
          st_shared_v4(chunk_at(rows_at, lane, c * 8 + v), make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]));
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        load_o(t_o + c * 32, have, r);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          __align__(16) T y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) from_f32(__uint_as_float(r[8 * v + e]) * inv, y[e]);
          st_shared_v4(chunk_at(rows_at, lane, c * 4 + v), *reinterpret_cast<const uint4*>(y));
        }
      }
    }
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < D / 8; ++i) {
      const int row = i * kStepRows + in_row;
      const unsigned long long to = __shfl_sync(0xffffffffu, mine, row);
      const uint4 v = ld_shared_v4(chunk_at(rows_at, row, chunk));
      if (to) *reinterpret_cast<uint4*>(to + round * (D * 2) + chunk * 16) = v;
    }
    __syncwarp();
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kKtThreads, 1) attention_kv_tile_kernel(const KvAttnParams p) {
  using L = KvTile<D>;
  constexpr int NS = L::kSlots;
  constexpr uint32_t kWCol = D == 64 ? 192 : 0;     // the weights' columns of a row tile: O takes 128 .. 128 + D
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* ring = sq + 2 * L::kTile;
  uint8_t* staged = ring + NS * L::kTile;                          // [converter warp][stage]
  float4* s_meta = reinterpret_cast<float4*>(staged + kKtConvWarps * L::kStages * L::kUnit);      // [block % 16][16 keys]: x scale, log2 vs, 1/vs or log2 vs, page
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_meta + kKtMeta * 8);
  uint64_t* q_full = bars;
  uint64_t* slot_full = bars + 1;
  uint64_t* slot_empty = slot_full + NS;
  uint64_t* s_full = slot_empty + NS;      // [tile]
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* meta_full = o_full + 2;        // [batch % 4]
  uint64_t* staged_full = meta_full + kKtMeta / kKtBatch;                     // [converter warp][stage]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staged_full + kKtConvWarps * L::kStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((1 + 2 * NS + 6 + kKtMeta / kKtBatch + kKtConvWarps * L::kStages) * 8 + 8 + kKtMeta / kKtBatch * 4 <= 384, "barriers' room");
  uint32_t* s_low = tmem_slot + 2;         // [batch % 4]: whether keys are to be summed from their scores

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

  // The converters' first lookups run under the set-up below: the pages of the units that a warp copies first, and
  // pages and scales of the first two batches of blocks (see there).
  const int units = 4 * n_blocks;
  const int seg_keys = min(p.c.page, kKtUnit), segs = kKtUnit / seg_keys;
  int look_page = -1, ahead_page[L::kStages];
  float look_k = 0.0f, look_v = 0.0f;
  auto look_pages = [&](int m) {
    const int key = (blk0 + m * kKtBatch) * kKtKeys + 16 * lane;
    look_page = -1;
    if (16 * m < units && key < len) look_page = kv_page(p.c, b, key >> p.c.page_shift);
  };
  auto look_scales = [&]() {
    if (look_page >= 0) {
      const int64_t ph = static_cast<int64_t>(look_page) * p.c.heads + hk;
      look_k = p.c.scale[0][ph];
      look_v = p.c.scale[1][ph];
    }
  };
  if (warp < kKtConvWarps) {
#pragma unroll
    for (int st = 0; st < L::kStages; ++st) {
      const int g = warp + st * kKtConvWarps, key = (blk0 + (g >> 2)) * kKtKeys + (g & 1) * kKtUnit + lane * seg_keys;
      ahead_page[st] = lane < segs && g < units && key < len ? kv_page(p.c, b, key >> p.c.page_shift) : -1;
    }
    if (warp < 2) {
      look_pages(warp);
      look_scales();
    }
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 32 * 4 * tiles);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&slot_full[s], kKtKeys / kKtUnit);
      mbar_init(&slot_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < kKtMeta / kKtBatch; ++s) mbar_init(&meta_full[s], 1);
    for (int s = 0; s < kKtConvWarps * L::kStages; ++s) mbar_init(&staged_full[s], 1);
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

  if (warp < kKtConvWarps) {
    // ----------------------------- codes to fp16 -----------------------------
    // The warps take half tiles (64 keys) in turn: unit g is half g & 1 of the
    // tile with ring position g >> 1 (even: K, odd: V, of block g >> 2).  A unit's
    // codes come by bulk copies (a page's codes of one head are contiguous) into
    // one of the warp's stages, kStages units ahead.  What no page holds is
    // converted as it lies there: codes are finite, and those keys weigh nothing.
    constexpr int kPerKey = D / 16;                        // vectors of 16 codes of a key
    constexpr int kVecs = kKtUnit * kPerKey / 32;          // of a unit, a lane
    constexpr int kKeyStep = 32 / kPerKey;
    const int key_in = lane / kPerKey, col = lane % kPerKey;
    const uint32_t seg_bytes = seg_keys * D;
    const uint32_t stage0 = smem_u32(staged + warp * L::kStages * L::kUnit);
    uint64_t* full = staged_full + warp * L::kStages;
    // Pages and scales are looked up for four blocks at a time, a lane for each 16 keys, two batches ahead, and in
    // three steps a unit apart, so that no load is waited for.  Batch m is the affair of the warp that has the
    // first unit of batch m - 2.  (Each warp looking up its own units' took 1400 cycles a unit.)
    auto write_meta = [&](int m) {
      float4 f = make_float4(1.0f, -INFINITY, 0.0f, __int_as_float(-1));       // no page: weight 0
      bool low = false;
      if (look_page >= 0) {   // a scale of zero: a page never written holds zeros
        const float v = fmaxf(look_v, kKvMinScale);
        const int poisoned = isnan(look_k) || isnan(look_v) ? kPoisoned : 0;
        low = v < kKvLowScale && !poisoned;
        f = make_float4(fmaxf(look_k, kKvMinScale) * fabsf(p.scale_log2), log2f(v), low ? log2f(v) : __frcp_rn(v),
                        __int_as_float(look_page | poisoned));
      }
      const unsigned lows = __ballot_sync(0xffffffffu, low);
      if (lane == 0) s_low[m % (kKtMeta / kKtBatch)] = lows;
      s_meta[(m * kKtBatch % kKtMeta) * 8 + lane] = f;
      __syncwarp();
      if (lane == 0) mbar_arrive(&meta_full[m % (kKtMeta / kKtBatch)]);
    };
    int known = -1;         // the last batch seen to be there
    auto know = [&](int g) {
      const int m = g >> 4;
      if (m <= known) return true;
      known = m;
      return static_cast<bool>(__all_sync(0xffffffffu, mbar_wait(&meta_full[m % (kKtMeta / kKtBatch)],
                                                                 (m / (kKtMeta / kKtBatch)) & 1, abort_flag)));
    };
    // what is known of the 16 keys `in` places into unit g
    auto page_of = [&](int g, int in) {
      return __float_as_int(s_meta[((g >> 2) % kKtMeta) * 8 + ((g & 1) * kKtUnit + in) / 16].w);
    };
    auto issue = [&](int g, int stage, int page) {   // lane j copies segment j
      const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], seg_bytes * __popc(there));
      __syncwarp();
      if (page >= 0) {
        const int key = (blk0 + (g >> 2)) * kKtKeys + (g & 1) * kKtUnit + lane * seg_keys;
        const int64_t off =
            ((static_cast<int64_t>(page & ~kPoisoned) * p.c.heads + hk) * p.c.page + (key & (p.c.page - 1))) * D;
        bulk_load(stage0 + stage * L::kUnit + lane * seg_bytes, p.c.code[(g >> 1) & 1] + off, seg_bytes,
                  smem_u32(&full[stage]));
      }
    };
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
#pragma unroll
    for (int st = 0; st < L::kStages; ++st)
      if (warp + st * kKtConvWarps < units) issue(warp + st * kKtConvWarps, st, ahead_page[st]), ++issued;
    if (warp < 2 && 16 * warp < units) write_meta(warp);
    bool ok = units == 0 || know(0);
    int g = warp;
    for (; ok && g < units; g += kKtConvWarps) {
      const bool is_v = (g >> 1) & 1;
      const int seq = g >> 1, s = seq % NS;
      const int after = g + L::kStages * kKtConvWarps;     // the unit that takes this stage next
      if ((g & 15) == 0) look_pages((g >> 4) + 2);
      if ((g & 15) == 3) look_scales();
      if ((g & 15) == 6 && 16 * ((g >> 4) + 2) < units) write_meta((g >> 4) + 2);
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag) &&
                                       mbar_wait(&slot_empty[s], ((seq / NS) & 1) ^ 1, abort_flag));
      if (!ok) break;
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
      const uint4* src = reinterpret_cast<const uint4*>(staged + (warp * L::kStages + stage) * L::kUnit) + lane;
#pragma unroll
      for (int i0 = 0; i0 < kVecs; i0 += 8) {
        uint4 codes[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) codes[i] = src[32 * (i0 + i)];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t w[4] = {codes[i].x ^ 0x80808080u, codes[i].y ^ 0x80808080u, codes[i].z ^ 0x80808080u,
                                 codes[i].w ^ 0x80808080u};
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[2 * e] = codes_to_h2(w[e], 0x4140);
            h[2 * e + 1] = codes_to_h2(w[e], 0x4342);
          }
          const int v = kVecs > 8 ? i & 1 : 0;
          st_shared_v4(at0[v] + (i0 + i) * kKeyStep * 128,
                       swap ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]));
          st_shared_v4(at1[v] + (i0 + i) * kKeyStep * 128,
                       swap ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]));
        }
      }
      // A page with a NaN scale gets NaN keys instead, so that it reaches the rows that see it and no other.
      if (!is_v) {
        const int page = lane < 4 ? page_of(g, 16 * lane) : -1;
        const unsigned poisoned = __ballot_sync(0xffffffffu, page >= kPoisoned);
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
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&slot_full[s]);
      if (after < units) {
        ok = know(after);
        if (ok) issue(after, stage, lane < segs ? page_of(after, lane * seg_keys) : -1);
      }
      if (++stage == L::kStages) stage = 0, phase ^= 1;
    }
    if (!ok) {   // a wait gave up: let every copy in flight land before the block's memory goes
      for (int st = 0; st < L::kStages; ++st) {
        const int last = g + st * kKtConvWarps;      // units g .. are the ones that may be in flight
        if (last < units && st < issued) mbar_wait(&full[(stage + st) % L::kStages], phase ^ (stage + st >= L::kStages ? 1u : 0u), nullptr);
      }
    }
  } else if (warp == 3) {
    // ------------------------------- MMA issuer -------------------------------
    if (elect_one_sync()) {
      constexpr uint32_t idesc_qk = make_idesc_f16(kKtRows, kKtKeys);
      constexpr uint32_t idesc_pv = make_idesc_f16(kKtRows, D) | (1u << 16);   // V is MN-major
      bool ok = n_blocks == 0 || mbar_poll(q_full, 0, abort_flag);
      auto have = [&](int seq) { return mbar_poll(&slot_full[seq % NS], (seq / NS) & 1, abort_flag); };
      auto issue_s = [&](int j, int t) {
        const int s = (2 * j) % NS;
        tc_fence_after();
        const uint32_t qb = smem_u32(sq + t * L::kTile), kb = smem_u32(ring + s * L::kTile);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_f16(tmem + t * 256, make_sw128_desc(qb + (k >> 2) * 16384) + 2 * (k & 3),
                  make_sw128_desc(kb + (k >> 2) * 16384) + 2 * (k & 3), idesc_qk, k > 0 ? 1u : 0u);
        tc_commit(&s_full[t]);
        if (t == tiles - 1) tc_commit(&slot_empty[s]);
      };
      if (n_blocks > 0) {
        ok = ok && have(0);
        for (int t = 0; t < tiles && ok; ++t) issue_s(0, t);
      }
      for (int j = 0; j < n_blocks && ok; ++j) {
        const int s = (2 * j + 1) % NS;
        // what is not there yet is waited for before the weights, off the tiles' chain, where the ring is deep enough
        ok = have(2 * j + 1) && (kWCol == 0 || j + 1 == n_blocks || have(2 * j + 2));
        for (int t = 0; t < tiles && ok; ++t) {
          if (!mbar_poll(&p_full[t], j & 1, abort_flag)) { ok = false; break; }
          // Dim 64 has columns for the weights beside the products', so the next products, which the softmax waits
          // for, go first.  Dim 128 has the weights where they go: they wait until these are used (nothing orders
          // products of different accumulators).
          if (kWCol != 0 && j + 1 < n_blocks) issue_s(j + 1, t);
          tc_fence_after();
          const uint32_t vb = smem_u32(ring + s * L::kTile);
#pragma unroll
          for (int k = 0; k < kKtKeys / 16; ++k) {
            // 64 dims of 16 keys are one swizzle atom column; the next 64 dims lie 16 KB further
            uint64_t vd = make_sw128_desc(vb + k * 16 * 128);
            vd = (vd & ~(uint64_t(0x3FFFu) << 16)) | (uint64_t(16384 >> 4) << 16);
            mma_f16_ts(tmem + t * 256 + 128, tmem + t * 256 + kWCol + 8 * k, vd, idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit(&o_full[t]);
          if (t == tiles - 1) tc_commit(&slot_empty[s]);
          if (kWCol == 0 && j + 1 < n_blocks) {
            ok = (t > 0 || have(2 * j + 2)) && mbar_poll(&o_full[t], j & 1, abort_flag);
            if (ok) issue_s(j + 1, t);
          }
        }
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
      // Blocks that need more than the usual are told by first_max alone, which a batch with low scales sets past every
      // key: a condition of its own in the loop costs it 2 to 5 %.
      constexpr int kLowBatch = 0x7fffffff;
      int first_max = 0;
      const int last_min = __reduce_min_sync(0xffffffffu, last);
      // Q rows to shared memory
      const uint32_t rows_at = smem_u32(sq + tile * L::kTile) + quad * 32 * 128;      // this warp's
      float back;
      {
        const T* mine = real ? static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + t * p.qs[2] : nullptr;
        // a negative scale turns the rows, so that larger products are larger scores
        back = load_rows<T, D>(mine, p.vec_q, p.scale_log2 < 0.0f ? -1.0f : 1.0f, rows_at);
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      auto wait_meta = [&](int m) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(smem_u32(&meta_full[m % (kKtMeta / kKtBatch)]),
                                                         (m / (kKtMeta / kKtBatch)) & 1, abort_flag));
        first_max = *const_cast<volatile uint32_t*>(s_low + m % (kKtMeta / kKtBatch)) ? kLowBatch : __reduce_max_sync(0xffffffffu, first);
      };
      if (n_blocks > 0) wait_meta(0);
      for (int j = 0; j < n_blocks; ++j) {
        // (dim 128: S(j) was issued after W V of block j - 1 was done, so O is whole)
        ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(smem_u32(&s_full[tile]), j & 1, abort_flag));
        uint32_t meta = smem_u32(s_meta + (j % kKtMeta) * 8);
        asm volatile("" : "+r"(meta));     // its loads stay below the wait
        // (after a wait that gave up the values mean nothing, but every warp keeps in step)
        tc_fence_after();
        const int key0 = (blk0 + j) * kKtKeys;
        if (key0 < first_max || key0 + kKtKeys > last_min) {
          mask_products(t_s, first - key0, last - key0);
          if (first_max == kLowBatch) {
            const float2 ml = low_sums(t_s, meta, back, m, l);
            m = ml.x, l = ml.y;
          }
        }
        // Against the maximum so far; only a row without one, or whose weights outgrow fp16's range by
        // their sums, looks for this block's.
        bool look = __any_sync(0xffffffffu, m == -INFINITY), moved = false;
        float alpha = 1.0f, sum;
        uint32_t w[64];
        while (true) {
          if (look) {
            const float4 r = look_row(t_s, meta, back, m, l);
            moved = r.x > m;
            m = r.x, alpha = r.y, l = r.z;
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          float most = 0.0f;
          sum = weights<0>(t_s, meta, back, ref, w, most);
          sum += weights<1>(t_s, meta, back, ref, w, most);
          if (look || !__any_sync(0xffffffffu, most > kKtMostWeight)) break;
          look = true;
        }
        l = __fmaf_rn(l, alpha, sum);
        // W V of block j - 1 is done: its weights' columns are free, and O is whole
        if (kWCol != 0 && j > 0)
          ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(smem_u32(&o_full[tile]), (j - 1) & 1, abort_flag));
        tmem_st64(t_s + kWCol, w);      // dim 128: over the products that they came from
        if (j > 0 && __any_sync(0xffffffffu, moved)) {
          tc_fence_after();
          rescale_row(t_o, D, alpha);
        }
        tmem_st_wait();
        tc_fence_before();
        if (ok) mbar_arrive(&p_full[tile]);
        if (j + 1 < n_blocks && (j + 1) % kKtBatch == 0) wait_meta((j + 1) / kKtBatch);      // under the next products
      }
      if (n_blocks > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait_u32(smem_u32(&o_full[tile]), (n_blocks - 1) & 1, abort_flag));
      const bool have = ok && n_blocks > 0;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (have) tc_fence_after();
      T* out = real ? static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] : nullptr;
      float* part = nullptr;
      if (real && p.part)
        part = p.part + ((((static_cast<int64_t>(split) * p.c.batch + b) * p.c.heads + hk) * g_rows) + full) * (D + 4);
      if (p.part || p.vec_out) {
        store_rows<T, D>(t_o, have, inv, out, part, p.part != nullptr, rows_at);   // over Q: every product with it is done
        if (part) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
      } else {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          load_o(t_o + c * 32, have, r);
          if (real) {
#pragma unroll
            for (int d = 0; d < 32; ++d) from_f32(__uint_as_float(r[d]) * inv, out[c * 32 + d]);
          }
          __syncwarp();     // the next load out of TMEM wants the whole warp
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
