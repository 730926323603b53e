// ops_attention_mma.cuh -- what the FP16 / BF16 attention kernels share: the ring
// of key and value slabs, operand packing, and the care for non-finite values in
// key tiles that are seen in part.
#pragma once

#include "ops_attention.cuh"

namespace svl {

// K and V travel in slabs of 128 keys x 64 columns, 128-byte swizzled.
constexpr int kSlabBytes = 16384, kSlabCols = 64;
constexpr int kSmemLimit = 232448;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kBehind = 8.0f;  // a maximum follows once it is 2^8 behind (log2 units)

// cap tanh(scale s / cap) of a raw score s in log2 units.  tanh y = y P(y^2) with
// P of degree 3 fitted to tanh(y) / y for |y| <= 0.35 (relative error 3.5e-08, below
// FP32's half step): multiply-adds on the FMA pipe, with the cap and scale in the
// coefficients.  The general form costs two of the 16 special functions a cycle
// that the softmax itself needs, and its error is of the cap's size.  A score takes
// it behind cap_limit (0.35 cap / scale), and by its own size alone: what else the
// tile holds (masked keys, other sequences, rows behind the tile) decides only
// whether the warp computes the general form at all.
constexpr double kTanhOdd[kCapTerms] = {0.9999999659298247, -0.3333243239119307, 0.1329601580300818, -0.04897000350211587};
constexpr double kTanhLimit = 0.35;
// where term i of it is 2^-25 of the whole: the limit without that term (its
// coefficient shrinks with the cap: caps above 2e5 at a scale of 1/8 lose the last one)
constexpr double kTanhWithout[kCapTerms] = {0.0, 2.9e-4, 0.0217, 0.092};
SVL_DEV float cap_odd(const AttnParams& p, float s) {
  const float z = __fmul_rn(s, s);
  return fmaf(z, fmaf(z, fmaf(z, p.cap_odd[3], p.cap_odd[2]), p.cap_odd[1]), p.cap_odd[0]);
}
// (rounded wherever it is used: not one half of a multiply-add)
SVL_DEV float capped_small(const AttnParams& p, float s) { return __fmul_rn(s, cap_odd(p, s)); }

// Two FP32 values in one register pair, and the packed forms of the FMA pipe.
SVL_DEV uint64_t two(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
SVL_DEV uint64_t two(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
SVL_DEV void apart(uint64_t v, uint32_t& lo, uint32_t& hi) { asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v)); }
SVL_DEV uint64_t mul_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SVL_DEV uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
SVL_DEV uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// cap_odd of four pairs, to the same bits.
struct CapOdd {
  uint64_t k[kCapTerms];
  SVL_DEV CapOdd(const AttnParams& p) {
#pragma unroll
    for (int i = 0; i < kCapTerms; ++i) k[i] = two(p.cap_odd[i], p.cap_odd[i]);
  }
  SVL_DEV void over(const uint64_t* s, uint64_t* r) const {
    uint64_t z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = mul_two(s[i], s[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fma_two(z[i], k[kCapTerms - 1], k[kCapTerms - 2]);
#pragma unroll
    for (int j = kCapTerms - 3; j >= 0; --j)
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = fma_two(z[i], r[i], k[j]);
  }
};

// capped_small over N values in place, eight at a time so that their chains
// overlap.
template <int N>
SVL_DEV void capped_small(const AttnParams& p, uint32_t* w) {
  const CapOdd odd(p);
#pragma unroll
  for (int c = 0; c < N; c += 8) {
    uint64_t s[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = two(w[c + 2 * i], w[c + 2 * i + 1]);
    odd.over(s, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) apart(mul_two(s[i], r[i]), w[c + 2 * i], w[c + 2 * i + 1]);
  }
}

// cap - 2 cap / (1 + e^2y); arg = 2 log2(e) scale / cap, cap2 = cap log2(e)
SVL_DEV float capped_large(float s, float arg, float cap2) {
  float r;  // of 1 .. infinity
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2_approx(s * arg)));
  return fmaf(-2.0f * cap2, r, cap2);
}
// The form that s's own size asks for: both are computed and one is selected, since
// lanes differ (a branch for each score: 1185 against 727 us where four scores of ten lie
// behind the limit).
SVL_DEV float by_size(const AttnParams& p, float s, float small, float large) {
  float r;
  asm("{\n.reg .pred p;\n.reg .f32 m;\nabs.f32 m, %3;\nsetp.le.f32 p, m, %4;\nselp.f32 %0, %1, %2, p;\n}"
      : "=f"(r)
      : "f"(small), "f"(large), "f"(s), "f"(p.cap_limit));
  return r;
}
SVL_DEV float capped_any(const AttnParams& p, float s, float arg, float cap2) {
  return by_size(p, s, capped_small(p, s), capped_large(s, arg, cap2));
}

SVL_DEV uint32_t pack2(__half, float lo, float hi) { return pack_half2(lo, hi); }
SVL_DEV uint32_t pack2(__nv_bfloat16, float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Keeps the larger magnitudes of each half; NaN stays.
SVL_DEV uint32_t max_abs(__half, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n.reg .b32 t;\nabs.f16x2 t, %2;\nmax.NaN.f16x2 %0, %1, t;\n}" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
SVL_DEV uint32_t max_abs(__nv_bfloat16, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n.reg .b32 t;\nabs.bf16x2 t, %2;\nmax.NaN.bf16x2 %0, %1, t;\n}" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Per packed pair: the sign bit of each half whose exponent is all ones.
SVL_DEV uint32_t non_finite(__half, uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
SVL_DEV uint32_t non_finite(__nv_bfloat16, uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

struct RingPos {
  uint32_t stage = 0, phase = 0;
  SVL_DEV void next(uint32_t stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// A position `slabs` further on (less than a turn).
SVL_DEV RingPos ahead(RingPos p, uint32_t slabs, uint32_t stages) {
  p.stage += slabs;
  if (p.stage >= stages) {
    p.stage -= stages;
    p.phase ^= 1;
  }
  return p;
}

// The non-finite values that the check took out of the segment's partly seen
// tiles, added to a row that sees them: 32 output columns.
template <typename T>
static __device__ __noinline__ void add_spoiled(const AttnParams& p, const AttnSegment& seg, const AttnSeq& s, uint32_t query,
                                         uint32_t col0, float* o) {
  const RowMask m = row_mask(p, s, query);
  for (uint32_t il = seg.list0; il < seg.list1; ++il) {
    const uint32_t e = p.lists[il];
    if (entry_sees(e, 0) != kSeesSome && entry_sees(e, 1) != kSeesSome) continue;
    for (uint32_t c = 0; c < kKeyTile; ++c) {
      const uint32_t j = entry_tile(e) * kKeyTile + c;
      if (j >= s.n_k) break;
      if (!sees(p, m, j, p.doc_k ? p.doc_k[s.k0 + j] : 0)) continue;
      const T* v = (const T*)p.v + (s.k0 + j) * p.ld_v + (uint64_t)seg.kvh * p.head_dim + col0;
      for (uint32_t d = 0; d < 32 && col0 + d < p.head_dim; ++d) {
        const float x = widen(v[d]);
        if (!isfinite(x)) o[d] += x;
      }
    }
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? (EncodeTiledFn)ptr
               : nullptr;
  }();
  return fn;
}

// [rows][heads][head_dim] with 128-byte swizzled boxes of 64 columns, box_heads
// heads and box_rows rows; columns behind the head read as zero.
inline bool head_map(CUtensorMap* map, const void* base, uint32_t dtype, uint64_t rows, uint64_t heads, uint64_t head_dim,
              uint64_t ld, uint32_t box_heads, uint32_t box_rows) {
  const cuuint64_t dims[3] = {head_dim, heads, rows}, strides[2] = {head_dim * 2, ld * 2};
  const cuuint32_t box[3] = {kSlabCols, box_heads, box_rows}, step[3] = {1, 1, 1};
  return encode_fn()(map, dtype == SVL_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     (void*)base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace svl
