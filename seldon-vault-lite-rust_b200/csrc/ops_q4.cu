// ops_q4.cu -- products of a few rows with a 4-bit weight matrix (svl_q4_* of
// include/svl_gpu.h): y[m, i] = sum_j x[m, j] (code[i, j] - zero[i, j / g])
// scale[i, j / g].
//
// A few rows are bound by reading the codes once (n k / 2 bytes), so the
// weights are the stationary operand of mma.sync m16n8k16: 16 weight rows x 16
// columns against up to 8 rows of x (n = 8).  (A tcgen05 tile has 128 rows of M
// and needs its operands in shared memory in the operand type; here the codes
// go from one 16-byte load straight into operand registers.)  code - zero is a
// whole number of at most 4 bits and sign, exact in FP16 and BF16, so a group's
// sum of products is FP32-exact up to its additions and the scale multiplies it
// once in FP32.  FP32 rows are cut into three BF16 parts of 8 bits each, which
// is exact for values of 2^-110 and more (BF16 ends at 2^-133, and what lies under
// that is cut off), and the parts are further columns of the product.
//
// 8192 x 28672 with groups of 128 and one BF16 row (121 MB): 36-38 us, 3.2-3.4 TB/s.
// The integer pipe bounds it: three shifts and four masks a word of eight codes at half
// an instruction a cycle and scheduler, 70-71% busy while the kernel runs.
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <vector>

#include "ops_common.cuh"

namespace svl {
namespace {

constexpr uint32_t kErrNonFinite = 1;

// The order of the product's columns inside a block of 64 is free as long as
// both operands have it.  Lane 4 g + q takes columns 8 q .. 8 q + 7 of each half
// block of 32 (the shortest group), four of them a step: steps 0 and 1 are the
// first half, 2 and 3 the second.  So its part of a 16-bit x row is two 16-byte
// loads and its codes of the block's 16 x 64 weights one: word w holds step w,
// for rows g and g + 8.  The two nibbles of an operand register lie 16 bits
// apart, where one mask takes both.
//
// A row block (16 weight rows) is a run of spans of 128 columns: two blocks'
// codes, and in arrays of their own the span's 128 / group scale pairs and
// zeros.  Rows and columns behind the matrix have code 0 and scale 0.
struct Q4Matrix {
  const uint4* codes;      // [row block][span][block][lane]
  const uint32_t* scales;  // [row block][span][group][8]: rows g (low half) and g + 8
  const uint8_t* zeros;    // the same, four bits each; NULL: 8
  uint32_t n, k, group, scale_dtype;
  __host__ __device__ uint32_t row_blocks() const { return (n + 15) / 16; }
  __host__ __device__ uint32_t spans() const { return (k + 127) / 128; }
  __host__ __device__ uint32_t span_groups() const { return 128 / group; }
};

// Nibble of a word that holds row g + 8 upper and the step's column c = 0..3:
// register upper + 2 (c / 2) of the operand, half c % 2.
SVL_DEV uint32_t nibble_at(uint32_t upper, uint32_t c) { return upper + 2 * (c >> 1) + 4 * (c & 1); }

// Plain codes, scales and zeros into the handle's order.
__global__ void q4_lay_out_kernel(const __grid_constant__ Q4Matrix m, const uint8_t* __restrict__ codes,
                                  const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros) {
  const uint64_t words = (uint64_t)m.row_blocks() * m.spans() * 256, step = (uint64_t)gridDim.x * blockDim.x;
  const uint64_t first = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  for (uint64_t i = first; i < words; i += step) {
    const uint32_t w = i & 3, lane = (i >> 2) & 31, half = (i >> 7) & 1;
    const uint64_t span = i >> 8;
    const uint64_t row = span / m.spans() * 16 + (lane >> 2);
    const uint64_t col = span % m.spans() * 128 + half * 64 + (w >> 1) * 32 + (lane & 3) * 8 + 4 * (w & 1);
    uint32_t word = 0;
    for (uint32_t upper = 0; upper < 2; ++upper)
      if (row + 8 * upper < m.n && col < m.k) {
        const uint8_t* src = codes + (row + 8 * upper) * (m.k / 2) + col / 2;
        for (uint32_t c = 0; c < 4; ++c)
          word |= (uint32_t)(src[c >> 1] >> (4 * (c & 1)) & 15) << (4 * nibble_at(upper, c));
      }
    ((uint32_t*)m.codes)[i] = word;
  }
  const uint32_t per_row = m.spans() * m.span_groups(), groups = m.k / m.group;
  for (uint64_t i = first; i < (uint64_t)m.row_blocks() * per_row * 8; i += step) {
    const uint64_t row = i / 8 / per_row * 16 + (i & 7), g = i / 8 % per_row;
    uint32_t s = 0, z = 0;
    for (uint32_t upper = 0; upper < 2; ++upper)
      if (row + 8 * upper < m.n && g < groups) {
        const uint64_t at = (row + 8 * upper) * groups + g;
        s |= (uint32_t)scales[at] << (16 * upper);
        if (zeros) z |= (uint32_t)(zeros[at] & 15) << (4 * upper);
      }
    ((uint32_t*)m.scales)[i] = s;
    if (zeros) ((uint8_t*)m.zeros)[i] = (uint8_t)z;
  }
}

// The reverse.
__global__ void q4_read_kernel(const __grid_constant__ Q4Matrix m, uint8_t* __restrict__ codes,
                               uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const uint64_t step = (uint64_t)gridDim.x * blockDim.x, first = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  for (uint64_t i = first; codes && i < (uint64_t)m.n * (m.k / 2); i += step) {
    const uint64_t row = i / (m.k / 2), col = i % (m.k / 2) * 2;
    const uint64_t block = (row / 16 * m.spans() + col / 128) * 2 + (col & 127) / 64;
    const uint32_t lane = (row & 7) * 4 + (col & 31) / 8, w = (col & 63) / 32 * 2 + (col & 7) / 4, upper = row >> 3 & 1;
    const uint32_t word = ((const uint32_t*)m.codes)[block * 128 + lane * 4 + w];
    codes[i] = (uint8_t)((word >> (4 * nibble_at(upper, col & 3)) & 15) | (word >> (4 * nibble_at(upper, (col & 3) + 1)) & 15) << 4);
  }
  const uint32_t per_row = m.spans() * m.span_groups(), groups = m.k / m.group;
  for (uint64_t i = first; i < (uint64_t)m.n * groups; i += step) {
    const uint64_t row = i / groups, at = (row / 16 * per_row + i % groups) * 8 + (row & 7);
    const uint32_t upper = row >> 3 & 1;
    if (scales) scales[i] = (uint16_t)(m.scales[at] >> (16 * upper));
    if (zeros) zeros[i] = m.zeros ? (uint8_t)(m.zeros[at] >> (4 * upper) & 15) : 8;
  }
}

SVL_DEV void mma_16816(__half, float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
SVL_DEV void mma_16816(__nv_bfloat16, float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// The same with nothing to add to.
SVL_DEV void mma_16816_first(__half, float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}
SVL_DEV void mma_16816_first(__nv_bfloat16, float* d, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}

// 16-bit operands of the product; FP32 rows take the BF16 form three times.
template <typename T>
struct Operand {
  using Type = T;
  static constexpr int kParts = 1;
};
template <>
struct Operand<float> {
  using Type = __nv_bfloat16;
  static constexpr int kParts = 3;
};

// A whole number q of 4 bits in a half: 1024 + q is FP16 0x6400 | q, 128 + q is
// BF16 0x4300 | q; the zero comes with the same offset, negated (the sign bit),
// and the sums are exact.
SVL_DEV uint32_t offset_bits(__half) { return 0x64006400u; }
SVL_DEV uint32_t offset_bits(__nv_bfloat16) { return 0x43004300u; }
SVL_DEV uint32_t plus(__half, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
SVL_DEV uint32_t plus(__nv_bfloat16, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x3f803f80u), "r"(b));
  return r;
}

// Part `part` of an FP32 value, as the high half of a word: its first 8
// significant bits, the next 8, the last 8 (cut, not rounded: nothing overflows).
SVL_DEV uint32_t bf16_part(float x, int part) {
  uint32_t hi = __float_as_uint(x) & 0xffff0000u;
  if (part > 0) {
    x -= __uint_as_float(hi);
    hi = __float_as_uint(x) & 0xffff0000u;
  }
  if (part > 1) {
    x -= __uint_as_float(hi);
    hi = __float_as_uint(x) & 0xffff0000u;
  }
  return hi;
}

// 8 values of a row of x as two steps' operand registers (two a step).
template <typename T>
SVL_DEV void pack_columns(const uint4* v, int part, uint32_t* b) {
  if constexpr (sizeof(T) == 2) {
    b[0] = v->x, b[1] = v->y, b[2] = v->z, b[3] = v->w;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x[4] = {__uint_as_float(v[i].x), __uint_as_float(v[i].y), __uint_as_float(v[i].z), __uint_as_float(v[i].w)};
      b[2 * i] = bf16_part(x[0], part) >> 16 | bf16_part(x[1], part);
      b[2 * i + 1] = bf16_part(x[2], part) >> 16 | bf16_part(x[3], part);
    }
  }
}
// From global memory, with the element's own alignment.
template <typename T>
SVL_DEV void load_columns(const T* row, int part, uint32_t* b) {
  uint4 v[sizeof(T) / 2];
  if constexpr (sizeof(T) == 2) {
    const uint16_t* e = (const uint16_t*)row;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    v[0] = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const uint32_t* e = (const uint32_t*)row;
    v[0] = make_uint4(e[0], e[1], e[2], e[3]);
    v[1] = make_uint4(e[4], e[5], e[6], e[7]);
  }
  pack_columns<T>(v, part, b);
}

// Asynchronous copies to shared memory.  `there` false: 16 zero bytes; with a
// source size of 0 the address is not looked at.
SVL_DEV void copy16(uint32_t smem, const void* src, bool there = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(src), "r"(there ? 16 : 0) : "memory");
}
SVL_DEV void copy4(uint32_t smem, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(src) : "memory");
}
SVL_DEV void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
SVL_DEV void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kWarps = 8;

// A span's weights in shared memory.
template <int GROUP>
struct Weights {
  static constexpr int kGroups = 128 / GROUP;
  uint4 code[2][32];
  uint32_t scale[kGroups][8];
  uint8_t zero[kGroups][8];
  uint8_t unused[128 - kGroups * 40 % 128];
};
static_assert(sizeof(Weights<32>) % 128 == 0 && sizeof(Weights<64>) % 128 == 0 && sizeof(Weights<128>) % 128 == 0,
              "whole lines");

// A lane's part in the copies of one row block's spans, one after another from
// `first` on.
template <int GROUP, bool ZEROS>
struct WeightCopies {
  using W = Weights<GROUP>;
  const uint4* code;
  const uint32_t* scale;
  const uint8_t* zero;
  SVL_DEV WeightCopies(const Q4Matrix& w, uint64_t rb, uint32_t first, int lane) {
    const uint64_t span = rb * w.spans() + first;
    code = w.codes + span * 64 + lane;
    scale = w.scales + span * W::kGroups * 8 + lane;
    if (ZEROS) zero = w.zeros + span * W::kGroups * 8 + lane * 4;
  }
  // Span `i` from here into shared memory; `to` includes this lane's 16 bytes.
  SVL_DEV void copy(uint32_t to, int i, int lane) const {
    copy16(to, code + i * 64);
    copy16(to + 512, code + i * 64 + 32);
    const uint32_t side = to - lane * 12;
    if (W::kGroups == 4 || lane < W::kGroups * 8) copy4(side + (uint32_t)offsetof(W, scale), scale + i * W::kGroups * 8);
    if (ZEROS && lane < W::kGroups * 2) copy4(side + (uint32_t)offsetof(W, zero), zero + i * W::kGroups * 8);
  }
  SVL_DEV void advance(int spans) {
    code += spans * 64;
    scale += spans * W::kGroups * 8;
    if (ZEROS) zero += spans * W::kGroups * 8;
  }
};

template <bool HALF>
SVL_DEV float2 scale_pair(uint32_t s) {
  return HALF ? unpack_half2(s) : make_float2(__uint_as_float(s << 16), __uint_as_float(s & 0xffff0000u));
}

// acc += (codes - zeros) . columns * scales over a span, a group at a time;
// b[block] are a lane's four steps of operand registers of a column tile.
// SETS column tiles share the unpacked weights.
template <typename Op, int GROUP, bool HALF, bool ZEROS, int SETS, typename Columns>
SVL_DEV void multiply_span(float (*acc)[4], const Weights<GROUP>& st, int lane, Columns&& columns) {
  const int g = lane >> 2;
  const uint32_t base = offset_bits(Op());
  uint32_t a[2][4][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint4 code = st.code[half][lane];
    const uint32_t word[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int group = (half * 64 + i / 2 * 32) / GROUP;
      uint32_t z0 = (base | 0x80008000u) + 0x00080008u, z1 = z0;
      if (ZEROS) {
        const uint32_t z = st.zero[group][g];
        z0 = (base | 0x80008000u) + (z & 15) * 0x10001u, z1 = (base | 0x80008000u) + (z >> 4) * 0x10001u;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) a[half][i][e] = plus(Op(), (word[i] >> (4 * e) & 0x000f000fu) | base, e & 1 ? z1 : z0);
    }
  }
  float2 scale[Weights<GROUP>::kGroups];
#pragma unroll
  for (int i = 0; i < Weights<GROUP>::kGroups; ++i) scale[i] = scale_pair<HALF>(st.scale[i][g]);
#pragma unroll
  for (int t = 0; t < SETS; ++t) {
    uint32_t b[2][8];
    columns(t, b);
    // a chain of products for each group, two for the span's only one
    constexpr int kChain = GROUP == 32 ? 2 : 4;
    float part[8 / kChain][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float* p = part[i / kChain];
      if (i % kChain == 0) mma_16816_first(Op(), p, a[i / 4][i % 4], b[i / 4] + 2 * (i % 4));
      else mma_16816(Op(), p, a[i / 4][i % 4], b[i / 4] + 2 * (i % 4));
    }
    if constexpr (GROUP == 128) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(part[0][e] + part[1][e], e < 2 ? scale[0].x : scale[0].y, acc[t][e]);
    } else {
#pragma unroll
      for (int i = 0; i < Weights<GROUP>::kGroups; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(part[i][e], e < 2 ? scale[i].x : scale[i].y, acc[t][e]);
    }
  }
}

// A span of x in shared memory: rows of 128 values whose 16-byte units change
// places in odd rows, so that the rows g and g + 1 that a quarter warp reads do
// not meet in a bank.
template <typename T>
struct XTile {
  static constexpr int kUnits = 8 * (int)sizeof(T), kBytes = 128 * (int)sizeof(T);
  static SVL_DEV int unit(int row, int u) { return row * kUnits + (u ^ (sizeof(T) == 2 ? (row & 1) << 2 : row & 1)); }
  // A lane's 8 columns of each half of each block, of one row: from byte offset
  // `even` in the even halves and `odd` in the odd ones.
  static SVL_DEV uint32_t offset(int row, int q, int half) { return unit(row, (half * 4 + q) * ((int)sizeof(T) / 2)) * 16; }
  static SVL_DEV void columns(const uint8_t* tile, uint32_t even, uint32_t odd, int part, uint32_t (*b)[8]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const uint4* from = (const uint4*)(tile + (h & 1 ? odd : even) + (h >> 1) * (kBytes / 2));
      uint4 v[sizeof(T) / 2];
      v[0] = from[0];
      // the neighbour of an FP32 unit is its partner in the row's order
      if constexpr (sizeof(T) == 4) v[1] = *(const uint4*)((uintptr_t)from ^ 16);
      pack_columns<T>(v, part, b[h >> 1] + 4 * (h & 1));
    }
  }
  // The same from global memory; columns behind the matrix are zero (k is a multiple of 32).
  static SVL_DEV void columns(const T* row, uint32_t col0, uint32_t k, int q, int part, uint32_t (*b)[8]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint32_t* to = b[h >> 1] + 4 * (h & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = 0;
      if (col0 + 32 * h < k) load_columns<T>(row + col0 + 32 * h + 8 * q, part, to);
    }
  }
};

// Copies by threads `tid` of N of spans of up to ROWS rows of x, one after
// another from `first` on.
template <typename T, int ROWS, int N>
struct XCopies {
  static constexpr int kUnits = XTile<T>::kUnits, kStep = N / kUnits, kCopies = (ROWS + kStep - 1) / kStep;
  static_assert(kStep % 2 == 0 || kStep == 1, "a thread's rows are all even or all odd, or alternate");
  const T* from;
  uint64_t stride;
  uint32_t to;
  int row, rows, whole;  // spans from here on that lie inside the matrix
  bool in_last;          // this thread's unit of the span behind them does
  SVL_DEV XCopies(const T* x, uint64_t ld, int rows_, uint32_t first, uint32_t k, int tid) {
    const int u = tid % kUnits;
    row = tid / kUnits;
    rows = rows_;
    from = x + row * ld + first * 128 + u * (16 / (int)sizeof(T));
    stride = kStep * ld;
    to = XTile<T>::unit(row, u) * 16;
    whole = (int)(k / 128) - (int)first;
    in_last = u * (16 / (int)sizeof(T)) < (int)(k % 128);
  }
  SVL_DEV void copy(uint32_t smem, int i) const {
    const bool there = i < whole || in_last;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      if (ROWS > 1 && c * kStep >= rows) break;
      if (row + c * kStep < rows) {
        // a step of one row changes the order of its units (FP32: neighbours)
        const uint32_t flip = kStep == 1 ? (c & 1) * 16 : 0;
        copy16(smem + (to ^ flip) + c * kStep * XTile<T>::kBytes, from + c * stride + i * 128, there);
      }
    }
  }
  SVL_DEV void advance(int spans) {
    from += spans * 128;
    whole -= spans;
  }
};

// Up to 16 columns (rows of x, or parts of them).  One block: 8 / split row
// blocks; `split` warps share one, take a run of its spans each and join their
// sums in shared memory, in a fixed order.  Each warp copies its own weights and
// rows of x ahead, so no barrier stands between load and product.  Tile columns
// behind the rows repeat the last one and are not written.  WIDE: x has rows of
// 16-byte units.
constexpr int few_stages(int cols) { return cols <= 8 ? 4 : 2; }  // so that two blocks fit an SM
template <typename T, int ROWS, int GROUP, bool HALF, bool ZEROS, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32, ROWS == 1 ? 3 : 2)
    q4_few_kernel(const __grid_constant__ Q4Matrix w, const T* __restrict__ x, uint64_t ld_x, uint32_t rows,
                  T* __restrict__ y, uint64_t ld_y, const uint32_t split) {
  using Op = typename Operand<T>::Type;
  constexpr int kParts = Operand<T>::kParts, NT = (ROWS * kParts + 7) / 8, kCols = NT * 8;
  constexpr int kStages = few_stages(ROWS * kParts);
  constexpr uint32_t kStage = sizeof(Weights<GROUP>) + (WIDE ? ROWS * XTile<T>::kBytes : 0);
  extern __shared__ __align__(128) uint8_t shared[];
  float* sums = (float*)shared;  // [warp][16][kCols], after the products
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint8_t* ring = shared + warp * kStages * kStage;
  const uint32_t ring_at = smem_u32(ring), spans = w.spans();
  const uint32_t rb = blockIdx.x * (kWarps / split) + warp / split, turn = warp % split;
  const bool mine = rb < w.row_blocks();
  const uint32_t first = (uint32_t)((uint64_t)spans * turn / split);
  const int count = mine ? (int)((uint64_t)spans * (turn + 1) / split) - (int)first : 0;
  float acc[NT][4] = {};

  WeightCopies<GROUP, ZEROS> weights(w, mine ? rb : 0, first, lane);
  XCopies<T, ROWS, 32> columns(x, ld_x, (int)rows, first, w.k, lane);
  // span `i` from where the copies stand, into a stage
  auto fetch = [&](int i, int stage, bool in) {
    if (in) {
      const uint32_t to = ring_at + stage * kStage;
      weights.copy(to + lane * 16, i, lane);
      if (WIDE) columns.copy(to + sizeof(Weights<GROUP>), i);
    }
    copies_commit();  // also empty: the count of groups in flight stays
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i, i, i < count);
  int row[NT], part[NT];
  uint32_t even[NT], odd[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    row[t] = ROWS == 1 ? 0 : min((t * 8 + g) / kParts, (int)rows - 1);
    part[t] = (t * 8 + g) % kParts;
    even[t] = sizeof(Weights<GROUP>) + XTile<T>::offset(row[t], q, 0);
    odd[t] = ROWS == 1 ? even[t] + XTile<T>::kBytes / 4 : sizeof(Weights<GROUP>) + XTile<T>::offset(row[t], q, 1);
  }
#pragma unroll 1
  for (int i = 0; i < count; i += kStages) {
#pragma unroll
    for (int u = 0; u < kStages; ++u) {
      if (i + u >= count) break;
      copies_wait<kStages - 2>();
      __syncwarp();
      // into the stage that every lane read a turn ago
      fetch(u + kStages - 1, (u + kStages - 1) % kStages, i + u + kStages - 1 < count);
      const uint8_t* st = ring + u * kStage;
      multiply_span<Op, GROUP, HALF, ZEROS, NT>(acc, *(const Weights<GROUP>*)st, lane, [&](int t, uint32_t(*b)[8]) {
        if constexpr (WIDE) XTile<T>::columns(st, even[t], odd[t], part[t], b);
        else XTile<T>::columns(x + row[t] * ld_x, (first + i + u) * 128, w.k, q, part[t], b);
      });
    }
    weights.advance(kStages);
    columns.advance(kStages);
  }
  copies_wait<0>();
  __syncthreads();  // the rings' memory becomes the sums'
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float* s = sums + (warp * 16 + g) * kCols + t * 8 + 2 * q;
    *(float2*)s = make_float2(acc[t][0], acc[t][1]);
    *(float2*)(s + 8 * kCols) = make_float2(acc[t][2], acc[t][3]);
  }
  __syncthreads();
  const int block_rows = 16 * (kWarps / split);
  for (int i = threadIdx.x; i < block_rows * (int)rows; i += kWarps * 32) {
    const int r = i % block_rows, m = i / block_rows;
    const uint64_t n = (uint64_t)blockIdx.x * block_rows + r;
    if (n >= w.n) continue;
    const float* from = sums + (r / 16 * split * 16 + r % 16) * kCols + m * kParts;
    float sum = 0.0f;
#pragma unroll
    for (int p = kParts - 1; p >= 0; --p)  // the smallest first
      for (uint32_t v = 0; v < split; ++v) sum += from[v * 16 * kCols + p];
    y[m * ld_y + n] = narrow<T>(sum);
  }
}

// More columns: the 8 warps take different row blocks of the same span, whose
// rows of x they share; the blocks of a cluster take a run of the spans each and
// join their sums through each other's shared memory, in a fixed order.
// FP32 rows are cut into their BF16 parts once for all warps (each warp for itself:
// 630 us at 14 rows, 4800 x 26496).
constexpr int kBlockStages = 3;
template <typename T, int NT, int GROUP, bool HALF, bool ZEROS>
__global__ void __launch_bounds__(kWarps * 32, NT == 4 ? 2 : 1)
    q4_many_kernel(const __grid_constant__ Q4Matrix w, const T* __restrict__ x, uint64_t ld_x, uint64_t rows,
                   T* __restrict__ y, uint64_t ld_y) {
  using Op = typename Operand<T>::Type;
  constexpr int kParts = Operand<T>::kParts, kCols = NT * 8, kRows = kCols / kParts, kBlockRows = 16 * kWarps;
  constexpr uint32_t kStage = kWarps * sizeof(Weights<GROUP>) + kRows * XTile<T>::kBytes;
  extern __shared__ __align__(128) uint8_t shared[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint32_t split = gridDim.z, turn = blockIdx.z;
  const uint64_t m0 = (uint64_t)blockIdx.y * kRows;
  const int rows_here = (int)min((uint64_t)kRows, rows - m0);
  const uint32_t rb = blockIdx.x * kWarps + warp;
  const bool mine = rb < w.row_blocks();
  const uint32_t first = (uint32_t)((uint64_t)w.spans() * turn / split);
  const int count = (int)((uint64_t)w.spans() * (turn + 1) / split) - (int)first;
  float acc[NT][4] = {};

  WeightCopies<GROUP, ZEROS> weights(w, mine ? rb : 0, first, lane);
  XCopies<T, kRows, kWarps * 32> columns(x + m0 * ld_x, ld_x, rows_here, first, w.k, threadIdx.x);
  auto fetch = [&](int stage, bool in) {
    if (in) {
      const uint32_t to = smem_u32(shared) + stage * kStage;
      if (mine) weights.copy(to + warp * sizeof(Weights<GROUP>) + lane * 16, 0, lane);
      columns.copy(to + kWarps * sizeof(Weights<GROUP>), 0);
      weights.advance(1);
      columns.advance(1);
    }
    copies_commit();
  };
  for (int i = 0; i < kBlockStages - 1; ++i) fetch(i, i < count);

  // the span's columns as the product takes them: as they came, or their parts
  using Tile = XTile<Op>;
  uint8_t* parts = shared + kBlockStages * kStage;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const uint8_t* st = shared + i % kBlockStages * kStage;
    copies_wait<kBlockStages - 2>();
    __syncthreads();  // everyone's copies of this stage are there, and everyone is done with the one before
    fetch((i + kBlockStages - 1) % kBlockStages, i + kBlockStages - 1 < count);
    const uint8_t* tile = st + kWarps * sizeof(Weights<GROUP>);
    if constexpr (kParts == 3) {
      for (int v = threadIdx.x; v < rows_here * 32; v += kWarps * 32) {
        const int row = v >> 5, u = v & 31;  // 4 columns
        const float4 x4 = *(const float4*)(tile + XTile<T>::unit(row, u) * 16);
        const float xs[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const uint2 w2 = make_uint2(bf16_part(xs[0], part) >> 16 | bf16_part(xs[1], part),
                                      bf16_part(xs[2], part) >> 16 | bf16_part(xs[3], part));
          *(uint2*)(parts + Tile::unit(row * 3 + part, u >> 1) * 16 + (u & 1) * 8) = w2;
        }
      }
      __syncthreads();
      tile = parts;
    }
    if (!mine) continue;
    multiply_span<Op, GROUP, HALF, ZEROS, NT>(
        acc, ((const Weights<GROUP>*)st)[warp], lane, [&](int t, uint32_t(*b)[8]) {
          const int c = min(t * 8 + g, rows_here * kParts - 1);
          Tile::columns(tile, Tile::offset(c, q, 0), Tile::offset(c, q, 1), 0, b);
        });
  }
  copies_wait<0>();
  __syncthreads();
  // [column][row]
  constexpr int kStride = kBlockRows + 4;
  float* sums = (float*)shared;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[(t * 8 + 2 * q + (e & 1)) * kStride + warp * 16 + g + 8 * (e >> 1)] = acc[t][e];
  if (split > 1) cluster_sync();
  else __syncthreads();
  // the blocks of the cluster share out the rows
  const int share = kBlockRows / split, from = turn * share;
  for (int i = threadIdx.x; i < share * rows_here; i += kWarps * 32) {
    const int row = from + i % share, m = i / share;
    const uint64_t n = (uint64_t)blockIdx.x * kBlockRows + row;
    if (n >= w.n) continue;
    float sum = 0.0f;
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)
      for (uint32_t v = 0; v < split; ++v) {
        const float* s = sums + (m * kParts + part) * kStride + row;
        float value;
        if (split == 1) value = *s;
        else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(map_to_rank(smem_u32(s), v)) : "memory");
        sum += value;
      }
    y[(m0 + m) * ld_y + n] = narrow<T>(sum);
  }
  if (split > 1) cluster_sync();  // no block leaves while another reads its sums
}

// One warp per group: its range, scale, zero and codes.
template <typename T>
__global__ void q4_quantize_kernel(const T* __restrict__ w, uint32_t n, uint32_t k, uint32_t group, int asymmetric,
                                   uint8_t* __restrict__ codes, uint16_t* __restrict__ scales,
                                   uint8_t* __restrict__ zeros, uint32_t* __restrict__ err) {
  const int lane = threadIdx.x & 31;
  const uint64_t groups = (uint64_t)n * (k / group), warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
  for (uint64_t g = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); g < groups; g += warps) {
    const T* in = w + g * group;
    float low = 0.0f, high = 0.0f;
    bool finite = true;
    for (uint32_t j = lane; j < group; j += 32) {
      const float v = widen(in[j]);
      finite &= isfinite(v);
      low = fminf(low, v);
      high = fmaxf(high, v);
    }
    low = -warp_max(-low);
    high = warp_max(high);
    if (!__all_sync(0xffffffffu, finite)) {
      if (lane == 0) atomicOr(err, kErrNonFinite);
      continue;
    }
    // 2^-7 of a step is lost when the scale is rounded to BF16's 8 bits: the
    // codes are chosen against the rounded scale and clamped.  The range of
    // two large FP32 values is halved first so that it cannot overflow.
    const float exact = asymmetric ? (high * 0.5f - low * 0.5f) * (2.0f / 15.0f) : fmaxf(-low, high) / 7.0f;
    uint32_t bits = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(exact));
    if (bits == 0 && exact > 0.0f) bits = 1;   // a scale below BF16's range keeps its smallest value
    if (bits >= 0x7f80u) bits = 0x7f7fu;       // and one above it its largest
    const float scale = __uint_as_float(bits << 16);
    const float zero = !asymmetric ? 8.0f : scale > 0.0f ? fminf(fmaxf(rintf(-low / scale), 0.0f), 15.0f) : 0.0f;
    for (uint32_t j = 2 * lane; j < group; j += 64) {
      uint32_t c[2];
      for (int e = 0; e < 2; ++e) {
        const float q = scale > 0.0f ? rintf(widen(in[j + e]) / scale) + zero : zero;
        c[e] = (uint32_t)fminf(fmaxf(q, asymmetric ? 0.0f : 1.0f), 15.0f);
      }
      codes[(g * group + j) / 2] = (uint8_t)(c[0] | c[1] << 4);
    }
    if (lane == 0) {
      scales[g] = (uint16_t)bits;
      if (zeros) zeros[g] = (uint8_t)zero;
    }
  }
}

struct Freed {
  void* p = nullptr;
  ~Freed() {
    if (p) cudaFree(p);
  }
};

}  // namespace
}  // namespace svl

struct svl_q4 {
  svl::Q4Matrix m{};
  int device = -1;
  void* block = nullptr;  // codes, scales and zeros
  ~svl_q4() { svl::free_block(device, block); }
  size_t code_bytes() const { return (size_t)m.n * (m.k / 2); }
  size_t group_count() const { return (size_t)m.n * (m.k / m.group); }
};

using svl::refuse;

namespace {

int q4_check(uint32_t n, uint32_t k, uint32_t group, uint32_t scale_dtype, char* err, size_t err_len) {
  if (group != 32 && group != 64 && group != 128) return refuse(SVL_USAGE, "group must be 32, 64 or 128", err, err_len);
  if (!n || !k || n >= 1u << 31 || k >= 1u << 31) return refuse(SVL_USAGE, "n and k must be 1..2^31 - 1", err, err_len);
  if (k % group) return refuse(SVL_USAGE, "k must be a multiple of the group", err, err_len);
  if (scale_dtype != SVL_DTYPE_F16 && scale_dtype != SVL_DTYPE_BF16)
    return refuse(SVL_USAGE, "scales must be F16 or BF16", err, err_len);
  return SVL_OK;
}

// Reserves the handle's memory on the current device.
int q4_reserve(svl_q4* w, int device, uint32_t n, uint32_t k, uint32_t group, uint32_t scale_dtype, bool zeros,
               char* err, size_t err_len) {
  w->device = device;
  w->m.n = n;
  w->m.k = k;
  w->m.group = group;
  w->m.scale_dtype = scale_dtype;
  const uint64_t rb = w->m.row_blocks();
  const size_t codes = rb * w->m.spans() * 1024, pairs = rb * w->m.spans() * w->m.span_groups() * 8;
  const cudaError_t e = cudaMalloc(&w->block, codes + pairs * 4 + (zeros ? pairs : 0));
  if (e != cudaSuccess) {
    w->block = nullptr;
    return svl::cuda_failure(e, err, err_len);
  }
  uint8_t* p = (uint8_t*)w->block;
  w->m.codes = (const uint4*)p;
  w->m.scales = (const uint32_t*)(p + codes);
  w->m.zeros = zeros ? p + codes + pairs * 4 : nullptr;
  return SVL_OK;
}

// Device memory for `bytes`, or `src` itself where it is this device's already.
bool is_on_device(const void* src, int device) {
  cudaPointerAttributes at{};
  if (cudaPointerGetAttributes(&at, src) == cudaSuccess) return at.type == cudaMemoryTypeDevice && at.device == device;
  cudaGetLastError();
  return false;
}
cudaError_t on_device(const void* src, size_t bytes, int device, svl::Freed& held, const void** out) {
  if (is_on_device(src, device)) {
    *out = src;
    return cudaSuccess;
  }
  cudaError_t e = cudaMalloc(&held.p, bytes);
  if (e == cudaSuccess) e = cudaMemcpy(held.p, src, bytes, cudaMemcpyDefault);
  *out = held.p;
  return e;
}

cudaError_t lay_out(const svl_q4& w, const void* codes, const void* scales, const void* zeros) {
  const uint64_t words = (uint64_t)w.m.row_blocks() * w.m.spans() * 256;
  svl::q4_lay_out_kernel<<<(unsigned)std::min<uint64_t>((words + 255) / 256, 148 * 8), 256>>>(
      w.m, (const uint8_t*)codes, (const uint16_t*)scales, (const uint8_t*)zeros);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? cudaStreamSynchronize(nullptr) : e;
}

constexpr uint32_t kSms = 148;

struct Rows {
  const void* x;
  uint64_t ld_x, rows;
  void* y;
  uint64_t ld_y;
};

template <typename T, int ROWS, int GROUP, bool HALF, bool ZEROS, bool WIDE>
cudaError_t launch_few(const svl::Q4Matrix& m, const Rows& r, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto kernel = svl::q4_few_kernel<T, ROWS, GROUP, HALF, ZEROS, WIDE>;
  constexpr int cols = ROWS * svl::Operand<T>::kParts;
  constexpr int stage = (int)sizeof(svl::Weights<GROUP>) + (WIDE ? ROWS * svl::XTile<T>::kBytes : 0);
  constexpr int ring = svl::few_stages(cols) * stage, sums = 16 * ((cols + 7) / 8) * 8 * 4;
  constexpr int smem = svl::kWarps * (ring > sums ? ring : sums);
  const cudaError_t e = smem_opt_in(kernel, smem, &done);
  if (e != cudaSuccess) return e;
  // Warps to a row block: as many as leave each a run of four spans, more where
  // there would not be a block for every SM.
  uint32_t split = 1;
  while (split < svl::kWarps && 2 * split <= m.spans() &&
         (m.spans() >= 8 * split || (uint64_t)m.row_blocks() * split < (uint64_t)kSms * svl::kWarps))
    split *= 2;
  const uint32_t per_block = svl::kWarps / split;
  const dim3 grid((m.row_blocks() + per_block - 1) / per_block);
  // without 16-byte units more rows come here too, so many at a time
  for (uint64_t m0 = 0; m0 < r.rows; m0 += ROWS) {
    const uint32_t now = (uint32_t)std::min<uint64_t>(r.rows - m0, ROWS);
    kernel<<<grid, svl::kWarps * 32, smem, st>>>(m, (const T*)r.x + m0 * r.ld_x, r.ld_x, now, (T*)r.y + m0 * r.ld_y,
                                                      r.ld_y, split);
    const cudaError_t f = cudaGetLastError();
    if (f != cudaSuccess) return f;
  }
  return cudaSuccess;
}

template <typename T, int NT, int GROUP, bool HALF, bool ZEROS>
cudaError_t launch_many(const svl::Q4Matrix& m, const Rows& r, cudaStream_t st) {
  constexpr uint32_t kRows = NT * 8 / svl::Operand<T>::kParts, kBlockRows = 16 * svl::kWarps;
  constexpr int ring = svl::kBlockStages * (svl::kWarps * (int)sizeof(svl::Weights<GROUP>) + kRows * svl::XTile<T>::kBytes);
  constexpr int all = ring + (svl::Operand<T>::kParts == 3 ? NT * 8 * 256 : 0);
  constexpr int sums = NT * 8 * (kBlockRows + 4) * 4, smem = all > sums ? all : sums;
  static std::atomic<uint64_t> done{0};
  auto kernel = svl::q4_many_kernel<T, NT, GROUP, HALF, ZEROS>;
  const cudaError_t e = smem_opt_in(kernel, smem, &done);
  if (e != cudaSuccess) return e;
  const uint32_t units = (m.row_blocks() + svl::kWarps - 1) / svl::kWarps;
  const uint64_t slabs = (r.rows + kRows - 1) / kRows;
  // Blocks of a cluster: up to 8, while all of them run at once and each has
  // two spans.
  uint32_t split = 1;
  while (split < 8 && split * 4 <= m.spans() && units * slabs * split * 2 <= kSms) split *= 2;
  // a grid's second dimension ends at 65535
  for (uint64_t m0 = 0; m0 < r.rows; m0 += 65535ull * kRows) {
    const uint64_t now = std::min<uint64_t>(r.rows - m0, 65535ull * kRows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units, (unsigned)((now + kRows - 1) / kRows), split);
    cfg.blockDim = dim3(svl::kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = split;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 1 : 0;
    const cudaError_t f = cudaLaunchKernelEx(&cfg, kernel, m, (const T*)r.x + m0 * r.ld_x, r.ld_x, now,
                                             (T*)r.y + m0 * r.ld_y, r.ld_y);
    if (f != cudaSuccess) return f;
  }
  return cudaSuccess;
}

template <typename T, int GROUP, bool HALF, bool ZEROS>
cudaError_t launch_rows(const svl::Q4Matrix& m, const Rows& r, cudaStream_t st) {
  constexpr int kParts = svl::Operand<T>::kParts;
  if (((uintptr_t)r.x | r.ld_x * sizeof(T)) % 16) return launch_few<T, 16 / kParts, GROUP, HALF, ZEROS, false>(m, r, st);
  if (r.rows == 1) return launch_few<T, 1, GROUP, HALF, ZEROS, true>(m, r, st);
  if (r.rows <= 8 / kParts) return launch_few<T, 8 / kParts, GROUP, HALF, ZEROS, true>(m, r, st);
  if (r.rows <= 16 / kParts) return launch_few<T, 16 / kParts, GROUP, HALF, ZEROS, true>(m, r, st);
  if (r.rows <= 32 / kParts) return launch_many<T, 4, GROUP, HALF, ZEROS>(m, r, st);
  return launch_many<T, 8, GROUP, HALF, ZEROS>(m, r, st);
}

template <typename T, int GROUP>
cudaError_t launch_group(const svl::Q4Matrix& m, const Rows& r, cudaStream_t st) {
  const bool half = m.scale_dtype == SVL_DTYPE_F16;
  if (m.zeros) return half ? launch_rows<T, GROUP, true, true>(m, r, st) : launch_rows<T, GROUP, false, true>(m, r, st);
  return half ? launch_rows<T, GROUP, true, false>(m, r, st) : launch_rows<T, GROUP, false, false>(m, r, st);
}

template <typename T>
cudaError_t launch_linear(const svl::Q4Matrix& m, const Rows& r, cudaStream_t st) {
  return m.group == 32   ? launch_group<T, 32>(m, r, st)
         : m.group == 64 ? launch_group<T, 64>(m, r, st)
                         : launch_group<T, 128>(m, r, st);
}

}  // namespace

extern "C" {

int svl_q4_create(int device, const uint8_t* codes, const void* scales, uint32_t scale_dtype, const uint8_t* zeros,
                  uint32_t n, uint32_t k, uint32_t group, svl_q4** out, char* err, size_t err_len) {
  if (!out) return refuse(SVL_USAGE, "null argument", err, err_len);
  *out = nullptr;
  if (!codes || !scales) return refuse(SVL_USAGE, "null argument", err, err_len);
  const int bad = q4_check(n, k, group, scale_dtype, err, err_len);
  if (bad) return bad;
  return svl::guarded(err, err_len, [&]() -> int {
    std::unique_ptr<svl_q4> w(new svl_q4());
    svl::DeviceGuard on(device);
    if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
    // read in place as 16-bit values; host memory is copied, from any address
    if ((uintptr_t)scales & 1 && is_on_device(scales, device)) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
    const int rc = q4_reserve(w.get(), device, n, k, group, scale_dtype, zeros != nullptr, err, err_len);
    if (rc) return rc;
    svl::Freed held[3];
    const void *dc = nullptr, *ds = nullptr, *dz = nullptr;
    cudaError_t e = on_device(codes, w->code_bytes(), device, held[0], &dc);
    if (e == cudaSuccess) e = on_device(scales, 2 * w->group_count(), device, held[1], &ds);
    if (e == cudaSuccess && zeros) e = on_device(zeros, w->group_count(), device, held[2], &dz);
    if (e == cudaSuccess) e = lay_out(*w, dc, ds, dz);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    *out = w.release();
    return SVL_OK;
  });
}

int svl_q4_quantize(int device, const svl_tensor_view* weight, uint32_t group, uint32_t asymmetric, svl_q4** out,
                    char* err, size_t err_len) {
  if (!out) return refuse(SVL_USAGE, "null argument", err, err_len);
  *out = nullptr;
  if (!weight || !weight->data) return refuse(SVL_USAGE, "null argument", err, err_len);
  if (weight->ndim != 2) return refuse(SVL_USAGE, "a 4-bit weight is 2-D", err, err_len);
  if (weight->dtype != SVL_DTYPE_F32 && weight->dtype != SVL_DTYPE_BF16)
    return refuse(SVL_USAGE, "a weight must be F32 or BF16", err, err_len);
  if (weight->shape[0] >= 1ull << 31 || weight->shape[1] >= 1ull << 31)
    return refuse(SVL_USAGE, "n and k must be 1..2^31 - 1", err, err_len);
  const uint32_t n = (uint32_t)weight->shape[0], k = (uint32_t)weight->shape[1];
  const int bad = q4_check(n, k, group, SVL_DTYPE_BF16, err, err_len);
  if (bad) return bad;
  return svl::guarded(err, err_len, [&]() -> int {
    std::unique_ptr<svl_q4> w(new svl_q4());
    svl::DeviceGuard on(device);
    if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
    const int rc = q4_reserve(w.get(), device, n, k, group, SVL_DTYPE_BF16, asymmetric != 0, err, err_len);
    if (rc) return rc;
    const size_t bytes = (size_t)n * k * svl::dtype_size(weight->dtype);
    svl::Freed in, flag, codes, scales, zeros;
    cudaError_t e = cudaMalloc(&in.p, bytes);
    if (e == cudaSuccess) e = cudaMalloc(&flag.p, 4);
    if (e == cudaSuccess) e = cudaMalloc(&codes.p, w->code_bytes());
    if (e == cudaSuccess) e = cudaMalloc(&scales.p, 2 * w->group_count());
    if (e == cudaSuccess && asymmetric) e = cudaMalloc(&zeros.p, w->group_count());
    if (e == cudaSuccess) e = cudaMemcpy(in.p, weight->data, bytes, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemset(flag.p, 0, 4);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    const unsigned grid = (unsigned)std::min<size_t>((w->group_count() + 7) / 8, 148 * 8);
    auto quantize = [&](auto kernel, auto* data) {
      kernel<<<grid, 256>>>(data, n, k, group, asymmetric != 0, (uint8_t*)codes.p, (uint16_t*)scales.p, (uint8_t*)zeros.p,
                            (uint32_t*)flag.p);
    };
    if (weight->dtype == SVL_DTYPE_F32) quantize(svl::q4_quantize_kernel<float>, (const float*)in.p);
    else quantize(svl::q4_quantize_kernel<__nv_bfloat16>, (const __nv_bfloat16*)in.p);
    uint32_t word = 0;
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(&word, flag.p, 4, cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && !word) e = lay_out(*w, codes.p, scales.p, zeros.p);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    if (word) return refuse(SVL_CORRUPT, "weight contains a non-finite value", err, err_len);
    *out = w.release();
    return SVL_OK;
  });
}

void svl_q4_destroy(svl_q4* weight) { delete weight; }

int svl_q4_read(const svl_q4* weight, uint32_t* n, uint32_t* k, uint32_t* group, uint32_t* scale_dtype,
                uint8_t* codes, void* scales, uint8_t* zeros, char* err, size_t err_len) {
  if (!weight) return refuse(SVL_USAGE, "null argument", err, err_len);
  const svl::Q4Matrix& m = weight->m;
  if (n) *n = m.n;
  if (k) *k = m.k;
  if (group) *group = m.group;
  if (scale_dtype) *scale_dtype = m.scale_dtype;
  if (!codes && !scales && !zeros) return SVL_OK;
  svl::DeviceGuard on(weight->device);
  svl::Freed dc, ds, dz;
  cudaError_t e = on.status;
  if (e == cudaSuccess && codes) e = cudaMalloc(&dc.p, weight->code_bytes());
  if (e == cudaSuccess && scales) e = cudaMalloc(&ds.p, 2 * weight->group_count());
  if (e == cudaSuccess && zeros) e = cudaMalloc(&dz.p, weight->group_count());
  if (e == cudaSuccess) {
    svl::q4_read_kernel<<<148 * 8, 256>>>(m, (uint8_t*)dc.p, (uint16_t*)ds.p, (uint8_t*)dz.p);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && codes) e = cudaMemcpy(codes, dc.p, weight->code_bytes(), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && scales) e = cudaMemcpy(scales, ds.p, 2 * weight->group_count(), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && zeros) e = cudaMemcpy(zeros, dz.p, weight->group_count(), cudaMemcpyDeviceToHost);
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

int svl_q4_linear_device(const svl_q4* weight, uint32_t dtype, const void* d_x, uint64_t ld_x, uint64_t rows,
                         void* d_y, uint64_t ld_y, void* stream, char* err, size_t err_len) {
  if (!weight) return refuse(SVL_USAGE, "null argument", err, err_len);
  if (!svl::is_operand_dtype(dtype)) return refuse(SVL_USAGE, "unknown dtype", err, err_len);
  if (rows >= 1ull << 31) return refuse(SVL_USAGE, "2^31 rows or more", err, err_len);
  if (!rows) return SVL_OK;
  if (!d_x || !d_y) return refuse(SVL_USAGE, "null argument", err, err_len);
  const svl::Q4Matrix& m = weight->m;
  if (ld_x < m.k || ld_y < m.n) return refuse(SVL_USAGE, "a row stride is shorter than its row", err, err_len);
  if (std::max(ld_x, ld_y) >= 1ull << 36) return refuse(SVL_USAGE, "a row stride is 2^36 or more", err, err_len);
  if (((uintptr_t)d_x | (uintptr_t)d_y) & (svl::dtype_size(dtype) - 1))
    return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  svl::DeviceGuard on(weight->device);
  if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
  cudaStream_t st = (cudaStream_t)stream;
  const Rows r{d_x, ld_x, rows, d_y, ld_y};
  const cudaError_t e = dtype == SVL_DTYPE_F32    ? launch_linear<float>(m, r, st)
                        : dtype == SVL_DTYPE_BF16 ? launch_linear<__nv_bfloat16>(m, r, st)
                                                  : launch_linear<__half>(m, r, st);
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

}  // extern "C"
