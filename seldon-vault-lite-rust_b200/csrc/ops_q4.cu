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
// is exact, and the parts are further columns of the product.
#include <algorithm>
#include <cmath>
#include <vector>

#include "ops_common.cuh"

namespace svl {
namespace {

constexpr uint32_t kErrNonFinite = 1;

SVL_DEV float scale_of(uint16_t bits, uint32_t dtype) {
  return dtype == SVL_DTYPE_F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
}

// The order of the product's columns inside a block of 64 is free as long as
// both operands have it.  Lane 4 g + q takes columns 8 q .. 8 q + 7 of each half
// block of 32 (the shortest group), four of them a step: steps 0 and 1 are the
// first half, 2 and 3 the second.  So its part of a 16-bit x row is two 16-byte
// loads and its codes of the block's 16 x 64 weights one: word w holds step w,
// for rows g and g + 8.  The two nibbles of an operand register lie 16 bits
// apart, where one mask takes both.
struct Q4Matrix {
  const uint4* codes;      // [row block of 16][column block of 64][lane]
  const uint32_t* scales;  // [row block][group][8]: rows g (low half) and g + 8
  const uint16_t* zeros;   // the same, a byte each; NULL: 8
  uint32_t n, k, group, scale_dtype;
  __host__ __device__ uint32_t row_blocks() const { return (n + 15) / 16; }
  __host__ __device__ uint32_t col_blocks() const { return (k + 63) / 64; }
  __host__ __device__ uint32_t groups() const { return k / group; }
};

// Nibble of a word that holds row g + 8 upper and the step's column c = 0..3:
// register upper + 2 (c / 2) of the operand, half c % 2.
SVL_DEV uint32_t nibble_at(uint32_t upper, uint32_t c) { return upper + 2 * (c >> 1) + 4 * (c & 1); }

// Plain codes, scales and zeros into the handle's order; rows and columns
// behind the matrix get code 0 and scale 0.
__global__ void q4_lay_out_kernel(const __grid_constant__ Q4Matrix m, const uint8_t* __restrict__ codes,
                                  const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros) {
  const uint64_t words = (uint64_t)m.row_blocks() * m.col_blocks() * 128, step = (uint64_t)gridDim.x * blockDim.x;
  const uint64_t first = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  for (uint64_t i = first; i < words; i += step) {
    const uint32_t w = i & 3, lane = (i >> 2) & 31;
    const uint64_t block = i >> 7;
    const uint64_t row = block / m.col_blocks() * 16 + (lane >> 2);
    const uint64_t col = block % m.col_blocks() * 64 + (w >> 1) * 32 + (lane & 3) * 8 + 4 * (w & 1);
    uint32_t word = 0;
    for (uint32_t upper = 0; upper < 2; ++upper)
      if (row + 8 * upper < m.n && col < m.k) {
        const uint8_t* src = codes + (row + 8 * upper) * (m.k / 2) + col / 2;
        for (uint32_t c = 0; c < 4; ++c)
          word |= (uint32_t)(src[c >> 1] >> (4 * (c & 1)) & 15) << (4 * nibble_at(upper, c));
      }
    ((uint32_t*)m.codes)[i] = word;
  }
  const uint64_t pairs = (uint64_t)m.row_blocks() * m.groups() * 8;
  for (uint64_t i = first; i < pairs; i += step) {
    const uint64_t row = i / 8 / m.groups() * 16 + (i & 7), g = i / 8 % m.groups();
    uint32_t s = 0, z = 0;
    for (uint32_t upper = 0; upper < 2; ++upper)
      if (row + 8 * upper < m.n) {
        const uint64_t at = (row + 8 * upper) * m.groups() + g;
        s |= (uint32_t)scales[at] << (16 * upper);
        if (zeros) z |= (uint32_t)(zeros[at] & 15) << (8 * upper);
      }
    ((uint32_t*)m.scales)[i] = s;
    if (zeros) ((uint16_t*)m.zeros)[i] = (uint16_t)z;
  }
}

// The reverse.
__global__ void q4_read_kernel(const __grid_constant__ Q4Matrix m, uint8_t* __restrict__ codes,
                               uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const uint64_t step = (uint64_t)gridDim.x * blockDim.x, first = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x;
  for (uint64_t i = first; codes && i < (uint64_t)m.n * (m.k / 2); i += step) {
    const uint64_t row = i / (m.k / 2), col = i % (m.k / 2) * 2;
    const uint64_t block = row / 16 * m.col_blocks() + col / 64;
    const uint32_t lane = (row & 7) * 4 + (col & 31) / 8, w = (col & 63) / 32 * 2 + (col & 7) / 4, upper = row >> 3 & 1;
    const uint32_t word = ((const uint32_t*)m.codes)[block * 128 + lane * 4 + w];
    codes[i] = (uint8_t)((word >> (4 * nibble_at(upper, col & 3)) & 15) | (word >> (4 * nibble_at(upper, (col & 3) + 1)) & 15) << 4);
  }
  for (uint64_t i = first; i < (uint64_t)m.n * m.groups(); i += step) {
    const uint64_t row = i / m.groups(), at = (row / 16 * m.groups() + i % m.groups()) * 8 + (row & 7);
    const uint32_t upper = row >> 3 & 1;
    if (scales) scales[i] = (uint16_t)(m.scales[at] >> (16 * upper));
    if (zeros) zeros[i] = m.zeros ? (uint8_t)(m.zeros[at] >> (8 * upper)) : 8;
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
// BF16 0x4300 | q; the zero comes with the same offset and both differences are
// exact.
SVL_DEV uint32_t offset_bits(__half) { return 0x64006400u; }
SVL_DEV uint32_t offset_bits(__nv_bfloat16) { return 0x43004300u; }
SVL_DEV uint32_t minus(__half, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
SVL_DEV uint32_t minus(__nv_bfloat16, uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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
template <typename T, bool WIDE>
SVL_DEV void load_columns(const T* row, int part, uint32_t* b) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (WIDE) {
      const uint4 v = *(const uint4*)row;
      b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
    } else {
      const uint16_t* v = (const uint16_t*)row;
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = (uint32_t)v[2 * i] | (uint32_t)v[2 * i + 1] << 16;
    }
  } else {
    float x[8];
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 v = *(const float4*)((const float*)row + 4 * i);
        x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = row[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = bf16_part(x[2 * i], part) >> 16 | bf16_part(x[2 * i + 1], part);
  }
}

constexpr int kWarps = 8;

// One block: 16 R weight rows against 8 NT columns (rows of x, or parts of
// them); its warps take the column blocks in turn and join their sums in shared
// memory, in a fixed order.  SHORT: groups of 32 (two a block of 64).
template <typename T, int NT, int R, bool SHORT, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32)
    q4_linear_kernel(const __grid_constant__ Q4Matrix w, const T* __restrict__ x, uint64_t ld_x, uint64_t rows,
                     T* __restrict__ y, uint64_t ld_y) {
  using Op = typename Operand<T>::Type;
  constexpr int kParts = Operand<T>::kParts, kCols = NT * 8, kRows = kCols / kParts;
  constexpr int kDeep = NT == 1 ? 4 : 2;  // column blocks in flight
  extern __shared__ float sums[];         // [warp][16 R][kCols]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const uint32_t col_blocks = w.col_blocks(), groups = w.groups(), row_blocks = w.row_blocks();
  const uint32_t rb0 = blockIdx.x * R;
  const uint64_t m0 = (uint64_t)blockIdx.y * kRows;
  float acc[R][NT][4] = {};

  for (uint32_t kb0 = warp; kb0 < col_blocks; kb0 += kWarps * kDeep) {
    uint4 code[kDeep][R];
    uint32_t scale[kDeep][R][SHORT ? 2 : 1], zero[kDeep][R][SHORT ? 2 : 1];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t kb = kb0 + d * kWarps, rb = rb0 + r;
        const bool in = kb < col_blocks && rb < row_blocks;
        code[d][r] = in ? __ldcs(w.codes + ((uint64_t)rb * col_blocks + kb) * 32 + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < (SHORT ? 2 : 1); ++h) {
          const uint32_t gr = SHORT ? 2 * kb + h : kb * 64 / w.group;
          const bool there = in && gr < groups;
          const uint64_t at = ((uint64_t)rb * groups + gr) * 8 + g;
          scale[d][r][h] = there ? __ldcs(w.scales + at) : 0;
          zero[d][r][h] = w.zeros ? (there ? __ldcs(w.zeros + at) : 0) : 0x0808;
        }
      }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const uint32_t kb = kb0 + d * kWarps;
      if (kb >= col_blocks) break;
      uint32_t a[R][4][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t word[4] = {code[d][r].x, code[d][r].y, code[d][r].z, code[d][r].w};
        const uint32_t base = offset_bits(Op());
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t z = zero[d][r][SHORT ? s >> 1 : 0];
          const uint32_t z0 = base + (z & 15) * 0x10001u, z1 = base + (z >> 8 & 15) * 0x10001u;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[r][s][i] = minus(Op(), (word[s] >> (4 * i) & 0x000f000fu) | base, i & 1 ? z1 : z0);
        }
      }
      const uint32_t col = kb * 64 + q * 8;
      const bool second = kb * 64 + 32 < w.k;  // k is a multiple of 32
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int c = t * 8 + g;
        const uint64_t m = m0 + c / kParts;
        uint32_t b[8] = {};
        if (m < rows && c / kParts < kRows) {
          const T* row = x + m * ld_x + col;
          load_columns<T, WIDE>(row, c % kParts, b);
          if (second) load_columns<T, WIDE>(row + 32, c % kParts, b + 4);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int h = 0; h < (SHORT ? 2 : 1); ++h) {
            float part[4] = {};
#pragma unroll
            for (int s = SHORT ? 2 * h : 0; s < (SHORT ? 2 * h + 2 : 4); ++s) mma_16816(Op(), part, a[r][s], b + 2 * s);
            const float s0 = scale_of((uint16_t)scale[d][r][h], w.scale_dtype);
            const float s1 = scale_of((uint16_t)(scale[d][r][h] >> 16), w.scale_dtype);
            acc[r][t][0] = fmaf(part[0], s0, acc[r][t][0]);
            acc[r][t][1] = fmaf(part[1], s0, acc[r][t][1]);
            acc[r][t][2] = fmaf(part[2], s1, acc[r][t][2]);
            acc[r][t][3] = fmaf(part[3], s1, acc[r][t][3]);
          }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* to = sums + ((warp * R + r) * 16 + g) * kCols + t * 8 + 2 * q;
      *(float2*)to = make_float2(acc[r][t][0], acc[r][t][1]);
      *(float2*)(to + 8 * kCols) = make_float2(acc[r][t][2], acc[r][t][3]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * R * kRows; i += kWarps * 32) {
    const int row = i % (16 * R), c = i / (16 * R);
    const uint64_t n = (uint64_t)rb0 * 16 + row, m = m0 + c;
    if (n >= w.n || m >= rows) continue;
    float sum = 0.0f;
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part)  // the smallest first
#pragma unroll
      for (int v = 0; v < kWarps; ++v) sum += sums[(v * R * 16 + row) * kCols + c * kParts + part];
    y[m * ld_y + n] = narrow<T>(sum);
  }
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
  ~svl_q4() {
    if (!block) return;
    svl::DeviceGuard on(device);
    cudaFree(block);
  }
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
  const size_t codes = rb * w->m.col_blocks() * 512, pairs = rb * w->m.groups() * 8;
  const cudaError_t e = cudaMalloc(&w->block, codes + pairs * 4 + (zeros ? pairs * 2 : 0));
  if (e != cudaSuccess) {
    w->block = nullptr;
    return svl::cuda_failure(e, err, err_len);
  }
  uint8_t* p = (uint8_t*)w->block;
  w->m.codes = (const uint4*)p;
  w->m.scales = (const uint32_t*)(p + codes);
  w->m.zeros = zeros ? (const uint16_t*)(p + codes + pairs * 4) : nullptr;
  return SVL_OK;
}

// Device memory for `bytes`, or `src` itself where it is this device's already.
cudaError_t on_device(const void* src, size_t bytes, int device, svl::Freed& held, const void** out) {
  cudaPointerAttributes at{};
  if (cudaPointerGetAttributes(&at, src) == cudaSuccess && at.type == cudaMemoryTypeDevice && at.device == device) {
    *out = src;
    return cudaSuccess;
  }
  cudaGetLastError();
  cudaError_t e = cudaMalloc(&held.p, bytes);
  if (e == cudaSuccess) e = cudaMemcpy(held.p, src, bytes, cudaMemcpyDefault);
  *out = held.p;
  return e;
}

cudaError_t lay_out(const svl_q4& w, const void* codes, const void* scales, const void* zeros) {
  const uint64_t words = (uint64_t)w.m.row_blocks() * w.m.col_blocks() * 128;
  svl::q4_lay_out_kernel<<<(unsigned)std::min<uint64_t>((words + 255) / 256, 148 * 8), 256>>>(
      w.m, (const uint8_t*)codes, (const uint16_t*)scales, (const uint8_t*)zeros);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? cudaStreamSynchronize(nullptr) : e;
}

template <typename T, int NT, int R, bool SHORT, bool WIDE>
cudaError_t launch_rows(const svl::Q4Matrix& m, const void* x, uint64_t ld_x, uint64_t rows, void* y, uint64_t ld_y,
                        cudaStream_t st) {
  constexpr uint32_t kRows = NT * 8 / svl::Operand<T>::kParts;
  constexpr int smem = svl::kWarps * R * 16 * NT * 8 * 4;
  static std::atomic<uint64_t> done{0};
  auto kernel = svl::q4_linear_kernel<T, NT, R, SHORT, WIDE>;
  if (smem > 48 * 1024) {
    const cudaError_t e = smem_opt_in(kernel, smem, &done);
    if (e != cudaSuccess) return e;
  }
  // a grid's second dimension ends at 65535
  for (uint64_t m0 = 0; m0 < rows; m0 += 65535ull * kRows) {
    const uint64_t now = std::min<uint64_t>(rows - m0, 65535ull * kRows);
    const dim3 grid((m.row_blocks() + R - 1) / R, (unsigned)((now + kRows - 1) / kRows));
    kernel<<<grid, svl::kWarps * 32, smem, st>>>(m, (const T*)x + m0 * ld_x, ld_x, now, (T*)y + m0 * ld_y, ld_y);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, bool SHORT, bool WIDE>
cudaError_t launch_linear(const svl::Q4Matrix& m, const void* x, uint64_t ld_x, uint64_t rows, void* y, uint64_t ld_y,
                          cudaStream_t st) {
  const uint64_t cols = rows * svl::Operand<T>::kParts;
  if (cols <= 8) return launch_rows<T, 1, 1, SHORT, WIDE>(m, x, ld_x, rows, y, ld_y, st);
  if (cols <= 16) return launch_rows<T, 2, 1, SHORT, WIDE>(m, x, ld_x, rows, y, ld_y, st);
  if (cols <= 32) return launch_rows<T, 4, 1, SHORT, WIDE>(m, x, ld_x, rows, y, ld_y, st);
  return launch_rows<T, 8, 2, SHORT, WIDE>(m, x, ld_x, rows, y, ld_y, st);
}

template <typename T>
cudaError_t launch_linear(const svl::Q4Matrix& m, const void* x, uint64_t ld_x, uint64_t rows, void* y, uint64_t ld_y,
                          cudaStream_t st) {
  const bool wide = ((uintptr_t)x | ld_x * sizeof(T)) % 16 == 0;
  if (m.group == 32)
    return wide ? launch_linear<T, true, true>(m, x, ld_x, rows, y, ld_y, st)
                : launch_linear<T, true, false>(m, x, ld_x, rows, y, ld_y, st);
  return wide ? launch_linear<T, false, true>(m, x, ld_x, rows, y, ld_y, st)
              : launch_linear<T, false, false>(m, x, ld_x, rows, y, ld_y, st);
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
  if (((uintptr_t)d_x | (uintptr_t)d_y) & (svl::dtype_size(dtype) - 1))
    return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  svl::DeviceGuard on(weight->device);
  if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == SVL_DTYPE_F32    ? launch_linear<float>(m, d_x, ld_x, rows, d_y, ld_y, st)
                        : dtype == SVL_DTYPE_BF16 ? launch_linear<__nv_bfloat16>(m, d_x, ld_x, rows, d_y, ld_y, st)
                                                  : launch_linear<__half>(m, d_x, ld_x, rows, d_y, ld_y, st);
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

}  // extern "C"
