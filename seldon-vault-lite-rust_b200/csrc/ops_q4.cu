// ops_q4.cu -- products of a few rows with a 4-bit weight matrix (svl_q4_* of
// include/svl_gpu.h): y[m, i] = sum_j x[m, j] (code[i, j] - zero[i, j / g])
// scale[i, j / g].
#include <algorithm>
#include <cmath>
#include <vector>

#include "ops_common.cuh"

namespace svl {
namespace {

constexpr uint32_t kErrNonFinite = 1;

struct Q4Matrix {
  const uint8_t* codes;   // [n][k / 2]
  const uint16_t* scales; // [n][k / group]
  const uint8_t* zeros;   // [n][k / group] or NULL
  uint32_t n, k, group, scale_dtype;
};

SVL_DEV float scale_of(uint16_t bits, uint32_t dtype) {
  return dtype == SVL_DTYPE_F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
}

// One warp per (output column, 4 rows of x).
template <typename T>
__global__ void q4_rows_kernel(const __grid_constant__ Q4Matrix w, const T* __restrict__ x, uint64_t ld_x,
                               uint64_t rows, T* __restrict__ y, uint64_t ld_y) {
  const int lane = threadIdx.x & 31;
  const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
  const uint64_t items = (uint64_t)w.n * ((rows + 3) / 4);
  for (uint64_t it = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += warps) {
    const uint64_t i = it % w.n, m0 = it / w.n * 4;
    const uint32_t groups = w.k / w.group;
    float acc[4] = {};
    for (uint32_t j = 2 * lane; j < w.k; j += 64) {
      const uint64_t g = i * groups + j / w.group;
      const uint8_t c = w.codes[i * (w.k / 2) + j / 2];
      const float s = scale_of(w.scales[g], w.scale_dtype), z = w.zeros ? (float)(w.zeros[g] & 15) : 8.0f;
      const float a = ((float)(c & 15) - z) * s, b = ((float)(c >> 4) - z) * s;
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (m0 + m < rows) {
          const T* row = x + (m0 + m) * ld_x;
          acc[m] = fmaf(widen(row[j]), a, fmaf(widen(row[j + 1]), b, acc[m]));
        }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float v = warp_sum(acc[m]);
      if (lane == 0 && m0 + m < rows) y[(m0 + m) * ld_y + i] = narrow<T>(v);
    }
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
  const size_t codes = (w->code_bytes() + 255) & ~(size_t)255, scales = (2 * w->group_count() + 255) & ~(size_t)255;
  const cudaError_t e = cudaMalloc(&w->block, codes + scales + (zeros ? w->group_count() : 0));
  if (e != cudaSuccess) {
    w->block = nullptr;
    return svl::cuda_failure(e, err, err_len);
  }
  uint8_t* p = (uint8_t*)w->block;
  w->m.codes = p;
  w->m.scales = (uint16_t*)(p + codes);
  w->m.zeros = zeros ? p + codes + scales : nullptr;
  return SVL_OK;
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
    cudaError_t e = cudaMemcpy((void*)w->m.codes, codes, w->code_bytes(), cudaMemcpyDefault);
    if (e == cudaSuccess) e = cudaMemcpy((void*)w->m.scales, scales, 2 * w->group_count(), cudaMemcpyDefault);
    if (e == cudaSuccess && zeros) e = cudaMemcpy((void*)w->m.zeros, zeros, w->group_count(), cudaMemcpyDefault);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
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
    svl::Freed in, flag;
    cudaError_t e = cudaMalloc(&in.p, bytes);
    if (e == cudaSuccess) e = cudaMalloc(&flag.p, 4);
    if (e == cudaSuccess) e = cudaMemcpy(in.p, weight->data, bytes, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaMemset(flag.p, 0, 4);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    const unsigned grid = (unsigned)std::min<size_t>((w->group_count() + 7) / 8, 148 * 8);
    if (weight->dtype == SVL_DTYPE_F32)
      svl::q4_quantize_kernel<float><<<grid, 256>>>((const float*)in.p, n, k, group, asymmetric != 0,
                                                    (uint8_t*)w->m.codes, (uint16_t*)w->m.scales,
                                                    (uint8_t*)w->m.zeros, (uint32_t*)flag.p);
    else
      svl::q4_quantize_kernel<__nv_bfloat16><<<grid, 256>>>((const __nv_bfloat16*)in.p, n, k, group, asymmetric != 0,
                                                            (uint8_t*)w->m.codes, (uint16_t*)w->m.scales,
                                                            (uint8_t*)w->m.zeros, (uint32_t*)flag.p);
    uint32_t word = 0;
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(&word, flag.p, 4, cudaMemcpyDeviceToHost);
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
  svl::DeviceGuard on(weight->device);
  cudaError_t e = on.status;
  if (e == cudaSuccess && codes) e = cudaMemcpy(codes, m.codes, weight->code_bytes(), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && scales) e = cudaMemcpy(scales, m.scales, 2 * weight->group_count(), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && zeros) {
    if (m.zeros)
      e = cudaMemcpy(zeros, m.zeros, weight->group_count(), cudaMemcpyDeviceToHost);
    else
      memset(zeros, 8, weight->group_count());
  }
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
  const unsigned grid = (unsigned)std::min<uint64_t>((m.n * ((rows + 3) / 4) + 7) / 8, 148 * 8);
  switch (dtype) {
    case SVL_DTYPE_F32:
      svl::q4_rows_kernel<float><<<grid, 256, 0, st>>>(m, (const float*)d_x, ld_x, rows, (float*)d_y, ld_y);
      break;
    case SVL_DTYPE_BF16:
      svl::q4_rows_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(m, (const __nv_bfloat16*)d_x, ld_x, rows,
                                                               (__nv_bfloat16*)d_y, ld_y);
      break;
    default:
      svl::q4_rows_kernel<__half><<<grid, 256, 0, st>>>(m, (const __half*)d_x, ld_x, rows, (__half*)d_y, ld_y);
      break;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

}  // extern "C"
