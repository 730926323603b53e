// ops_rope.cu -- rotary positions with several axes (svl_rope_* of
// include/svl_gpu.h).
//
// A pair (x, y) of axis a becomes (x cos - y sin, y cos + x sin) at the angle
// position * f.  The angle in turns, position * f / 2 pi, is needed modulo 1
// only, so f / 2 pi is kept as a 64-bit binary fraction of a turn and the
// product with an integer position wraps in 64-bit arithmetic: the reduction
// is exact for every int32 position (the fraction's own rounding, 2^-65 of a
// turn a position, reaches 2^-34 of a turn at 2^31), and FP32 sees an angle in
// [-1/2, 1/2) turns.
#include <cmath>

#include "ops_common.cuh"

#pragma nv_diag_suppress 20208  // long double: host code only

namespace svl {
namespace {

constexpr int kMaxPairs = SVL_ROPE_MAX_HEAD_DIM / 2;

// Passed by value: the tables travel in the launch's own parameters, so the
// handle owns no device memory and a captured launch keeps its copy.
struct RopeTables {
  uint64_t turn[kMaxPairs];  // frequency: fraction of a turn per position, times 2^64
  uint16_t first[kMaxPairs], second[kMaxPairs];
  uint8_t axis[kMaxPairs];
  uint32_t n_pairs, head_dim;
};

struct RopeTensor {
  const void* in;
  void* out;
  uint64_t ld_in, ld_out;
  uint32_t heads;
};

SVL_DEV float2 angle_of(int32_t position, uint64_t turn) {
  const uint64_t phase = (uint64_t)(int64_t)position * turn;
  const float half_turns = (float)(int32_t)(phase >> 32) * 0x1p-31f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c, s);
}

// One thread per (token, head, pair); the last threads of a head copy the
// dimensions behind the pairs.
template <typename T>
__global__ void rope_kernel(const __grid_constant__ RopeTables tab, const __grid_constant__ RopeTensor q,
                            const __grid_constant__ RopeTensor k, const int32_t* __restrict__ positions,
                            uint64_t n_tokens) {
  const uint32_t pass = tab.head_dim - 2 * tab.n_pairs, per_head = tab.n_pairs + pass;
  const uint64_t per_token = (uint64_t)(q.heads + k.heads) * per_head;
  for (uint64_t i = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; i < n_tokens * per_token;
       i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t t = i / per_token;
    const uint32_t r = (uint32_t)(i % per_token), p = r % per_head;
    uint32_t h = r / per_head;
    const bool is_k = h >= q.heads;
    h -= is_k ? q.heads : 0;
    const RopeTensor& x = is_k ? k : q;
    const T* in = (const T*)x.in + t * x.ld_in + (uint64_t)h * tab.head_dim;
    T* out = (T*)x.out + t * x.ld_out + (uint64_t)h * tab.head_dim;
    if (p >= tab.n_pairs) {
      out[p + tab.n_pairs] = in[p + tab.n_pairs];
      continue;
    }
    const float2 cs = angle_of(positions[tab.axis[p] * n_tokens + t], tab.turn[p]);
    const float a = widen(in[tab.first[p]]), b = widen(in[tab.second[p]]);
    out[tab.first[p]] = narrow<T>(a * cs.x - b * cs.y);
    out[tab.second[p]] = narrow<T>(b * cs.x + a * cs.y);
  }
}

}  // namespace
}  // namespace svl

struct svl_rope {
  svl::RopeTables tab;
  uint32_t n_axes;
};

using svl::refuse;

extern "C" {

int svl_rope_create(const svl_rope_config* config, svl_rope** out, char* err, size_t err_len) {
  if (!config || !out) return refuse(SVL_USAGE, "null argument", err, err_len);
  *out = nullptr;
  const svl_rope_config& c = *config;
  if (c.head_dim < 2 || c.head_dim > SVL_ROPE_MAX_HEAD_DIM)
    return refuse(SVL_USAGE, "head_dim is outside 2..=512", err, err_len);
  if (c.n_axes < 1 || c.n_axes > SVL_ROPE_MAX_AXES) return refuse(SVL_USAGE, "n_axes is outside 1..=4", err, err_len);
  if (c.arrangement > SVL_ROPE_INTERLEAVED) return refuse(SVL_USAGE, "unknown arrangement", err, err_len);
  if (c.reserved) return refuse(SVL_USAGE, "svl_rope_config.reserved must be zero", err, err_len);
  uint64_t n = 0;
  for (uint32_t a = 0; a < c.n_axes; ++a) {
    if (!c.pairs[a]) return refuse(SVL_USAGE, "every axis needs a pair", err, err_len);
    n += c.pairs[a];
    if ((a == 0 || c.arrangement == SVL_ROPE_SPLIT) && !(std::isfinite(c.theta[a]) && c.theta[a] > 0))
      return refuse(SVL_USAGE, "theta must be finite and positive", err, err_len);
  }
  if (2 * n > c.head_dim) return refuse(SVL_USAGE, "the axes' pairs do not fit the head", err, err_len);
  return svl::guarded(err, err_len, [&]() -> int {
    svl_rope* r = new svl_rope();
    svl::RopeTables& t = r->tab;
    r->n_axes = c.n_axes;
    t.n_pairs = (uint32_t)n;
    t.head_dim = c.head_dim;
    auto put = [&](uint32_t p, uint32_t axis, uint32_t first, uint32_t second, double theta, uint32_t i, uint32_t of) {
      // frequency / 2 pi, kept modulo 1 with 64 bits behind the point
      const long double f = powl((long double)theta, -(long double)i / of) / 6.283185307179586476925286766559L;
      const long double scaled = ldexpl(f - floorl(f), 64);
      t.turn[p] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
      t.axis[p] = (uint8_t)axis;
      t.first[p] = (uint16_t)first;
      t.second[p] = (uint16_t)second;
    };
    uint32_t p = 0;
    if (c.arrangement == SVL_ROPE_SPLIT) {
      for (uint32_t a = 0; a < c.n_axes; ++a) {
        const uint32_t start = 2 * p, na = c.pairs[a];
        for (uint32_t i = 0; i < na; ++i, ++p) put(p, a, start + i, start + i + na, c.theta[a], i, na);
      }
    } else if (c.arrangement == SVL_ROPE_SECTIONS) {
      for (uint32_t a = 0; a < c.n_axes; ++a)
        for (uint32_t i = 0; i < c.pairs[a]; ++i, ++p) put(p, a, p, p + (uint32_t)n, c.theta[0], p, (uint32_t)n);
    } else {
      for (uint32_t round = 0; p < n; ++round)
        for (uint32_t a = 0; a < c.n_axes; ++a)
          if (round < c.pairs[a]) {
            put(p, a, p, p + (uint32_t)n, c.theta[0], p, (uint32_t)n);
            ++p;
          }
    }
    *out = r;
    return SVL_OK;
  });
}

void svl_rope_destroy(svl_rope* rope) { delete rope; }

int svl_rope_apply_device(const svl_rope* rope, int device, uint32_t dtype, const int32_t* d_positions,
                          uint64_t n_tokens, const void* d_q, uint64_t ld_q, uint32_t q_heads, void* d_q_out,
                          uint64_t ld_q_out, const void* d_k, uint64_t ld_k, uint32_t k_heads, void* d_k_out,
                          uint64_t ld_k_out, void* stream, char* err, size_t err_len) {
  if (!rope) return refuse(SVL_USAGE, "null argument", err, err_len);
  if (!svl::is_operand_dtype(dtype)) return refuse(SVL_USAGE, "unknown dtype", err, err_len);
  if (n_tokens >= 1ull << 31) return refuse(SVL_USAGE, "n_tokens is 2^31 or more", err, err_len);
  const uint64_t hd = rope->tab.head_dim;
  const uintptr_t mask = svl::dtype_size(dtype) - 1;
  svl::RopeTensor q{d_q, d_q_out, ld_q, ld_q_out, q_heads}, k{d_k, d_k_out, ld_k, ld_k_out, k_heads};
  for (const svl::RopeTensor* x : {&q, &k}) {
    if (!x->heads || !n_tokens) continue;
    if (!x->in || !x->out || !d_positions) return refuse(SVL_USAGE, "null argument", err, err_len);
    if (x->heads > 65535) return refuse(SVL_USAGE, "more than 65535 heads", err, err_len);
    if (x->ld_in < x->heads * hd || x->ld_out < x->heads * hd)
      return refuse(SVL_USAGE, "a row stride is shorter than its heads", err, err_len);
    if (((uintptr_t)x->in | (uintptr_t)x->out) & mask) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
    if (x->in == x->out && x->ld_in != x->ld_out)
      return refuse(SVL_USAGE, "in place needs one row stride", err, err_len);
  }
  if (!n_tokens || (!q_heads && !k_heads)) return SVL_OK;
  svl::DeviceGuard on(device);
  if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
  const uint64_t work = n_tokens * (q_heads + k_heads) * (hd - rope->tab.n_pairs);
  const dim3 grid((unsigned)std::min<uint64_t>((work + 255) / 256, 148 * 8));
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case SVL_DTYPE_F32: svl::rope_kernel<float><<<grid, 256, 0, st>>>(rope->tab, q, k, d_positions, n_tokens); break;
    case SVL_DTYPE_BF16:
      svl::rope_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(rope->tab, q, k, d_positions, n_tokens);
      break;
    default: svl::rope_kernel<__half><<<grid, 256, 0, st>>>(rope->tab, q, k, d_positions, n_tokens); break;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

}  // extern "C"
