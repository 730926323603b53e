// ops_rope.cu -- rotary positions with several axes (svl_rope_* of
// include/svl_gpu.h).
//
// A pair (x, y) of axis a becomes (x cos - y sin, y cos + x sin) at the angle
// position * f.  The angle in turns, position * f / 2 pi, is needed modulo 1
// only, so f / 2 pi is kept as a 64-bit binary fraction of a turn and the
// product with an integer position wraps in 64-bit arithmetic: the reduction
// is exact for the stored fraction at every int32 position.  The fraction is cut
// at 2^-64 of a turn, which reaches 2^-33 at 2^31; f / 2 pi itself is computed
// with 64 significant bits, so where f exceeds a turn (bases below 1) its error
// is 2^-63 f / 2 pi a position: under 2^-27 of a turn at 2^31 for kLeastTheta,
// whose largest frequency is 20.4 turns.  sine and cosine see the phase cut at
// 2^-32 of a turn and rounded to FP32 in [-1/2, 1/2] turns, at most 2^-26 off.
#include <cmath>

#include "ops_common.cuh"

#pragma nv_diag_suppress 20208  // long double: host code only

namespace svl {
namespace {

constexpr int kMaxPairs = SVL_ROPE_MAX_HEAD_DIM / 2;
constexpr double kLeastTheta = 1.0 / 128;

// Passed by value: the tables travel in the launch's own parameters, so the
// handle owns no device memory and a captured launch keeps its copy.
struct RopeTables {
  uint64_t turn[kMaxPairs];  // frequency: fraction of a turn per position, times 2^64
  uint8_t axis[kMaxPairs];
  // Runs of pairs that lie next to each other: pair p of run r is (first[r] +
  // p - start[r], second[r] + p - start[r]).
  uint32_t start[SVL_ROPE_MAX_AXES], first[SVL_ROPE_MAX_AXES], second[SVL_ROPE_MAX_AXES];
  uint32_t n_runs, n_pairs, head_dim;
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

// Bytes of the tables in shared memory.
__host__ __device__ inline uint32_t rope_tables_bytes(uint32_t n) { return (n * 9 + 15) / 16 * 16; }

// V values in one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// A block takes `per_block` tokens: their cosines and sines go into shared
// memory once, for all heads; then its threads walk the (token, head)s in memory
// order, V pairs a thread.  Bound by reading and writing the rows once.  (A
// thread that keeps the angles of one token and turns them in several heads saves
// the shared memory, but spreads the block's accesses over that many rows at a
// time: 173 against 130 us for 65536 BF16 rows of 20 heads of 128, 5.1-5.2 TB/s.)  The last vectors
// of a head copy the dimensions behind the pairs.
template <typename T, int V>
__global__ void __launch_bounds__(512)
    rope_kernel(const __grid_constant__ RopeTables tab, const __grid_constant__ RopeTensor q,
                const __grid_constant__ RopeTensor k, const int32_t* __restrict__ positions, const uint32_t n_tokens,
                const uint32_t per_block) {
  using P = Pack<T, V>;
  constexpr int kQuads = V >= 4 ? V / 4 : 1, kWide = V >= 4 ? 4 : V;  // values of an access of the angles
  using A = Pack<float, kWide>;
  extern __shared__ __align__(16) uint8_t shared[];
  const uint32_t n = tab.n_pairs, pair_vectors = (n + V - 1) / V;
  uint64_t* turn = (uint64_t*)shared;
  uint8_t* axis = (uint8_t*)(turn + n);
  // [token][cosine, sine][quad][vector]: neighbouring vectors are neighbours in each access
  A* angles = (A*)(shared + rope_tables_bytes(n));
  // Lanes that index the launch's parameters apart from each other are served
  // one by one, so a warp copies one entry after another first.
  for (uint32_t i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5)
    if ((threadIdx.x & 31) == 0) {
      turn[i] = tab.turn[i];
      axis[i] = tab.axis[i];
    }
  __syncthreads();
  const uint32_t t0 = blockIdx.x * per_block, tokens = min(per_block, n_tokens - t0);
  for (uint32_t i = threadIdx.x; i < tokens * n; i += blockDim.x) {
    const uint32_t t = i / n, p = i - t * n;
    const float2 cs = angle_of(positions[(uint64_t)axis[p] * n_tokens + t0 + t], turn[p]);
    A* at = angles + (2 * t * kQuads + p % V / kWide) * pair_vectors + p / V;
    at->v[p % kWide] = cs.x;
    at[kQuads * pair_vectors].v[p % kWide] = cs.y;
  }
  __syncthreads();
  const uint32_t vectors = (tab.head_dim - n) / V, lanes = blockDim.x / vectors;  // (token, head)s at a time
  const uint32_t v = threadIdx.x % vectors;
  if (threadIdx.x >= lanes * vectors) return;
  const bool turns = v * V < n;
  uint32_t first = n + v * V, second = 0;  // behind the pairs: dimension 2 n + ..
  if (turns) {
    uint32_t r = 0;
    while (r + 1 < tab.n_runs && v * V >= tab.start[r + 1]) ++r;
    first = tab.first[r] + v * V - tab.start[r];
    second = tab.second[r] + v * V - tab.start[r];
  }
  const uint32_t heads = q.heads + k.heads;
  uint32_t t = 0, h = threadIdx.x / vectors;
  while (true) {
    while (h >= heads) {
      h -= heads;
      ++t;
    }
    if (t >= tokens) break;
    const bool is_k = h >= q.heads;
    const RopeTensor& x = is_k ? k : q;
    const uint64_t at = (uint64_t)(h - (is_k ? q.heads : 0)) * tab.head_dim;
    const T* in = (const T*)x.in + (t0 + t) * x.ld_in + at;
    T* out = (T*)x.out + (t0 + t) * x.ld_out + at;
    P a = *(const P*)(in + first);
    if (turns) {
      P b = *(const P*)(in + second);
      const A* cs = angles + 2 * t * kQuads * pair_vectors + v;
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const A c = cs[u * pair_vectors], s = cs[(kQuads + u) * pair_vectors];
#pragma unroll
        for (int e = 0; e < kWide; ++e) {
          const float x0 = widen(a.v[u * kWide + e]), y0 = widen(b.v[u * kWide + e]);
          a.v[u * kWide + e] = narrow<T>(x0 * c.v[e] - y0 * s.v[e]);
          b.v[u * kWide + e] = narrow<T>(y0 * c.v[e] + x0 * s.v[e]);
        }
      }
      *(P*)(out + second) = b;
    }
    *(P*)(out + first) = a;
    h += lanes;
  }
}

template <typename T, int V>
cudaError_t launch_rope(const RopeTables& tab, const RopeTensor& q, const RopeTensor& k, const int32_t* positions,
                        uint32_t n_tokens, cudaStream_t st) {
  const uint32_t n = tab.n_pairs, vectors = (tab.head_dim - n) / V, heads = q.heads + k.heads;
  // whole heads of vectors (at most 511); about kTurns (token, head)s a thread,
  // the angles in 24 KB, and for few tokens a block each
  constexpr uint32_t kTurns = 12;
  const uint32_t threads = std::max(vectors, 256 / vectors * vectors);
  uint32_t per_block = std::max(1u, std::min(kTurns * (threads / vectors) / heads, 24u * 1024 / (8 * n)));
  per_block = std::min(per_block, std::max(1u, n_tokens / (148 * 2)));
  rope_kernel<T, V><<<(n_tokens + per_block - 1) / per_block, threads,
                      rope_tables_bytes(n) + (size_t)per_block * ((n + V - 1) / V * V) * 8, st>>>(tab, q, k, positions,
                                                                                                 n_tokens, per_block);
  return cudaGetLastError();
}

// The widest vector that divides every offset, stride and address.
template <typename T>
cudaError_t launch_rope(const RopeTables& tab, const RopeTensor& q, const RopeTensor& k, const int32_t* positions,
                        uint32_t n_tokens, cudaStream_t st) {
  uint64_t all = tab.head_dim | tab.n_pairs;
  for (uint32_t r = 0; r < tab.n_runs; ++r) all |= tab.start[r] | tab.first[r] | tab.second[r];
  for (const RopeTensor* x : {&q, &k})
    if (x->heads) all |= x->ld_in | x->ld_out | (uintptr_t)x->in / sizeof(T) | (uintptr_t)x->out / sizeof(T);
  if constexpr (sizeof(T) == 2)
    if (all % 8 == 0) return launch_rope<T, 8>(tab, q, k, positions, n_tokens, st);
  if (all % 4 == 0) return launch_rope<T, 4>(tab, q, k, positions, n_tokens, st);
  if (all % 2 == 0) return launch_rope<T, 2>(tab, q, k, positions, n_tokens, st);
  return launch_rope<T, 1>(tab, q, k, positions, n_tokens, st);
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
    if ((a == 0 || c.arrangement == SVL_ROPE_SPLIT) && !(std::isfinite(c.theta[a]) && c.theta[a] >= svl::kLeastTheta))
      return refuse(SVL_USAGE, "theta must be finite and at least 1/128", err, err_len);
  }
  if (2 * n > c.head_dim) return refuse(SVL_USAGE, "the axes' pairs do not fit the head", err, err_len);
  return svl::guarded(err, err_len, [&]() -> int {
    svl_rope* r = new svl_rope();
    svl::RopeTables& t = r->tab;
    r->n_axes = c.n_axes;
    t.n_pairs = (uint32_t)n;
    t.head_dim = c.head_dim;
    auto put = [&](uint32_t p, uint32_t axis, double theta, uint32_t i, uint32_t of) {
      // frequency / 2 pi, kept modulo 1 with 64 bits behind the point
      const long double f = powl((long double)theta, -(long double)i / of) / 6.283185307179586476925286766559L;
      const long double scaled = ldexpl(f - floorl(f), 64);
      t.turn[p] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
      t.axis[p] = (uint8_t)axis;
    };
    uint32_t p = 0;
    if (c.arrangement == SVL_ROPE_SPLIT) {
      t.n_runs = c.n_axes;
      for (uint32_t a = 0; a < c.n_axes; ++a) {
        t.start[a] = p;
        t.first[a] = 2 * p;
        t.second[a] = 2 * p + c.pairs[a];
        for (uint32_t i = 0; i < c.pairs[a]; ++i, ++p) put(p, a, c.theta[a], i, c.pairs[a]);
      }
    } else {
      t.n_runs = 1;
      t.second[0] = (uint32_t)n;
      if (c.arrangement == SVL_ROPE_SECTIONS) {
        for (uint32_t a = 0; a < c.n_axes; ++a)
          for (uint32_t i = 0; i < c.pairs[a]; ++i, ++p) put(p, a, c.theta[0], p, (uint32_t)n);
      } else {
        for (uint32_t round = 0; p < n; ++round)
          for (uint32_t a = 0; a < c.n_axes; ++a)
            if (round < c.pairs[a]) {
              put(p, a, c.theta[0], p, (uint32_t)n);
              ++p;
            }
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
    if (std::max(x->ld_in, x->ld_out) >= 1ull << 36) return refuse(SVL_USAGE, "a row stride is 2^36 or more", err, err_len);
    if (((uintptr_t)x->in | (uintptr_t)x->out) & mask) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
    if (x->in == x->out && x->ld_in != x->ld_out)
      return refuse(SVL_USAGE, "in place needs one row stride", err, err_len);
    if ((uintptr_t)d_positions & 3) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  }
  if (!n_tokens || (!q_heads && !k_heads)) return SVL_OK;
  svl::DeviceGuard on(device);
  if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
  cudaStream_t st = (cudaStream_t)stream;
  const uint32_t n = (uint32_t)n_tokens;
  const cudaError_t e = dtype == SVL_DTYPE_F32    ? svl::launch_rope<float>(rope->tab, q, k, d_positions, n, st)
                        : dtype == SVL_DTYPE_BF16 ? svl::launch_rope<__nv_bfloat16>(rope->tab, q, k, d_positions, n, st)
                                                  : svl::launch_rope<__half>(rope->tab, q, k, d_positions, n, st);
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

}  // extern "C"
