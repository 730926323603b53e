// ops_attention.cu -- attention with capped scores, a distance bias, document,
// prefix, order and window masks (svl_attention_* of include/svl_gpu.h): the
// plan, the kernel for every type and head size, and the join of cut key axes.
#include <cmath>
#include <climits>
#include <vector>

#include "ops_attention_mma.cuh"

namespace svl {
namespace {

// ------------------------------------------------------ the general kernel --
//
// One pass over the keys with the running maximum and sum of each row's
// softmax, in FP32 throughout.  A block takes 32 rows, or 8 where 32 would leave
// SMs without a block (one 32-token query of 4 heads of 256: 22 us with 4 blocks,
// 10.8 us with 16).
constexpr int kGenRows = 32, kGenFewRows = 8, kGenKeys = 32, kGenThreads = 256;

// Row stride of the staged operands in floats: a multiple of 4 whose quarter
// is odd, so that eight rows' 16-byte reads touch all banks once.
__host__ __device__ inline uint32_t gen_stride(uint32_t head_dim) {
  const uint32_t quarters = (head_dim + 3) / 4;
  return 4 * (quarters | 1);
}
inline size_t gen_smem(uint32_t head_dim, int rows) {
  return (size_t)(rows + 2 * kGenKeys) * gen_stride(head_dim) * 4 + rows * (kGenKeys + 4) * 4 + 3 * rows * 4 + kGenKeys * 4;
}

// A warp's copy of one operand row into shared memory as FP32, zero behind the
// head and for rows that are not there.  `wide`: FP32 rows of 16-byte units.
template <typename T>
SVL_DEV void gen_row(float* to, const T* from, uint32_t hd, uint32_t stride, bool there, bool wide, int lane) {
  if (wide) {
#pragma unroll
    for (uint32_t u = 0; u < kAttnMaxHead / 128; ++u) {
      const uint32_t d = 128 * u + 4 * lane;
      if (d >= stride) break;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (there && d < hd) x = *(const float4*)(from + d);
      *(float4*)(to + d) = x;
    }
  } else {
    for (uint32_t d = lane; d < stride; d += 32) to[d] = there && d < hd ? widen(from[d]) : 0.0f;
  }
}

template <typename T, int ROWS>
__global__ void __launch_bounds__(kGenThreads, 2) attention_general_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ float sm[];
  const uint32_t hd = p.head_dim, stride = gen_stride(hd);
  float* sq = sm;
  float* sk = sq + ROWS * stride;
  float* sv = sk + kGenKeys * stride;
  float* sp = sv + kGenKeys * stride;        // scores, then weights; masked: -1
  float* s_max = sp + ROWS * (kGenKeys + 4);
  float* s_sum = s_max + ROWS;
  float* s_old = s_sum + ROWS;           // what the row's earlier sums are worth now
  int32_t* s_doc = (int32_t*)(s_old + ROWS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* gq = (const T*)p.q;
  const T* gk = (const T*)p.k;
  const T* gv = (const T*)p.v;
  const bool wide = sizeof(T) == 4 && ((p.ld_q | p.ld_k | p.ld_v | hd) % 4 == 0) &&
                    ((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0;

  for (uint32_t is = p.block_segments[blockIdx.x]; is < p.block_segments[blockIdx.x + 1]; ++is) {
    const AttnSegment seg = p.segments[is];
    const AttnSeq s = p.seqs[seg.seq];
    __syncthreads();
#pragma unroll
    for (int r = warp; r < ROWS; r += kGenThreads / 32) {
      const uint32_t row = seg.row0 + r;
      gen_row(sq + r * stride, gq + (s.q0 + row / p.group) * p.ld_q + (uint64_t)(seg.kvh * p.group + row % p.group) * hd, hd,
              stride, r < (int)seg.rows, wide, lane);
    }
    if (tid < ROWS) {
      s_max[tid] = -INFINITY;
      s_sum[tid] = 0.0f;
    }
    // this thread's scores: rows M ty .. x keys tx, tx + 32 / M
    constexpr int M = ROWS == 32 ? 2 : 1, kSpan = kGenKeys / M, kOwn = ROWS / 8;
    const int ty = tid / kSpan, tx = tid % kSpan;
    RowMask mask[M];
    float slope[M];
#pragma unroll
    for (int a = 0; a < M; ++a) {
      const uint32_t row = seg.row0 + min(M * ty + a, (int)seg.rows - 1);
      mask[a] = row_mask(p, s, row / p.group);
      slope[a] = p.slopes ? p.slopes[seg.kvh * p.group + row % p.group] : 0.0f;
    }
    // this thread's output: kOwn rows from kOwn warp on, columns 128 c + 4 lane ..
    float acc[kOwn][4][4] = {};

    for (uint32_t il = seg.list0; il < seg.list1; ++il) {
      const uint32_t entry = p.lists[il];
      const bool some = entry_sees(entry, 0) != kSeesAll;
      for (uint32_t sub = 0; sub < kKeyTile; sub += kGenKeys) {
        const uint32_t j0 = entry_tile(entry) * kKeyTile + sub;
        if (j0 >= s.n_k) break;
        __syncthreads();
#pragma unroll
        for (int j = warp; j < kGenKeys; j += kGenThreads / 32) {
          const uint64_t row = s.k0 + j0 + j, col = (uint64_t)seg.kvh * hd;
          const bool there = j0 + j < s.n_k;
          gen_row(sk + j * stride, gk + row * p.ld_k + col, hd, stride, there, wide, lane);
          gen_row(sv + j * stride, gv + row * p.ld_v + col, hd, stride, there, wide, lane);
        }
        if (tid < kGenKeys) s_doc[tid] = p.doc_k && j0 + tid < s.n_k ? p.doc_k[s.k0 + j0 + tid] : 0;
        __syncthreads();
        // four sums of every fourth dimension over 64 dimensions at a time: a rounding
        // is of a sum of 16 products, not of the whole head
        float dot[M][M] = {};
        for (uint32_t d0 = 0; d0 < hd; d0 += 64) {
          float4 part[M][M] = {};
          const uint32_t d1 = min(d0 + 64, hd);
#pragma unroll 4
          for (uint32_t d = d0; d < d1; d += 4) {  // the strides' padding is zero
            float4 a[M], b[M];
#pragma unroll
            for (int u = 0; u < M; ++u) {
              a[u] = *(const float4*)(sq + (M * ty + u) * stride + d);
              b[u] = *(const float4*)(sk + (tx + kSpan * u) * stride + d);
            }
#pragma unroll
            for (int u = 0; u < M; ++u)
#pragma unroll
              for (int w = 0; w < M; ++w) {
                part[u][w].x = fmaf(a[u].x, b[w].x, part[u][w].x);
                part[u][w].y = fmaf(a[u].y, b[w].y, part[u][w].y);
                part[u][w].z = fmaf(a[u].z, b[w].z, part[u][w].z);
                part[u][w].w = fmaf(a[u].w, b[w].w, part[u][w].w);
              }
          }
#pragma unroll
          for (int u = 0; u < M; ++u)
#pragma unroll
            for (int w = 0; w < M; ++w) dot[u][w] += (part[u][w].x + part[u][w].y) + (part[u][w].z + part[u][w].w);
        }
#pragma unroll
        for (int u = 0; u < M; ++u)
#pragma unroll
          for (int w = 0; w < M; ++w) {
            const uint32_t j = j0 + tx + kSpan * w;
            float t = dot[u][w] * p.scale;
            if (p.cap > 0.0f) t = p.cap * tanhf(t / p.cap);
            if (p.slopes) t -= slope[u] * fabsf((float)(mask[u].place - (int64_t)j));
            // a NaN score is a visible key's own: it has to survive the maximum
            if (some && !sees(p, mask[u], j, s_doc[tx + kSpan * w])) t = -INFINITY;
            sp[(M * ty + u) * (kGenKeys + 4) + tx + kSpan * w] = t;
          }
        __syncthreads();
        for (int r = kOwn * warp; r < kOwn * warp + kOwn; ++r) {
          const float t = sp[r * (kGenKeys + 4) + lane];
          const float before = s_max[r], m = fmaxf(before, warp_max(t));
          // rows that have seen nothing keep -inf, and their weights are 0
          const float base = m == -INFINITY ? 0.0f : m;
          const float w = expf(t - base);
          const float sum = warp_sum(w);
          __syncwarp();
          sp[r * (kGenKeys + 4) + lane] = t == -INFINITY ? -1.0f : w;
          if (lane == 0) {
            const float old = expf(before - base);
            s_old[r] = old;
            s_sum[r] = s_sum[r] * old + sum;
            s_max[r] = m;
          }
        }
        __syncwarp();  // a warp's rows are its own from here on
#pragma unroll
        for (int r = 0; r < kOwn; ++r) {
          const float old = s_old[kOwn * warp + r];
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][c][e] *= old;
        }
#pragma unroll 4
        for (int j = 0; j < kGenKeys; ++j) {
          float w[kOwn];
          bool seen[kOwn];
#pragma unroll
          for (int r = 0; r < kOwn; ++r) {
            w[r] = sp[(kOwn * warp + r) * (kGenKeys + 4) + j];
            seen[r] = !(w[r] < 0.0f);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t d = 128 * c + 4 * lane;
            if (d >= hd) continue;
            const float4 x = *(const float4*)(sv + j * stride + d);
#pragma unroll
            for (int r = 0; r < kOwn; ++r)
              if (seen[r]) {  // a masked value is not multiplied by zero: it may be NaN
                acc[r][c][0] = fmaf(w[r], x.x, acc[r][c][0]);
                acc[r][c][1] = fmaf(w[r], x.y, acc[r][c][1]);
                acc[r][c][2] = fmaf(w[r], x.z, acc[r][c][2]);
                acc[r][c][3] = fmaf(w[r], x.w, acc[r][c][3]);
              }
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      const uint32_t in_seg = kOwn * warp + r, row = seg.row0 + in_seg;
      if (in_seg >= seg.rows) continue;
      const float sum = s_sum[in_seg], m = s_max[in_seg];
      const bool empty = m == -INFINITY && sum == 0.0f;
      const float inv = empty ? 0.0f : 1.0f / sum, lse = empty ? -INFINITY : m + logf(sum);
      const uint64_t token = s.q0 + row / p.group;
      const uint32_t head = seg.kvh * p.group + row % p.group;
      const uint64_t part = (uint64_t)(seg.slot < 0 ? 0 : seg.slot) * p.slot_rows + in_seg;
      if (lane == 0) {
        if (seg.slot >= 0) p.part_lse[part] = lse;
        else if (p.lse) p.lse[token * p.q_heads + head] = lse;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t d = 128 * c + 4 * lane + e;
          if (d >= hd) continue;
          const float o = empty ? 0.0f : acc[r][c][e] * inv;
          if (seg.slot >= 0) p.part_o[part * hd + d] = o;
          else ((T*)p.out)[token * p.ld_out + (uint64_t)head * hd + d] = narrow<T>(o);
        }
    }
  }
}

// ---------------------------------------------------------------- the join --
//
// out = sum_s e^(lse_s - lse) out_s with lse = log sum_s e^lse_s: one block a
// row.  Its weights go to shared memory a batch at a time, and the threads take
// the columns, so that the loads of a batch do not wait for one another.
constexpr int kJoinThreads = 128, kJoinBatch = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const __grid_constant__ AttnParams p) {
  __shared__ float weight[kJoinBatch], all[2][kJoinThreads / 32];
  pdl_wait();  // the parts; launch_pdl's rule
  const AttnJoin j = p.joins[blockIdx.x];
  const uint32_t r = blockIdx.y;
  if (r >= j.rows) return;
  const AttnSeq s = p.seqs[j.seq];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row = j.row0 + r, head = j.kvh * p.group + row % p.group;
  const uint64_t token = s.q0 + row / p.group;
  const float* lse = p.part_lse + (uint64_t)j.slot0 * p.slot_rows + r;
  const float* part = p.part_o + ((uint64_t)j.slot0 * p.slot_rows + r) * p.head_dim;
  const uint64_t lse_step = p.slot_rows, part_step = (uint64_t)p.slot_rows * p.head_dim;
  float m = -INFINITY;
  for (uint32_t c = tid; c < j.slots; c += kJoinThreads) m = fmaxf(m, lse[c * lse_step]);
  m = warp_max(m);
  if (lane == 0) all[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w) m = fmaxf(m, all[0][w]);
  const float base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, o[kAttnMaxHead / kJoinThreads] = {};
  for (uint32_t c0 = 0; c0 < j.slots; c0 += kJoinBatch) {
    const uint32_t n = min((uint32_t)kJoinBatch, j.slots - c0);
    __syncthreads();
    if (tid < (int)n) {
      // NaN where a part's rows are; -1: a part in which the row sees nothing
      const float part_lse = lse[(c0 + tid) * lse_step], w = expf(part_lse - base);
      weight[tid] = part_lse == -INFINITY ? -1.0f : w;
      sum += w;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAttnMaxHead / kJoinThreads; ++u) {
      const uint32_t d = u * kJoinThreads + tid;
      if (d >= p.head_dim) break;
#pragma unroll 8
      for (uint32_t c = 0; c < n; ++c) {
        const float x = part[(c0 + c) * part_step + d];
        if (!(weight[c] < 0.0f)) o[u] = fmaf(weight[c], x, o[u]);
      }
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) all[1][warp] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += all[1][w];
  const bool empty = sum == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int u = 0; u < kAttnMaxHead / kJoinThreads; ++u) {
    const uint32_t d = u * kJoinThreads + tid;
    if (d < p.head_dim) ((T*)p.out)[token * p.ld_out + (uint64_t)head * p.head_dim + d] = narrow<T>(o[u] * inv);
  }
  if (tid == 0 && p.lse) p.lse[token * p.q_heads + head] = empty ? -INFINITY : base + logf(sum);
}

}  // namespace
}  // namespace svl

struct svl_attention_plan {
  svl::AttnParams p{};
  int device = -1;
  uint32_t dtype = 0;
  enum Kernel { kGeneral, kTiles, kRows } kernel = kGeneral;
  uint32_t max_join_rows = 0;
  uint64_t workspace = 0;
  void* block = nullptr;
  ~svl_attention_plan() { svl::free_block(device, block); }
};

using svl::refuse;

namespace {

using svl::AttnJoin;
using svl::AttnSegment;
using svl::AttnSeq;
using svl::kKeyTile;

// The smallest and largest document of a run of rows, padding apart.
struct DocRange {
  int32_t low = INT_MAX, high = -1;
  bool padding = false;
  void add(int32_t d) {
    if (d < 0) {
      padding = true;
      return;
    }
    low = std::min(low, d);
    high = std::max(high, d);
  }
  bool any() const { return high >= 0; }
};

struct Schedule {
  std::vector<AttnSeq> seqs;
  std::vector<AttnSegment> segments;
  std::vector<uint32_t> block_segments, lists;
  std::vector<AttnJoin> joins;
  uint32_t slots = 0, max_join_rows = 0;
};

// Rows row0 .. row0 + rows - 1 of a sequence against every key tile: appends
// the tiles that some row sees to `list`.
void list_keys(const svl_attention_config& c, const AttnSeq& s, uint32_t group, uint32_t row0, uint32_t rows,
               uint32_t tile_rows, const int32_t* doc_q, const std::vector<DocRange>& key_docs,
               std::vector<uint32_t>& list) {
  const int64_t shift = (int64_t)s.n_k - s.n_q;
  struct Tile {
    int64_t first, last;  // places of its queries
    DocRange docs;
    bool exists;
  } tile[2];
  for (int t = 0; t < 2; ++t) {
    tile[t].exists = (uint64_t)t * tile_rows < rows;
    if (!tile[t].exists) continue;
    const uint32_t q0 = (row0 + t * tile_rows) / group, q1 = (row0 + std::min(rows, (t + 1) * tile_rows) - 1) / group;
    tile[t].first = q0 + shift;
    tile[t].last = q1 + shift;
    if (doc_q)
      for (uint32_t i = q0; i <= q1; ++i) tile[t].docs.add(doc_q[s.q0 + i]);
  }
  const uint32_t n_tiles = (uint32_t)(((uint64_t)s.n_k + kKeyTile - 1) / kKeyTile);
  auto classify = [&](const Tile& t, uint32_t kt) -> uint32_t {
    if (!t.exists || (doc_q && !t.docs.any())) return svl::kSeesNone;
    const int64_t j0 = (int64_t)kt * kKeyTile, j1 = std::min<int64_t>(j0 + kKeyTile, s.n_k) - 1;
    const DocRange* kd = doc_q ? &key_docs[kt] : nullptr;
    if (kd && !kd->any()) return svl::kSeesNone;
    const bool whole = j1 - j0 + 1 == (int64_t)kKeyTile && (!kd || (!kd->padding && !t.docs.padding));
    if (j1 < (int64_t)s.prefix) return whole ? svl::kSeesAll : svl::kSeesSome;
    if (j0 < (int64_t)s.prefix) return svl::kSeesSome;
    if (c.causal && j0 > t.last) return svl::kSeesNone;
    if (c.window >= 0 && (j1 < t.first - c.window || j0 > t.last + c.window)) return svl::kSeesNone;
    if (kd && (kd->high < t.docs.low || kd->low > t.docs.high)) return svl::kSeesNone;
    if (!whole || (c.causal && j1 > t.first)) return svl::kSeesSome;
    if (c.window >= 0 && (j0 < t.last - c.window || j1 > t.first + c.window)) return svl::kSeesSome;
    if (kd && (kd->low != kd->high || t.docs.low != t.docs.high || kd->low != t.docs.low)) return svl::kSeesSome;
    return svl::kSeesAll;
  };
  // tiles outside the prefix and outside every row's order and window hold no visible key
  const int64_t last = tile[1].exists ? tile[1].last : tile[0].last;
  int64_t from = 0, to = n_tiles;
  if (c.window >= 0) from = std::max<int64_t>(0, tile[0].first - c.window) / kKeyTile;
  if (c.window >= 0) to = std::min<int64_t>(to, std::max<int64_t>(-1, last + c.window) / kKeyTile + 1);
  if (c.causal) to = std::min<int64_t>(to, std::max<int64_t>(-1, last) / kKeyTile + 1);
  const int64_t ahead = std::min<int64_t>(n_tiles, ((int64_t)s.prefix + kKeyTile - 1) / kKeyTile);
  auto add = [&](uint32_t kt) {
    const uint32_t a = classify(tile[0], kt), b = classify(tile[1], kt);
    if (a || b) list.push_back(kt | a << 28 | b << 30);
  };
  for (int64_t kt = 0; kt < ahead; ++kt) add((uint32_t)kt);
  for (int64_t kt = std::max(from, ahead); kt < to; ++kt) add((uint32_t)kt);
}

// A segment costs its key tiles and about two tiles more for its queries,
// first scores and output.
constexpr uint64_t kSegmentTiles = 2;
// Parts of a cut key axis are at least this many tiles.
constexpr uint32_t kMinPart = 2;
// What the join's launch costs, in key tiles.
constexpr uint64_t kJoinTiles = 3;

Schedule schedule(const svl_attention_config& c, const uint64_t* cu_q, const uint64_t* cu_k, uint32_t batch,
                  const uint64_t* prefix, const int32_t* doc_q, const int32_t* doc_k, uint32_t tile_rows,
                  uint32_t row_tiles, uint32_t workers) {
  Schedule out;
  const uint32_t group = c.q_heads / c.kv_heads;
  struct Task {
    uint32_t seq, row0, rows, list0, list1;
  };
  std::vector<Task> tasks;
  std::vector<DocRange> key_docs;
  std::vector<uint32_t> list;
  uint64_t cost = 0;
  uint32_t longest = 0;
  for (uint32_t b = 0; b < batch; ++b) {
    AttnSeq s{};
    s.q0 = cu_q[b];
    s.k0 = cu_k[b];
    s.n_q = (uint32_t)(cu_q[b + 1] - cu_q[b]);
    s.n_k = (uint32_t)(cu_k[b + 1] - cu_k[b]);
    s.prefix = prefix ? (uint32_t)std::min<uint64_t>(prefix[b], s.n_k) : 0;
    out.seqs.push_back(s);
    key_docs.clear();
    if (doc_k && s.n_q)
      for (uint32_t j = 0; j < s.n_k; ++j) {
        if (j % kKeyTile == 0) key_docs.emplace_back();
        key_docs.back().add(doc_k[s.k0 + j]);
      }
    const uint64_t rows = (uint64_t)s.n_q * group;
    for (uint64_t r = 0; r < rows; r += (uint64_t)tile_rows * row_tiles) {
      Task t{b, (uint32_t)r, (uint32_t)std::min<uint64_t>(rows - r, (uint64_t)tile_rows * row_tiles), 0, 0};
      list.clear();
      list_keys(c, s, group, t.row0, t.rows, tile_rows, doc_q, key_docs, list);
      // neighbours often see the same keys in the same way
      const size_t n = list.size(), at = tasks.empty() ? 0 : tasks.back().list0;
      if (!tasks.empty() && tasks.back().list1 - at == n && std::equal(list.begin(), list.end(), out.lists.begin() + at)) {
        t.list0 = (uint32_t)at;
      } else {
        t.list0 = (uint32_t)out.lists.size();
        out.lists.insert(out.lists.end(), list.begin(), list.end());
        if (out.lists.size() > UINT32_MAX / 2) throw std::bad_alloc();
      }
      t.list1 = t.list0 + (uint32_t)n;
      longest = std::max(longest, (uint32_t)n);
      cost += (n + kSegmentTiles) * c.kv_heads;
      tasks.push_back(t);
    }
  }
  // Whole key axes first; where the longest is more than a worker's even
  // share, parts of a share and of fractions of it, and of all these the
  // division whose most loaded worker has least to do.
  struct Piece {
    AttnSegment seg;
    uint64_t cost;
  };
  struct Division {
    std::vector<Piece> pieces;
    std::vector<std::vector<uint32_t>> of;  // per worker
    std::vector<AttnJoin> joins;
    uint32_t slots = 0, max_join_rows = 0;
    uint64_t makespan = 0;
  };
  auto divide = [&](uint32_t part) {
    Division d;
    for (const Task& t : tasks)
      for (uint32_t h = 0; h < c.kv_heads; ++h) {
        const uint32_t n = t.list1 - t.list0;
        const uint32_t parts = std::max(1u, std::min(n / kMinPart, (uint32_t)(((uint64_t)n + part - 1) / part)));
        if (parts > 1) {
          d.joins.push_back({t.seq, h, t.row0, t.rows, d.slots, parts});
          d.max_join_rows = std::max(d.max_join_rows, t.rows);
        }
        for (uint32_t i = 0; i < parts; ++i) {
          const uint32_t a = t.list0 + (uint32_t)((uint64_t)n * i / parts);
          const uint32_t b = t.list0 + (uint32_t)((uint64_t)n * (i + 1) / parts);
          d.pieces.push_back({{t.seq, h, t.row0, t.rows, a, b, parts > 1 ? (int32_t)d.slots++ : -1, 0},
                              b - a + kSegmentTiles});
        }
      }
    // longest first to the least loaded worker
    std::stable_sort(d.pieces.begin(), d.pieces.end(), [](const Piece& a, const Piece& b) { return a.cost > b.cost; });
    d.of.resize(std::min<size_t>(workers, d.pieces.size()));
    std::vector<std::pair<uint64_t, uint32_t>> heap;  // (load, worker), least on top
    for (uint32_t w = 0; w < d.of.size(); ++w) heap.emplace_back(0, w);
    auto more = [](const std::pair<uint64_t, uint32_t>& a, const std::pair<uint64_t, uint32_t>& b) { return a > b; };
    for (uint32_t i = 0; i < d.pieces.size(); ++i) {
      std::pop_heap(heap.begin(), heap.end(), more);
      d.of[heap.back().second].push_back(i);
      heap.back().first += d.pieces[i].cost;
      d.makespan = std::max(d.makespan, heap.back().first);
      std::push_heap(heap.begin(), heap.end(), more);
    }
    if (!d.joins.empty()) d.makespan += kJoinTiles;
    return d;
  };
  const uint64_t share = std::max<uint64_t>(1, (cost + workers - 1) / workers);
  Division best = divide(UINT32_MAX);
  if (longest > share)
    for (uint32_t fraction = 1; fraction <= 8; fraction *= 2) {
      Division d = divide((uint32_t)std::max<uint64_t>(kMinPart, share / fraction));
      if (d.makespan < best.makespan) best = std::move(d);
    }
  out.block_segments.push_back(0);
  for (const auto& w : best.of) {
    for (uint32_t i : w) out.segments.push_back(best.pieces[i].seg);
    out.block_segments.push_back((uint32_t)out.segments.size());
  }
  out.joins = std::move(best.joins);
  out.slots = best.slots;
  out.max_join_rows = best.max_join_rows;
  return out;
}

int check_offsets(const uint64_t* cu, uint32_t batch, const char* name, char* err, size_t err_len) {
  if (cu[0]) return refuse(SVL_USAGE, std::string(name) + " must start at 0", err, err_len);
  for (uint32_t b = 0; b < batch; ++b)
    if (cu[b + 1] < cu[b]) return refuse(SVL_USAGE, std::string(name) + " must not fall", err, err_len);
  if (cu[batch] >= 1ull << 40) return refuse(SVL_LIMIT_EXCEEDED, std::string(name) + " is 2^40 or more", err, err_len);
  return SVL_OK;
}

template <typename T, int ROWS>
cudaError_t launch_general(const svl::AttnParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto kernel = svl::attention_general_kernel<T, ROWS>;
  const cudaError_t e = smem_opt_in(kernel, (int)svl::gen_smem(svl::kAttnMaxHead, ROWS), &done);
  if (e != cudaSuccess) return e;
  kernel<<<p.blocks, svl::kGenThreads, svl::gen_smem(p.head_dim, ROWS), st>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_general(const svl::AttnParams& p, cudaStream_t st) {
  return p.slot_rows == svl::kGenRows ? launch_general<T, svl::kGenRows>(p, st) : launch_general<T, svl::kGenFewRows>(p, st);
}

template <typename T>
cudaError_t launch_join(const svl::AttnParams& p, uint32_t rows, cudaStream_t st) {
  return launch_pdl(svl::attention_join_kernel<T>, dim3(p.n_joins, rows), dim3(svl::kJoinThreads), 0, st, p);
}

// Blocks of the general kernel an SM takes (its shared memory allows two at
// head sizes up to 256).
constexpr uint32_t kGeneralBlocksPerSm = 2;

}  // namespace

extern "C" {

int svl_attention_plan_create(int device, const svl_attention_config* config, const uint64_t* cu_q,
                              const uint64_t* cu_k, uint32_t batch, const uint64_t* prefix, const int32_t* doc_q,
                              const int32_t* doc_k, const float* slopes, svl_attention_plan** out, char* err,
                              size_t err_len) {
  if (!out) return refuse(SVL_USAGE, "null argument", err, err_len);
  *out = nullptr;
  if (!config || !cu_q) return refuse(SVL_USAGE, "null argument", err, err_len);
  const svl_attention_config& c = *config;
  if (!svl::is_operand_dtype(c.dtype)) return refuse(SVL_USAGE, "unknown dtype", err, err_len);
  if (!c.kv_heads || c.kv_heads > 65535) return refuse(SVL_USAGE, "kv_heads is outside 1..=65535", err, err_len);
  if (!c.q_heads || c.q_heads % c.kv_heads || c.q_heads / c.kv_heads > 65535)
    return refuse(SVL_USAGE, "q_heads must be a multiple of kv_heads (at most 65535 times)", err, err_len);
  if (!c.head_dim || c.head_dim > svl::kAttnMaxHead) return refuse(SVL_USAGE, "head_dim is outside 1..=512", err, err_len);
  // within these every product that the kernels form of scale, cap, slope and a
  // distance below 2^31 is finite in FP32
  if (!(c.scale >= 1e-30f && c.scale <= 1e30f)) return refuse(SVL_USAGE, "scale is outside 1e-30..=1e30", err, err_len);
  if (!(c.cap == 0 || (c.cap >= 1e-30f && c.cap <= 1e30f && (double)c.scale / c.cap <= 1e30)))
    return refuse(SVL_USAGE, "cap is neither 0 nor in 1e-30..=1e30 with scale / cap at most 1e30", err, err_len);
  if (c.causal > 1) return refuse(SVL_USAGE, "causal must be 0 or 1", err, err_len);
  for (uint32_t r : c.reserved)
    if (r) return refuse(SVL_USAGE, "svl_attention_config.reserved must be zero", err, err_len);
  const bool own_keys = cu_k != nullptr;
  if (!own_keys) cu_k = cu_q;
  if (!doc_k && doc_q && !own_keys) doc_k = doc_q;
  if (!doc_q != !doc_k) return refuse(SVL_USAGE, "documents need both queries and keys", err, err_len);
  int rc = check_offsets(cu_q, batch, "cu_q", err, err_len);
  if (!rc) rc = check_offsets(cu_k, batch, "cu_k", err, err_len);
  if (rc) return rc;
  const uint32_t group = c.q_heads / c.kv_heads;
  for (uint32_t b = 0; b < batch; ++b)
    if (cu_k[b + 1] - cu_k[b] >= 1ull << 31 || (cu_q[b + 1] - cu_q[b]) >= (1ull << 31) / group)
      return refuse(SVL_LIMIT_EXCEEDED, "a sequence has 2^31 or more keys or query rows", err, err_len);
  if (slopes)
    for (uint32_t h = 0; h < c.q_heads; ++h)
      if (!(std::fabs(slopes[h]) <= 1e20f)) return refuse(SVL_USAGE, "slopes are outside -1e20..=1e20", err, err_len);
  return svl::guarded(err, err_len, [&]() -> int {
    std::unique_ptr<svl_attention_plan> plan(new svl_attention_plan());
    svl::DeviceGuard on(device);
    if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
    plan->device = device;
    plan->dtype = c.dtype;
    int sms = 0;
    cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    uint32_t tile_rows = svl::kGenRows, row_tiles = 1, per_sm = kGeneralBlocksPerSm;
    if (svl::attention_tc_takes(c, cu_q[batch], cu_k[batch])) {
      uint64_t most = 0;
      for (uint32_t b = 0; b < batch; ++b) most = std::max(most, (cu_q[b + 1] - cu_q[b]) * group);
      per_sm = 1;
      plan->kernel = svl_attention_plan::kRows;
      tile_rows = svl::attention_rows_takes(c.head_dim, most);
      if (!tile_rows) {
        plan->kernel = svl_attention_plan::kTiles;
        tile_rows = svl::attention_tc_tile_rows(group);
        row_tiles = svl::attention_tc_row_tiles(c.head_dim);
      }
    } else {
      uint64_t blocks = 0;
      for (uint32_t b = 0; b < batch; ++b)
        blocks += ((cu_q[b + 1] - cu_q[b]) * group + svl::kGenRows - 1) / svl::kGenRows * c.kv_heads;
      if (blocks < (uint64_t)sms) tile_rows = svl::kGenFewRows;
    }
    const Schedule s = schedule(c, cu_q, cu_k, batch, prefix, doc_q, doc_k, tile_rows, row_tiles, (uint32_t)sms * per_sm);
    svl::AttnParams& p = plan->p;
    p.slot_rows = tile_rows * row_tiles;
    // one block of device memory, one copy
    std::vector<uint8_t> host;
    auto put = [&](const void* data, size_t bytes) {
      const size_t at = (host.size() + 15) & ~(size_t)15;
      host.resize(at + bytes);
      if (bytes) std::memcpy(host.data() + at, data, bytes);
      return at;
    };
    const uint64_t n_q = cu_q[batch], n_k = cu_k[batch];
    const uint32_t no_error = 0;
    const size_t at_err = put(&no_error, 4), at_seqs = put(s.seqs.data(), s.seqs.size() * sizeof(AttnSeq)),
                 at_segments = put(s.segments.data(), s.segments.size() * sizeof(AttnSegment)),
                 at_blocks = put(s.block_segments.data(), s.block_segments.size() * 4),
                 at_lists = put(s.lists.data(), s.lists.size() * 4),
                 at_joins = put(s.joins.data(), s.joins.size() * sizeof(AttnJoin)),
                 at_slopes = put(slopes, slopes ? c.q_heads * 4 : 0), at_doc_q = put(doc_q, doc_q ? n_q * 4 : 0),
                 at_doc_k = put(doc_k, doc_k ? n_k * 4 : 0);
    e = cudaMalloc(&plan->block, host.size());
    if (e != cudaSuccess) {
      plan->block = nullptr;
      return svl::cuda_failure(e, err, err_len);
    }
    e = cudaMemcpy(plan->block, host.data(), host.size(), cudaMemcpyHostToDevice);
    // a copy from pageable memory may return before it has landed, and a stream
    // that does not wait for the default one may be the first to read it
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
    uint8_t* base = (uint8_t*)plan->block;
    p.err = (uint32_t*)(base + at_err);
    p.seqs = (const AttnSeq*)(base + at_seqs);
    p.segments = (const AttnSegment*)(base + at_segments);
    p.block_segments = (const uint32_t*)(base + at_blocks);
    p.lists = (const uint32_t*)(base + at_lists);
    p.joins = (const AttnJoin*)(base + at_joins);
    p.slopes = slopes ? (const float*)(base + at_slopes) : nullptr;
    p.doc_q = doc_q ? (const int32_t*)(base + at_doc_q) : nullptr;
    p.doc_k = doc_k ? (const int32_t*)(base + at_doc_k) : nullptr;
    p.blocks = (uint32_t)s.block_segments.size() - 1;
    p.n_joins = (uint32_t)s.joins.size();
    // a minute, and 4 s more for each 2^17 key tiles of the longest block (30 us a
    // tile): whole tiles alone, as 32 heads over 2^21 tokens have, outlast any fixed limit
    uint64_t most_tiles = 0;
    for (uint32_t b = 0; b < p.blocks; ++b) {
      uint64_t tiles = 0;
      for (uint32_t i = s.block_segments[b]; i < s.block_segments[b + 1]; ++i) tiles += s.segments[i].list1 - s.segments[i].list0;
      most_tiles = std::max(most_tiles, tiles);
    }
    p.check_waits = 15 + (uint32_t)(most_tiles >> 17);
    p.q_heads = c.q_heads;
    p.kv_heads = c.kv_heads;
    p.group = group;
    p.head_dim = c.head_dim;
    p.total_q = n_q;
    p.total_k = n_k;
    p.scale = c.scale;
    p.cap = c.cap;
    if (c.cap > 0) {
      const double k = (double)c.scale / c.cap;
      double power = (double)c.cap * 1.4426950408889634 * k;
      // A coefficient too large for FP32 leaves every score to the general form.  One
      // too small is left out, and the polynomial ends where it would be 2^-25 of it.
      bool held = true;
      double limit = svl::kTanhLimit;
      for (int i = 0; i < svl::kCapTerms; ++i, power *= k * k) {
        const bool small = std::fabs(power * svl::kTanhOdd[i]) < 1e-37;
        if (small) limit = std::min(limit, svl::kTanhWithout[i]);
        held &= std::fabs(power) < 1e37;
        p.cap_odd[i] = held && !small ? (float)(power * svl::kTanhOdd[i]) : 0.0f;
      }
      p.cap_limit = held ? (float)std::min(limit / k, 1.8e19) : -1.0f;  // whose square is finite
    }
    p.causal = (int32_t)c.causal;
    p.window = c.window;
    plan->max_join_rows = s.max_join_rows;
    // outputs of every slot's rows, then their log sums
    plan->workspace = ((uint64_t)s.slots * p.slot_rows * (c.head_dim + 1) * 4 + 15) & ~15ull;
    p.part_lse = (float*)((uint64_t)s.slots * p.slot_rows * c.head_dim * 4);  // offset; run adds the base
    *out = plan.release();
    return SVL_OK;
  });
}

void svl_attention_plan_destroy(svl_attention_plan* plan) { delete plan; }

int svl_attention_plan_workspace(const svl_attention_plan* plan, uint64_t* bytes) {
  if (!plan || !bytes) return SVL_USAGE;
  *bytes = plan->workspace;
  return SVL_OK;
}

int svl_attention_device(const svl_attention_plan* plan, const void* d_q, uint64_t ld_q, const void* d_k,
                         uint64_t ld_k, const void* d_v, uint64_t ld_v, void* d_out, uint64_t ld_out, float* d_lse,
                         void* d_workspace, uint64_t workspace_bytes, void* stream, char* err, size_t err_len) {
  if (!plan) return refuse(SVL_USAGE, "null argument", err, err_len);
  svl::AttnParams p = plan->p;
  if (!p.total_q) return SVL_OK;
  if (!d_q || !d_out || (p.total_k && (!d_k || !d_v))) return refuse(SVL_USAGE, "null argument", err, err_len);
  const uint64_t q_width = (uint64_t)p.q_heads * p.head_dim, k_width = (uint64_t)p.kv_heads * p.head_dim;
  if (ld_q < q_width || ld_out < q_width || (p.total_k && (ld_k < k_width || ld_v < k_width)))
    return refuse(SVL_USAGE, "a row stride is shorter than its heads", err, err_len);
  if (std::max(std::max(ld_q, ld_out), p.total_k ? std::max(ld_k, ld_v) : 0) >= 1ull << 36)
    return refuse(SVL_USAGE, "a row stride is 2^36 or more", err, err_len);
  const uint64_t size = svl::dtype_size(plan->dtype);
  const bool wide = size == 2 && p.head_dim % 8 == 0;
  const uint64_t align = wide ? 16 : size;
  const uint64_t strides = ld_q | ld_out | (p.total_k ? ld_k | ld_v : 0);
  const uintptr_t pointers = (uintptr_t)d_q | (uintptr_t)d_out | (p.total_k ? (uintptr_t)d_k | (uintptr_t)d_v : 0);
  if (pointers & (align - 1)) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  if (wide && strides % 8) return refuse(SVL_USAGE, "row strides must be multiples of 8", err, err_len);
  if ((uintptr_t)d_lse & 3) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  if (plan->workspace) {
    if (!d_workspace || workspace_bytes < plan->workspace)
      return refuse(SVL_USAGE, "the workspace is smaller than svl_attention_plan_workspace", err, err_len);
    if ((uintptr_t)d_workspace & 15) return refuse(SVL_USAGE, "misaligned pointer", err, err_len);
  }
  p.q = d_q;
  p.k = d_k;
  p.v = d_v;
  p.out = d_out;
  p.lse = d_lse;
  p.ld_q = ld_q;
  p.ld_k = ld_k;
  p.ld_v = ld_v;
  p.ld_out = ld_out;
  p.part_o = (float*)d_workspace;
  p.part_lse = (float*)((uintptr_t)d_workspace + (uintptr_t)plan->p.part_lse);
  svl::DeviceGuard on(plan->device);
  if (on.status != cudaSuccess) return svl::cuda_failure(on.status, err, err_len);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = plan->kernel == svl_attention_plan::kRows    ? svl::attention_rows_launch(p, plan->dtype, st)
                  : plan->kernel == svl_attention_plan::kTiles ? svl::attention_tc_launch(p, plan->dtype, st)
                  : plan->dtype == SVL_DTYPE_F32  ? launch_general<float>(p, st)
                  : plan->dtype == SVL_DTYPE_BF16 ? launch_general<__nv_bfloat16>(p, st)
                                                  : launch_general<__half>(p, st);
  if (e == cudaSuccess && p.n_joins)
    e = plan->dtype == SVL_DTYPE_F32    ? launch_join<float>(p, plan->max_join_rows, st)
        : plan->dtype == SVL_DTYPE_BF16 ? launch_join<__nv_bfloat16>(p, plan->max_join_rows, st)
                                        : launch_join<__half>(p, plan->max_join_rows, st);
  return e == cudaSuccess ? SVL_OK : svl::cuda_failure(e, err, err_len);
}

int svl_attention_check(const svl_attention_plan* plan, char* err, size_t err_len) {
  if (!plan) return refuse(SVL_USAGE, "null argument", err, err_len);
  svl::DeviceGuard on(plan->device);
  uint32_t word = 0;
  cudaError_t e = on.status;
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&word, plan->p.err, 4, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && word) e = cudaMemset(plan->p.err, 0, 4);
  if (e == cudaSuccess && word) e = cudaStreamSynchronize(nullptr);
  if (e != cudaSuccess) return svl::cuda_failure(e, err, err_len);
  std::string message;
  const int rc = svl::status_from_device(word, &message);
  return rc ? refuse(rc, message, err, err_len) : SVL_OK;
}

}  // extern "C"
