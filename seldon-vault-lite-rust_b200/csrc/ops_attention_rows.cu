// ops_attention_rows.cu -- the FP16 / BF16 attention kernel of svl_attention_*
// for few query rows (single tokens) over long key axes.
//
// Bound by reading K and V once.  A 128-row tensor-core tile would leave the
// softmax of a handful of rows to a handful of threads, so the rows are the 16
// rows of mma.sync m16n8k16 instead: all lanes share the scores.  Two teams of
// four warps take every other 128-key tile, 32 keys a warp, and each warp keeps
// the running maximum, sum and output of its own keys in registers, joined at the
// end.
// K and V come by TMA through a ring of 16 KB slabs that a thread of a third
// warpgroup keeps full across tiles and segments; its registers go to the teams.
// One row of 32 query and 8 key heads of 128 over 8 caches of 13135-64537 keys
// (1.25 GB): 250-258 us, 4.8-5.0 TB/s; bound by the chains of two warps a scheduler,
// which issue in 27% of the cycles, then by memory.
#include "ops_attention_mma.cuh"

namespace svl {
namespace {

// Warpgroup 0 loads; 1 and 2 are the teams.
constexpr int kThreads = 384, kMmaWarps = 8, kTeam = kMmaWarps / 2, kKeys = 2;  // 16s of keys a warp
constexpr int kRegs = 168;  // of a thread at launch
constexpr int kRegsLoad = 40, kRegsTeam = 232;
static_assert(kRegsLoad + 2 * kRegsTeam == 3 * kRegs, "registers move inside the launch's own");

// MT tiles of 16 rows.
template <int HDP, int MT>
struct Smem {
  static constexpr int kStages = 9, kRowBytes = HDP * 2 + 16;
  alignas(1024) uint8_t ring[kStages * kSlabBytes];
  float join[4][MT * 16][HDP];  // a join's outputs
  uint8_t q[MT * 16 * kRowBytes];
  float join_max[4][MT * 16], join_sum[4][MT * 16];
  uint64_t full[kStages], empty[kStages];
  uint32_t spoiled;
};
static_assert(sizeof(Smem<256, 1>) + 1024 <= kSmemLimit && sizeof(Smem<128, 2>) + 1024 <= kSmemLimit, "shared memory");

SVL_DEV void ldmatrix(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
SVL_DEV void ldmatrix_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
SVL_DEV void mma(__half, float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SVL_DEV void mma(__nv_bfloat16, float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SVL_DEV void teams_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Zeroes the non-finite halves of an operand register.
template <typename T>
SVL_DEV bool clean(uint32_t& w) {
  const uint32_t bad = non_finite(T(), w);
  if (!bad) return false;
  w &= ~((bad >> 15) * 0xffffu);
  return true;
}

template <typename T, int HDP, int MT>
__global__ void __launch_bounds__(kThreads, 1)
    attention_rows_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v) {
  using Sm = Smem<HDP, MT>;
  constexpr int kStages = Sm::kStages;
  extern __shared__ uint8_t raw[];
  Sm& sm = *(Sm*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slabs = (p.head_dim + kSlabCols - 1) / kSlabCols, steps = (p.head_dim + 15) / 16;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kTeam);
    }
    sm.spoiled = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  pdl_trigger();
  const uint32_t seg0 = p.block_segments[blockIdx.x], seg1 = p.block_segments[blockIdx.x + 1];

  if (warp < 4) {
    setmaxnreg_dec<kRegsLoad>();
    if (threadIdx.x == 0) {
      RingPos at;
      uint32_t issued = 0;
      bool ok = true;
      for (uint32_t is = seg0; ok && is < seg1; ++is) {
        const uint32_t list0 = p.segments[is].list0, list1 = p.segments[is].list1, kvh = p.segments[is].kvh;
        const uint64_t k0 = p.seqs[p.segments[is].seq].k0;
        uint32_t next = list0 < list1 ? p.lists[list0] : 0;
        for (uint32_t il = list0; ok && il < list1; ++il) {
          const int32_t row = (int32_t)(k0 + (uint64_t)entry_tile(next) * kKeyTile);
          if (il + 1 < list1) next = p.lists[il + 1];
          for (int i = 0; i < 2 * slabs; ++i) {
            if (!mbar_wait(&sm.empty[at.stage], at.phase ^ 1, p.err)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&sm.full[at.stage], kSlabBytes);
            tma_load_3d(sm.ring + at.stage * kSlabBytes, i < slabs ? &map_k : &map_v, &sm.full[at.stage],
                        (i < slabs ? i : i - slabs) * kSlabCols, (int32_t)kvh, row);
            ++issued;
            at.next(kStages);
          }
        }
      }
      if (!ok) {
        // copies in flight land before the CTA leaves
        RingPos back;
        for (uint32_t i = 0; i < issued; ++i) {
          if (i + kStages >= issued) mbar_wait(&sm.full[back.stage], back.phase, p.err);
          back.next(kStages);
        }
      }
    }
    return;
  }
  setmaxnreg_inc<kRegsTeam>();
  const int tid = threadIdx.x - 128, warp_in = warp - 4;
  const int g = lane >> 2, c2 = (lane & 3) * 2, mi = lane >> 3, mr = lane & 7;
  const bool capped = p.cap > 0.0f, biased = p.slopes != nullptr;
  const float scale2 = p.scale * kLog2e, cap2 = p.cap * kLog2e, cap_arg = capped ? 2.0f * scale2 / p.cap : 0.0f;
  const uint32_t q_at = smem_u32(sm.q) + ((mi & 1) * 8 + mr) * Sm::kRowBytes + (mi >> 1) * 16;
  // this warp's keys of a slab: K by (8 keys, 8 columns) blocks, V by the same transposed
  const int team = warp_in / kTeam, key0 = warp_in % kTeam * 16 * kKeys;
  const uint32_t k_row = key0 + (mi >> 1) * 8 + mr, v_row = key0 + (mi & 1) * 8 + mr;
  RingPos pos;
  uint32_t slabs0 = 0;  // the CTA's slabs before this segment
  bool dead = false;    // a wait ran out: no more waits, but every step is taken
  auto wait = [&]() {
    if (!dead && !mbar_wait(&sm.full[pos.stage], pos.phase, p.err)) dead = true;
    __syncwarp();
  };
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.empty[pos.stage]);
    pos.next(kStages);
  };

  for (uint32_t is = seg0; is < seg1; ++is) {
    const AttnSegment seg = p.segments[is];
    const AttnSeq s = p.seqs[seg.seq];
    teams_sync();  // the last segment's rows and flags are read
    for (int i = tid; i < MT * 16 * (HDP / 8); i += kMmaWarps * 32) {
      const int r = i / (HDP / 8), d = i % (HDP / 8) * 8;
      uint4 w = make_uint4(0, 0, 0, 0);
      const uint32_t row = seg.row0 + r;
      if (r < (int)seg.rows && d < (int)p.head_dim)
        w = *(const uint4*)((const T*)p.q + (s.q0 + row / p.group) * p.ld_q +
                            (uint64_t)(seg.kvh * p.group + row % p.group) * p.head_dim + d);
      *(uint4*)(sm.q + r * Sm::kRowBytes + d * 2) = w;
    }
    if (tid == 0) sm.spoiled = 0;
    // this thread's rows: g and g + 8 of each row tile
    RowMask mask[MT][2];
    float slope2[MT][2], m[MT][2], l[MT][2], o[MT][HDP / 8][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t row = seg.row0 + min((uint32_t)(t * 16 + u * 8 + g), seg.rows - 1);
        mask[t][u] = row_mask(p, s, row / p.group);
        slope2[t][u] = biased ? p.slopes[seg.kvh * p.group + row % p.group] * kLog2e : 0.0f;
        m[t][u] = -INFINITY;
        l[t][u] = 0.0f;
      }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int d = 0; d < HDP / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][d][e] = 0.0f;
    teams_sync();

    // the query operand stays in registers where there is room
    constexpr bool kKeepQ = HDP * MT <= 128;
    uint32_t qa[kKeepQ ? MT : 1][kKeepQ ? HDP / 16 : 1][4];
    if constexpr (kKeepQ) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k) ldmatrix(qa[t][k], q_at + t * 16 * Sm::kRowBytes + k * 32);
    }
    uint32_t next = seg.list0 + team < seg.list1 ? p.lists[seg.list0 + team] : 0;
#pragma unroll 1
    for (uint32_t il = seg.list0 + team; il < seg.list1; il += 2) {
      const uint32_t entry = next;
      if (il + 2 < seg.list1) next = p.lists[il + 2];
      const uint32_t at = slabs0 + (il - seg.list0) * 2 * slabs;
      pos.stage = at % kStages;
      pos.phase = at / kStages & 1;
      const uint32_t j0 = entry_tile(entry) * kKeyTile + key0;
      const bool some = entry_sees(entry, 0) == kSeesSome;
      // scores: tiles of 8 keys
      float sc[MT][2 * kKeys][4] = {};
#pragma unroll
      for (int c = 0; c < HDP / kSlabCols; ++c) {
        if (c >= slabs) break;
        wait();
        const uint32_t slab = smem_u32(sm.ring) + pos.stage * kSlabBytes + k_row * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c * 4 + k >= steps) break;
          uint32_t b[kKeys][4];
#pragma unroll
          for (int n = 0; n < kKeys; ++n) ldmatrix(b[n], slab + n * 2048 + ((2 * k + (mi & 1)) ^ mr) * 16);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t a[4];
            if constexpr (kKeepQ) {
#pragma unroll
              for (int i = 0; i < 4; ++i) a[i] = qa[t][c * 4 + k][i];
            } else {
              ldmatrix(a, q_at + t * 16 * Sm::kRowBytes + (c * 4 + k) * 32);
            }
#pragma unroll
            for (int n = 0; n < kKeys; ++n) {
              mma(T(), sc[t][2 * n], a, b[n][0], b[n][1]);
              mma(T(), sc[t][2 * n + 1], a, b[n][2], b[n][3]);
            }
          }
        }
        done();
      }
      uint32_t pa[MT][kKeys][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (capped) {
          float most = 0.0f;
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(sc[t][n][e]));
          if (__any_sync(0xffffffffu, most > p.cap_limit)) {
#pragma unroll
            for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[t][n][e] = capped_any(p, sc[t][n][e], cap_arg, cap2);
          } else {
#pragma unroll
            for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[t][n][e] = capped_small(p, sc[t][n][e]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][n][e] *= scale2;
        }
        if (biased) {
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int64_t gap = mask[t][e >> 1].place - (int64_t)(j0 + n * 8 + c2 + (e & 1));
              sc[t][n][e] = fmaf(-slope2[t][e >> 1], fabsf((float)gap), sc[t][n][e]);
            }
        }
        if (some) {
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t j = j0 + n * 8 + c2 + (e & 1);
              if (!sees(p, mask[t][e >> 1], j, p.doc_k && j < s.n_k ? __ldg(p.doc_k + s.k0 + j) : 0))
                sc[t][n][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n) top = fmax3(top, sc[t][n][2 * u], sc[t][n][2 * u + 1]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          float factor = 1.0f;
          if (top > m[t][u] + kBehind || (m[t][u] == -INFINITY && top > -INFINITY)) {
            factor = m[t][u] == -INFINITY ? 0.0f : ex2_approx(m[t][u] - top);
            m[t][u] = top;
          }
          if (__any_sync(0xffffffffu, factor != 1.0f)) {
            l[t][u] *= factor;
#pragma unroll
            for (int d = 0; d < HDP / 8; ++d) {
              o[t][d][2 * u] *= factor;
              o[t][d][2 * u + 1] *= factor;
            }
          }
          const float base = m[t][u] == -INFINITY ? 0.0f : m[t][u];
#pragma unroll
          for (int n = 0; n < 2 * kKeys; ++n) {
            const float x = ex2_approx(sc[t][n][2 * u] - base), y = ex2_approx(sc[t][n][2 * u + 1] - base);
            l[t][u] += x + y;
            pa[t][n >> 1][2 * (n & 1) + u] = pack2(T(), x, y);
          }
        }
      }
      bool found = false;
#pragma unroll
      for (int c = 0; c < HDP / kSlabCols; ++c) {
        if (c >= slabs) break;
        wait();
        const uint32_t slab = smem_u32(sm.ring) + pos.stage * kSlabBytes + v_row * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (c * 4 + k >= steps) break;
          uint32_t b[kKeys][4];
#pragma unroll
          for (int n = 0; n < kKeys; ++n) {
            ldmatrix_t(b[n], slab + n * 2048 + ((2 * k + (mi >> 1)) ^ mr) * 16);
            if (some) {
#pragma unroll
              for (int i = 0; i < 4; ++i) found |= clean<T>(b[n][i]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < kKeys; ++n) {
              mma(T(), o[t][(c * 4 + k) * 2], pa[t][n], b[n][0], b[n][1]);
              mma(T(), o[t][(c * 4 + k) * 2 + 1], pa[t][n], b[n][2], b[n][3]);
            }
        }
        done();
      }
      if (some && __any_sync(0xffffffffu, found) && lane == 0) atomicOr(&sm.spoiled, 1u);
    }
    slabs0 += (seg.list1 - seg.list0) * 2 * slabs;
    // A row's sum lies over its four lanes; then the warps join in halves: the
    // upper half hands maximum, sum and output over, the lower half adds them.
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[t][u] += __shfl_xor_sync(0xffffffffu, l[t][u], 1);
        l[t][u] += __shfl_xor_sync(0xffffffffu, l[t][u], 2);
      }
#pragma unroll 1
    for (int half = kMmaWarps / 2; half >= 1; half /= 2) {
      if (warp_in >= half && warp_in < 2 * half) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = t * 16 + u * 8 + g;
            if (c2 == 0) {
              sm.join_max[warp_in - half][r] = m[t][u];
              sm.join_sum[warp_in - half][r] = l[t][u];
            }
#pragma unroll
            for (int d = 0; d < HDP / 8; ++d)
              *(float2*)&sm.join[warp_in - half][r][d * 8 + c2] = make_float2(o[t][d][2 * u], o[t][d][2 * u + 1]);
          }
      }
      teams_sync();
      if (warp_in < half) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = t * 16 + u * 8 + g;
            const float other = sm.join_max[warp_in][r], top = fmaxf(m[t][u], other);
            const float mine = m[t][u] == -INFINITY ? 0.0f : ex2_approx(m[t][u] - top);
            const float theirs = other == -INFINITY ? 0.0f : ex2_approx(other - top);
            // a sum that is NaN with a maximum of -inf (every score NaN) stays
            const float their_sum = sm.join_sum[warp_in][r];
            l[t][u] = (l[t][u] != l[t][u] || their_sum != their_sum) ? NAN : l[t][u] * mine + their_sum * theirs;
            m[t][u] = top;
#pragma unroll
            for (int d = 0; d < HDP / 8; ++d) {
              const float2 w = *(const float2*)&sm.join[warp_in][r][d * 8 + c2];
              // nothing is taken from a side without weight: what it holds is 0
              if (mine != 1.0f) o[t][d][2 * u] *= mine, o[t][d][2 * u + 1] *= mine;
              o[t][d][2 * u] = fmaf(w.x, theirs, o[t][d][2 * u]);
              o[t][d][2 * u + 1] = fmaf(w.y, theirs, o[t][d][2 * u + 1]);
            }
          }
      }
      teams_sync();
    }
    if (warp_in != 0) continue;
    const bool spoiled = sm.spoiled != 0;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t in_seg = t * 16 + u * 8 + g;
        if (in_seg >= seg.rows) continue;
        const uint32_t row = seg.row0 + in_seg, query = row / p.group, head = seg.kvh * p.group + row % p.group;
        const uint64_t token = s.q0 + query, part = (uint64_t)(seg.slot < 0 ? 0 : seg.slot) * p.slot_rows + in_seg;
        const bool empty = m[t][u] == -INFINITY && l[t][u] == 0.0f;
        const float inv = empty ? 0.0f : 1.0f / l[t][u];
        const float lse = empty ? -INFINITY : kLn2 * ((m[t][u] == -INFINITY ? 0.0f : m[t][u]) + log2f(l[t][u]));
        if (c2 == 0) {
          if (seg.slot >= 0) p.part_lse[part] = lse;
          else if (p.lse) p.lse[token * p.q_heads + head] = lse;
        }
#pragma unroll
        for (int d = 0; d < HDP / 8; ++d) {
          const uint32_t col = d * 8 + c2;
          if (col >= p.head_dim) break;
          float2 w = make_float2(empty ? 0.0f : o[t][d][2 * u] * inv, empty ? 0.0f : o[t][d][2 * u + 1] * inv);
          if (spoiled) {
            float extra[32];
            for (int i = 0; i < 32; ++i) extra[i] = 0.0f;
            add_spoiled<T>(p, seg, s, query, col, extra);
            w.x += extra[0];
            w.y += extra[1];
          }
          if (seg.slot >= 0) *(float2*)(p.part_o + part * p.head_dim + col) = w;
          else *(uint32_t*)((T*)p.out + token * p.ld_out + (uint64_t)head * p.head_dim + col) = pack2(T(), w.x, w.y);
        }
      }
  }
}

template <typename T, int HDP, int MT>
cudaError_t launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int smem = (int)sizeof(Smem<HDP, MT>) + 1024;
  const cudaError_t e = smem_opt_in(attention_rows_kernel<T, HDP, MT>, smem, &done);
  if (e != cudaSuccess) return e;
  // setmaxnreg hands the launch's own registers on: an increase beyond them never ends
  static std::atomic<int> fits{-1};
  if (fits.load() < 0) {
    cudaFuncAttributes fa{};
    const cudaError_t f = cudaFuncGetAttributes(&fa, attention_rows_kernel<T, HDP, MT>);
    if (f != cudaSuccess) return f;
    fits.store(fa.numRegs == kRegs);
  }
  if (!fits.load()) return cudaErrorInvalidConfiguration;
  CUtensorMap k, v;
  // without keys there is nothing to load: any valid map will do
  const bool keys = p.total_k > 0;
  if (!encode_fn() ||
      !head_map(&k, keys ? p.k : p.q, dtype, keys ? p.total_k : 1, keys ? p.kv_heads : 1, p.head_dim, keys ? p.ld_k : p.ld_q,
                1, kKeyTile) ||
      !head_map(&v, keys ? p.v : p.q, dtype, keys ? p.total_k : 1, keys ? p.kv_heads : 1, p.head_dim, keys ? p.ld_v : p.ld_q,
                1, kKeyTile))
    return cudaErrorInvalidValue;
  attention_rows_kernel<T, HDP, MT><<<p.blocks, kThreads, smem, st>>>(p, k, v);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  const bool two = p.slot_rows > 16;
  if (p.head_dim <= 64) return two ? launch<T, 64, 2>(p, dtype, st) : launch<T, 64, 1>(p, dtype, st);
  if (p.head_dim <= 128) return two ? launch<T, 128, 2>(p, dtype, st) : launch<T, 128, 1>(p, dtype, st);
  return launch<T, 256, 1>(p, dtype, st);
}

}  // namespace

uint32_t attention_rows_takes(uint32_t head_dim, uint64_t rows) {
  return rows <= 16 ? 16 : rows <= 32 && head_dim <= 128 ? 32 : 0;
}

cudaError_t attention_rows_launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  return dtype == SVL_DTYPE_F16 ? launch<__half>(p, dtype, st) : launch<__nv_bfloat16>(p, dtype, st);
}

}  // namespace svl
