// ops_attention_tc.cu -- the FP16 / BF16 attention kernel of svl_attention_*
// on the 5th-generation tensor cores.
//
// One persistent CTA per SM walks its segments (rows of one key-value head
// against a list of 128-key tiles).  A row tile is up to 128 (query, head of
// the group) rows, so every head of a group reads a key tile once.  Head
// sizes up to 128: two row tiles share each key tile, one softmax warpgroup
// each, so that one tile's products run under the other's softmax.  Head sizes
// up to 256: one row tile with two score buffers, its 128 columns split between
// the two warpgroups.
//
//   S = Q K^T  128 x 128 into TMEM (kind::f16, FP32 accumulators)
//   softmax    one row per thread: running maximum m and sum l; weights
//              P = 2^(t - m) rounded to the type over S's own columns.  m
//              follows the row's maximum only once it is more than 2^8 behind,
//              so O is rarely rescaled; the weights stay below 2^8.
//   O += P V   P from TMEM, V from shared memory
//
// K and V come through one ring of 16 KB slabs (128 keys x 64 columns), in
// the order in which the products take them.  Key tiles that some row sees
// only in part are checked for non-finite values of V, which a weight of zero
// would turn into NaN: two warps zero them in shared memory before the product,
// and the epilogue adds them back to the rows that see them.
#include "ops_attention_mma.cuh"

namespace svl {
namespace {

constexpr int kThreads = 384;  // warpgroup 0: loads, MMAs, checks; 1 and 2: softmax
constexpr int kRegsControl = 72, kRegsSoftmax = 216;  // 72 + 2 * 216 = 3 * 168

template <int HDP>
struct Shape {
  static constexpr int kRowTiles = HDP <= 128 ? 2 : 1;
  static constexpr int kAhead = HDP <= 128 ? 1 : 2;       // score tiles of a row tile in flight
  static constexpr int kSlabs = HDP / kSlabCols;          // of a K or V tile
  static constexpr int kStages = HDP == 64 ? 12 : HDP == 128 ? 10 : 9;
  static constexpr int kCols = 128 / (3 - kRowTiles);     // score columns of a softmax thread
  static constexpr int kOutCols = kRowTiles == 2 ? HDP : HDP / 2;  // output columns of a softmax thread
  static constexpr uint32_t kOutTmem = 256;
};

struct Mailbox {
  uint32_t slab, segment;
};

template <int HDP>
struct Smem {
  alignas(1024) uint8_t q[Shape<HDP>::kRowTiles * Shape<HDP>::kSlabs * kSlabBytes];
  uint8_t ring[Shape<HDP>::kStages * kSlabBytes];
  uint64_t full[Shape<HDP>::kStages], empty[Shape<HDP>::kStages];
  uint64_t drained, q_full, q_empty, s_full[2], p_ready[2], pv_done[2], check_req, check_done;
  uint32_t tmem;
  Mailbox mail;
  uint32_t spoiled[2];  // 1 + the CTA's last segment of that parity with non-finite values
  float row_max[HDP > 128 ? 2 : 1][2][HDP > 128 ? 128 : 1];
};
static_assert(sizeof(Smem<64>) + 1024 <= kSmemLimit && sizeof(Smem<128>) + 1024 <= kSmemLimit &&
                  sizeof(Smem<256>) + 1024 <= kSmemLimit,
              "shared memory");

// The low `n` bits (none for n <= 0, all for n >= 32).
SVL_DEV uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }

// kind::f16 with A in tensor memory.
SVL_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

SVL_DEV void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const uint32_t tile_rows) {
  using Sh = Shape<HDP>;
  constexpr int kTiles = Sh::kRowTiles, kAhead = Sh::kAhead;
  const int slabs = (p.head_dim + kSlabCols - 1) / kSlabCols;  // of a K or V tile
  const uint32_t stages = Sh::kStages / slabs * slabs;          // whole tiles: theirs lie in one piece
  extern __shared__ uint8_t raw[];
  Smem<HDP>& sm = *(Smem<HDP>*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < (int)stages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.drained, 1);
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_ready[i], kTiles == 2 ? 4 : 8);
      mbar_init(&sm.pv_done[i], 1);
    }
    mbar_init(&sm.check_req, 1);
    mbar_init(&sm.check_done, 64);
    sm.spoiled[0] = sm.spoiled[1] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const uint32_t seg0 = p.block_segments[blockIdx.x], seg1 = p.block_segments[blockIdx.x + 1];

  if (warp < 4) {
    setmaxnreg_dec<kRegsControl>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------- loads --
      const uint32_t q_bytes = tile_rows * 128;  // of one slab
      RingPos pos;
      uint32_t n_segs = 0, issued = 0;
      bool ok = true;
      auto slabs_of = [&](const CUtensorMap* map, uint32_t kvh, int64_t row) {
        for (int s = 0; ok && s < slabs; ++s) {
          if (!mbar_wait(&sm.empty[pos.stage], pos.phase ^ 1, p.err)) {
            ok = false;
            return;
          }
          mbar_arrive_expect_tx(&sm.full[pos.stage], kSlabBytes);
          tma_load_3d(sm.ring + pos.stage * kSlabBytes, map, &sm.full[pos.stage], s * kSlabCols, (int32_t)kvh, (int32_t)row);
          ++issued;
          pos.next(stages);
        }
      };
      for (uint32_t is = seg0; ok && is < seg1; ++is) {
        const AttnSegment seg = p.segments[is];
        const AttnSeq s = p.seqs[seg.seq];
        const uint32_t n = seg.list1 - seg.list0;
        if (!n) continue;
        if (!mbar_wait(&sm.q_empty, (n_segs & 1) ^ 1, p.err)) {
          ok = false;
          break;
        }
        ++n_segs;
        const int tiles = kTiles == 2 && seg.rows > tile_rows ? 2 : 1;
        mbar_arrive_expect_tx(&sm.q_full, tiles * slabs * q_bytes);
        for (int t = 0; t < tiles; ++t)
          for (int c = 0; c < slabs; ++c)
            tma_load_3d(sm.q + (t * Sh::kSlabs + c) * kSlabBytes, &map_q, &sm.q_full, c * kSlabCols,
                        (int32_t)(seg.kvh * p.group), (int32_t)(s.q0 + (seg.row0 + t * tile_rows) / p.group));
        auto key_row = [&](uint32_t j) { return (int64_t)s.k0 + (int64_t)entry_tile(p.lists[seg.list0 + j]) * kKeyTile; };
        for (uint32_t j = 0; j < (uint32_t)kAhead && j < n; ++j) slabs_of(&map_k, seg.kvh, key_row(j));
        for (uint32_t j = 0; ok && j < n; ++j) {
          slabs_of(&map_v, seg.kvh, key_row(j));
          if (j + kAhead < n) slabs_of(&map_k, seg.kvh, key_row(j + kAhead));
        }
      }
      if (!ok) {
        // copies in flight land before the CTA leaves
        RingPos back;
        for (uint32_t i = 0; i < issued; ++i) {
          if (i + stages >= issued) mbar_wait(&sm.full[back.stage], back.phase, p.err);
          back.next(stages);
        }
        if (n_segs) mbar_wait(&sm.q_full, (n_segs - 1) & 1, p.err);
      }
    } else if (warp == 1 && lane == 0) {
      // -------------------------------------------------------------- MMAs --
      constexpr uint32_t kType = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? (1u << 7 | 1u << 10) : 0u;
      const uint32_t idesc_s = idesc_f16(128, 128, 0) | kType;
      const uint32_t q_smem = smem_u32(sm.q), ring_smem = smem_u32(sm.ring);
      const uint32_t hd = p.head_dim;
      RingPos pos;
      uint32_t n_segs = 0, n_checks = 0;
      uint32_t taken[2] = {0, 0};  // p_ready phases
      bool ok = true;
      const int k_steps = (hd + 15) / 16;
      const uint32_t idesc_o = idesc_f16(128, k_steps * 16, 1) | kType;
      // shared-memory descriptors at the first byte; addresses go in in 16s
      const uint64_t q_desc = sdesc(q_smem, 16, 1024, kLayoutSW128), k_desc = sdesc(ring_smem, 16, 1024, kLayoutSW128);
      // V, keys by columns: 64 columns a slab, 16 keys (2 KB) a step
      const uint64_t v_desc = sdesc(ring_smem, kSlabBytes, 1024, kLayoutSW128);
      auto scores = [&](int t, int buf, RingPos at, bool release) {
        uint64_t a = q_desc + t * (Sh::kSlabs * kSlabBytes / 16), b = k_desc + at.stage * (kSlabBytes / 16);
        for (int c = 0; c < slabs; ++c, a += kSlabBytes / 16, b += kSlabBytes / 16) {
          if (!mbar_wait(&sm.full[at.stage], at.phase, p.err)) {
            ok = false;
            return;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c * 4 + k < k_steps) mma_f16(tmem + buf * 128, a + k * 2, b + k * 2, idesc_s, (c | k) != 0);
          if (release) mma_commit(&sm.empty[at.stage]);
          at.next(stages);
        }
        mma_commit(&sm.s_full[buf]);
      };
      auto outputs = [&](int t, int buf, RingPos at, bool accumulate, bool release) {
        const uint64_t b = v_desc + at.stage * (kSlabBytes / 16);
        for (int c = 0; c < slabs; ++c)
          if (!mbar_wait(&sm.full[at.stage + c], at.phase, p.err)) {
            ok = false;
            return;
          }
        tc_fence_after();
        const uint32_t d = tmem + Sh::kOutTmem + t * HDP;
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_f16_ts(d, tmem + buf * 128 + k * 8, b + k * 128, idesc_o, accumulate || k);
        if (release)
          for (int c = 0; c < slabs; ++c) mma_commit(&sm.empty[at.stage + c]);
        mma_commit(&sm.pv_done[buf]);
      };
      // Asks the check warps for a V tile at `at`, once it is there.
      auto ask = [&](RingPos at) {
        for (int c = 0; ok && c < slabs; ++c) {
          const RingPos slab = ahead(at, c, stages);
          if (!mbar_wait(&sm.full[slab.stage], slab.phase, p.err)) ok = false;
        }
        if (!ok) return;
        sm.mail = {at.stage | at.phase << 31, n_segs};
        mbar_arrive(&sm.check_req);
      };
      auto some = [](uint32_t e) { return entry_sees(e, 0) == kSeesSome || entry_sees(e, 1) == kSeesSome; };
      uint32_t g = 0;  // score tiles (one row tile)
      for (uint32_t is = seg0; ok && is < seg1; ++is) {
        const AttnSegment seg = p.segments[is];
        const uint32_t n = seg.list1 - seg.list0;
        if (!n) continue;
        const uint32_t* list = p.lists + seg.list0;
        if (!mbar_wait(&sm.q_full, n_segs & 1, p.err)) {
          ok = false;
          break;
        }
        ++n_segs;
        uint32_t e = list[0], e1 = n > 1 ? list[1] : 0;
        bool checking = false;
        auto checked = [&]() {
          if (!checking) return;
          checking = false;
          if (!mbar_wait(&sm.check_done, n_checks++ & 1, p.err)) ok = false;
        };
        if constexpr (kTiles == 2) {
          auto sees_any = [&](uint32_t x, int t) { return entry_sees(x, t) != kSeesNone; };
          bool started[2] = {false, false};
          for (int t = 0; t < 2; ++t)
            if (sees_any(e, t)) scores(t, t, pos, t == 1 || !sees_any(e, 1));
          if (n == 1) mma_commit(&sm.q_empty);
          pos = ahead(pos, slabs, stages);
          for (uint32_t j = 0; ok && j < n; ++j) {
            const uint32_t e2 = j + 2 < n ? list[j + 2] : 0;  // in flight under this tile's waits
            const RingPos v = pos, k = ahead(pos, slabs, stages);
            const bool more = j + 1 < n;
            if (some(e)) {
              ask(v);
              checking = ok;
            }
            for (int t = 0; ok && t < 2; ++t) {
              if (sees_any(e, t)) {
                if (!mbar_wait(&sm.p_ready[t], taken[t]++ & 1, p.err)) ok = false;
                checked();
                if (!ok) break;
                tc_fence_after();
                outputs(t, t, v, started[t], t == 1 || !sees_any(e, 1));
                started[t] = true;
              }
              if (more && sees_any(e1, t)) scores(t, t, k, t == 1 || !sees_any(e1, 1));
            }
            if (j + 2 == n) mma_commit(&sm.q_empty);
            pos = ahead(pos, more ? 2 * slabs : slabs, stages);
            e = e1;
            e1 = e2;
          }
        } else {
          scores(0, g & 1, pos, true);
          pos = ahead(pos, slabs, stages);
          if (n > 1) {
            scores(0, (g + 1) & 1, pos, true);
            pos = ahead(pos, slabs, stages);
          }
          if (n <= 2) mma_commit(&sm.q_empty);
          for (uint32_t j = 0; ok && j < n; ++j, ++g) {
            const uint32_t e2 = j + 2 < n ? list[j + 2] : 0;
            const int buf = g & 1;
            if (some(e)) {
              ask(pos);
              checking = ok;
            }
            if (!mbar_wait(&sm.p_ready[buf], taken[buf]++ & 1, p.err)) ok = false;
            checked();
            if (!ok) break;
            tc_fence_after();
            outputs(0, buf, pos, j > 0, true);
            pos = ahead(pos, slabs, stages);
            if (j + 2 < n) {
              scores(0, buf, pos, true);
              pos = ahead(pos, slabs, stages);
              if (j + 3 == n) mma_commit(&sm.q_empty);
            }
            e = e1;
            e1 = e2;
          }
        }
      }
      sm.mail = {~0u, 0};
      mbar_arrive(&sm.check_req);
      if (!ok) {  // products in flight end before the CTA leaves
        mma_commit(&sm.drained);
        mbar_wait(&sm.drained, 0, p.err);
      }
    } else if (warp >= 2) {
      // ------------------------------------------------------------ checks --
      const int tid = threadIdx.x - 64;
      for (uint32_t round = 0;; ++round) {
        // between two checks lies any number of fully seen tiles: the limit is 15 times a wait's
        bool got = false;
        for (int i = 0; !got && i < 15; ++i) got = mbar_wait(&sm.check_req, round & 1, nullptr);
        if (!got) {
          atomicOr(p.err, SVL_DEVERR_TIMEOUT);
          break;
        }
        const Mailbox mail = sm.mail;
        if (mail.slab == ~0u) break;
        RingPos at;
        at.stage = mail.slab & 0x7fffffffu;
        at.phase = mail.slab >> 31;
        bool found = false;
        for (int c = 0; c < slabs; ++c) {
          mbar_wait(&sm.full[at.stage], at.phase, p.err);  // passed already: orders this thread's reads
          uint4* slab = (uint4*)(sm.ring + at.stage * kSlabBytes);
          uint32_t most[4] = {};
#pragma unroll 8
          for (int i = 0; i < kSlabBytes / 16 / 64; ++i) {
            const uint4 w = slab[i * 64 + tid];
            most[0] = max_abs(T(), most[0], w.x);
            most[1] = max_abs(T(), most[1], w.y);
            most[2] = max_abs(T(), most[2], w.z);
            most[3] = max_abs(T(), most[3], w.w);
          }
          if (non_finite(T(), most[0]) | non_finite(T(), most[1]) | non_finite(T(), most[2]) | non_finite(T(), most[3])) {
            found = true;
#pragma unroll 1
            for (int i = 0; i < kSlabBytes / 16 / 64; ++i) {
              const uint4 w = slab[i * 64 + tid];
              auto zero = [](uint32_t x) { return x & ~((non_finite(T(), x) >> 15) * 0xffffu); };
              slab[i * 64 + tid] = make_uint4(zero(w.x), zero(w.y), zero(w.z), zero(w.w));
            }
          }
          at.next(stages);
        }
        if (found) sm.spoiled[mail.segment & 1] = mail.segment;
        fence_async_smem();
        mbar_arrive(&sm.check_done);
      }
    }
  } else {
    // -------------------------------------------------------------- softmax --
    setmaxnreg_inc<kRegsSoftmax>();
    const int wg = (warp - 4) >> 2, lg = warp & 3;
    const int t = kTiles == 2 ? wg : 0;        // row tile
    const int half = kTiles == 2 ? 0 : wg;     // column half
    const int r = lg * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(lg * 32) << 16);
    const uint32_t out_addr = lane_addr + Sh::kOutTmem + (kTiles == 2 ? t * HDP : half * Sh::kOutCols);
    constexpr int kCols = Sh::kCols;
    const bool capped = p.cap > 0.0f, biased = p.slopes != nullptr, plain = !capped && !biased;
    const float scale2 = p.scale * kLog2e;
    const float unit = plain ? scale2 : 1.0f;  // log2 units of a score as it is kept
    const float cap2 = p.cap * kLog2e, cap_arg = capped ? 2.0f * scale2 / p.cap : 0.0f;
    const float behind = kBehind / unit;
    uint32_t g = 0;       // tiles of this warpgroup
    uint32_t n_segs = 0;
    bool dead = false;    // a wait ran out: no more waits, but every step is taken
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      if (!dead && !mbar_wait(bar, phase, p.err)) dead = true;
      __syncwarp();
    };
    // The product of tile g - 1, which takes all earlier ones with it.  A barrier
    // for each score buffer: with one for both, the product before it could be
    // outstanding too, and the parity of the phase would not tell them apart.
    auto product_done = [&]() {
      if (kTiles == 2) wait(&sm.pv_done[t], (g - 1) & 1);
      else wait(&sm.pv_done[(g - 1) & 1], (g - 1) >> 1 & 1);
    };
    for (uint32_t is = seg0; is < seg1; ++is) {
      const AttnSegment seg = p.segments[is];
      const AttnSeq s = p.seqs[seg.seq];
      if (seg.list1 > seg.list0) ++n_segs;
      if (t * tile_rows >= seg.rows) continue;
      const uint32_t in_seg = t * tile_rows + r;
      const bool live = r < (int)tile_rows && in_seg < seg.rows;
      const uint32_t row = seg.row0 + (live ? in_seg : 0), query = row / p.group, head = seg.kvh * p.group + row % p.group;
      const RowMask mask = row_mask(p, s, query);
      const bool sighted = live && mask.doc >= 0;
      const int64_t last = sighted ? min((int64_t)s.n_k - 1, p.causal ? mask.place
                                                             : p.window >= 0 ? mask.place + p.window
                                                                             : (int64_t)s.n_k - 1)
                                   : -1;
      const int64_t first = p.window >= 0 ? max((int64_t)0, mask.place - p.window) : 0;
      const uint32_t prefix = sighted ? s.prefix : 0;
      const float slope2 = biased ? p.slopes[head] * kLog2e : 0.0f;
      float m = -INFINITY, l = 0.0f;
      bool started = false;
      uint32_t entry = seg.list0 < seg.list1 ? p.lists[seg.list0] : 0;
      for (uint32_t il = seg.list0; il < seg.list1; ++il) {
        const uint32_t e = entry;
        if (il + 1 < seg.list1) entry = p.lists[il + 1];
        const uint32_t see = entry_sees(e, t);
        if (see == kSeesNone) continue;
        const int buf = kTiles == 2 ? t : (int)(g & 1);
        wait(&sm.s_full[buf], (kTiles == 2 ? g : g >> 1) & 1);
        tc_fence_after();
        const uint32_t s_addr = lane_addr + buf * 128;
        uint32_t w[kCols];
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_ld32_nowait(s_addr + half * kCols + c * 32, w + c * 32);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) tmem_regs_after_wait(w + c * 32);
        auto x = [&](int c) { return __uint_as_float(w[c]); };
        const int64_t j0 = (int64_t)entry_tile(e) * kKeyTile + half * kCols;
        if (capped) {
          float most = 0.0f;
#pragma unroll
          for (int c = 0; c < kCols; c += 2) most = fmax3(most, fabsf(x(c)), fabsf(x(c + 1)));
          if (__any_sync(0xffffffffu, most > p.cap_limit)) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) w[c] = __float_as_uint(capped_any(x(c), cap_arg, cap2));
          } else {
            capped_small<kCols>(p, w);
          }
        }
        if (biased) {
          const float gap = (float)(mask.place - j0), by = capped ? 1.0f : scale2;
          // the distance |gap - c| is linear in c unless the row's own place lies inside the tile
          if (__all_sync(0xffffffffu, gap >= (float)(kCols - 1) || gap <= 0.0f)) {
            const float rise = gap > 0.0f ? slope2 : -slope2;
            const uint64_t by2 = two(by, by), rise2 = two(rise, rise), start2 = two(-rise * gap, -rise * gap);
#pragma unroll
            for (int c = 0; c < kCols; c += 8) {
              uint64_t t2[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) t2[i] = fma_two(rise2, two((float)(c + 2 * i), (float)(c + 2 * i + 1)), start2);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                apart(fma_two(two(w[c + 2 * i], w[c + 2 * i + 1]), by2, t2[i]), w[c + 2 * i], w[c + 2 * i + 1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < kCols; ++c) w[c] = __float_as_uint(fmaf(x(c), by, -slope2 * fabsf(gap - (float)c)));
          }
        }
        if (see == kSeesSome) {
          const int lo = (int)max((int64_t)0, min(first - j0, (int64_t)kCols));
          const int hi = (int)max((int64_t)-1, min(last - j0, (int64_t)kCols - 1));
          const int pre = (int)max((int64_t)0, min((int64_t)prefix - j0, (int64_t)kCols));
          const int n = (int)max((int64_t)0, min((int64_t)s.n_k - j0, (int64_t)kCols));
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            // one bit a key
            uint32_t bits = bits_below(hi + 1 - c) & ~bits_below(lo - c);
            const uint32_t ahead = bits_below(pre - c);
            if (p.doc_k) {
              // a lane loads a key's document; each document of the 32 in turn gives its keys to its rows
              const int32_t d = c + lane < n ? __ldg(p.doc_k + s.k0 + j0 + c + lane) : -1;
              const uint32_t member = __ballot_sync(0xffffffffu, d >= 0);
              uint32_t own = 0;
              for (uint32_t left = member; left;) {
                const int32_t one = __shfl_sync(0xffffffffu, d, __ffs(left) - 1);
                const uint32_t its = __ballot_sync(0xffffffffu, d == one);
                if (one == mask.doc) own = its;
                left &= ~its;
              }
              bits = (ahead | (bits & own)) & member;
            } else {
              bits |= ahead;
            }
            if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(bits >> i & 1)) w[c + i] = __float_as_uint(-INFINITY);
          }
        }
        float mx[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          constexpr int kPart = kCols / 4;
          mx[u] = x(u * kPart);
#pragma unroll
          for (int c = 1; c + 1 < kPart; c += 2) mx[u] = fmax3(mx[u], x(u * kPart + c), x(u * kPart + c + 1));
          mx[u] = fmaxf(mx[u], x(u * kPart + kPart - 1));
        }
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if constexpr (kTiles == 1) {
          // both halves of a row follow one maximum
          sm.row_max[g & 1][half][r] = top;
          tc_fence_before();  // both halves are read before either is written over
          pair_sync(1 + lg);
          tc_fence_after();
          top = fmaxf(top, sm.row_max[g & 1][half ^ 1][r]);
        }
        float factor = 1.0f;
        if (top > m + behind || (m == -INFINITY && top > -INFINITY)) {
          factor = m == -INFINITY ? 0.0f : ex2_approx((m - top) * unit);
          m = top;
        }
        if (started && __any_sync(0xffffffffu, factor != 1.0f)) {
          product_done();  // O stands still until this tile's weights are handed over
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < Sh::kOutCols; c += 32) {
            float o[32];
            tmem_ld32(out_addr + c, o);
#pragma unroll
            for (int u = 0; u < 32; ++u) o[u] *= factor;
            tmem_st32(out_addr + c, o);
          }
        }
        started = true;
        __syncwarp();
        const float base = m == -INFINITY ? 0.0f : m * unit;
        const uint64_t unit2 = two(unit, unit), base2 = two(-base, -base);
        uint64_t sum[4] = {0, 0, 0, 0};  // pairs of 0.0f
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 16; u += 4) {
            uint64_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fma_two(two(w[c + 2 * (u + i)], w[c + 2 * (u + i) + 1]), unit2, base2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a, b;
              apart(y[i], a, b);
              const float ea = ex2_approx(__uint_as_float(a)), eb = ex2_approx(__uint_as_float(b));
              sum[i] = add_two(sum[i], two(ea, eb));
              pk[u + i] = pack2(T(), ea, eb);
            }
          }
          tmem_st16(s_addr + (half * kCols + c) / 2, pk);
        }
        uint32_t part[2];
        apart(add_two(add_two(sum[0], sum[1]), add_two(sum[2], sum[3])), part[0], part[1]);
        l = l * factor + (__uint_as_float(part[0]) + __uint_as_float(part[1]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_ready[buf]);
        ++g;
      }
      // ------------------------------------------------------------ epilogue --
      if constexpr (kTiles == 1) {
        const int at = g & 1;  // the next tile writes the other parity's slot first
        sm.row_max[at][half][r] = l;
        pair_sync(1 + lg);
        l += sm.row_max[at][half ^ 1][r];
        pair_sync(1 + lg);
      }
      if (started) product_done();
      tc_fence_after();
      const bool spoiled = started && sm.spoiled[n_segs & 1] == n_segs;
      const bool empty = !started || (m == -INFINITY && l == 0.0f);
      const float inv = empty ? 0.0f : 1.0f / l;
      const float lse = empty ? -INFINITY : kLn2 * ((m == -INFINITY ? 0.0f : m * unit) + log2f(l));
      const uint64_t token = s.q0 + query;
      const uint64_t part = (uint64_t)(seg.slot < 0 ? 0 : seg.slot) * p.slot_rows + in_seg;
      if (live && half == 0) {
        if (seg.slot >= 0) p.part_lse[part] = lse;
        else if (p.lse) p.lse[token * p.q_heads + head] = lse;
      }
#pragma unroll 1
      for (int c = 0; c < Sh::kOutCols; c += 32) {
        const uint32_t col0 = (kTiles == 1 ? half * Sh::kOutCols : 0) + c;
        if (col0 >= p.head_dim) break;
        float o[32];
        if (started) {
          tmem_ld32(out_addr + c, o);
        }
#pragma unroll
        for (int u = 0; u < 32; ++u) o[u] = empty ? 0.0f : o[u] * inv;
        if (spoiled) {
          float extra[32];
#pragma unroll
          for (int u = 0; u < 32; ++u) extra[u] = o[u];
          if (live) add_spoiled<T>(p, seg, s, query, col0, extra);
#pragma unroll
          for (int u = 0; u < 32; ++u) o[u] = extra[u];
        }
        if (live && seg.slot >= 0) {
          float* dst = p.part_o + part * p.head_dim + col0;
#pragma unroll
          for (int u = 0; u < 32; u += 4)
            if (col0 + u < p.head_dim) *(float4*)(dst + u) = make_float4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        } else if (live) {
          T* dst = (T*)p.out + token * p.ld_out + (uint64_t)head * p.head_dim + col0;
#pragma unroll
          for (int u = 0; u < 32; u += 8)
            if (col0 + u < p.head_dim)
              *(uint4*)(dst + u) = make_uint4(pack2(T(), o[u], o[u + 1]), pack2(T(), o[u + 2], o[u + 3]),
                                              pack2(T(), o[u + 4], o[u + 5]), pack2(T(), o[u + 6], o[u + 7]));
        }
        __syncwarp();  // TMEM loads are the whole warp's
      }
      tc_fence_before();  // O is read before the next segment's first weights are handed over
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int HDP>
cudaError_t launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int smem = (int)sizeof(Smem<HDP>) + 1024;
  const cudaError_t e = smem_opt_in(attention_tc_kernel<T, HDP>, smem, &done);
  if (e != cudaSuccess) return e;
  // the registers that setmaxnreg hands over have to come out of the launch's own: an increase beyond them never ends
  static std::atomic<int> fits{-1};
  if (fits.load() < 0) {
    cudaFuncAttributes fa{};
    const cudaError_t f = cudaFuncGetAttributes(&fa, attention_tc_kernel<T, HDP>);
    if (f != cudaSuccess) return f;
    fits.store(kRegsControl + 2 * kRegsSoftmax <= 3 * fa.numRegs && kRegsControl <= fa.numRegs &&
               fa.numRegs <= kRegsSoftmax);
  }
  if (!fits.load()) return cudaErrorInvalidConfiguration;
  const uint32_t rows = attention_tc_tile_rows(p.group);
  CUtensorMap q, k, v;
  if (!encode_fn() ||
      !head_map(&q, p.q, dtype, p.total_q, p.q_heads, p.head_dim, p.ld_q, p.group, rows / p.group) ||
      !head_map(&k, p.total_k ? p.k : p.q, dtype, p.total_k ? p.total_k : 1, p.total_k ? p.kv_heads : 1, p.head_dim,
                p.total_k ? p.ld_k : p.ld_q, 1, kKeyTile) ||
      !head_map(&v, p.total_k ? p.v : p.q, dtype, p.total_k ? p.total_k : 1, p.total_k ? p.kv_heads : 1, p.head_dim,
                p.total_k ? p.ld_v : p.ld_q, 1, kKeyTile))
    return cudaErrorInvalidValue;
  attention_tc_kernel<T, HDP><<<p.blocks, kThreads, smem, st>>>(p, q, k, v, rows);
  return cudaGetLastError();
}

}  // namespace

bool attention_tc_takes(const svl_attention_config& c, uint64_t total_q, uint64_t total_k) {
  // a TMA coordinate is an int32, and a box of 128 rows starts at most there
  return c.dtype != SVL_DTYPE_F32 && c.head_dim % 8 == 0 && c.head_dim <= 256 && c.q_heads / c.kv_heads <= 128 &&
         total_q < (1ull << 31) - 256 && total_k < (1ull << 31) - 256;
}

uint32_t attention_tc_tile_rows(uint32_t group) { return 128 / group * group; }
uint32_t attention_tc_row_tiles(uint32_t head_dim) { return head_dim <= 128 ? 2 : 1; }

cudaError_t attention_tc_launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  const bool half = dtype == SVL_DTYPE_F16;
  if (p.head_dim <= 64) return half ? launch<__half, 64>(p, dtype, st) : launch<__nv_bfloat16, 64>(p, dtype, st);
  if (p.head_dim <= 128) return half ? launch<__half, 128>(p, dtype, st) : launch<__nv_bfloat16, 128>(p, dtype, st);
  return half ? launch<__half, 256>(p, dtype, st) : launch<__nv_bfloat16, 256>(p, dtype, st);
}

}  // namespace svl
