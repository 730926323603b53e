// ops_attention_tc.cu -- the FP16 / BF16 attention kernel of svl_attention_*
// on the 5th-generation tensor cores.
//
// One persistent CTA per SM walks its segments (rows of one key-value head
// against a list of 128-key tiles).  A row tile is up to 128 (query, head of the
// group) rows, so every head of a group reads a key tile once.  Head sizes up to
// 128: two row tiles share each key tile, so that one tile's products run under
// the other's softmax.  Head sizes up to 256: one row tile with two score
// buffers.  Two softmax warpgroups share a row tile, 64 of a key tile's columns
// each: with one of them a scheduler has a single softmax warp for each row tile,
// whose chains of dependent instructions do not fill it (2 sequences of 6000-8192
// tokens, 16 query and 2 key heads of 128, causal behind a prefix, capped: 597 us
// with one, 538 with two at the same state of the rest).
//
//   S = Q K^T  128 x 128 into TMEM (kind::f16, FP32 accumulators)
//   softmax    half a row per thread: running maximum m and sum l; weights
//              P = 2^(t - m) rounded to the type over S's own columns.  m
//              follows the row's maximum only once it is more than 2^8 behind,
//              so O is rarely rescaled; the weights stay below 2^8.
//   O += P V   P from TMEM, V from shared memory
//
// K and V tiles come through one ring, in slabs of 128 keys x 64 columns, in the
// order in which the products take them.  Key tiles that some row sees
// only in part are checked for non-finite values of V, which a weight of zero
// would turn into NaN: two warps zero them in shared memory before the product,
// and the epilogue adds them back to the rows that see them.
//
// What bounds it: the round from a row tile's scores through its softmax and back
// to the products.  On that case (437-474 us from box to box, 730-790 TFLOP/s
// counted over visible pairs) the products alone, with the softmax only handing
// over, take 307 us; S reads both operands from shared memory, 8 KB a 64-cycle step,
// which is all its bandwidth.  Of 440 us, leaving out the cap's polynomial saves 63,
// the maximum 45, the exponentials 26.  On a shorter such batch the tensor pipe is
// active 36% of the cycles, the special functions 37%, and a scheduler issues in 54%.
#include "ops_attention_mma.cuh"

namespace svl {
namespace {

constexpr int kCols = 64;  // score columns of a softmax thread
// Behind this size (log2 units) a score and its bias are rounded before the maximum
// is subtracted.  Below it the subtraction may share a multiply-add with the product
// and the bias may run along the columns in steps: the maximum and the exponents then
// differ by up to 16 2^-24 of the size, at most 1, where a weight has to stay below 2^16.
// The rows of a warp (all of one sequence) share the choice.
constexpr float kMild = 1048576.0f;
// Tensor-memory columns of the weights of keys 16 k ..: each thread's lie over its own scores.
SVL_DEV uint32_t weights_at(int k) { return k * 16 / kCols * kCols + k * 16 % kCols / 2; }

template <int HDP>
struct Shape {
  static constexpr int kRowTiles = HDP <= 128 ? 2 : 1;
  static constexpr int kAhead = HDP <= 128 ? 1 : 2;       // score tiles of a row tile in flight
  static constexpr int kSlabs = HDP / kSlabCols;          // of a K or V tile
  static constexpr int kRingSlabs = HDP == 64 ? 11 : 9;
  static constexpr int kOutCols = HDP / 2;                // output columns of a softmax thread
  static constexpr uint32_t kOutTmem = 256;
  // warpgroup 0: loads, MMAs, checks; the others: softmax
  static constexpr int kSoftmax = 2 * kRowTiles, kThreads = 128 * (1 + kSoftmax);
  static constexpr int kRegs = kRowTiles == 2 ? 96 : 168;  // of a thread at launch: 65536 / kThreads, in eights
  static constexpr int kRegsControl = kRowTiles == 2 ? 64 : 72;
  static constexpr int kRegsSoftmax = kRowTiles == 2 ? 104 : 216;
  static_assert(kRegsControl + kSoftmax * kRegsSoftmax == (1 + kSoftmax) * kRegs, "registers move inside the launch's own");
};

// What the check warps are asked for: a ring stage with its phase in the top bit
// (all ones: nothing more), and for each row tile that sees the key tile its turn:
// 1 for the first segment of the CTA in which the row tile sees a key, 2 for the
// next such segment, and so on; 0 if it does not see this key tile.
struct Mailbox {
  uint32_t stage, turn[2];
};

template <int HDP>
struct Smem {
  alignas(1024) uint8_t q[Shape<HDP>::kRowTiles * Shape<HDP>::kSlabs * kSlabBytes];
  uint8_t ring[Shape<HDP>::kRingSlabs * kSlabBytes];
  uint64_t full[Shape<HDP>::kRingSlabs], empty[Shape<HDP>::kRingSlabs];
  uint64_t drained, q_full, q_empty, s_full[2], p_ready[2], pv_done[2], check_req, check_done;
  uint32_t tmem;
  Mailbox mail;
  // [row tile][parity]: its last turn of that parity with non-finite values.  A check
  // for turn k + 2 follows the products of turn k + 1, which wait for the weights of all
  // of the row tile's warps, and these have read the flag of turn k by then.
  uint32_t spoiled[2][2];
  float shared_row[2][Shape<HDP>::kRowTiles][2][128];  // [parity][row tile][half]: maxima, sums
};
static_assert(sizeof(Smem<64>) + 1024 <= kSmemLimit && sizeof(Smem<128>) + 1024 <= kSmemLimit &&
                  sizeof(Smem<256>) + 1024 <= kSmemLimit,
              "shared memory");

// A step of the transposition of four lanes' four units: lanes l and l ^ D swap
// the off-diagonal blocks of theirs.
template <int D>
SVL_DEV void exchange(uint4* v, int lane) {
  const bool upper = lane & D;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (u & D) continue;
    uint4 give = upper ? v[u] : v[u | D];
    give.x = __shfl_xor_sync(0xffffffffu, give.x, D);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, D);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, D);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, D);
    if (upper) v[u] = give;
    else v[u | D] = give;
  }
}

SVL_DEV float fmin3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The low `n` bits (none for n <= 0, all for n >= 32).
SVL_DEV uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }

// A value that is the same in every lane, as one that the compiler knows to be.
SVL_DEV uint32_t one_of(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

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

// FULL: heads of HDP columns, not fewer.
template <typename T, int HDP, bool FULL>
__global__ void __launch_bounds__(Shape<HDP>::kThreads, 1)
    attention_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const uint32_t tile_rows) {
  using Sh = Shape<HDP>;
  constexpr int kTiles = Sh::kRowTiles, kAhead = Sh::kAhead;
  const int slabs = FULL ? HDP / kSlabCols : (p.head_dim + kSlabCols - 1) / kSlabCols;  // of a K or V tile
  const uint32_t stages = Sh::kRingSlabs / slabs, stage_bytes = slabs * kSlabBytes;         // a stage is a tile
  extern __shared__ uint8_t raw[];
  Smem<HDP>& sm = *(Smem<HDP>*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = one_of(threadIdx.x >> 5), lane = threadIdx.x & 31;

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
      mbar_init(&sm.p_ready[i], 8);
      mbar_init(&sm.pv_done[i], 1);
    }
    mbar_init(&sm.check_req, 1);
    mbar_init(&sm.check_done, 64);
    for (int i = 0; i < 4; ++i) sm.spoiled[i / 2][i % 2] = 0;
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
    setmaxnreg_dec<Sh::kRegsControl>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------- loads --
      const uint32_t q_bytes = tile_rows * 128;  // of one slab
      RingPos pos;
      uint32_t n_segs = 0, issued = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, uint32_t kvh, int64_t row) {
        if (!mbar_wait(&sm.empty[pos.stage], pos.phase ^ 1, p.err)) {
          ok = false;
          return;
        }
        mbar_arrive_expect_tx(&sm.full[pos.stage], stage_bytes);
        for (int c = 0; c < slabs; ++c)
          tma_load_3d(sm.ring + pos.stage * stage_bytes + c * kSlabBytes, map, &sm.full[pos.stage], c * kSlabCols,
                      (int32_t)kvh, (int32_t)row);
        ++issued;
        pos.next(stages);
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
        for (uint32_t j = 0; ok && j < (uint32_t)kAhead && j < n; ++j) load(&map_k, seg.kvh, key_row(j));
        for (uint32_t j = 0; ok && j < n; ++j) {
          load(&map_v, seg.kvh, key_row(j));
          if (ok && j + kAhead < n) load(&map_k, seg.kvh, key_row(j + kAhead));
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
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMAs --
      // The whole warp walks the products and one of its threads issues them: the
      // instruction takes its descriptors from uniform registers, which a branch
      // that one thread takes alone does not compute in (200 cycles a product).
      constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7 | 1u << 10) : 0u;
      const uint32_t idesc_s = idesc_f16(128, 128, 0) | kType;
      const int k_steps = FULL ? HDP / 16 : (p.head_dim + 15) / 16;
      const uint32_t idesc_o = idesc_f16(128, k_steps * 16, 1) | kType;
      // shared-memory descriptors at the first byte; addresses go in in 16s
      const uint64_t q_desc = sdesc(smem_u32(sm.q), 16, 1024, kLayoutSW128);
      const uint64_t k_desc = sdesc(smem_u32(sm.ring), 16, 1024, kLayoutSW128);
      // V, keys by columns: 64 columns a slab, 16 keys (2 KB) a step
      const uint64_t v_desc = sdesc(smem_u32(sm.ring), kSlabBytes, 1024, kLayoutSW128);
      RingPos pos;
      uint32_t n_segs = 0, n_checks = 0, turn[2] = {0, 0};
      uint32_t taken[2] = {0, 0};  // p_ready phases
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t phase) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, phase, p.err));
      };
      // by one thread: S of a row tile against the K tile at `at`; the last row tile gives the K tile back
      auto scores = [&](int t, int buf, RingPos at, bool release) {
        const uint64_t a = q_desc + t * (Sh::kSlabs * kSlabBytes / 16), b = k_desc + at.stage * (stage_bytes / 16);
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k)
          if (FULL || k < k_steps) {
            const int step = k / 4 * (kSlabBytes / 16) + k % 4 * 2;
            mma_f16(tmem + buf * 128, a + step, b + step, idesc_s, k != 0);
          }
        mma_commit(&sm.s_full[buf]);
        if (release) mma_commit(&sm.empty[at.stage]);
      };
      // by one thread: O of a row tile += P V
      auto outputs = [&](int t, int buf, RingPos at, bool accumulate, bool release) {
        const uint64_t b = v_desc + at.stage * (stage_bytes / 16);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_f16_ts(tmem + Sh::kOutTmem + t * HDP, tmem + buf * 128 + weights_at(k), b + k * 128, idesc_o,
                     k ? 1 : accumulate);
        mma_commit(&sm.pv_done[buf]);
        if (release) mma_commit(&sm.empty[at.stage]);
      };
      // Asks the check warps for the V tile at `at`, which is there, for the turns of the two row tiles.
      bool checking = false;
      auto ask = [&](RingPos at, uint32_t turn0, uint32_t turn1) {
        if (ok && lane == 0) {
          sm.mail = {at.stage | at.phase << 31, {turn0, turn1}};
          mbar_arrive(&sm.check_req);
        }
        __syncwarp();
        checking = ok;
      };
      auto checked = [&]() {
        if (checking) wait(&sm.check_done, n_checks++ & 1);
        checking = false;
      };
      auto some = [](uint32_t e) { return entry_sees(e, 0) == kSeesSome || entry_sees(e, 1) == kSeesSome; };
      uint32_t g = 0;  // score tiles (one row tile)
      for (uint32_t is = seg0; ok && is < seg1; ++is) {
        const uint32_t list0 = one_of(p.segments[is].list0), n = one_of(p.segments[is].list1) - list0;
        if (!n) continue;
        const uint32_t* list = p.lists + list0;
        // entries come a tile ahead of their use
        uint32_t e = one_of(list[0]), e1 = n > 1 ? one_of(list[1]) : 0;
        wait(&sm.q_full, n_segs & 1);
        ++n_segs;
        wait(&sm.full[pos.stage], pos.phase);
        if constexpr (kTiles == 2) {
          auto sees_any = [&](uint32_t x, int t) { return entry_sees(x, t) != kSeesNone; };
          bool started[2] = {false, false};
          tc_fence_after();
          if (ok && elect_one()) {
            if (sees_any(e, 0)) scores(0, 0, pos, !sees_any(e, 1));
            if (sees_any(e, 1)) scores(1, 1, pos, true);
            if (n == 1) mma_commit(&sm.q_empty);
          }
          __syncwarp();
          pos.next(stages);
          for (uint32_t j = 0; ok && j < n; ++j) {
            const uint32_t e2 = j + 2 < n ? list[j + 2] : 0;
            const bool more = j + 1 < n;
            const RingPos v = pos, k = ahead(pos, 1, stages);
            wait(&sm.full[v.stage], v.phase);
            if (more) wait(&sm.full[k.stage], k.phase);
            if (some(e)) ask(v, sees_any(e, 0) ? turn[0] + !started[0] : 0, sees_any(e, 1) ? turn[1] + !started[1] : 0);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const bool now = sees_any(e, t), then = more && sees_any(e1, t);
              if (now) {
                wait(&sm.p_ready[t], taken[t]++ & 1);
                checked();
              }
              tc_fence_after();
              if (ok && elect_one()) {
                if (now) outputs(t, t, v, started[t], t == 1 || !sees_any(e, 1));
                if (then) scores(t, t, k, t == 1 || !sees_any(e1, 1));
              }
              __syncwarp();
              turn[t] += now && !started[t];
              started[t] |= now;
            }
            if (j + 2 == n && ok && elect_one()) mma_commit(&sm.q_empty);
            pos = ahead(pos, more ? 2 : 1, stages);
            e = e1;
            e1 = one_of(e2);
          }
        } else {
          tc_fence_after();
          if (ok && elect_one()) scores(0, g & 1, pos, true);
          __syncwarp();
          pos.next(stages);
          if (n > 1) {
            wait(&sm.full[pos.stage], pos.phase);
            tc_fence_after();
            if (ok && elect_one()) scores(0, (g + 1) & 1, pos, true);
            __syncwarp();
            pos.next(stages);
          }
          if (n <= 2 && ok && elect_one()) mma_commit(&sm.q_empty);
          for (uint32_t j = 0; ok && j < n; ++j, ++g) {
            const uint32_t e2 = j + 2 < n ? list[j + 2] : 0;
            const int buf = g & 1;
            wait(&sm.full[pos.stage], pos.phase);
            if (some(e)) ask(pos, n_segs, 0);  // every key tile of the list is seen: a turn a segment
            wait(&sm.p_ready[buf], taken[buf]++ & 1);
            checked();
            tc_fence_after();
            if (ok && elect_one()) outputs(0, buf, pos, j > 0, true);
            __syncwarp();
            pos.next(stages);
            if (j + 2 < n) {
              wait(&sm.full[pos.stage], pos.phase);
              tc_fence_after();
              if (ok && elect_one()) {
                scores(0, buf, pos, true);
                if (j + 3 == n) mma_commit(&sm.q_empty);
              }
              __syncwarp();
              pos.next(stages);
            }
            e = e1;
            e1 = one_of(e2);
          }
        }
      }
      if (lane == 0) {
        sm.mail = {~0u, {0, 0}};
        mbar_arrive(&sm.check_req);
        if (!ok) {  // products in flight end before the CTA leaves
          mma_commit(&sm.drained);
          mbar_wait(&sm.drained, 0, p.err);
        }
      }
      __syncwarp();
    } else if (warp >= 2) {
      // ------------------------------------------------------------ checks --
      const int tid = threadIdx.x - 64;
      for (uint32_t round = 0;; ++round) {
        // between two checks lies any number of fully seen tiles: the limit goes by the block's tiles
        bool got = false;
        for (uint32_t i = 0; !got && i < p.check_waits; ++i) got = mbar_wait(&sm.check_req, round & 1, nullptr);
        if (!got) {
          atomicOr(p.err, SVL_DEVERR_TIMEOUT);
          break;
        }
        const Mailbox mail = sm.mail;
        if (mail.stage == ~0u) break;
        RingPos at;
        at.stage = mail.stage & 0x7fffffffu;
        at.phase = mail.stage >> 31;
        bool found = false;
        mbar_wait(&sm.full[at.stage], at.phase, p.err);  // passed already: orders this thread's reads
        for (int c = 0; c < slabs; ++c) {
          uint4* slab = (uint4*)(sm.ring + at.stage * stage_bytes + c * kSlabBytes);
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
        }
        if (found)
          for (int t = 0; t < 2; ++t)
            if (mail.turn[t]) sm.spoiled[t][mail.turn[t] & 1] = mail.turn[t];
        fence_async_smem();
        mbar_arrive(&sm.check_done);
      }
    }
  } else {
    // -------------------------------------------------------------- softmax --
    setmaxnreg_inc<Sh::kRegsSoftmax>();
    const int wg = (warp - 4) >> 2, lg = warp & 3;
    const int t = wg >> 1, half = wg & 1;  // row tile, columns
    const int r = lg * 32 + lane;
    const int pair = 1 + t * 4 + lg;       // the barrier of the two warps of these rows
    const uint32_t lane_addr = tmem + ((uint32_t)(lg * 32) << 16);
    const uint32_t out_addr = lane_addr + Sh::kOutTmem + t * HDP + half * Sh::kOutCols;
    const bool capped = p.cap > 0.0f, biased = p.slopes != nullptr, plain = !capped && !biased;
    // capped_large is off by up to 2^-20 of the cap, and a weight must stay below
    // 2^16 (FP16): from the largest raw score on (below) only with caps that leave
    // that error under 2^1; higher ones take the maximum of the transformed scores
    const bool mild_cap = p.cap <= 1e6f;
    const float scale2 = p.scale * kLog2e;
    const float cap2 = p.cap * kLog2e, cap_arg = capped ? 2.0f * scale2 / p.cap : 0.0f;
    uint32_t g = 0;       // tiles of this warpgroup
    uint32_t turn = 0;    // segments in which this row tile has seen a key
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
        const int64_t j0 = (int64_t)entry_tile(e) * kKeyTile + half * kCols;
        // a lane loads two keys' documents, under the wait for the scores
        int32_t docs[2] = {-1, -1};
        if (p.doc_k && see == kSeesSome) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (j0 + 32 * h + lane < (int64_t)s.n_k) docs[h] = __ldg(p.doc_k + s.k0 + j0 + 32 * h + lane);
        }
        const uint32_t s_addr = lane_addr + buf * 128 + half * kCols;
        // Tiles that a row sees whole need nothing but the maximum (and, for the
        // cap, the minimum) here, and their scores are transformed where they are
        // exponentiated.  The distance is linear over columns that the row's own
        // place does not lie among; the bias has to be mild over them.  In all other
        // cases the transformed scores go back to TMEM.
        const float gap = (float)(mask.place - j0);
        const bool apart_from = (gap >= (float)(kCols - 1) || gap <= 0.0f) && fabsf(slope2) * (fabsf(gap) + kCols) <= kMild;
        const bool direct = see == kSeesAll && (plain || (capped != biased && (capped ? mild_cap : __all_sync(0xffffffffu, apart_from))));
        const float rise = gap > 0.0f ? slope2 : -slope2;  // direct bias: -slope |gap - c| = rise (c - gap)
        wait(&sm.s_full[buf], (kTiles == 2 ? g : g >> 1) & 1);
        tc_fence_after();
        float top = -INFINITY;
        bool small = true;   // every score within the cap's polynomial
        bool raw = direct;   // the scores in TMEM stay as they are
        if (direct) {
          float low = INFINITY;
#pragma unroll 1
          for (int c0 = 0; c0 < kCols; c0 += 32) {
            uint32_t w[32];
            tmem_ld32_nowait(s_addr + c0, w);
            tmem_ld_wait();
            tmem_regs_after_wait(w);
            auto x = [&](int c) { return __uint_as_float(w[c]); };
            if (biased) {
              const uint64_t by2 = two(scale2, scale2), rise2 = two(2.0f * rise, 2.0f * rise);
              uint64_t t2 = two(rise * ((float)c0 - gap), rise * ((float)c0 - gap) + rise);
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                apart(fma_two(two(w[c], w[c + 1]), by2, t2), w[c], w[c + 1]);
                t2 = add_two(t2, rise2);
              }
            }
            float mx[2] = {x(0), x(1)};
#pragma unroll
            for (int c = 2; c < 32; c += 4) {
              mx[0] = fmax3(mx[0], x(c), x(c + 1));
              if (c + 2 < 32) mx[1] = fmax3(mx[1], x(c + 2), x(c + 3));
            }
            top = fmax3(top, mx[0], mx[1]);
            if (capped) {
              float mn[2] = {x(0), x(1)};
#pragma unroll
              for (int c = 2; c < 32; c += 4) {
                mn[0] = fmin3(mn[0], x(c), x(c + 1));
                if (c + 2 < 32) mn[1] = fmin3(mn[1], x(c + 2), x(c + 3));
              }
              low = fmin3(low, mn[0], mn[1]);
            }
          }
          if (plain) top *= scale2;
          if (capped) {
            small = !__any_sync(0xffffffffu, live && fmaxf(top, -low) > p.cap_limit);
            // the cap keeps the order
            const float by = small ? capped_small(p, top) : capped_any(p, top, cap_arg, cap2);
            top = top == -INFINITY ? top : by;
          } else {
            raw = !__any_sync(0xffffffffu, live && fabsf(top) > kMild);
            if (!raw) top = -INFINITY;
          }
        }
        if (!raw)
#pragma unroll 1
        for (int c0 = 0; c0 < kCols; c0 += 32) {
          uint32_t w[32];
          tmem_ld32_nowait(s_addr + c0, w);
          tmem_ld_wait();
          tmem_regs_after_wait(w);
          auto x = [&](int c) { return __uint_as_float(w[c]); };
          if (capped) {
            float most = 0.0f;
#pragma unroll
            for (int c = 0; c < 32; c += 2) most = fmax3(most, fabsf(x(c)), fabsf(x(c + 1)));
            if (__any_sync(0xffffffffu, live && most > p.cap_limit)) {
#pragma unroll
              for (int c = 0; c < 32; ++c) w[c] = __float_as_uint(capped_any(p, x(c), cap_arg, cap2));
            } else {
              capped_small<32>(p, w);
            }
          }
          if (biased) {
            const float from = gap - (float)c0, by = capped ? 1.0f : scale2;
#pragma unroll
            for (int c = 0; c < 32; ++c) w[c] = __float_as_uint(fmaf(x(c), by, -slope2 * fabsf(from - (float)c)));
          } else if (!capped) {
#pragma unroll
            for (int c = 0; c < 32; ++c) w[c] = __float_as_uint(x(c) * scale2);
          }
          if (see == kSeesSome) {
            const int64_t j = j0 + c0;
            // one bit a key
            uint32_t bits = bits_below((int)max((int64_t)0, min(last + 1 - j, (int64_t)32))) &
                            ~bits_below((int)max((int64_t)0, min(first - j, (int64_t)32)));
            const uint32_t ahead = bits_below((int)max((int64_t)0, min((int64_t)prefix - j, (int64_t)32)));
            if (p.doc_k) {
              // each document of the 32 in turn gives its keys to its rows
              const int32_t d = c0 ? docs[1] : docs[0];
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
            if (!__all_sync(0xffffffffu, bits == 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(bits >> i & 1)) w[i] = __float_as_uint(-INFINITY);
            }
          }
          float mx[2] = {x(0), x(1)};
#pragma unroll
          for (int c = 2; c < 32; c += 4) {
            mx[0] = fmax3(mx[0], x(c), x(c + 1));
            if (c + 2 < 32) mx[1] = fmax3(mx[1], x(c + 2), x(c + 3));
          }
          top = fmax3(top, mx[0], mx[1]);
          __syncwarp();
          tmem_st32(s_addr + c0, w);
          tmem_st_wait();
        }
        // both halves of a row follow one maximum
        sm.shared_row[g & 1][t][half][r] = top;
        pair_sync(pair);
        top = fmaxf(top, sm.shared_row[g & 1][t][half ^ 1][r]);
        float factor = 1.0f;
        if (top > m + kBehind || (m == -INFINITY && top > -INFINITY)) {
          factor = m == -INFINITY ? 0.0f : ex2_approx(m - top);
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
        turn += !started;
        started = true;
        __syncwarp();
        const float base = m == -INFINITY ? 0.0f : m;
        uint64_t sum[2] = {0, 0};  // pairs of 0.0f
        // 2^(t - m) of 32 columns; `exponents` makes four pairs of t - m from four of scores
        auto weights = [&](auto&& exponents) {
#pragma unroll 1
          for (int c0 = 0; c0 < kCols; c0 += 32) {
            uint32_t w[32], pk[16];
            tmem_ld32_nowait(s_addr + c0, w);
            tmem_ld_wait();
            tmem_regs_after_wait(w);
#pragma unroll
            for (int u = 0; u < 16; u += 4) {
              uint64_t y[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = two(w[2 * (u + i)], w[2 * (u + i) + 1]);
              exponents(y, c0 + 2 * u);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t a, b;
                apart(y[i], a, b);
                const float ea = ex2_approx(__uint_as_float(a)), eb = ex2_approx(__uint_as_float(b));
                sum[i & 1] = add_two(sum[i & 1], two(ea, eb));
                pk[u + i] = pack2(T(), ea, eb);
              }
            }
            tmem_st16(s_addr + c0 / 2, pk);  // over what this warp has read of these columns
          }
        };
        const uint64_t base2 = two(-base, -base);
        if (!raw) {
          weights([&](uint64_t* y, int) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = add_two(y[i], base2);
          });
        } else if (capped) {
          if (small) {
            const CapOdd odd(p);
            weights([&](uint64_t* y, int) {
              uint64_t r[4];
              odd.over(y, r);
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = fma_two(y[i], r[i], base2);
            });
          } else {
            // the same bits as above for each score within the limit
            auto exponent = [&](uint32_t w) {
              const float s = __uint_as_float(w);
              return by_size(p, s, fmaf(s, cap_odd(p, s), -base), capped_large(s, cap_arg, cap2) - base);
            };
            weights([&](uint64_t* y, int) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t a, b;
                apart(y[i], a, b);
                y[i] = two(exponent(a), exponent(b));
              }
            });
          }
        } else {
          // biased: rise (c - gap); plain: no rise
          const float up = biased ? rise : 0.0f, start = biased ? -rise * gap - base : -base;
          const uint64_t by2 = two(scale2, scale2), up2 = two(2.0f * up, 2.0f * up);
          weights([&](uint64_t* y, int c) {
            if (biased) {
              uint64_t t2 = two(fmaf(up, (float)c, start), fmaf(up, (float)(c + 1), start));
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                y[i] = fma_two(y[i], by2, t2);
                t2 = add_two(t2, up2);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = fma_two(y[i], by2, base2);
            }
          });
        }
        uint32_t part[2];
        apart(add_two(sum[0], sum[1]), part[0], part[1]);
        l = l * factor + (__uint_as_float(part[0]) + __uint_as_float(part[1]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_ready[buf]);
        ++g;
      }
      // ------------------------------------------------------------ epilogue --
      {
        const int at = g & 1;  // not the last tile's slot, and the next tile writes this one after the barrier
        sm.shared_row[at][t][half][r] = l;
        pair_sync(pair);
        l += sm.shared_row[at][t][half ^ 1][r];
        pair_sync(pair);
      }
      if (started) product_done();
      tc_fence_after();
      const bool spoiled = started && sm.spoiled[t][turn & 1] == turn;
      const bool empty = !started || (m == -INFINITY && l == 0.0f);
      const float inv = empty ? 0.0f : 1.0f / l;
      const float lse = empty ? -INFINITY : kLn2 * ((m == -INFINITY ? 0.0f : m) + log2f(l));
      const uint64_t token = s.q0 + query;
      const uint64_t part = (uint64_t)(seg.slot < 0 ? 0 : seg.slot) * p.slot_rows + in_seg;
      const uint64_t row_at = live ? token * p.ld_out + (uint64_t)head * p.head_dim : ~0ull;
      if (live && half == 0) {
        if (seg.slot >= 0) p.part_lse[part] = lse;
        else if (p.lse) p.lse[token * p.q_heads + head] = lse;
      }
#pragma unroll 1
      for (int c = 0; c < Sh::kOutCols; c += 32) {
        const uint32_t col0 = half * Sh::kOutCols + c;
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
        }
        if (seg.slot < 0) {
          // Four lanes exchange their rows' 16-byte units, so that they write 64
          // contiguous bytes of one row after another.
          uint4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            v[u] = make_uint4(pack2(T(), o[8 * u], o[8 * u + 1]), pack2(T(), o[8 * u + 2], o[8 * u + 3]),
                              pack2(T(), o[8 * u + 4], o[8 * u + 5]), pack2(T(), o[8 * u + 6], o[8 * u + 7]));
          exchange<1>(v, lane);
          exchange<2>(v, lane);
          const uint32_t col = col0 + 8 * (lane & 3);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint64_t to = __shfl_sync(0xffffffffu, row_at, (lane & ~3) + u);
            if (to != ~0ull && col < p.head_dim) *(uint4*)((T*)p.out + to + col) = v[u];
          }
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

template <typename T, int HDP, bool FULL>
cudaError_t launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int smem = (int)sizeof(Smem<HDP>) + 1024;
  const cudaError_t e = smem_opt_in(attention_tc_kernel<T, HDP, FULL>, smem, &done);
  if (e != cudaSuccess) return e;
  // the registers that setmaxnreg hands over have to come out of the launch's own: an increase beyond them never ends
  static std::atomic<int> fits{-1};
  if (fits.load() < 0) {
    cudaFuncAttributes fa{};
    const cudaError_t f = cudaFuncGetAttributes(&fa, attention_tc_kernel<T, HDP, FULL>);
    if (f != cudaSuccess) return f;
    fits.store(fa.numRegs == Shape<HDP>::kRegs);
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
  attention_tc_kernel<T, HDP, FULL><<<p.blocks, Shape<HDP>::kThreads, smem, st>>>(p, q, k, v, rows);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const AttnParams& p, uint32_t dtype, cudaStream_t st) {
  const uint32_t hd = p.head_dim;
  if (hd <= 64) return hd == 64 ? launch<T, 64, true>(p, dtype, st) : launch<T, 64, false>(p, dtype, st);
  if (hd <= 128) return hd == 128 ? launch<T, 128, true>(p, dtype, st) : launch<T, 128, false>(p, dtype, st);
  return hd == 256 ? launch<T, 256, true>(p, dtype, st) : launch<T, 256, false>(p, dtype, st);
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
  return dtype == SVL_DTYPE_F16 ? launch<__half>(p, dtype, st) : launch<__nv_bfloat16>(p, dtype, st);
}

}  // namespace svl
