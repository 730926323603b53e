// ops_attention.cuh -- the schedule that an svl_attention_plan puts on the
// device, shared by the plan's host code and the attention kernels.
#pragma once

#include "ops_common.cuh"

namespace svl {

constexpr uint32_t kKeyTile = 128;    // keys of a tile, counted from the sequence's first key
constexpr uint32_t kAttnMaxHead = 512;
constexpr int kCapTerms = 4;          // of the capped score's polynomial

// How a row tile sees a key tile.
enum : uint32_t { kSeesNone = 0, kSeesAll = 1, kSeesSome = 2 };

// An entry of a segment's key list: the key tile, and how each of the
// segment's two row tiles sees it.
SVL_DEV uint32_t entry_tile(uint32_t e) { return e & 0x0fffffffu; }
SVL_DEV uint32_t entry_sees(uint32_t e, int row_tile) { return (e >> (28 + 2 * row_tile)) & 3u; }

struct AttnSeq {
  uint64_t q0, k0;      // first packed query and key
  uint32_t n_q, n_k;
  uint32_t prefix, unused;
};

// Rows of a segment are (query, head of the group) pairs of one key-value
// head, the group innermost: row r is query r / group, head kvh * group +
// r % group.  So all rows of a tile read the same keys.
struct AttnSegment {
  uint32_t seq, kvh;
  uint32_t row0, rows;
  uint32_t list0, list1;  // key list entries
  int32_t slot;           // partial results go to this workspace slot; -1: to the output
  uint32_t unused;
};

// Rows whose key axis was cut: slots slot0 .. slot0 + slots - 1 are joined.
struct AttnJoin {
  uint32_t seq, kvh, row0, rows, slot0, slots;
};

struct AttnParams {
  const AttnSeq* seqs;
  const AttnSegment* segments;
  const uint32_t* block_segments;  // blocks + 1 offsets
  const uint32_t* lists;
  const AttnJoin* joins;
  const int32_t* doc_q;  // NULL without documents
  const int32_t* doc_k;
  const float* slopes;   // NULL without a distance bias
  uint32_t* err;
  uint32_t blocks, n_joins, slot_rows;
  uint32_t check_waits;  // a check warp's patience, in waits (4 s)
  uint32_t q_heads, kv_heads, group, head_dim;
  uint64_t total_q, total_k;
  float scale, cap;
  float cap_odd[kCapTerms], cap_limit;  // capped_small() of the FP16 / BF16 kernels
  int32_t causal, window;
  // one call's operands
  const void *q, *k, *v;
  void* out;
  float* lse;
  float* part_o;    // [slot][slot_rows][head_dim], normalised
  float* part_lse;  // [slot][slot_rows]
  uint64_t ld_q, ld_k, ld_v, ld_out;
};

// What a query row needs to know to tell which keys it sees.
struct RowMask {
  int64_t place;  // p
  int32_t doc;
  uint32_t n_k, prefix;
};

SVL_DEV RowMask row_mask(const AttnParams& p, const AttnSeq& s, uint32_t query) {
  RowMask m;
  m.place = (int64_t)query + s.n_k - s.n_q;
  m.doc = p.doc_q ? p.doc_q[s.q0 + query] : 0;
  m.n_k = s.n_k;
  m.prefix = s.prefix;
  return m;
}

// doc: the key's document (0 without documents); j may lie behind the end.
SVL_DEV bool sees(const AttnParams& p, const RowMask& m, uint32_t j, int32_t doc) {
  const int64_t gap = m.place - (int64_t)j;
  const bool near = (!p.causal || gap >= 0) && (p.window < 0 || (gap <= p.window && -gap <= p.window));
  const bool ahead = j < m.prefix;
  return j < m.n_k && m.doc >= 0 && doc >= 0 && (ahead || (near && doc == m.doc));
}

// The tcgen05 kernel for FP16 and BF16 (ops_attention_tc.cu).
bool attention_tc_takes(const svl_attention_config& c, uint64_t total_q, uint64_t total_k);
// Rows of a row tile (whole queries: a multiple of the group) and row tiles of
// a segment.
uint32_t attention_tc_tile_rows(uint32_t group);
uint32_t attention_tc_row_tiles(uint32_t head_dim);
cudaError_t attention_tc_launch(const AttnParams& p, uint32_t dtype, cudaStream_t st);
// The same types with few rows (ops_attention_rows.cu): the rows of a tile that
// takes a sequence of `rows` (query, head of the group) rows, or 0.
uint32_t attention_rows_takes(uint32_t head_dim, uint64_t rows);
cudaError_t attention_rows_launch(const AttnParams& p, uint32_t dtype, cudaStream_t st);

}  // namespace svl
