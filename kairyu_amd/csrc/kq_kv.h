// Paged e4m3 key/value cache: what its append and its attention share.
//
// Codes are [pages][kv heads][page size][head dim] e4m3 bytes, one tensor for
// keys and one for values, and scales fp32 [pages][kv heads] each: a page of one
// head is one contiguous tile of page_size * head_dim bytes and one scale.  A
// sequence's tokens lie in the pages its row of the block table names, in order.
// Sequence b's new rows are rows [cu[b], cu[b + 1]) of the packed activations and
// the last tokens of its lengths[b]: row r sits at position
// lengths[b] - (cu[b + 1] - r).
#pragma once

#include "kq_common.h"

namespace kq {

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int64_t pages;
  int kv_heads, page_shift;  // page size: 1 << page_shift tokens
};

struct KvBatch {
  const int32_t* table;  // [seqs][table_width], row pitch table_ld
  const int32_t* cu;     // [seqs + 1]
  const int32_t* lengths;
  int64_t table_ld;
  int seqs, table_width;
  int rows;  // rows of the packed activations; those at or past cu[seqs] are padding
};

struct KvSeq {
  int row0, rows;  // new rows
  int first;       // position of the first (negative: more rows than tokens)
  int tokens;      // tokens the table can hold of the sequence's length
};

KQ_DEV KvSeq kv_seq(const KvBatch& b, int s, int page_shift) {
  KvSeq q;
  // row bounds held within the tensor whatever cu says
  const int lo = min(max(b.cu[s], 0), b.rows), hi = min(max(b.cu[s + 1], lo), b.rows);
  const int len = max(b.lengths[s], 0);
  q.row0 = lo;
  q.rows = hi - lo;
  q.first = len - q.rows;
  const int64_t most = (int64_t)b.table_width << page_shift;
  q.tokens = (int)(len < most ? len : most);
  return q;
}

// The same for one sequence of the whole wave, in scalar registers.
KQ_DEV KvSeq kv_seq_uniform(const KvBatch& b, int s, int page_shift) {
  KvSeq q = kv_seq(b, s, page_shift);
  q.row0 = __builtin_amdgcn_readfirstlane(q.row0);
  q.rows = __builtin_amdgcn_readfirstlane(q.rows);
  q.first = __builtin_amdgcn_readfirstlane(q.first);
  q.tokens = __builtin_amdgcn_readfirstlane(q.tokens);
  return q;
}

// The page that holds `slot` of sequence s (slot < table_width), or -1 where the
// entry names none.
KQ_DEV int kv_page(const KvBatch& b, const KvCache& c, int s, int slot) {
  const int p = b.table[(int64_t)s * b.table_ld + slot];
  return p >= 0 && p < c.pages ? p : -1;
}

// Sum over lanes 0..l, in registers (DPP row shifts, then the rows' last lanes
// broadcast to the rows behind them).
template <int CTRL, int ROWS>
KQ_DEV int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, ROWS == 0xf);
}
KQ_DEV int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr:1
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast:15
  return dpp_add<0x143, 0xc>(v);  // row_bcast:31
}

// The sequence that unit `u` falls to when sequence s has count(s) units, found by
// a wave together (64 sequences at a time: one load and a scan, where a binary
// search would wait for a load at each of its steps), and its index there; -1 past
// the last unit.  Uniform.
template <typename F>
KQ_DEV int kv_find(int64_t u, int seqs, int& local, F count) {
  int64_t base = 0;
  for (int s0 = 0; s0 < seqs; s0 += 64) {
    const int s = s0 + lane_id();
    const int c = s < seqs ? count(s) : 0;
    const int incl = wave_scan(c);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (u < base + total) {
      const int at = (int)__builtin_ctzll(__ballot(base + incl > u));
      local = (int)(u - base) - (__builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(c, at));
      return s0 + at;
    }
    base += total;
  }
  local = 0;
  return -1;
}

// The sequence of `row` and, in `units`, sum of count(s) over those before it; -1
// for padding.
template <typename F>
KQ_DEV int kv_of_row(int row, const KvBatch& b, int page_shift, int64_t& units, F count) {
  units = 0;
  for (int s0 = 0; s0 < b.seqs; s0 += 64) {
    const int s = s0 + lane_id();
    const KvSeq q = kv_seq(b, min(s, b.seqs - 1), page_shift);
    const int c = s < b.seqs ? count(s) : 0;
    const int incl = wave_scan(c);
    const uint64_t here = __ballot(s < b.seqs && row >= q.row0 && row < q.row0 + q.rows);
    if (here != 0) {
      const int at = (int)__builtin_ctzll(here);
      units += __builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(c, at);
      return s0 + at;
    }
    units += __builtin_amdgcn_readlane(incl, 63);
  }
  return -1;
}

// Host checks that append and attention share; set_error and a status on failure.
int kv_check(const char* what, int dtype, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
             int64_t page_size, int64_t pages, int64_t seqs, int64_t table_width, int64_t table_ld);

}  // namespace kq
