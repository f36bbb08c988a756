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
  const int len = min(max(b.lengths[s], 0), 0x7fff0000);  // (positions a few steps on stay within 32 bits)
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

// The sequences of a batch, one a lane: up to 64 are loaded once and then looked at in
// registers; more are read again, 64 at a time.
struct KvLanes {
  const KvBatch& b;
  int shift;
  KvSeq mine;
  bool held;

  KQ_DEV KvLanes(const KvBatch& batch, int page_shift) : b(batch), shift(page_shift), mine{}, held(batch.seqs <= 64) {
    if (held && lane_id() < b.seqs) mine = kv_seq(b, lane_id(), shift);
  }
  // sequence s0 + lane (no rows past the last)
  KQ_DEV KvSeq at_lane(int s0) const {
    if (held) return mine;
    KvSeq q{};
    if (s0 + lane_id() < b.seqs) q = kv_seq(b, s0 + lane_id(), shift);
    return q;
  }
  // sequence s, in scalar registers
  KQ_DEV KvSeq operator[](int s) const {
    if (!held) return kv_seq_uniform(b, s, shift);
    KvSeq q;
    q.row0 = __builtin_amdgcn_readlane(mine.row0, s);
    q.rows = __builtin_amdgcn_readlane(mine.rows, s);
    q.first = __builtin_amdgcn_readlane(mine.first, s);
    q.tokens = __builtin_amdgcn_readlane(mine.tokens, s);
    return q;
  }
  // Units of all sequences, count(q) of each (0 for one without rows).
  template <typename F>
  KQ_DEV int total(F count) const {
    int sum = 0;
    for (int s0 = 0; s0 < b.seqs; s0 += 64) sum += __builtin_amdgcn_readlane(wave_scan(count(at_lane(s0))), 63);
    return sum;
  }
  // The sequence that unit `u` falls to, found by the wave together (one load and a scan
  // per 64 sequences, where a binary search would wait for a load at each of its steps),
  // and its index there; -1 past the last unit.
  template <typename F>
  KQ_DEV int find(int u, int& local, F count) const {
    int base = 0;
    for (int s0 = 0; s0 < b.seqs; s0 += 64) {
      const int c = count(at_lane(s0));
      const int incl = wave_scan(c);
      const int all = __builtin_amdgcn_readlane(incl, 63);
      if (u < base + all) {
        const int at = (int)__builtin_ctzll(__ballot(base + incl > u));
        local = u - base - (__builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(c, at));
        return s0 + at;
      }
      base += all;
    }
    local = 0;
    return -1;
  }
  // The sequence of `row` and, in `units`, the units of those before it; -1 for padding.
  template <typename F>
  KQ_DEV int of_row(int row, int& units, F count) const {
    units = 0;
    for (int s0 = 0; s0 < b.seqs; s0 += 64) {
      const KvSeq q = at_lane(s0);
      const int c = count(q);
      const int incl = wave_scan(c);
      const uint64_t here = __ballot(row >= q.row0 && row < q.row0 + q.rows);
      if (here != 0) {
        const int at = (int)__builtin_ctzll(here);
        units += __builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(c, at);
        return s0 + at;
      }
      units += __builtin_amdgcn_readlane(incl, 63);
    }
    return -1;
  }
};

// A value of the whole wave in a scalar register (quotients come out of the vector unit).
KQ_DEV int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Four codes of stored tokens on a coarser scale: code * ratio (below 1), rounded again;
// NaN codes stay.
KQ_DEV uint32_t move4(uint32_t w, float ratio) {
  uint32_t nan = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((w >> (8 * e) & 0x7fu) == 0x7fu) nan |= 0xffu << (8 * e);
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)(w & ~nan), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)(w & ~nan), true);
  return (pack4_e4m3(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio) & ~nan) | (w & nan);
}
KQ_DEV u32x4 move16(u32x4 w, float ratio) { return u32x4{move4(w[0], ratio), move4(w[1], ratio), move4(w[2], ratio), move4(w[3], ratio)}; }

// Host checks that the cache's entries share; set_error and a status on failure.
int kv_check(const char* what, int dtype, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
             int64_t page_size, int64_t pages, int64_t seqs, int64_t table_width, int64_t table_ld);

}  // namespace kq
