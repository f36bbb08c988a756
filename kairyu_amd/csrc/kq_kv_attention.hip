// Attention over the paged e4m3 cache.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = exp(scale * q . k_t - max) over the tokens
// a row sees, in one pass with a running maximum.  Key codes enter the products as
// they are and the page's scale multiplies the finished dot product; the value scale
// joins the exponent instead, w_t = log2(e) scale k_scale (q . code_t) + log2 v_scale,
// so that exp2(w_t - max w + lift) multiplies the value's codes whatever the scales of
// the pages are; the denominator adds the same over v_scale.  Maxima, denominators and
// outputs are held in fp32, and the lift, which a row's sums all have, cancels.
//
// Weights enter the products with the values as fp16: 11 bits, 8 with bf16, which fp16
// rows would show.  fp16 ends 2^-14 (11 bits) or 2^-25 (anything) below one, and a token
// that most of the mass goes to may have a value of nearly zero, so that the others' tail
// is the answer: the lift takes the largest weights towards the top of fp16's range, and
// a weight keeps its 11 bits down to 2^-23 of the largest and some down to 2^-34 (tiles of
// 128; 2^-29 and 2^-40 in tiles of 16).
#include "kq_kv.h"

#include <algorithm>
#include <type_traits>

namespace kq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
  const uint16_t* q;
  int64_t q_ld, q_hs;
  uint16_t* out;  // [rows][heads][D]
  float* part;    // partial outputs of split sequences, null: none can be split
  float scale;    // magnitude times log2 e, at least 2^-60: times a page's scale it stays positive
  uint32_t q_sign;  // the softmax scale's sign, for two 16-bit elements
  int heads, causal, window;
  int most_blocks;  // no batch has more
  int shares;     // workgroups per kv head that the batch's tokens are dealt to
  int block_shift;  // log2 of the 64-token steps of a block
  float* big_part;  // partial outputs of the large tiles, null: their tokens are not split
  int few;          // rows * group up to which a sequence goes to tiles of 16 rows
  int big_tiles;    // large tiles per kv head that the grid has room for
  int splits;       // parts that a large tile's tokens are cut into
};

constexpr int kBigRows = 128;  // rows of a large tile, 32 a wave

// log2 of the largest weight.  Tiles of 16 have the exact maximum.  Tiles of 128 move theirs
// when a lane's 16 weights of a half step may add up to more than fp16 holds, 128 of 2^9: a
// larger lift leaves less room and moves it more often (8192 rows behind 12288 tokens and 24
// windows of heads of 64 with lifts of 5, 8, 9 and 11: 1092, 1101, 1107 and 1119 us, 52.5, 53.2,
// 54.8 and 57.3; weights of at most one, which are lost, 1080 and 51.0).
constexpr float kLift = 15.0f, kBigLift = 9.0f, kBigMost = 65504.0f;
// Beyond this magnitude of the maximum, log2 of a value scale and the lift drown in a score's
// last bits: tiles of 128 then form each exponent from the rounded score, as tiles of 16 do.
constexpr float kCoarse = 0x1p20f;

// e4m3 codes widened to the 16-bit type of a product (exact in both)
template <int DT>
KQ_DEV u32x4 widen_codes(uint32_t lo, uint32_t hi) {
  u32x4 r;
  if (DT == KQ_DTYPE_BF16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  }
  return r;
}

template <int DT>
KQ_DEV f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if (DT == KQ_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Bytes of four dwords transposed: out[j] holds byte j of in[0..3].
KQ_DEV void transpose4(const uint32_t in[4], uint32_t out[4]) {
  const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u), d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Maximum and sum over the four lanes that hold one column (l, l ^ 16, l ^ 32, l ^ 48).
KQ_DEV float column_max(float v) {
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
KQ_DEV float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// A sequence's rows (new tokens x the group's query heads) go to tiles of 16, and the
// tokens that they see to blocks (of 256; or so long that a tile is one block, and nothing
// is to be joined, where no sequence can look at more than kWhole or kWholeMany tokens).
// The blocks of all tiles, one after the other, are dealt to `shares` workgroups per kv
// head in equal runs, so that every workgroup streams the same number of bytes whatever
// the lengths are.  A run covers whole tiles, written at once, and at most two parts of
// tiles: the end of one begun before it (part 0) and the beginning of one that goes on
// behind it (part 1).
struct Deal {
  const AttendArgs& a;
  int group;

  // 64-token step of the first token that any row sees
  KQ_DEV int first(const KvSeq& q) const { return a.window > 0 ? max(q.first + 1 - a.window, 0) >> 6 : 0; }
  // at least one, so that rows that see nothing are written as well
  KQ_DEV int blocks(const KvSeq& q) const { return (max(((q.tokens + 63) >> 6) - first(q), 1) + (1 << a.block_shift) - 1) >> a.block_shift; }
  KQ_DEV int tiles(const KvSeq& q) const {
    const int items = q.rows * group;
    return items <= a.few ? (items + 15) >> 4 : 0;
  }
  KQ_DEV int operator()(const KvSeq& q) const { return tiles(q) * blocks(q); }
  // blocks of a workgroup: the same in every one
  KQ_DEV int run(const KvLanes& lanes) const {
    // (held to what a batch can have, whatever the row bounds say)
    const uint32_t all = min((uint32_t)lanes.total(*this), (uint32_t)a.most_blocks);
    return scalar((int)((all + (uint32_t)a.shares - 1) / (uint32_t)a.shares));
  }
};
struct BigTiles {
  const AttendArgs& a;
  int group;
  KQ_DEV int operator()(const KvSeq& q) const {
    const int items = q.rows * group;
    return items > a.few ? (items + kBigRows - 1) / kBigRows : 0;
  }
};

// Large tiles by the tokens that they see, most first, so that the last workgroups to start
// are the shortest.  Tile k of a sequence sees min(tokens, first + ((k + 1) * kBigRows - 1) /
// group + 1) of them (or all), which grows with k: how many of its tiles see at least 64 T
// is a matter of a product and a shift.
struct LongestFirst {
  const AttendArgs& a;
  const KvLanes& lanes;
  int group;

  KQ_DEV int at_least(const KvSeq& q, int t) const {
    const int tiles = BigTiles{a, group}(q);
    if (t <= 0) return tiles;
    if (tiles == 0 || q.tokens >> 6 < t) return 0;
    const int row = 64 * t - 1 - q.first;  // the first that sees 64 t
    if (!a.causal || row <= 0) return tiles;
    return row < q.rows ? tiles - row * group / kBigRows : 0;
  }
  // The tile of a rank: its sequence (-1 past the last) and its index there.
  KQ_DEV int find(int rank, int& tile) const {
    if (rank >= lanes.total(BigTiles{a, group})) return -1;
    int t = 0, end = (int)wave_max_u32_dpp((uint32_t)(lanes.at_lane(0).tokens >> 6)) + 1;
    while (end - t > 1) {  // (at most 25 times)
      const int mid = (t + end) >> 1;
      if (lanes.total([&](const KvSeq& q) { return at_least(q, mid); }) > rank)
        t = mid;
      else
        end = mid;
    }
    rank -= lanes.total([&](const KvSeq& q) { return at_least(q, t + 1); });
    const int s = lanes.find(rank, tile, [&](const KvSeq& q) { return at_least(q, t) - at_least(q, t + 1); });
    const KvSeq q = lanes[s];
    tile += BigTiles{a, group}(q) - at_least(q, t);
    return s;
  }
};

// Whether any of tokens [from, to) is there.  Scores over a token of no page are 0 * q, NaN
// where the query is not finite, though the row does not see it: a lane whose sum is NaN
// looks at the pages again, and takes the sum for empty if there are none.
KQ_DEV bool any_there(const int32_t* pages, int64_t count, int from, int to, int shift) {
  for (int i = from >> shift; from < to && i <= (to - 1) >> shift; ++i)
    if (pages[i] >= 0 && pages[i] < count) return true;
  return false;
}

// What waves have put in LDS is there for all of them; loads from memory stay in flight.
KQ_DEV void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Rows of no sequence are zero: those of one kv head, dealt to `of` workgroups.
template <int D>
KQ_DEV void zero_padding(const AttendArgs& a, const KvBatch& batch, int head, int group, int nth, int of, int threads) {
  const int last = batch.seqs > 0 ? min(max(batch.cu[batch.seqs], 0), batch.rows) : 0;
  const int first = batch.seqs > 0 ? min(max(batch.cu[0], 0), last) : 0;
  const int words = group * D / 2;
  for (int i = nth; i < first + batch.rows - last; i += of) {
    const int64_t row = i < first ? i : last + (i - first);
    uint32_t* dst = (uint32_t*)(a.out + (row * a.heads + head * group) * D);
    for (int j = (int)threadIdx.x; j < words; j += threads) dst[j] = 0;
  }
}

// One workgroup: its run of blocks of one kv head, tile by tile; its four waves take
// a tile's steps of 16 * NT tokens in turn.
//
// Products run transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32 MFMAs: lane
// (c, b) = (l % 16, l / 16) then holds scores of query row c for tokens 4b..4b+3 of
// each 16-token tile, which are, for two tiles, just the eight tokens that it has to
// hand over as its part of P^T: no score leaves its lane.  Keys and values go from
// memory to registers; a lane loads D / 16 bytes of each of its tokens' values and
// transposes them by bytes (the order of d within an output tile is free: row c of
// tile j is d = c * D / 16 + j, so a lane ends up with neighbouring elements).
//
// Loads go through buffer resources of one page's tile whose size ends at the
// sequence's last token: slots past it, pages that are none and steps past the run
// read as zero without a branch.  They are marked non-temporal: a token is read once by
// a tile and most sequences have one (64 ragged contexts 51.2 -> 46.5 us, 3 x 131001
// tokens 158 -> 139; two tiles a sequence, which then share less, 66 -> 69).
//
// Bound by HBM on long contexts: 3 x 131001 tokens on 8 kv heads of 128, 805 MB, take
// 124 us (6.5 TB/s); 64 of up to 6000 on 4, 186 MB, 40 (4.6), where starting, the first
// loads' latency and the last part's merge are 8 of them.  A single context of 700 tokens
// takes 8-10 us, its three steps' latency.
template <int D, int DT, int NT, int PP>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 3)
kv_attend_rows_kernel(AttendArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
                      const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int KS = D / 32;   // MFMA steps along a key
  constexpr int VD = D / 64;   // dwords of a token's value a lane holds
  constexpr int OT = D / 16;   // output tiles
  constexpr int ST = 16 * NT;  // tokens of a step
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * LD];
  const int lane = lane_id(), wave = scalar(wave_id()), c = lane & 15, b = lane >> 4;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int head = (int)blockIdx.y;

  zero_padding<D>(a, batch, head, group, (int)blockIdx.x, (int)gridDim.x, 256);
  const KvLanes lanes(batch, shift);
  const Deal deal{a, group};
  const int run = deal.run(lanes), run_end = ((int)blockIdx.x + 1) * run;
  int block = (int)blockIdx.x * run;
  int within = 0;  // blocks of the sequence, then of the tile, before `block`
  int s = lanes.find(block, within, deal);
  if (s < 0) return;
  KvSeq q = lanes[s];
  int blocks = deal.blocks(q), tile = scalar(within / blocks);
  within -= tile * blocks;
  const int64_t tile_bytes = (int64_t)D << shift;
  const int in_page = (1 << shift) - 1;
  const int k_lane = c * D + 16 * b, v_lane = 4 * b * D + c * (D / 16);

  // One part of a tile: its bounds, its rows of Q, and its loads on their way.
  int from, to, lo, hi, lo_all, hi_all, part_blocks;
  const int32_t* pages;
  u32x4 qf[KS];
  int id;                   // lane l: the page that holds the step's tokens from l % PP * (ST / PP) on
  u32x4 kx[NT][D / 64];     // a step's keys and values, and their pages' scales (0: no tokens there)
  uint32_t vx[NT * 4][VD];
  float ks, vs;
  // pages of the step at t
  const int nth_page = PP == 1 ? 0 : (lane & (PP - 1)) * (ST / PP);
  auto pages_of = [&](int t) { id = pages[min(t + nth_page, max(hi - 1, 0)) >> shift]; };
  int head_tile, size;
  auto place = [&](int t) {
    const int at = t + nth_page, page = PP == 1 ? scalar(id) : id;
    const bool there = page >= 0 && page < (int)cache.pages && at < hi;
    head_tile = (there ? page : 0) * cache.kv_heads + head;
    size = there ? min(q.tokens - (at & ~in_page), in_page + 1) * D : 0;
  };
  auto of_page = [&](int v, int p) { return PP == 1 ? v : __builtin_amdgcn_readlane(v, p); };
  auto scale_of = [&](const float* scales) {
    if constexpr (PP == 1) return __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(scales + head_tile, size != 0 ? 4 : 0), 0, 0, 0));
    const int end = (int)cache.pages * cache.kv_heads * 4;  // (an offset there reads 0)
    return __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(scales, end), size != 0 ? 4 * head_tile : end, 0, 0));
  };
  auto load_keys = [&](int t) {
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      const i32x4 src = make_rsrc(cache.k + of_page(head_tile, p) * tile_bytes, of_page(size, p));
      const int off = ((t + p * (ST / PP)) & in_page) * D;
#pragma unroll
      for (int i = p * (NT / PP); i < (p + 1) * (NT / PP); ++i)
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
          kx[i][h] = __builtin_bit_cast(u32x4, kq_rbl_v4i32(src, k_lane + 64 * h, off + (i - p * (NT / PP)) * 16 * D, kAuxNT));
    }
    ks = scale_of(k_scale);
    vs = scale_of(v_scale);
  };
  auto load_values = [&](int t) {
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      const i32x4 src = make_rsrc(cache.v + of_page(head_tile, p) * tile_bytes, of_page(size, p));
      const int off = ((t + p * (ST / PP)) & in_page) * D;
#pragma unroll
      for (int i = p * (NT / PP); i < (p + 1) * (NT / PP); ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int so = off + (i - p * (NT / PP)) * 16 * D;
          if constexpr (VD == 1) {
            vx[4 * i + r][0] = (uint32_t)kq_rbl_i32(src, v_lane + r * D, so, kAuxNT);
          } else if constexpr (VD == 2) {
            const i32x2 w = kq_rbl_v2i32(src, v_lane + r * D, so, kAuxNT);
            vx[4 * i + r][0] = (uint32_t)w[0];
            vx[4 * i + r][1] = (uint32_t)w[1];
          } else {
            const i32x4 w = kq_rbl_v4i32(src, v_lane + r * D, so, kAuxNT);
#pragma unroll
            for (int d = 0; d < VD; ++d) vx[4 * i + r][d] = (uint32_t)w[d];
          }
        }
    }
  };
  auto begin_part = [&] {
    const int item = tile * 16 + c;  // this lane's column: row item / group, head item % group
    const bool real = item < q.rows * group;
    const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
    const int pos = q.first + row;
    // tokens [from, to) of this column; [lo, hi) of the part; [lo_all, hi_all) of every row
    to = a.causal ? min(q.tokens, pos + 1) : q.tokens;
    from = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
    const int row_lo = scalar(tile * 16 / group), row_hi = min(q.rows - 1, scalar((tile * 16 + 15) / group));
    hi = a.causal ? min(q.tokens, q.first + row_hi + 1) : q.tokens;
    lo = a.window > 0 ? max(q.first + row_lo + 1 - a.window, 0) : 0;
    hi_all = a.causal ? min(q.tokens, q.first + row_lo + 1) : q.tokens;
    lo_all = a.window > 0 ? max(q.first + row_hi + 1 - a.window, 0) : 0;
    part_blocks = min(blocks - within, run_end - block);
    const int begin = deal.first(q) * 64 + (within << (6 + a.block_shift));
    hi = (int)min((int64_t)hi, (int64_t)begin + ((int64_t)part_blocks << (6 + a.block_shift)));
    lo = max(lo & ~63, begin);
    pages = table + (int64_t)s * batch.table_ld;
    const int t = lo + ST * wave;
    pages_of(t);
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = u32x4{0, 0, 0, 0};
    if (real) {
      const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
      for (int i = 0; i < KS; ++i) qf[i] = *(const u32x4*)(src + 64 * (i >> 1) + 16 * b + 8 * (i & 1)) ^ a.q_sign;
    }
    place(t);
    load_keys(t);
    load_values(t);
    pages_of(t + 4 * ST);
  };

  f32x4 o[OT];
  float top, sum;
  auto step = [&](int t) {
    f32x4 w[NT];
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < KS / 2; ++h) {
        acc = mfma16<DT>(widen_codes<DT>(kx[i][h][0], kx[i][h][1]), qf[2 * h], acc);
        acc = mfma16<DT>(widen_codes<DT>(kx[i][h][2], kx[i][h][3]), qf[2 * h + 1], acc);
      }
      w[i] = acc;
    }
    float inv_v[PP];
    const float lane_shift = __builtin_amdgcn_logf(vs), lane_scale = ks * a.scale;  // (-inf where there are no tokens)
    const float lane_inv = vs > 0.0f ? __builtin_amdgcn_rcpf(vs) : 0.0f;
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      auto of = [&](float v) { return __uint_as_float((uint32_t)of_page((int)__float_as_uint(v), p)); };
      const float shift_v = of(lane_shift), scale = of(lane_scale);
      inv_v[p] = of(lane_inv);
#pragma unroll
      for (int i = p * (NT / PP); i < (p + 1) * (NT / PP); ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[i][r] = fmaf(w[i][r], scale, shift_v);
    }
    // the keys' registers take the next step's while this one goes on, the values' then theirs
    place(t + 4 * ST);
    load_keys(t + 4 * ST);
    pages_of(t + 8 * ST);
    if (t < lo_all || t + ST > hi_all) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = t + 16 * i + 4 * b + r;
          if (token < from || token >= to) w[i][r] = -__builtin_inff();
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, w[i][r]);
    m = column_max(m);
    if (__ballot(m > top) != 0) {
      m = fmaxf(m, top);
      const float keep = __builtin_amdgcn_exp2f(top - (m == -__builtin_inff() ? 0.0f : m));
      sum *= keep;
#pragma unroll
      for (int j = 0; j < OT; ++j) o[j] *= keep;
      top = m;
    }
    const float base = top == -__builtin_inff() ? 0.0f : top;
    u32x4 p[NT / 2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) w[i][r] = __builtin_amdgcn_exp2f((w[i][r] - base) + kLift);  // (the difference exact: at most kLift)
      sum = fmaf(w[i][0] + w[i][1] + w[i][2] + w[i][3], inv_v[i / (NT / PP)], sum);
      p[i >> 1][2 * (i & 1)] = pack_act2(w[i][0], w[i][1], KQ_DTYPE_F16);
      p[i >> 1][2 * (i & 1) + 1] = pack_act2(w[i][2], w[i][3], KQ_DTYPE_F16);
    }
#pragma unroll
    for (int d = 0; d < VD; ++d)
#pragma unroll
      for (int g = 0; g < NT / 2; ++g) {
        uint32_t in[2][4], out[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int r = 0; r < 4; ++r) in[e][r] = vx[8 * g + 4 * e + r][d];
          transpose4(in[e], out[e]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[4 * d + j] = mfma16<KQ_DTYPE_F16>(widen_codes<KQ_DTYPE_F16>(out[0][j], out[1][j]), p[g], o[4 * d + j]);
      }
    load_values(t + 4 * ST);
  };

  begin_part();
  while (true) {
#pragma unroll
    for (int j = 0; j < OT; ++j) o[j] = f32x4{0, 0, 0, 0};
    top = -__builtin_inff();
    sum = 0.0f;
    for (int t = lo + ST * wave; t < hi; t += 4 * ST) step(t);
    sum = column_sum(sum);
    if (sum != sum && !any_there(pages, cache.pages, max(from, lo), min(to, hi), shift)) {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < OT; ++j) o[j] = f32x4{0, 0, 0, 0};
    }

    // the next part's loads travel while this one's waves meet
    const KvSeq old = q;
    const int old_tile = tile, old_within = within;
    const bool whole = part_blocks == blocks;
    block += part_blocks;
    within = 0;
    bool more = block < run_end;
    if (more && ++tile >= deal.tiles(q)) {
      tile = 0;
      do {
        more = ++s < batch.seqs;
        if (!more) break;
        q = lanes[s];
      } while (deal.tiles(q) == 0);
      blocks = deal.blocks(q);
    }
    if (more) begin_part();

    // the waves' parts meet in LDS, added in wave order
    float* mine = lds + (wave * 16 + c) * LD;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < OT; j += 4)
        *(f32x4*)(mine + (4 * b + r) * OT + j) = f32x4{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
    if (b == 0) {
      mine[D] = top;
      mine[D + 1] = sum;
    }
    meet();
    for (int i = (int)threadIdx.x; i < 16 * (D / 2); i += 256) {
      const int col = i / (D / 2), d = 2 * (i - col * (D / 2));
      const int it = old_tile * 16 + col;
      if (it >= old.rows * group) break;
      float m = -__builtin_inff();
#pragma unroll
      for (int v = 0; v < 4; ++v) m = fmaxf(m, lds[(v * 16 + col) * LD + D]);
      const float base = m == -__builtin_inff() ? 0.0f : m;
      float ox = 0.0f, oy = 0.0f, l = 0.0f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float* part = lds + (v * 16 + col) * LD;
        const float f = __builtin_amdgcn_exp2f(part[D] - base);
        ox += part[d] * f;
        oy += part[d + 1] * f;
        l += part[D + 1] * f;
      }
      if (!whole) {
        float* dst = a.part + ((((int64_t)head * a.shares + (int)blockIdx.x) * 2 + (old_within == 0)) * 16 + col) * LD;
        *(f32x2_t*)(dst + d) = f32x2_t{ox, oy};
        if (d == 0) *(f32x2_t*)(dst + D) = f32x2_t{m, l};
        continue;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees no token is zero)
      const int rw = it / group;
      uint32_t* dst = (uint32_t*)(a.out + ((int64_t)(old.row0 + rw) * a.heads + head * group + (it - rw * group)) * D + d);
      *dst = pack_act2(ox * inv, oy * inv, DT);
    }
    if (!more) return;
    meet();
  }
}

// The parts of split tiles joined in the order of their tokens, one wave per row and
// query head: of every row, or of the 16-row tiles alone where no large tile is split.
// Latency: 5 us for 64 contexts, most of it the launch and two dependent loads.
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv_attend_join_kernel(AttendArgs a, KvCache cache, KvBatch batch, int small_tiles) {
  constexpr int LD = D + 4, PER = D / 64;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int at = (int)blockIdx.x * 4 + scalar(wave_id());
  const KvLanes lanes(batch, shift);
  const Deal deal{a, group};
  int s, item, head, block = 0, above = 0;  // blocks, and large tiles, of the sequences before s
  if (small_tiles > 0) {
    const int column = scalar(at / cache.kv_heads);
    head = at - column * cache.kv_heads;
    int tile;
    s = lanes.find(column >> 4, tile, [&](const KvSeq& q) { return deal.tiles(q); });
    if (s < 0) return;
    item = tile * 16 + (column & 15);
    if (item >= lanes[s].rows * group) return;
    lanes.of_row(lanes[s].row0, block, deal);
  } else {
    const int row = scalar(at / a.heads), qh = at - row * a.heads;
    if (row >= batch.rows) return;
    head = scalar(qh / group);
    s = lanes.of_row(row, block, deal);
    if (s < 0) return;
    item = (row - lanes[s].row0) * group + (qh - head * group);
    if (a.splits > 1) lanes.of_row(row, above, BigTiles{a, group});
  }
  const KvSeq q = lanes[s];
  const float* src;
  int chunks;
  const bool big = q.rows * group > a.few;
  if (big) {
    if (a.splits == 1) return;
    chunks = a.splits;
    const int tile = item / kBigRows;
    if (above + tile >= a.big_tiles) return;  // (row bounds that go back: past the grid)
    src = a.big_part + ((((int64_t)head * a.big_tiles + above + tile) * a.splits) * kBigRows + item - tile * kBigRows) * LD;
  } else {
    if (a.part == nullptr) return;  // (one block each)
    const int run = max(deal.run(lanes), 1), blocks = deal.blocks(q);
    block += (item >> 4) * blocks;
    // (within the shares also where row bounds that go back make counts wrap)
    const int x0 = min(max(scalar(block / run), 0), a.shares - 1);
    chunks = min(max(scalar((block + blocks - 1) / run), x0), a.shares - 1) - x0 + 1;
    if (chunks == 1) return;  // written already
    // part 1 of the run it begins in, then part 0 of those behind
    src = a.part + ((((int64_t)head * a.shares + x0) * 2 + 1) * 16 + (item & 15)) * LD;
  }
  auto at_part = [&](int i) { return src + (big ? (int64_t)i * kBigRows : i == 0 ? 0 : (int64_t)(2 * i - 1) * 16) * LD; };
  const int row = q.row0 + scalar(item / group), qh = head * group + item % group;
  float m = -__builtin_inff();
  for (int i = lane_id(); i < chunks; i += 64) m = fmaxf(m, at_part(i)[D]);
  m = wave_max(m);
  const float base = m == -__builtin_inff() ? 0.0f : m;
  float x[PER], l = 0.0f;
#pragma unroll
  for (int d = 0; d < PER; ++d) x[d] = 0.0f;
#pragma unroll 4
  for (int i = 0; i < chunks; ++i) {
    const float* p = at_part(i);
    const float f = __builtin_amdgcn_exp2f(p[D] - base);
    l += p[D + 1] * f;
#pragma unroll
    for (int d = 0; d < PER; ++d) x[d] += p[PER * lane_id() + d] * f;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* dst = a.out + ((int64_t)row * a.heads + qh) * D + PER * lane_id();
#pragma unroll
  for (int d = 0; d < PER; ++d) dst[d] = f32_to_out(x[d] * inv, DT);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT>
KQ_DEV f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if (DT == KQ_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One workgroup: a tile of 32 rows a wave of one sequence and kv head, over the tokens
// that it sees or one of `splits` parts of them, 64 at a step.  (With eight waves, which
// share what a step widens, 8192 rows behind 12288 tokens took 1087 us and with four 1100,
// but 1024 of 1024 42.7 and 31.6: fewer tiles fill the chip unevenly.)
//
// 8192 rows behind 12288 tokens, 32 heads over 8 of 128, 1.1 TFLOP: 1105-1150 us, 1.0
// PFLOP/s.  No unit bounds it alone: the matrix cores are busy for 47% of that, LDS for 52%,
// the vector unit, with about 100 instructions a half step of 32 tokens, 16 of them
// exponentials, for about half.  Widening and staging account for 27% of the time, the
// products with the values for 20%, exponentials for 8% (copies timed without them).
// Waves past a sequence's rows compute like the others: where rows are few, as long as
// the longest tile (24 windows of 1024 tokens, heads of 64: 53 us, 35% of the waves empty).
//
// The same transposed products as above on 32x32x16 MFMAs.  A step's keys and values
// are shared by the waves: they are widened once, keys to Q's type in rows of one
// token, values to fp16 in rows of one d whose tokens stand in the order in which the
// lanes of S^T hold them (for each 16: 0-3, 8-11, then 4-7, 12-15), so that both are
// read as 16-byte MFMA operands; rows are padded by 16 bytes, which spreads eight
// lanes' reads over all banks.
template <int D, int DT>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2)
kv_attend_tiles_kernel(AttendArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
                       const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int KS = D / 16;            // MFMA steps along a key
  constexpr int OT = D / 32;            // output tiles
  constexpr int KLD = 2 * D + 16;       // bytes of a key's row
  constexpr int VLD = 2 * 64 + 16;      // bytes of a d's row of values
  constexpr int KB = 64 * KLD, VB = D * VLD, BUF = KB + VB + 64;  // ... and 4 x (scale, log2 of the value scale, its inverse)
  constexpr int KC = D / 64;            // 16-byte chunks of one token's key a thread moves
  constexpr int VY = D / 16, VC = VY / 4;  // bytes and dwords of each of four tokens' values a thread moves
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) char smem[2 * BUF];
  const int wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int lane = lane_id(), c = lane & 31, h = lane >> 5, tid = (int)threadIdx.x;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  // kv heads side by side, so that (for up to 8 of them) an XCD's workgroups share
  // theirs through its L2; the tiles with the most tokens first
  const int rest = scalar((int)blockIdx.x / cache.kv_heads), head = (int)blockIdx.x - rest * cache.kv_heads;
  const int above = scalar(rest / a.splits), part = rest - above * a.splits, nth = a.big_tiles - 1 - above;
  if (a.few == 0) zero_padding<D>(a, batch, head, group, rest, a.big_tiles * a.splits, 256);  // (no other kernel does)
  const KvLanes lanes(batch, shift);
  int tile;
  const int s = a.splits == 1 && a.window == 0 && batch.seqs > 1 && lanes.held
                    ? LongestFirst{a, lanes, group}.find(above, tile)
                    : lanes.find(nth, tile, BigTiles{a, group});
  if (s < 0) return;
  const KvSeq q = lanes[s];
  const int item = tile * kBigRows + wave * 32 + c;
  const bool real = item < q.rows * group;
  const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
  const int pos = q.first + row;
  // tokens [from, to) of this column, [lo_all, hi_all) of every row of the tile, [lo, hi) of any
  const int to = a.causal ? min(q.tokens, pos + 1) : q.tokens;
  const int from = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
  const int first_row = scalar(tile * kBigRows / group);
  const int last_row = min(q.rows - 1, scalar((tile * kBigRows + kBigRows - 1) / group));
  int hi = a.causal ? max(min(q.tokens, q.first + last_row + 1), 0) : q.tokens;
  int lo = a.window > 0 ? max(q.first + first_row + 1 - a.window, 0) & ~63 : 0;
  const int hi_all = a.causal ? min(q.tokens, q.first + first_row + 1) : q.tokens;
  const int lo_all = a.window > 0 ? max(q.first + last_row + 1 - a.window, 0) : 0;
  if (a.splits > 1) {
    const int n = hi > lo ? (hi - lo + 63) >> 6 : 0, per = scalar((n + a.splits - 1) / a.splits);
    lo += part * per * 64;
    hi = min(hi, lo + per * 64);
  }

  u32x4 qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) qf[i] = u32x4{0, 0, 0, 0};
  if (real) {
    const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *(const u32x4*)(src + 16 * i + 8 * h) ^ a.q_sign;
  }

  // what this thread moves: D / 4 bytes of one token's key, D / 16 of four tokens' values;
  // a wave moves one 16-token tile, which lies in one page.  Row R of the values is
  // d = R % 16 * VY + R / 16: any order of d does, and neighbouring lanes then write
  // neighbouring rows.
  const int k_tok = tid / 4, v_grp = tid / 16, v_c = tid % 16;
  const int k_lane = (k_tok % 16) * D + (tid % 4) * (D / 4), v_lane = 4 * (v_grp % 4) * D + v_c * VY;
  const int v_pos = (v_grp >> 2) * 16 + (v_grp & 1) * 8 + ((v_grp >> 1) & 1) * 4;
  const int tile_shift = shift + (D == 64 ? 6 : D == 128 ? 7 : 8);  // log2 of a page's bytes
  const int in_page = (1 << shift) - 1;
  const int32_t* pages = table + (int64_t)s * batch.table_ld;
  auto page_at = [&](int t) { return pages[min(t + 16 * wave, max(hi - 1, 0)) >> shift]; };
  u32x4 kr[KC];
  uint32_t vr[4][VC];
  float sc_k = 0.0f, sc_v = 0.0f;
  // a step's page of this wave: its tile, the bytes before the sequence's end (slots past
  // it hold whatever was there, NaN perhaps; the resources end before them) and the offset
  struct Place {
    int head_tile, size, off;
  };
  auto place_of = [&](int t, int page_) {
    const int page = __builtin_amdgcn_readfirstlane(page_), at = t + 16 * wave;
    const bool there = page >= 0 && page < (int)cache.pages && at < hi;
    Place p;
    p.head_tile = (there ? page : 0) * cache.kv_heads + head;
    p.size = there ? min(q.tokens - (at & ~in_page), in_page + 1) * D : 0;
    p.off = (at & in_page) * D;
    return p;
  };
  auto fetch_k = [&](const Place& p) {
    const i32x4 src = make_rsrc(cache.k + ((int64_t)p.head_tile << tile_shift), (uint32_t)p.size);
#pragma unroll
    for (int i = 0; i < KC; ++i) kr[i] = __builtin_bit_cast(u32x4, kq_rbl_v4i32(src, k_lane + 16 * i, p.off, 0));
    // (a vector load, which the barriers do not wait for; 0 where there is no page)
    sc_k = __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(k_scale + p.head_tile, p.size != 0 ? 4 : 0), 0, 0, 0));
  };
  auto fetch_v = [&](const Place& p) {
    const i32x4 src = make_rsrc(cache.v + ((int64_t)p.head_tile << tile_shift), (uint32_t)p.size);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (VC == 1) {
        vr[r][0] = (uint32_t)kq_rbl_i32(src, v_lane + r * D, p.off, 0);
      } else if constexpr (VC == 2) {
        const i32x2 w = kq_rbl_v2i32(src, v_lane + r * D, p.off, 0);
        vr[r][0] = (uint32_t)w[0];
        vr[r][1] = (uint32_t)w[1];
      } else {
        const i32x4 w = kq_rbl_v4i32(src, v_lane + r * D, p.off, 0);
#pragma unroll
        for (int i = 0; i < VC; ++i) vr[r][i] = (uint32_t)w[i];
      }
    }
    sc_v = __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(v_scale + p.head_tile, p.size != 0 ? 4 : 0), 0, 0, 0));
  };
  auto put_k = [&](char* buf) {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      char* dst = buf + k_tok * KLD + 2 * ((tid % 4) * (D / 4) + 16 * i);
      *(u32x4*)dst = widen_codes<DT>(kr[i][0], kr[i][1]);
      *(u32x4*)(dst + 16) = widen_codes<DT>(kr[i][2], kr[i][3]);
    }
    if (lane == 0) ((float*)(buf + KB + VB))[wave] = sc_k > 0.0f ? sc_k * a.scale : 1.0f;
  };
  auto put_v = [&](char* buf) {
#pragma unroll
    for (int i = 0; i < VC; ++i) {
      const uint32_t in[4] = {vr[0][i], vr[1][i], vr[2][i], vr[3][i]};
      uint32_t out[4];
      transpose4(in, out);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x2 w = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(out[j], 1.0f, false)),
                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(out[j], 1.0f, true))};
        *(u32x2*)(buf + KB + ((4 * i + j) * 16 + v_c) * VLD + 2 * v_pos) = w;
      }
    }
    if (lane == 0) {
      float* dst = (float*)(buf + KB + VB) + 4 + wave;
      dst[0] = __builtin_amdgcn_logf(sc_v);
      dst[4] = sc_v > 0.0f ? __builtin_amdgcn_rcpf(sc_v) : 0.0f;
    }
  };
  f32x16 o[OT];
#pragma unroll
  for (int j = 0; j < OT; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;
  float top = -__builtin_inff(), sum = 0.0f;
  float ref = -kBigLift;  // what exponents are formed against: top (0 while there is none) - kBigLift

  // the keys of 32 tokens, half i of the step in buf, and their scores
  u32x4 kx[KS];
  auto read_keys = [&](const char* buf, int i) {
#pragma unroll
    for (int k = 0; k < KS; ++k) kx[k] = *(const u32x4*)(buf + (32 * i + c) * KLD + 32 * k + 16 * h);
  };
  auto dots = [&](f32x16& w) {
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) w = mfma32<DT>(kx[k], qf[k], w);
  };
  auto mask = [&](int t, f32x16& w) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int token = t + 8 * (e >> 2) + 4 * h + (e & 3);
      if (token < from || token >= to) w[e] = -__builtin_inff();
    }
  };
  // Their weights by an earlier maximum: it only has to keep them from overflowing, so it
  // moves where they may add up to more than kBigMost (seldom after the first steps), no weight
  // waits for this step's maximum and none is computed.  l adds up the denominator's share
  // before the weights are rounded to fp16, in fp32: a page of small values has a small
  // value scale, and weights that are 0 in fp16 may be what the denominator consists of.
  // (l is the weights times 1 / value scale of either 16-token tile, so that none is above
  // l / min(iv); a tile without a page has 0 there and only makes the maximum move early.)
  auto weight_pair = [&](int i, f32x2_t ks, f32x2_t shift_v, f32x2_t iv, const f32x16& w, float& l) {
    const int g = i >> 2;
    const float x = __builtin_amdgcn_exp2f(fmaf(w[2 * i], ks[g], shift_v[g]));
    const float y = __builtin_amdgcn_exp2f(fmaf(w[2 * i + 1], ks[g], shift_v[g]));
    l = i == 0 ? (x + y) * iv[g] : fmaf(x + y, iv[g], l);
    return pack_act2(x, y, KQ_DTYPE_F16);
  };
  auto base_of = [](float m) { return m == -__builtin_inff() ? 0.0f : m; };
  // Scores of the next 32 tokens with the weights of these between the products, an MFMA to
  // every pair or two: the order is pinned.
  auto dots_under_weights = [&](f32x16& next, f32x2_t ks, f32x2_t lv, f32x2_t iv, const f32x16& w, u32x4 (&p)[2], float& l) {
    const f32x2_t shift_v = {lv[0] - ref, lv[1] - ref};
#pragma unroll
    for (int e = 0; e < 16; ++e) next[e] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      next = mfma32<DT>(kx[k], qf[k], next);
#pragma unroll
      for (int i = 8 * k / KS; i < 8 * (k + 1) / KS; ++i) p[i >> 2][i & 3] = weight_pair(i, ks, shift_v, iv, w, l);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(l));  // (not behind the branch that may compute them anew)
  };
  auto limit = [&](f32x2_t ks, f32x2_t lv, f32x2_t iv, const f32x16& w, u32x4 (&p)[2], float& l) {
    if (__ballot(l > kBigMost * fminf(iv[0], iv[1]) || !(fabsf(top) <= kCoarse)) == 0) return;
    // a 16-token tile's scale is positive, so its largest score is its largest dot product's
    float x[2] = {w[0], w[8]};
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      x[0] = fmaxf(x[0], w[e]);
      x[1] = fmaxf(x[1], w[8 + e]);
    }
    float m = fmaxf(fmaf(x[0], ks[0], lv[0]), fmaf(x[1], ks[1], lv[1]));
    const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(top, fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
    const float keep = __builtin_amdgcn_exp2f(top - base_of(m));
    sum *= keep;
#pragma unroll
    for (int j = 0; j < OT; ++j) o[j] *= keep;
    top = m;
    const float base = base_of(m);
    ref = base - kBigLift;
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // (exact differences, of at most kBigLift with it)
      const int g = i >> 2;
      const float u = __builtin_amdgcn_exp2f((fmaf(w[2 * i], ks[g], lv[g]) - base) + kBigLift);
      const float v = __builtin_amdgcn_exp2f((fmaf(w[2 * i + 1], ks[g], lv[g]) - base) + kBigLift);
      l = i == 0 ? (u + v) * iv[g] : fmaf(u + v, iv[g], l);
      p[i >> 2][i & 3] = pack_act2(u, v, KQ_DTYPE_F16);
    }
  };
  u32x4 vx[2][OT];
  auto read_values = [&](const char* buf, int i) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < OT; ++j) vx[k][j] = *(const u32x4*)(buf + KB + (32 * j + c) * VLD + 64 * i + 32 * k + 16 * h);
  };
  auto add_values = [&](const u32x4 (&p)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < OT; ++j) o[j] = mfma32<KQ_DTYPE_F16>(vx[k][j], p[k], o[j]);
  };
  auto pair_at = [&](const char* buf, int which, int i) { return *(const f32x2_t*)(buf + KB + VB + 16 * which + 8 * i); };

  // Half steps of 32 tokens, each one's weights computed while the next one's scores are:
  // the matrix cores have work from the wave itself, not from the other one on its SIMD
  // alone.  The next step's keys reach LDS before its first half is needed, in the middle
  // of this step, and its values at the end.
  if (lo < hi) {
    Place here = place_of(lo, page_at(lo));
    fetch_k(here);
    fetch_v(here);
    put_k(smem);
    put_v(smem);
    here = place_of(lo + 64, page_at(lo + 64));
    fetch_k(here);
    fetch_v(here);
    int next_page = page_at(lo + 128);
    meet();
    f32x16 x, y;
    read_keys(smem, 0);
    dots(x);
    int which = 0;
    auto step = [&](int t, auto masked) {
      const char* buf = smem + which * BUF;
      char* next = smem + (which ^ 1) * BUF;
      u32x4 p[2];
      float l;
      {
        const f32x2_t ks = pair_at(buf, 0, 0), lv = pair_at(buf, 1, 0), iv = pair_at(buf, 2, 0);
        read_keys(buf, 1);
        if constexpr (masked) mask(t, x);
        dots_under_weights(y, ks, lv, iv, x, p, l);
        read_values(buf, 0);
        limit(ks, lv, iv, x, p, l);
        add_values(p);
        sum += l;
        put_k(next);
        here = place_of(t + 128, next_page);
        fetch_k(here);
      }
      meet();
      {
        const f32x2_t ks = pair_at(buf, 0, 1), lv = pair_at(buf, 1, 1), iv = pair_at(buf, 2, 1);
        read_keys(next, 0);
        if constexpr (masked) mask(t + 32, y);
        dots_under_weights(x, ks, lv, iv, y, p, l);
        read_values(buf, 1);
        limit(ks, lv, iv, y, p, l);
        add_values(p);
        sum += l;
        put_v(next);
        fetch_v(here);
        next_page = page_at(t + 192);
      }
      meet();
      which ^= 1;
    };
    // steps that every row of the tile sees whole need no mask: those between
    int t = lo;
    for (; t < hi && t < lo_all; t += 64) step(t, std::true_type{});
    for (; t + 64 <= min(hi, hi_all); t += 64) step(t, std::false_type{});
    for (; t < hi; t += 64) step(t, std::true_type{});
  }
  sum += __shfl_xor(sum, 32, 64);
  if (sum != sum && !any_there(pages, cache.pages, max(from, lo), min(to, hi), shift)) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < OT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;
  }

  if (!real) return;
  // element e of tile j: row R = 32 j + 8 (e / 4) + 4 h + e % 4 of the values, so that
  // elements e and e + 8 are neighbouring d
  auto store = [&](auto put) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int j = 0; j < OT; ++j) put((8 * (e >> 2) + 4 * h + (e & 3)) * VY + 2 * j, o[j][e], o[j][8 + e]);
  };
  if (a.splits > 1) {
    float* dst = a.big_part + ((((int64_t)head * a.big_tiles + nth) * a.splits + part) * kBigRows + wave * 32 + c) * LD;
    store([&](int d, float x, float y) { *(f32x2_t*)(dst + d) = f32x2_t{x, y}; });
    if (h == 0) *(f32x2_t*)(dst + D) = f32x2_t{top, sum};
    return;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that sees no token is zero)
  uint16_t* dst = a.out + ((int64_t)(q.row0 + row) * a.heads + head * group + qh) * D;
  store([&](int d, float x, float y) { *(uint32_t*)(dst + d) = pack_act2(x * inv, y * inv, DT); });
}

// Workgroups that fill the chip: CUs times what the registers let a CU hold.
constexpr int rows_slots(int64_t dim) { return 256 * (dim == 256 ? 2 : 3); }

constexpr int64_t tile_slots(int64_t dim) { return 256 * (dim == 64 ? 3 : dim == 128 ? 2 : 1); }

// Tokens up to which sequences of few rows go to large tiles as well, a launch and a join
// less, where there are no more than 64 tokens to a new row and the tiles are few (32 heads
// over 8 of 128: 24 sequences of up to 300 rows behind 2000 tokens 103 -> 94 us, 12 of 64
// behind 1000 45 -> 32; but a prompt of 512 rows beside one token behind 2000 37 -> 47, behind
// 8000 42 -> 81, beside 100 tokens behind 1000 66 -> 81)
constexpr int64_t kAlone = 2048, kAloneTokens = 64;

// rows * group up to which a sequence goes to tiles of 16 rows, which stream its
// tokens once per tile (24 sequences behind 3000 tokens, 4 heads a kv head: 5 rows 65 us
// either way; 15 rows 79 in large tiles, 113 in small ones).  That is for sequences that
// fill the chip.  Few of them fall off at this limit, since large tiles are cut no finer
// than 1024 tokens: one behind 1000, 4096 and 16384, 32 heads over 8 of 128, 8 rows 15, 18
// and 31 us and 9 rows 27, 31 and 35; heads of 256, 8 over 1, 4 rows 22, 16 and 23 and
// 8 rows 52, 58 and 60; four behind 16384 do not (8 rows 65, 9 rows 60).
constexpr int kFewItems = 32;

// Tokens up to which one workgroup reads a tile's whole: a second launch costs 4 us of host
// time (16 contexts of up to 700 tokens on 8 kv heads 11.9 us whole, 13.1 shared out; 4 of
// 1000 13.4 and 12.7).  By the table's width, which is all that the host knows: in a table
// for 32768 tokens those 16 contexts take 14.5 us instead of 11.1, six prompts of kAlone's
// kind 82 instead of 71.
constexpr int64_t kWhole = 1024;
// ... and where a window makes the tiles alike and they fill the chip by themselves (64 single
// tokens on 4 kv heads of 128, windows of 900, 1400 and 1900: 16.7, 21.5 and 25.7 us whole,
// 25.4, 31.7 and 37.9 shared out; 4 on 8 kv heads, 1400: 17.1 and 13.4)
constexpr int64_t kWholeMany = 2048;

struct Plan {
  bool rows, tiles;  // which kernels run
  int few, shares, splits, block_shift;
  int64_t big_tiles, small_tiles;  // small_tiles: 16-row tiles that may need joining (0: look at every row)
  size_t part, big_part;  // bytes
};

// From what the host knows: rows and sequences, not their lengths.  `alone`: large tiles
// take every sequence, however few its rows are.
static Plan plan_with(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size, int64_t width,
                      int64_t seqs, int64_t window, bool alone) {
  Plan p{};
  const int64_t group = heads / kv_heads, items = rows * group, tokens = width * page_size;
  // tokens that some rows of a sequence can look at, from their first step on
  auto span_of = [&](int64_t most_rows) { return window > 0 ? std::min(tokens, window + most_rows + 64) : tokens; };
  int64_t span = span_of(rows);
  if (rows <= seqs || items <= kFewItems) {  // single tokens (no more rows than sequences)
    p.rows = true;
    p.few = 0x7fffffff;
  } else {
    p.rows = !alone && seqs > 1;
    p.tiles = true;
    p.few = p.rows ? kFewItems : 0;
    // (no sequence of more than `few` items ends more than one tile short)
    const int64_t ends = std::min<int64_t>(seqs, items / (p.few + 1));
    p.big_tiles = (items + ends * (kBigRows - 1)) / kBigRows;
    // few tiles: cut their tokens until every workgroup slot has some, but not below 1024 each: a cut costs the
    // second launch and the partial sums' way through memory (32 heads over 8 of 128 channels, one sequence: 512 rows
    // behind 4096 tokens 130 us whole, 70 cut; 1024 rows behind 8192 on 4 heads 250 and 166; 1024 rows of 1024 42 and
    // 52; fewer rows than these would want finer cuts, see kFewItems)
    const int64_t most = std::max<int64_t>(span_of(kBigRows) / 1024, 1);
    p.splits = (int)std::min<int64_t>(most, std::max<int64_t>(1, tile_slots(dim) / std::max<int64_t>(1, p.big_tiles * kv_heads)));
    span = span_of(std::max<int64_t>(kFewItems / group, 1));
  }
  p.splits = std::max(p.splits, 1);
  if (p.rows && p.splits == 1) p.small_tiles = p.tiles ? std::min<int64_t>(rows * group, seqs * (kFewItems / 16)) : 0;
  p.shares = (int)std::max<int64_t>(rows_slots(dim) / kv_heads, 1);
  const bool whole = span <= (window > 0 && seqs * kv_heads >= 256 ? kWholeMany : kWhole);
  p.block_shift = 2;
  while (whole && (64LL << p.block_shift) < span) ++p.block_shift;  // (no tile in two blocks: they would need `part`)
  if (p.rows && !whole) p.part = sizeof(float) * (size_t)(p.shares * kv_heads * 2 * 16 * (dim + 4));
  if (p.splits > 1) p.big_part = sizeof(float) * (size_t)(p.big_tiles * kv_heads * p.splits * kBigRows * (dim + 4));
  return p;
}

static Plan plan_of(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size, int64_t width,
                    int64_t seqs, int64_t window) {
  const int64_t tokens = width * page_size, span = window > 0 ? std::min(tokens, window + kFewItems + 64) : tokens;
  const int64_t tiles = rows * (heads / kv_heads) / kBigRows + seqs;
  return plan_with(rows, heads, kv_heads, dim, page_size, width, seqs, window,
                   span <= kAlone && kAloneTokens * rows >= seqs * span && tiles * kv_heads <= 2 * tile_slots(dim));
}

template <int D, int DT, int NT, int PP>
static void launch_rows(const AttendArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  hipLaunchKernelGGL((kv_attend_rows_kernel<D, DT, NT, PP>), dim3((unsigned)a.shares, (unsigned)c.kv_heads), dim3(256), 0, st, a,
                     c, b, b.table, c.k_scale, c.v_scale);
}

template <int D, int DT>
static void launch(const AttendArgs& a, const Plan& p, const KvCache& c, const KvBatch& b, hipStream_t st) {
  constexpr int NT = D == 256 ? 2 : 4;  // (registers)
  const int page = 1 << c.page_shift;
  if (p.rows) {
    if (page >= 16 * NT)
      launch_rows<D, DT, NT, 1>(a, c, b, st);
    else if (page == 8 * NT)
      launch_rows<D, DT, NT, 2>(a, c, b, st);
    else if constexpr (NT == 4)
      launch_rows<D, DT, NT, 4>(a, c, b, st);
  }
  if (p.tiles)
    hipLaunchKernelGGL((kv_attend_tiles_kernel<D, DT>), dim3((unsigned)(p.big_tiles * p.splits * c.kv_heads)), dim3(256), 0,
                       st, a, c, b, b.table, c.k_scale, c.v_scale);
  if (a.part != nullptr || a.big_part != nullptr) {
    const int64_t waves = p.small_tiles > 0 ? (int64_t)p.small_tiles * 16 * c.kv_heads : (int64_t)b.rows * a.heads;
    hipLaunchKernelGGL((kv_attend_join_kernel<D, DT>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a, c, b,
                       (int)p.small_tiles);
  }
}

template <int D>
static void launch_dtype(const AttendArgs& a, const Plan& p, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  if (dtype == KQ_DTYPE_BF16)
    launch<D, KQ_DTYPE_BF16>(a, p, c, b, st);
  else
    launch<D, KQ_DTYPE_F16>(a, p, c, b, st);
}

}  // namespace kq

using namespace kq;

extern "C" size_t kq_kv_attention_workspace_size(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                                 int64_t page_size, int64_t table_width, int64_t seqs) {
  if (rows < 1 || heads < 1 || kv_heads < 1 || dim < 1 || page_size < 1 || table_width < 0 || seqs < 0) return 0;
  size_t most = 0;  // (a window needs no more than none)
  for (const bool alone : {false, true}) {
    const Plan p = plan_with(rows, heads, kv_heads, dim, page_size, table_width, seqs, 0, alone);
    most = std::max(most, p.part + p.big_part);
  }
  return most;
}

extern "C" int kq_kv_attention(const void* q, int64_t q_ld, int64_t q_hs, int dtype, int64_t rows, int64_t heads,
                               int64_t kv_heads, int64_t dim, const uint8_t* k_cache, const uint8_t* v_cache,
                               const float* k_scale, const float* v_scale, int64_t pages, int64_t page_size,
                               const int32_t* table, int64_t table_ld, int64_t table_width, const int32_t* cu,
                               const int32_t* lengths, int64_t seqs, float scale, int causal, int64_t window, void* out,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "kq_kv_attention";
  int rc = kv_check(what, dtype, rows, heads, kv_heads, dim, page_size, pages, seqs, table_width, table_ld);
  if (rc) return rc;
  if (!(fabsf(scale) <= 0x1p100f)) {
    set_error("%s: scale %g", what, (double)scale);
    return KQ_EINVAL;
  }
  if (window < 0 || window > (1 << 30) || (window > 0 && !causal)) {
    set_error("%s: window %lld (a window is of causal attention)", what, (long long)window);
    return KQ_EINVAL;
  }
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) % 16 != 0 ||
      (q_ld | q_hs) % 8 != 0) {
    set_error("%s: tensors need 16-byte aligned rows and heads", what);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  const bool empty = seqs == 0 || pages == 0 || table_width == 0;  // every row is zero
  Plan p = plan_of(rows, heads, kv_heads, dim, page_size, table_width, seqs, window);
  if (empty) {
    p = Plan{};
    p.rows = true;
    p.shares = (int)std::min<int64_t>(rows, 1024);
  }
  if (p.part + p.big_part > 0 && (workspace == nullptr || workspace_bytes < p.part + p.big_part)) {
    set_error("%s: workspace of %zu bytes is too small", what, workspace_bytes);
    return KQ_EWORKSPACE;
  }
  // threads of one launch, and blocks of all tiles of 16 (beside large ones: of few rows a sequence)
  const int64_t few_tiles = empty || !p.rows ? 0 : p.tiles ? seqs * (kFewItems / 16) : rows * (heads / kv_heads) / 16 + seqs;
  const int64_t blocks = few_tiles * ((table_width * page_size + 255) / 256);
  if (rows * heads * 64 >= (1LL << 32) || p.big_tiles * p.splits * kv_heads * 512 >= (1LL << 32) || blocks >= (1LL << 30)) {
    set_error("%s: %lld rows of %lld heads over up to %lld tokens are past the supported range", what, (long long)rows,
              (long long)heads, (long long)(table_width * page_size));
    return KQ_EINVAL;
  }
  AttendArgs a{};
  a.q = (const uint16_t*)q;
  a.q_ld = q_ld, a.q_hs = q_hs;
  a.out = (uint16_t*)out;
  a.part = p.part > 0 ? (float*)workspace : nullptr;
  a.big_part = p.big_part > 0 ? (float*)((char*)workspace + p.part) : nullptr;
  a.scale = fmaxf(fabsf(scale) * 1.44269504088896340736f, 0x1p-60f);
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.heads = (int)heads, a.causal = causal != 0, a.window = (int)window;
  a.most_blocks = (int)blocks;
  a.shares = p.shares, a.block_shift = p.block_shift, a.few = p.few, a.big_tiles = (int)p.big_tiles, a.splits = p.splits;
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  const KvCache c{(uint8_t*)k_cache, (uint8_t*)v_cache, (float*)k_scale, (float*)v_scale, pages, (int)kv_heads, shift};
  // (without pages or table columns no sequence is looked at and all rows are padding)
  const KvBatch b{table, cu, lengths, table_ld, empty ? 0 : (int)seqs, (int)table_width, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  if (dim == 64)
    launch_dtype<64>(a, p, c, b, dtype, st);
  else if (dim == 128)
    launch_dtype<128>(a, p, c, b, dtype, st);
  else
    launch_dtype<256>(a, p, c, b, dtype, st);
  return check_launch(what);
}
