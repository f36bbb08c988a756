// Attention of drafted tokens that branch, over the paged e4m3 cache.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = exp(scale * q . k_t - max) over the tokens a row
// sees: those before its sequence's new ones (from its position less the window on), and
// the new ones whose bit its mask holds.  Scores, scales and weights are formed as in
// attention over prompts and single tokens: w_t = log2(e) scale k_scale (q . code_t) +
// log2 v_scale, exp2(w_t - max w + lift) in fp16 (11 bits down to 2^-29 of the largest and
// some down to 2^-40, in tiles of 64 and 128 columns 2^-23 and 2^-34) times the value's codes,
// the denominator in fp32 from weights not yet rounded over v_scale, maxima, denominators and
// outputs in fp32.  The width of a tile follows the batch, so that a tree's last bits may differ
// from one batch to another.
//
// Times are of calls in a captured graph, joins included, unless they are said to be of one kernel
// under the profiler, where kernels take up to a tenth longer.
#include "kq_kv_attend.h"

#include <algorithm>
#include <type_traits>

namespace kq {

struct TreeArgs {
  const uint16_t* q;
  int64_t q_ld, q_hs;
  uint16_t* out;  // [rows][heads][D]
  const uint32_t* mask;  // [rows][words]
  const int32_t* positions;
  float* part;    // partial outputs of split tiles, null: none can be split
  float scale;    // magnitude times log2 e, at least 2^-60: times a page's scale it stays positive
  uint32_t q_sign;  // the softmax scale's sign, for two 16-bit elements
  int words, heads, window;
  int most_blocks;  // no batch has more
  int shares;     // workgroups per kv head that the batch's tokens are dealt to
  int block_shift;  // log2 of the 64-token steps of a block
  int alike;      // whether every workgroup gets one part of one tile
  int near;       // whether neighbouring shares go to one XCD
};

constexpr float kLift = 15.0f;  // log2 of the largest weight

// A sequence's rows (drafted tokens x the group's query heads) go to tiles of TW, the
// tokens that they see to blocks.  Where no batch has more tiles than there are workgroups to a
// kv head, tiles are cut into parts of as few blocks as gives every part a workgroup of its
// own.  Otherwise, and in tiles of 16 columns, the blocks of all tiles, one after the other, are
// dealt to the workgroups in equal runs: whole tiles, and at most two parts of tiles.  Parts that
// are not whole go through memory: those that do not begin their tile to a workgroup's place 0,
// the others to place 1.  (A workgroup with two parts begins twice, 8 us, and finding the length
// of parts takes 1: 32 trees of up to 32 rows behind 6000 tokens, 32 heads over 4, in runs 102 us,
// in parts of one length 96; one tree of 16 rows behind 4000, 32 heads over 8, 18.9 and 19.9.)
template <int TW>
struct TreeDeal {
  const TreeArgs& a;
  int group;

  // 64-token step of the first token that any row sees
  KQ_DEV int first(const KvSeq& q) const { return a.window > 0 ? max(q.first + 1 - a.window, 0) >> 6 : 0; }
  KQ_DEV int blocks(const KvSeq& q) const { return (max(((q.tokens + 63) >> 6) - first(q), 1) + (1 << a.block_shift) - 1) >> a.block_shift; }
  KQ_DEV int tiles(const KvSeq& q) const { return (q.rows * group + TW - 1) / TW; }
  KQ_DEV int operator()(const KvSeq& q) const { return tiles(q) * blocks(q); }
  KQ_DEV int parts(const KvSeq& q, int length) const { return (int)((uint32_t)(blocks(q) + length - 1) / (uint32_t)length); }
  // blocks of all tiles (held to what a batch can have, whatever the row bounds say)
  KQ_DEV int all(const KvLanes& lanes) const { return (int)min((uint32_t)lanes.total(*this), (uint32_t)a.most_blocks); }
  KQ_DEV int run(const KvLanes& lanes) const { return scalar((int)(((uint32_t)all(lanes) + (uint32_t)a.shares - 1) / (uint32_t)a.shares)); }
  // blocks of a part: the fewest that need no more parts than there are workgroups
  KQ_DEV int length(const KvLanes& lanes) const {
    const KvSeq q = lanes.at_lane(0);
    const int tiles_ = tiles(q), blocks_ = blocks(q);  // (of the lane's sequence, while a wave holds them all)
    const int most = all(lanes), spare = a.shares - lanes.total([&](const KvSeq& p) { return tiles(p); });
    int lo = max((int)((uint32_t)(most + a.shares - 1) / (uint32_t)a.shares), 1);
    // (a tile has at most one part that is not full; without spare workgroups every tile is one)
    int hi = max(spare > 0 ? (int)((uint32_t)(most + spare - 1) / (uint32_t)spare)
                           : (int)(((int64_t)lanes.b.table_width << lanes.shift) >> (6 + a.block_shift)) + 2, lo);
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const int parts_ = lanes.held ? __builtin_amdgcn_readlane(wave_scan(tiles_ * (int)((uint32_t)(blocks_ + mid - 1) / (uint32_t)mid)), 63)
                                    : lanes.total([&](const KvSeq& p) { return tiles(p) * parts(p, mid); });
      if (parts_ <= a.shares)
        hi = mid;
      else
        lo = mid + 1;
    }
    return scalar(lo);
  }
};

// Workgroups go to the 8 XCDs in turn: those of one take neighbouring shares, so that the tiles of
// a tree that read the same tokens at the same time do so through one L2 (16 trees of 64 columns
// behind 900 tokens 20.8 us, 24.1 in turn; 16 of 512 behind 6000 134 and 137).  Where several tiles of
// a sequence are cut by runs, equal parts of them are far apart, and meet more often in turn (one tree
// of 64 columns behind 16000 tokens 32 and 27).
KQ_DEV int share_of(const TreeArgs& a, int x, int shares) {
  if (!a.near || x >= shares) return x;
  const int xcd = x & 7, each = shares >> 3, more = shares & 7;
  return xcd * each + min(xcd, more) + (x >> 3);
}

// A workgroup's blocks: from `within` of `tile` of sequence s (-1: none) on, `end` - `block` of them.
struct TreeRun {
  int share, s, tile, within, blocks, block, end;
  KvSeq q;
};
template <int TW>
KQ_DEV TreeRun run_of(const TreeArgs& a, const KvLanes& lanes, const TreeDeal<TW>& deal, int x) {
  TreeRun r{};
  if (a.alike) {
    const int length = deal.length(lanes);
    int unit;
    r.share = share_of(a, x, a.shares);
    r.s = lanes.find(r.share, unit, [&](const KvSeq& q) { return deal.tiles(q) * deal.parts(q, length); });
    if (r.s < 0) return r;
    r.q = lanes[r.s];
    r.blocks = deal.blocks(r.q);
    const int tiles = scalar(deal.tiles(r.q)), nth = scalar(unit / tiles);  // (all tiles' first parts, then their second)
    r.tile = unit - nth * tiles;
    r.within = nth * length;
    r.end = min(length, r.blocks - r.within);
    return r;
  }
  const int all = deal.all(lanes), run = max(scalar((int)(((uint32_t)all + (uint32_t)a.shares - 1) / (uint32_t)a.shares)), 1);
  r.share = share_of(a, x, scalar((int)((uint32_t)(all + run - 1) / (uint32_t)run)));  // (of those with blocks)
  r.block = r.share * run;
  r.end = r.block + run;
  int unit;
  r.s = lanes.find(r.block, unit, deal);
  if (r.s < 0) return r;
  r.q = lanes[r.s];
  r.blocks = deal.blocks(r.q);
  r.tile = scalar(unit / r.blocks);
  r.within = unit - r.tile * r.blocks;
  return r;
}

// A row's mask with all ones before it, for the tokens before the new ones, and none behind.
// The load is always in range and may be on its way long before the word is asked for.
KQ_DEV uint32_t load_word(const uint32_t* mask, int words, int at) { return mask[min(max(at, 0), words - 1)]; }
KQ_DEV uint32_t word_at(uint32_t loaded, int words, int at) { return at < 0 ? ~0u : at < words ? loaded : 0u; }
// 32 bits from bit `shift` of two words on.
KQ_DEV uint32_t bits_at(uint32_t lo, uint32_t hi, int shift) { return (uint32_t)(((uint64_t)hi << 32 | lo) >> (shift & 31)); }

// Bits of tokens 0..31 from the n-th on.
KQ_DEV uint32_t tokens_from(int n) { return n <= 0 ? ~0u : n >= 32 ? 0u : ~0u << n; }

// The wave's priority by how far its workgroup is through its part: the CU serves the older of two
// workgroups first (with equal parts, it was through in 94 us and the other in 121, alone at the end),
// so the one that is ahead gives way.  16 trees of 512 columns behind 6000 tokens 135 -> 132 us, 32 of
// up to 256 95 -> 92, 24 windows of 1024 15.9 -> 15.5.
KQ_DEV void give_way(int done, int all) {
  if (2 * done < all)
    __builtin_amdgcn_s_setprio(3);
  else if (4 * done < 3 * all)
    __builtin_amdgcn_s_setprio(2);
  else if (10 * done < 9 * all)
    __builtin_amdgcn_s_setprio(1);
  else
    __builtin_amdgcn_s_setprio(0);
}

// One workgroup: its run of blocks of one kv head, tile by tile; its four waves take a
// tile's steps of 16 * NT tokens in turn, each for all of the tile's 16 * MT columns, so that
// a token is loaded and widened once for all of them, and by one wave.
//
// The products run transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32 MFMAs: lane (c, b) =
// (l % 16, l / 16) holds scores of columns c of the MT tiles for tokens 4b..4b+3 of each 16,
// which are what it hands over as its part of P^T.  Loads go from memory to registers through
// resources of one page's tile that end at the sequence's last token.
//
// Bound by its chain of steps, not by bytes.  One tree of 12 rows behind 900 tokens, 32 heads over
// 8 of 128, eight waves to a tile: 13.2 us (1.9 MB, which 0.4 would do).  Of them, by time stamps, 0.5 are
// bounds and padding, 0.7 the deal, 2.4 table, pages and the first keys, 2.2 the rest of the first step (its
// values, the next step's keys), 2.0 the second, 2.1 until all waves' parts are in LDS, 1.0 merge and
// store, and 2.2 lie between the end of one launch and the start of the next.  24 windows of 1024, 16 heads of
// 64: 15.5 us, 3.0 TB/s.
template <int D, int DT, int NT, int PP, int MT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : D * MT <= 64 ? 3 : D * MT <= 256 ? 2 : 1)
kv_tree_kernel(TreeArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
               const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int KS = D / 32;   // MFMA steps along a key
  constexpr int VD = D / 64;   // dwords of a token's value a lane holds
  constexpr int OT = D / 16;   // output tiles
  constexpr int ST = 16 * NT;  // tokens of a step
  constexpr int TW = 16 * MT;
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds[WAVES * 16 * LD];
  const int lane = lane_id(), wave = scalar(wave_id()), c = lane & 15, b = lane >> 4;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int head = (int)blockIdx.y;

  const KvLanes lanes(batch, shift);
  zero_padding<D>(a, batch, head, group, (int)blockIdx.x, (int)gridDim.x, 64 * WAVES);
  const TreeDeal<TW> deal{a, group};
  const TreeRun given = run_of(a, lanes, deal, (int)blockIdx.x);
  if (given.s < 0) return;
  KvSeq q = given.q;
  int s = given.s, tile = given.tile, within = given.within, blocks = given.blocks, block = given.block;
  const int run_end = given.end;
  const int64_t tile_bytes = (int64_t)D << shift;
  const int in_page = (1 << shift) - 1;
  const int k_lane = c * D + 16 * b, v_lane = 4 * b * D + c * (D / 16);

  // One part of a tile: its bounds, its rows of Q, and its loads on their way.
  int from[MT];             // first token that a column sees (past all: the column sees none)
  const uint32_t* bits[MT];
  int lo, hi, lo_all, part_blocks;
  const int32_t* pages;
  u32x4 qf[MT][KS];
  int id;                   // lane l: the page that holds the step's tokens from l % PP * (ST / PP) on
  u32x4 kx[NT][D / 64];     // a step's keys and values, and their pages' scales (0: no tokens there)
  uint32_t vx[NT * 4][VD];
  float ks, vs;
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
          kx[i][h] = __builtin_bit_cast(u32x4, kq_rbl_v4i32(src, k_lane + 64 * h, off + (i - p * (NT / PP)) * 16 * D, 0));
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
            vx[4 * i + r][0] = (uint32_t)kq_rbl_i32(src, v_lane + r * D, so, 0);
          } else if constexpr (VD == 2) {
            const i32x2 w = kq_rbl_v2i32(src, v_lane + r * D, so, 0);
            vx[4 * i + r][0] = (uint32_t)w[0];
            vx[4 * i + r][1] = (uint32_t)w[1];
          } else {
            const i32x4 w = kq_rbl_v4i32(src, v_lane + r * D, so, 0);
#pragma unroll
            for (int d = 0; d < VD; ++d) vx[4 * i + r][d] = (uint32_t)w[d];
          }
        }
    }
  };
  auto begin_loads = [&] {
    hi = q.tokens;
    part_blocks = min(blocks - within, run_end - block);
    const int begin = deal.first(q) * 64 + (within << (6 + a.block_shift));
    hi = (int)min((int64_t)hi, (int64_t)begin + ((int64_t)part_blocks << (6 + a.block_shift)));
    lo = begin;
    pages = table + (int64_t)s * batch.table_ld;
    const int t = lo + ST * wave;
    pages_of(t);
    uint32_t most_from = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int item = tile * TW + 16 * m + c;  // this lane's column: row item / group, head item % group
      const bool real = item < q.rows * group;
      const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
      const int pos = a.positions[q.row0 + row];
      bits[m] = a.mask + (int64_t)(q.row0 + row) * a.words;
      from[m] = !real ? 0 : pos < 0 ? 0x7fffffff : a.window > 0 ? min(max(max(pos, q.first) - (a.window - 1), 0), max(q.first, 0)) : 0;
      most_from = max(most_from, (uint32_t)from[m]);
      // (columns past the rows compute the first one's again, and are not stored)
      const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
      for (int i = 0; i < KS; ++i) qf[m][i] = *(const u32x4*)(src + 64 * (i >> 1) + 16 * b + 8 * (i & 1)) ^ a.q_sign;
    }
    lo_all = (int)wave_max_u32_dpp(most_from);
    place(t);
    load_keys(t);
    load_values(t);
    pages_of(t + WAVES * ST);
  };

  // a step's words of the masks, a step ahead, where it is not seen whole
  int last;
  uint32_t word[MT][NT / 2 + 1];
  auto words_of = [&](int t) {
    if (t + ST <= last) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g <= NT / 2; ++g) word[m][g] = load_word(bits[m], a.words, ((t - q.first) >> 5) + g);
  };
  auto begin_part = [&] {
    begin_loads();
    last = min(q.first, q.tokens);  // (steps that end at or before it are seen whole, but for a window)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g <= NT / 2; ++g) word[m][g] = 0;
    words_of(lo + ST * wave);
  };

  f32x4 o[MT][OT];
  float top[MT], sum[MT];
  auto step = [&](int t) {
    f32x4 w[MT][NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int m = 0; m < MT; ++m) w[m][i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < KS / 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x4 key = widen_codes<DT>(kx[i][h][2 * e], kx[i][h][2 * e + 1]);
#pragma unroll
          for (int m = 0; m < MT; ++m) w[m][i] = mfma16<DT>(key, qf[m][2 * h + e], w[m][i]);
        }
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
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = p * (NT / PP); i < (p + 1) * (NT / PP); ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) w[m][i][r] = fmaf(w[m][i][r], scale, shift_v);
    }
    // the keys' registers take the next step's while this one goes on, the values' then theirs
    place(t + WAVES * ST);
    load_keys(t + WAVES * ST);
    pages_of(t + 2 * WAVES * ST);
    if (t < lo_all || t + ST > last) {
      const int node = t - q.first, at = node >> 5;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int g = 0; g < NT / 2; ++g) {  // 32 tokens
          const int token = t + 32 * g;
          uint32_t seen = bits_at(word_at(word[m][g], a.words, at + g), word_at(word[m][g + 1], a.words, at + g + 1), node);
          seen = (seen & tokens_from(from[m] - token) & ~tokens_from(q.tokens - token)) >> (4 * b);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool sees = seen & (1u << (16 * (e >> 2) + (e & 3)));
            w[m][2 * g + (e >> 2)][e & 3] = sees ? w[m][2 * g + (e >> 2)][e & 3] : -__builtin_inff();
          }
        }
    }
    words_of(t + WAVES * ST);
    u32x4 p[MT][NT / 2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float most = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, w[m][i][r]);
      most = column_max(most);
      if (__ballot(most > top[m]) != 0) {
        most = fmaxf(most, top[m]);
        const float keep = __builtin_amdgcn_exp2f(top[m] - (most == -__builtin_inff() ? 0.0f : most));
        sum[m] *= keep;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[m][j] *= keep;
        top[m] = most;
      }
      const float base = top[m] == -__builtin_inff() ? 0.0f : top[m];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) w[m][i][r] = __builtin_amdgcn_exp2f((w[m][i][r] - base) + kLift);  // (the difference exact: at most kLift)
        sum[m] = fmaf(w[m][i][0] + w[m][i][1] + w[m][i][2] + w[m][i][3], inv_v[i / (NT / PP)], sum[m]);
        p[m][i >> 1][2 * (i & 1)] = pack_act2(w[m][i][0], w[m][i][1], KQ_DTYPE_F16);
        p[m][i >> 1][2 * (i & 1) + 1] = pack_act2(w[m][i][2], w[m][i][3], KQ_DTYPE_F16);
      }
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
        for (int j = 0; j < 4; ++j) {
          const u32x4 value = widen_codes<KQ_DTYPE_F16>(out[0][j], out[1][j]);
#pragma unroll
          for (int m = 0; m < MT; ++m) o[m][4 * d + j] = mfma16<KQ_DTYPE_F16>(value, p[m][g], o[m][4 * d + j]);
        }
      }
    load_values(t + WAVES * ST);
  };
  // Whether a column sees any token of this part that is there (its sum is NaN).
  auto sees_any = [&](int m) {
    if (any_there(pages, cache.pages, max(from[m], lo), min(max(q.first, 0), hi), shift)) return true;
    if (from[m] == 0x7fffffff) return false;
    for (int t = max(max(q.first, 0), lo); t < hi; ++t) {
      const int node = t - q.first;
      if ((word_at(load_word(bits[m], a.words, node >> 5), a.words, node >> 5) >> (node & 31) & 1) &&
          any_there(pages, cache.pages, t, t + 1, shift))
        return true;
    }
    return false;
  };

  begin_part();
  while (true) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int j = 0; j < OT; ++j) o[m][j] = f32x4{0, 0, 0, 0};
      top[m] = -__builtin_inff();
      sum[m] = 0.0f;
    }
    for (int t = lo + ST * wave; t < hi; t += WAVES * ST) {
      if constexpr (WAVES == 4) give_way((t - lo) >> 6, (hi - lo) >> 6);
      step(t);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sum[m] = column_sum(sum[m]);
      if (sum[m] != sum[m] && !sees_any(m)) {
        sum[m] = 0.0f;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[m][j] = f32x4{0, 0, 0, 0};
      }
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

    // the waves' parts meet in LDS, 16 columns at a time, added in wave order
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float* mine = lds + (wave * 16 + c) * LD;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < OT; j += 4)
          *(f32x4*)(mine + (4 * b + r) * OT + j) = f32x4{o[m][j][r], o[m][j + 1][r], o[m][j + 2][r], o[m][j + 3][r]};
      if (b == 0) {
        mine[D] = top[m];
        mine[D + 1] = sum[m];
      }
      meet();
      for (int i = (int)threadIdx.x; i < 16 * (D / 2); i += 64 * WAVES) {
        const int col = i / (D / 2), d = 2 * (i - col * (D / 2));
        const int it = old_tile * TW + 16 * m + col;
        if (it >= old.rows * group) break;
        float most = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < WAVES; ++v) most = fmaxf(most, lds[(v * 16 + col) * LD + D]);
        const float base = most == -__builtin_inff() ? 0.0f : most;
        float ox = 0.0f, oy = 0.0f, l = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
          const float* part = lds + (v * 16 + col) * LD;
          const float f = __builtin_amdgcn_exp2f(part[D] - base);
          ox += part[d] * f;
          oy += part[d + 1] * f;
          l += part[D + 1] * f;
        }
        if (!whole) {
          float* dst = a.part + ((((int64_t)head * a.shares + given.share) * 2 + (old_within == 0)) * TW + 16 * m + col) * LD;
          *(f32x2_t*)(dst + d) = f32x2_t{ox, oy};
          if (d == 0) *(f32x2_t*)(dst + D) = f32x2_t{most, l};
          continue;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees no token is zero)
        const int rw = it / group;
        uint32_t* dst = (uint32_t*)(a.out + ((int64_t)(old.row0 + rw) * a.heads + head * group + (it - rw * group)) * D + d);
        *dst = pack_act2(ox * inv, oy * inv, DT);
      }
      if (m + 1 < MT || more) meet();
    }
    if (!more) return;
  }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT>
KQ_DEV f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if (DT == KQ_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// log2 of the weights' lift in these tiles, whose maximum moves only when a lane's 16 weights
// may add up to more than fp16 holds, and the maximum's magnitude from which exponents are
// formed as exact differences.
constexpr float kTileLift = 9.0f, kTileMost = 65504.0f, kCoarse = 0x1p20f;

// One workgroup: its run of blocks of one kv head, tile by tile, tiles of 32 * CG columns.
// A step's tokens, 32 for each of TG = 4 / CG groups, are widened once for the whole
// workgroup, keys to Q's type in rows of one token and values to fp16 in rows of one d; a
// wave takes 32 columns and 32 tokens of it on 32x32x16 MFMAs.  So a wave's columns
// bound what LDS and the widening cost, and the workgroup's what memory does.
//
// The transposed products keep scores in the lane that hands them over as weights: lane
// (c, h) = (l % 32, l / 32) holds column c's scores of tokens 8 i + 4 h + 0..3, i < 4, which
// is the order (of each 16: 0-3, 8-11, then 4-7, 12-15) that the rows of values have.
//
// A step's weights are computed between the products of the next step's scores.  Codes
// travel two steps ahead in registers, keys reach LDS a step before values, and
// one barrier ends a step: it has read keys i + 1 and values i, and written keys i + 2 and
// values i + 1 where keys i and values i - 1 were.
//
// MFMAs (39% busy), vector instructions (48%) and LDS (44%) bound it in turn, with two workgroups
// to a CU by their registers: 32 tokens of 128 columns take a CU 1310 cycles of some 512 of MFMA.
// Two trees of 48 rows behind 100000 tokens, 28 heads over 4 of 128: 186 to 192 us on different cards,
// 0.72 PFLOP/s in the middle (0.83 with the columns past 336 that pad the last tile); 32 of up to 32 behind up to 6000, 32
// over 4: 93 us, 0.46 PFLOP/s, as parts end unevenly and tiles are padded to 128.  Joins are 11 us of each
// under the profiler.
template <int D, int DT, int CG>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2)
kv_tree_tiles_kernel(TreeArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
                     const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int TG = 4 / CG, ST = 64, TW = 32 * CG;
  constexpr int KS = D / 16;            // MFMA steps along a key
  constexpr int OT = D / 32;            // output tiles
  constexpr int KLD = 2 * D + 16;       // bytes of a key's row: 16 more spread eight lanes' reads over all banks
  constexpr int VLD = 2 * ST + 16;      // bytes of a d's row of values
  constexpr int KB = ST * KLD, VB = D * VLD + 64;  // a buffer of keys; of values, and per 16 tokens scale, log2 of the value scale, its inverse
  constexpr int KC = D / 64;            // 16-byte chunks of one token's key a thread moves
  constexpr int VY = D / 16, VC = VY / 4;  // bytes and dwords of each of four tokens' values a thread moves
  constexpr int LD = D + 4;
  constexpr int MERGE = 4 * 32 * LD * 4;  // every wave's columns at the end of a part
  constexpr int LDS = 2 * (KB + VB) > MERGE ? 2 * (KB + VB) : MERGE;
  __shared__ __attribute__((aligned(16))) char smem[LDS];
  const int wave = scalar(wave_id()), cg = wave % CG, tg = wave / CG;
  const int lane = lane_id(), c = lane & 31, h = lane >> 5, tid = (int)threadIdx.x;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int head = (int)blockIdx.y;
  const KvLanes lanes(batch, shift);
  zero_padding<D>(a, batch, head, group, (int)blockIdx.x, (int)gridDim.x, 256);
  const TreeDeal<TW> deal{a, group};
  const TreeRun given = run_of(a, lanes, deal, (int)blockIdx.x);
  if (given.s < 0) return;
  KvSeq q = given.q;
  int s = given.s, tile = given.tile, within = given.within, blocks = given.blocks, block = given.block;
  const int run_end = given.end;

  // what this thread moves: D / 4 bytes of a token's key, D / 16 of four tokens' values; a
  // wave moves 16 tokens, which lie in one page.  Row R of the values is d = R % 16 * VY + R / 16,
  // so that neighbouring lanes write neighbouring rows.
  const int k_tok = tid / 4, v_grp = tid / 16, v_c = tid % 16;
  const int k_lane = (k_tok % 16) * D + (tid % 4) * (D / 4), v_lane = 4 * (v_grp % 4) * D + v_c * VY;
  const int v_pos = (v_grp >> 2) * 16 + (v_grp & 1) * 8 + ((v_grp >> 1) & 1) * 4;
  const int tile_shift = shift + (D == 64 ? 6 : D == 128 ? 7 : 8);  // log2 of a page's bytes
  const int in_page = (1 << shift) - 1;

  while (true) {
    const int item = tile * TW + cg * 32 + c;
    const bool real = item < q.rows * group;
    const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
    const int pos = a.positions[q.row0 + row];
    const uint32_t* bits = a.mask + (int64_t)(q.row0 + row) * a.words;
    const int from = !real ? 0 : pos < 0 ? 0x7fffffff : a.window > 0 ? min(max(max(pos, q.first) - (a.window - 1), 0), max(q.first, 0)) : 0;
    const int part_blocks = min(blocks - within, run_end - block);
    const int lo = deal.first(q) * 64 + (within << (6 + a.block_shift));
    const int hi = (int)min((int64_t)q.tokens, (int64_t)lo + ((int64_t)part_blocks << (6 + a.block_shift)));
    const int32_t* pages = table + (int64_t)s * batch.table_ld;
    u32x4 qf[KS];  // (columns past the rows compute the first one's again, and are not stored)
    const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *(const u32x4*)(src + 16 * i + 8 * h);

    auto page_at = [&](int t) { return pages[min(t + 16 * wave, max(hi - 1, 0)) >> shift]; };
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
    u32x4 kr[KC];
    uint32_t vr[4][VC];
    float sc_k = 0.0f, sc_v = 0.0f;
    auto fetch_k = [&](const Place& p) {
      const i32x4 src = make_rsrc(cache.k + ((int64_t)p.head_tile << tile_shift), (uint32_t)p.size);
#pragma unroll
      for (int i = 0; i < KC; ++i) kr[i] = __builtin_bit_cast(u32x4, kq_rbl_v4i32(src, k_lane + 16 * i, p.off, 0));
    };
    auto fetch_v = [&](const Place& p) {
      const i32x4 src = make_rsrc(cache.v + ((int64_t)p.head_tile << tile_shift), (uint32_t)p.size);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (VC == 1) {
          vr[r][0] = (uint32_t)kq_rbl_i32(src, v_lane + r * D, p.off, 0);
        } else if constexpr (VC == 2) {
          const i32x2 x = kq_rbl_v2i32(src, v_lane + r * D, p.off, 0);
          vr[r][0] = (uint32_t)x[0], vr[r][1] = (uint32_t)x[1];
        } else {
          const i32x4 x = kq_rbl_v4i32(src, v_lane + r * D, p.off, 0);
#pragma unroll
          for (int i = 0; i < VC; ++i) vr[r][i] = (uint32_t)x[i];
        }
      }
      // (vector loads, which the barriers do not wait for; 0 where there is no page)
      sc_k = __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(k_scale + p.head_tile, p.size != 0 ? 4 : 0), 0, 0, 0));
      sc_v = __builtin_bit_cast(float, kq_rbl_i32(make_rsrc(v_scale + p.head_tile, p.size != 0 ? 4 : 0), 0, 0, 0));
    };
    auto put_k = [&](char* buf) {
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        char* dst = buf + k_tok * KLD + 2 * ((tid % 4) * (D / 4) + 16 * i);
        *(u32x4*)dst = widen_codes<DT>(kr[i][0], kr[i][1]);
        *(u32x4*)(dst + 16) = widen_codes<DT>(kr[i][2], kr[i][3]);
      }
    };
    auto put_v = [&](char* buf) {
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const uint32_t in[4] = {vr[0][i], vr[1][i], vr[2][i], vr[3][i]};
        uint32_t out[4];
        transpose4(in, out);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x2 x = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(out[j], 1.0f, false)),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(out[j], 1.0f, true))};
          *(u32x2*)(buf + ((4 * i + j) * 16 + v_c) * VLD + 2 * v_pos) = x;
        }
      }
      if (lane == 0) {
        float* dst = (float*)(buf + D * VLD) + wave;
        dst[0] = sc_k > 0.0f ? sc_k * a.scale : 1.0f;
        dst[4] = __builtin_amdgcn_logf(sc_v);
        dst[8] = sc_v > 0.0f ? __builtin_amdgcn_rcpf(sc_v) : 0.0f;
      }
    };
    f32x16 o[OT];
#pragma unroll
    for (int j = 0; j < OT; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;
    float top = -__builtin_inff(), sum = 0.0f;
    float ref = -kTileLift;  // what exponents are formed against: top (0 while there is none) - kTileLift

    // operands of 32 tokens of a step, its half `i`
    auto key_of = [&](const char* buf, int i, int k) { return *(const u32x4*)(buf + (32 * i + c) * KLD + 32 * k + 16 * h); };
    auto value_of = [&](const char* buf, int i, int k, int j) { return *(const u32x4*)(buf + (32 * j + c) * VLD + 64 * i + 32 * k + 16 * h); };
    // Weights by an earlier maximum, which only has to keep them from overflowing; l adds up
    // the denominator's share in fp32, weights times 1 / value scale.
    auto weight_pair = [&](int i, f32x2_t ks, f32x2_t shift_v, f32x2_t iv, const f32x16& w, float& l) {
      const int g = i >> 2;
      const float x = __builtin_amdgcn_exp2f(fmaf(w[2 * i], ks[g], shift_v[g]));
      const float y = __builtin_amdgcn_exp2f(fmaf(w[2 * i + 1], ks[g], shift_v[g]));
      l = i == 0 ? (x + y) * iv[g] : fmaf(x + y, iv[g], l);
      return pack_act2(x, y, KQ_DTYPE_F16);
    };
    auto base_of = [](float m) { return m == -__builtin_inff() ? 0.0f : m; };
    // (a tile's scale is positive, so its largest score is its largest dot product's)
    auto limit = [&](f32x2_t ks, f32x2_t lv, f32x2_t iv, const f32x16& w, u32x4 (&p)[2], float& l) {
      if (__ballot(l > kTileMost * fminf(iv[0], iv[1]) || !(fabsf(top) <= kCoarse)) == 0) return;
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
      ref = base - kTileLift;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // (exact differences, of at most kTileLift with it)
        const int g = i >> 2;
        const float u = __builtin_amdgcn_exp2f((fmaf(w[2 * i], ks[g], lv[g]) - base) + kTileLift);
        const float v = __builtin_amdgcn_exp2f((fmaf(w[2 * i + 1], ks[g], lv[g]) - base) + kTileLift);
        l = i == 0 ? (u + v) * iv[g] : fmaf(u + v, iv[g], l);
        p[i >> 2][i & 3] = pack_act2(u, v, KQ_DTYPE_F16);
      }
    };

    auto keys = [&](int which) { return smem + which * KB; };
    auto values = [&](int which) { return smem + 2 * KB + which * VB; };
    f32x16 x, y;
    if (lo < hi) {
      const int last = min(q.first, q.tokens);  // (what ends at or before it is seen whole)
      const int lo_all = (int)wave_max_u32_dpp((uint32_t)from);
      Place at = place_of(lo, page_at(lo));
      fetch_k(at);
      fetch_v(at);
      int next_page = page_at(lo + ST), page = page_at(lo + 2 * ST);
      // the words of the mask for 32 tokens, asked for while those before are at work
      uint32_t word0 = 0, word1 = 0;
      auto words_of = [&](int t) {
        if (t + 32 <= last) return;
        const int at = (t - q.first) >> 5;
        word0 = load_word(bits, a.words, at);
        word1 = load_word(bits, a.words, at + 1);
      };
      words_of(lo + 32 * tg);
      put_k(keys(0));
      put_v(values(0));
      at = place_of(lo + ST, next_page);
      fetch_k(at);
      if constexpr (TG > 1) {
        put_k(keys(1));
        fetch_v(at);
        at = place_of(lo + 2 * ST, page);
        fetch_k(at);
        next_page = page_at(lo + 3 * ST);
      } else {
        fetch_v(at);
        next_page = page;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) qf[i] ^= a.q_sign;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.0f;
      meet();
#pragma unroll
      for (int k = 0; k < KS; ++k) x = mfma32<DT>(key_of(keys(0), tg, k), qf[k], x);
      // 32 tokens from t on, half i of a step whose values are in `vals`: their weights from the
      // scores `now`, between the products that give the next ones' scores
      auto half = [&](int t, int i, const char* vals, f32x16& now, f32x16& next, const char* next_keys, int next_i, int next_t) {
        const char* scales = vals + D * VLD + 8 * i;
        const f32x2_t ks = *(const f32x2_t*)scales, lv = *(const f32x2_t*)(scales + 16), iv = *(const f32x2_t*)(scales + 32);
        u32x4 kx[4];  // (four of the operands ahead)
#pragma unroll
        for (int k = 0; k < 4; ++k) kx[k] = key_of(next_keys, next_i, k);
        if (t < lo_all || t + 32 > last) {
          const int node = t - q.first, at = node >> 5;
          const uint32_t seen = bits_at(word_at(word0, a.words, at), word_at(word1, a.words, at + 1), node) & tokens_from(from - t) &
                                ~tokens_from(q.tokens - t);
#pragma unroll
          for (int e = 0; e < 16; ++e) now[e] = seen >> (4 * h) & (1u << (8 * (e >> 2) + (e & 3))) ? now[e] : -__builtin_inff();
        }
        words_of(next_t);
        u32x4 w[2];
        float l;
        const f32x2_t shift_v = {lv[0] - ref, lv[1] - ref};
#pragma unroll
        for (int e = 0; e < 16; ++e) next[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          next = mfma32<DT>(kx[k & 3], qf[k], next);
          if (k + 4 < KS) kx[k & 3] = key_of(next_keys, next_i, k + 4);
#pragma unroll
          for (int j = 8 * k / KS; j < 8 * (k + 1) / KS; ++j) w[j >> 2][j & 3] = weight_pair(j, ks, shift_v, iv, now, l);
          __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(l));  // (not behind the branch that may compute them anew)
        u32x4 vx[2][OT];
#pragma unroll
        for (int j = 0; j < OT; ++j) vx[0][j] = value_of(vals, i, 0, j);
        limit(ks, lv, iv, now, w, l);
#pragma unroll
        for (int j = 0; j < OT; ++j) vx[1][j] = value_of(vals, i, 1, j);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < OT; ++j) o[j] = mfma32<KQ_DTYPE_F16>(vx[k][j], w[k], o[j]);
        sum += l;
      };
      if constexpr (TG > 1) {
        meet();  // (keys 0 are read)
        // step n of parity p: reads keys n + 1 and values n, writes keys n + 2 and values n + 1
        // where keys n and values n - 1 were
        auto step = [&](int t, f32x16& now, f32x16& next, auto p_) {
          constexpr int p = decltype(p_)::value;
          half(t + 32 * tg, tg, values(p), now, next, keys(1 - p), tg, t + ST + 32 * tg);
          put_k(keys(p));
          put_v(values(1 - p));
          fetch_v(at);
          at = place_of(t + 3 * ST, next_page);
          fetch_k(at);
          next_page = page_at(t + 4 * ST);
          meet();
        };
        for (int t = lo; t < hi; t += 2 * ST) {  // (a step past the end finds no page and adds nothing)
          if constexpr (D != 256) give_way((t - lo) >> 6, (hi - lo) >> 6);
          step(t, x, y, std::integral_constant<int, 0>{});
          step(t + ST, y, x, std::integral_constant<int, 1>{});
        }
      } else {
        // both halves of a step: keys n + 1 reach LDS between them, values n + 1 at the end
        int which = 0;
        for (int t = lo; t < hi; t += ST) {
          if constexpr (D != 256) give_way((t - lo) >> 6, (hi - lo) >> 6);
          half(t, 0, values(which), x, y, keys(which), 1, t + 32);
          put_k(keys(which ^ 1));
          at = place_of(t + 2 * ST, next_page);
          fetch_k(at);
          next_page = page_at(t + 3 * ST);
          meet();
          half(t + 32, 1, values(which), y, x, keys(which ^ 1), 0, t + 64);
          put_v(values(which ^ 1));
          fetch_v(at);
          meet();
          which ^= 1;
        }
      }
    }
    sum += __shfl_xor(sum, 32, 64);
    if (sum != sum) {
      bool any = any_there(pages, cache.pages, max(from, lo), min(max(q.first, 0), hi), shift);
      for (int t = max(max(q.first, 0), lo); !any && from != 0x7fffffff && t < hi; ++t) {
        const int node = t - q.first;
        any = (word_at(load_word(bits, a.words, node >> 5), a.words, node >> 5) >> (node & 31) & 1) &&
              any_there(pages, cache.pages, t, t + 1, shift);
      }
      if (!any) {
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < OT; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[j][e] = 0.0f;
      }
    }
    // The waves' columns meet in LDS in the order of d, and are added in the order of their
    // tokens by threads that write whole rows.  Element e of tile j is row R = 32 j + 8 (e / 4) +
    // 4 h + e % 4 of the values: elements e and e + 8 of all tiles are neighbouring d.
    constexpr int N = 2 * OT;
    float* mine = (float*)smem + (wave * 32 + c) * LD;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v[N];
#pragma unroll
      for (int j = 0; j < OT; ++j) {
        v[2 * j] = o[j][e];
        v[2 * j + 1] = o[j][8 + e];
      }
      float* dst = mine + (8 * (e >> 2) + 4 * h + (e & 3)) * VY;
#pragma unroll
      for (int i = 0; i < N; i += 4) *(f32x4*)(dst + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    }
    if (h == 0) mine[D] = top, mine[D + 1] = sum;
    meet();
    const bool whole = part_blocks == blocks;
    float* part = a.part + ((((int64_t)head * a.shares + given.share) * 2 + (within == 0)) * TW) * LD;
#pragma unroll 1
    for (int i = tid; i < TW * (D / 4); i += 256) {
      const int col = i / (D / 4), d = 4 * (i - col * (D / 4)), it = tile * TW + col;
      if (it >= q.rows * group) break;
      const float* from_ = (const float*)smem + col * LD;
      float most = from_[D];
#pragma unroll
      for (int g = 1; g < TG; ++g) most = fmaxf(most, from_[g * TW * LD + D]);
      f32x4 v = {0, 0, 0, 0};
      float l = 0.0f;
#pragma unroll
      for (int g = 0; g < TG; ++g) {
        const float f = TG == 1 ? 1.0f : __builtin_amdgcn_exp2f(from_[g * TW * LD + D] - base_of(most));
        const f32x4 more = *(const f32x4*)(from_ + g * TW * LD + d);
        l += from_[g * TW * LD + D + 1] * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += more[e] * f;
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees no token is zero)
        const int rw = it / group;
        uint16_t* dst = a.out + ((int64_t)(q.row0 + rw) * a.heads + head * group + (it - rw * group)) * D + d;
        *(u32x2*)dst = u32x2{pack_act2(v[0] * inv, v[1] * inv, DT), pack_act2(v[2] * inv, v[3] * inv, DT)};
      } else {
        *(f32x4*)(part + (int64_t)col * LD + d) = v;
        if (d == 0) *(f32x2_t*)(part + (int64_t)col * LD + D) = f32x2_t{most, l};
      }
    }
    block += part_blocks;
    within = 0;
    if (block >= run_end) return;
    if (++tile >= deal.tiles(q)) {
      tile = 0;
      do {
        if (++s >= batch.seqs) return;
        q = lanes[s];
      } while (deal.tiles(q) == 0);
      blocks = deal.blocks(q);
    }
    meet();  // (LDS is read to the end)
  }
}

// The parts of split tiles joined in the order of their tokens: a workgroup takes COLS columns
// of one tile, a thread four neighbouring d of each of E columns.  Latency: finding the tile's parts,
// then their loads, eight a thread on their way: 7.5 us for 16 trees of up to 24 rows, 12 for 32 of up to
// 32 (28 MB of parts), both under the profiler.
template <int D, int DT, int TW>
__global__ void __launch_bounds__(256)
kv_tree_join_kernel(TreeArgs a, KvCache cache, KvBatch batch) {
  constexpr int LD = D + 4, PER = D / 4, E = TW * PER >= 512 ? 2 : 1, COLS = 256 * E / PER;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int head = (int)blockIdx.y, column0 = (int)blockIdx.z * COLS;
  const KvLanes lanes(batch, shift);
  const TreeDeal<TW> deal{a, group};
  int tile;
  const int s = lanes.find((int)blockIdx.x, tile, [&](const KvSeq& q) { return deal.tiles(q); });
  if (s < 0) return;
  const KvSeq q = lanes[s];
  if (tile * TW + column0 >= q.rows * group) return;
  // its parts and the workgroup of the first (within the shares also where row bounds that go
  // back make counts wrap)
  int x0 = 0, chunks = 0, apart = 1;
  const int blocks = deal.blocks(q);
  if (a.alike) {
    const int length = deal.length(lanes), parts = scalar(deal.parts(q, length));
    lanes.of_row(q.row0, x0, [&](const KvSeq& p) { return deal.tiles(p) * deal.parts(p, length); });
    x0 = min(max(x0 + tile, 0), a.shares - 1);
    apart = scalar(deal.tiles(q));
    chunks = min(parts, (int)((uint32_t)(a.shares - 1 - x0) / (uint32_t)apart) + 1);
  } else {
    const int run = max(deal.run(lanes), 1);
    int block = 0;  // blocks before the tile's
    lanes.of_row(q.row0, block, deal);
    block += tile * blocks;
    x0 = min(max(scalar(block / run), 0), a.shares - 1);
    chunks = min(max(scalar((block + blocks - 1) / run), x0), a.shares - 1) - x0 + 1;
  }
  if (chunks == 1) return;  // written already
  // place 1 of the workgroup it begins in, then place 0 of those behind
  const float* src = a.part + ((((int64_t)head * a.shares + x0) * 2 + 1) * TW + column0) * LD;
  auto at_part = [&](int i) { return src + (i == 0 ? 0 : (int64_t)(2 * i * apart - 1) * TW) * LD; };
  float m[E], l[E];
  f32x4 x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    m[e] = -__builtin_inff(), l[e] = 0.0f;
    x[e] = f32x4{0, 0, 0, 0};
  }
  constexpr int U = 8 / E;  // parts on their way at once
  for (int i0 = 0; i0 < chunks; i0 += U) {
    f32x4 v[U][E];
    f32x2_t has[U][E];  // a part's maximum and denominator
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i0 + i >= chunks) break;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = (int)threadIdx.x + 256 * e, col = at / PER;
        const float* p = at_part(i0 + i) + col * LD;
        has[i][e] = *(const f32x2_t*)(p + D);
        v[i][e] = *(const f32x4*)(p + 4 * (at - col * PER));
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i0 + i >= chunks) break;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float most = fmaxf(m[e], has[i][e][0]), base = most == -__builtin_inff() ? 0.0f : most;
        const float keep = __builtin_amdgcn_exp2f(m[e] - base), f = __builtin_amdgcn_exp2f(has[i][e][0] - base);
        m[e] = most;
        l[e] = l[e] * keep + has[i][e][1] * f;
        x[e] = x[e] * keep + v[i][e] * f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = (int)threadIdx.x + 256 * e, col = at / PER, item = tile * TW + column0 + col;
    if (item >= q.rows * group) return;
    const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
    const int row = item / group;
    uint16_t* dst = a.out + ((int64_t)(q.row0 + row) * a.heads + head * group + (item - row * group)) * D + 4 * (at - col * PER);
    *(u32x2*)dst = u32x2{pack_act2(x[e][0] * inv, x[e][1] * inv, DT), pack_act2(x[e][2] * inv, x[e][3] * inv, DT)};
  }
}

// Blocks of 16 columns and 256 tokens up to which the tiles are of 16 columns whatever the trees
// are: a step of theirs is the shortest, and they fill the chip with the least (one tree of 64
// rows x heads behind 4000 and 16000 tokens, 8 kv heads of 128: 19 and 27 us, in tiles of 64 28
// and 39; one of 256 behind 4000 24 and 32; but 16 of up to 96 behind 3000 65, in tiles of 128 44).
constexpr int64_t kFewBlocks = 2560;
// Tokens up to which one workgroup reads a tile's whole and nothing is joined, where that leaves
// tiles of 16 (one tree of 48 behind 900 tokens 13 us, cut 14; 48 of 64 behind up to 900, in tiles of
// 64, 39 and 51), and under a window, which makes the tiles alike, where they fill the chip (24
// windows of 1024, 16 heads of 64: 16 us whole, 23 cut).  By the table's width, which is all that
// the host knows; under a window by the batch's rows in place of a sequence's, so that the form changes with
// the batch (of such trees of 16 rows 60 are whole, 29.3 us, and 61 cut, 32.5; 128 take 67, their bytes 58).
constexpr int64_t kWhole = 1024, kWholeMany = 2048;

struct TreePlan {
  int columns;  // of a tile: 16 or 32 (a wave holds them all), 64 or 128 (the workgroup does)
  int waves;    // of a workgroup
  int shares, block_shift;
  bool alike, near;
  size_t part;  // bytes
};

// Workgroups that registers and LDS let a CU hold, on all of them.
static int64_t tree_slots(int columns, int waves, int64_t dim) {
  return 256 * (columns > 32 ? (dim == 256 ? 1 : 2) : waves == 8 ? 1 : dim * columns <= 1024 ? 3 : dim * columns <= 4096 ? 2 : 1);
}
static int tree_shares(int64_t slots, int64_t kv_heads) { return (int)std::max<int64_t>(slots / kv_heads, 1); }
// Bytes of the parts of split tiles.
static size_t tree_parts(int shares, int64_t kv_heads, int columns, int64_t dim) {
  return sizeof(float) * (size_t)(shares * kv_heads * 2 * columns * (dim + 4));
}

// From what the host knows: rows and sequences, not their lengths.
static TreePlan tree_plan(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size, int64_t width,
                          int64_t seqs, int64_t window) {
  TreePlan p{};
  const int64_t items = rows * (heads / kv_heads), each = (items + std::max<int64_t>(seqs, 1) - 1) / std::max<int64_t>(seqs, 1);
  const int64_t tokens = width * page_size, span = window > 0 ? std::min(tokens, window + rows + 64) : tokens;
  auto tiles = [&](int64_t columns) { return (items / columns + seqs) * kv_heads; };
  if (tiles(16) * ((span + 255) / 256) <= kFewBlocks)
    p.columns = 16;
  else
    p.columns = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
  const bool whole = (span <= kWhole && (p.columns == 16 || tiles(p.columns) >= 256)) ||
                     (window > 0 && span <= kWholeMany && p.columns == 16 && tiles(16) >= 256);
  // eight waves to a tile while there is at most one for a CU (four trees of 64 behind 900 tokens 14
  // us, with four waves 19; 16 of them 26 and 24)
  p.waves = whole && p.columns == 16 && tiles(16) <= 256 ? 8 : 4;
  const int64_t slots = tree_slots(p.columns, p.waves, dim);
  p.shares = tree_shares(slots, kv_heads);
  p.alike = p.columns > 16 && tiles(p.columns) <= p.shares * kv_heads;
  p.near = p.alike || (whole ? each > p.columns : each <= p.columns);
  // parts of one length: blocks of what a workgroup's loop takes at once.  Runs: of 256 tokens, or of 512 where
  // those still give every workgroup one, so that tiles are cut less often
  p.block_shift = p.alike ? (p.columns > 64 ? 0 : 1) : tiles(p.columns) * ((span + 511) / 512) >= slots ? 3 : 2;
  while (whole && (64LL << p.block_shift) < span) ++p.block_shift;  // (no tile in two blocks: they would need `part`)
  if (!whole) p.part = tree_parts(p.shares, kv_heads, p.columns, dim);
  return p;
}

template <int D, int DT, int MT, int WAVES>
static void launch_rows(const TreeArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  constexpr int NT = D == 256 || MT > 1 ? 2 : 4;  // (registers)
  const int page = 1 << c.page_shift;
  const dim3 grid((unsigned)a.shares, (unsigned)c.kv_heads);
  if (page >= 16 * NT)
    hipLaunchKernelGGL((kv_tree_kernel<D, DT, NT, 1, MT, WAVES>), grid, dim3(64 * WAVES), 0, st, a, c, b, b.table, c.k_scale, c.v_scale);
  else if (page == 8 * NT)
    hipLaunchKernelGGL((kv_tree_kernel<D, DT, NT, 2, MT, WAVES>), grid, dim3(64 * WAVES), 0, st, a, c, b, b.table, c.k_scale, c.v_scale);
  else if constexpr (NT == 4)
    hipLaunchKernelGGL((kv_tree_kernel<D, DT, NT, 4, MT, WAVES>), grid, dim3(64 * WAVES), 0, st, a, c, b, b.table, c.k_scale, c.v_scale);
}

template <int D, int DT, int CG>
static void launch_tiles(const TreeArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  hipLaunchKernelGGL((kv_tree_tiles_kernel<D, DT, CG>), dim3((unsigned)a.shares, (unsigned)c.kv_heads), dim3(256), 0, st, a, c, b,
                     b.table, c.k_scale, c.v_scale);
}

template <int D, int DT, int TW>
static void launch_join(const TreeArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  if (a.part == nullptr) return;
  constexpr int COLS = 1024 * (TW * D >= 2048 ? 2 : 1) / D;
  const int64_t tiles = std::min<int64_t>((int64_t)b.rows * (a.heads / c.kv_heads) / TW + b.seqs, b.rows * (int64_t)a.heads);
  hipLaunchKernelGGL((kv_tree_join_kernel<D, DT, TW>), dim3((unsigned)tiles, (unsigned)c.kv_heads, (TW + COLS - 1) / COLS), dim3(256),
                     0, st, a, c, b);
}

template <int D, int DT>
static void launch_tree(const TreeArgs& a, const TreePlan& p, const KvCache& c, const KvBatch& b, hipStream_t st) {
  if (p.columns == 16) {
    if (p.waves == 8)
      launch_rows<D, DT, 1, 8>(a, c, b, st);
    else
      launch_rows<D, DT, 1, 4>(a, c, b, st);
    launch_join<D, DT, 16>(a, c, b, st);
  } else if (p.columns == 32) {
    launch_rows<D, DT, 2, 4>(a, c, b, st);
    launch_join<D, DT, 32>(a, c, b, st);
  } else if (p.columns == 64) {
    launch_tiles<D, DT, 2>(a, c, b, st);
    launch_join<D, DT, 64>(a, c, b, st);
  } else {
    launch_tiles<D, DT, 4>(a, c, b, st);
    launch_join<D, DT, 128>(a, c, b, st);
  }
}

template <int D>
static void launch_tree_dtype(const TreeArgs& a, const TreePlan& p, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  if (dtype == KQ_DTYPE_BF16)
    launch_tree<D, KQ_DTYPE_BF16>(a, p, c, b, st);
  else
    launch_tree<D, KQ_DTYPE_F16>(a, p, c, b, st);
}

}  // namespace kq

using namespace kq;

extern "C" size_t kq_kv_tree_attention_workspace_size(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                                      int64_t page_size, int64_t table_width, int64_t seqs) {
  if (rows < 1 || heads < 1 || kv_heads < 1 || dim < 1 || page_size < 1 || table_width < 0 || seqs < 0) return 0;
  // A window changes the plan in two ways: tiles are read whole and need nothing (as all are that are
  // whole without one), or they are of 16 columns where wider ones would be taken without it, which have
  // more workgroups where the kv heads do not divide them (10 heads of 256: 51 of 16 columns, 25 of 32).
  const size_t part = tree_plan(rows, heads, kv_heads, dim, page_size, table_width, seqs, 0).part;
  return part == 0 ? 0 : std::max(part, tree_parts(tree_shares(tree_slots(16, 4, dim), kv_heads), kv_heads, 16, dim));
}

extern "C" int kq_kv_tree_attention(const void* q, int64_t q_ld, int64_t q_hs, int dtype, int64_t rows, int64_t heads,
                                    int64_t kv_heads, int64_t dim, const uint8_t* k_cache, const uint8_t* v_cache,
                                    const float* k_scale, const float* v_scale, int64_t pages, int64_t page_size,
                                    const int32_t* table, int64_t table_ld, int64_t table_width, const int32_t* cu,
                                    const int32_t* lengths, int64_t seqs, const int32_t* mask, int64_t words,
                                    const int32_t* positions, float scale, int64_t window, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* what = "kq_kv_tree_attention";
  int rc = kv_check(what, dtype, rows, heads, kv_heads, dim, page_size, pages, seqs, table_width, table_ld);
  if (rc) return rc;
  if (!(fabsf(scale) <= 0x1p100f)) {
    set_error("%s: scale %g", what, (double)scale);
    return KQ_EINVAL;
  }
  if (window < 0 || window > (1 << 30) || words < 1 || words > 32) {
    set_error("%s: window %lld, masks of %lld words (1 to 32 are supported)", what, (long long)window, (long long)words);
    return KQ_EINVAL;
  }
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) % 16 != 0 ||
      (q_ld | q_hs) % 8 != 0) {
    set_error("%s: tensors need 16-byte aligned rows and heads", what);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  const bool empty = seqs == 0 || pages == 0 || table_width == 0;  // every row is zero
  TreePlan p = tree_plan(rows, heads, kv_heads, dim, page_size, table_width, seqs, window);
  if (empty) p.part = 0;
  if (p.part > 0 && (workspace == nullptr || workspace_bytes < p.part)) {
    set_error("%s: workspace of %zu bytes is too small", what, workspace_bytes);
    return KQ_EWORKSPACE;
  }
  // threads of one launch, and blocks of all tiles
  const int64_t tiles = empty ? 0 : rows * (heads / kv_heads) / p.columns + seqs;
  const int64_t blocks = tiles * (((table_width * page_size - 1) >> (6 + p.block_shift)) + 1);
  if (rows * heads * 64 >= (1LL << 32) || tiles >= (1LL << 24) || blocks >= (1LL << 30)) {
    set_error("%s: %lld rows of %lld heads over up to %lld tokens are past the supported range", what, (long long)rows,
              (long long)heads, (long long)(table_width * page_size));
    return KQ_EINVAL;
  }
  TreeArgs a{};
  a.q = (const uint16_t*)q;
  a.q_ld = q_ld, a.q_hs = q_hs;
  a.out = (uint16_t*)out;
  a.mask = (const uint32_t*)mask, a.words = (int)words, a.positions = positions;
  a.part = p.part > 0 ? (float*)workspace : nullptr;
  a.scale = fmaxf(fabsf(scale) * 1.44269504088896340736f, 0x1p-60f);
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  a.heads = (int)heads, a.window = (int)window;
  a.most_blocks = (int)blocks;
  a.shares = p.shares, a.block_shift = p.block_shift, a.alike = p.alike, a.near = p.near;
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  const KvCache c{(uint8_t*)k_cache, (uint8_t*)v_cache, (float*)k_scale, (float*)v_scale, pages, (int)kv_heads, shift};
  // (without pages or table columns no sequence is looked at and all rows are padding)
  const KvBatch b{table, cu, lengths, table_ld, empty ? 0 : (int)seqs, (int)table_width, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  if (dim == 64)
    launch_tree_dtype<64>(a, p, c, b, dtype, st);
  else if (dim == 128)
    launch_tree_dtype<128>(a, p, c, b, dtype, st);
  else
    launch_tree_dtype<256>(a, p, c, b, dtype, st);
  return check_launch(what);
}
