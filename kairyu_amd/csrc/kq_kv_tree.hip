// Attention of drafted tokens that branch, over the paged e4m3 cache.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = exp(scale * q . k_t - max) over the tokens a row
// sees: those before its sequence's new ones (from its position less the window on), and
// the new ones whose bit its mask holds.  Scores, scales and weights are formed as in
// attention over prompts and single tokens: w_t = log2(e) scale k_scale (q . code_t) +
// log2 v_scale, exp2(w_t - max w + lift) in fp16 (11 bits down to 2^-29 of the largest,
// some down to 2^-40) times the value's codes, the denominator in fp32 from weights not yet
// rounded over v_scale, maxima, denominators and outputs in fp32.
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
};

constexpr float kLift = 15.0f;  // log2 of the largest weight

// A sequence's rows (drafted tokens x the group's query heads) go to tiles of TW, the
// tokens that they see to blocks, and the blocks of all tiles, one after the other, to
// `shares` workgroups per kv head in equal runs: whole tiles, written at once, and at most two
// parts of tiles, the end of one begun before (part 0) and the beginning of one that goes on
// (part 1).
template <int TW>
struct TreeDeal {
  const TreeArgs& a;
  int group;

  // 64-token step of the first token that any row sees
  KQ_DEV int first(const KvSeq& q) const { return a.window > 0 ? max(q.first + 1 - a.window, 0) >> 6 : 0; }
  KQ_DEV int blocks(const KvSeq& q) const { return (max(((q.tokens + 63) >> 6) - first(q), 1) + (1 << a.block_shift) - 1) >> a.block_shift; }
  KQ_DEV int tiles(const KvSeq& q) const { return (q.rows * group + TW - 1) / TW; }
  KQ_DEV int operator()(const KvSeq& q) const { return tiles(q) * blocks(q); }
  KQ_DEV int run(const KvLanes& lanes) const {
    // (held to what a batch can have, whatever the row bounds say)
    const uint32_t all = min((uint32_t)lanes.total(*this), (uint32_t)a.most_blocks);
    return scalar((int)((all + (uint32_t)a.shares - 1) / (uint32_t)a.shares));
  }
};

// Words `at` of a row's mask with all ones before it: tokens before the new ones are seen.
KQ_DEV uint32_t mask_word(const uint32_t* mask, int words, int at) { return at < 0 ? ~0u : at < words ? mask[at] : 0u; }

// One workgroup: its run of blocks of one kv head, tile by tile; its four waves take a
// tile's steps of 16 * NT tokens in turn, each for all of the tile's 16 * MT columns, so that
// a token is loaded and widened once for all of them, and by one wave.
//
// The products run transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32 MFMAs: lane (c, b) =
// (l % 16, l / 16) holds scores of columns c of the MT tiles for tokens 4b..4b+3 of each 16,
// which are what it hands over as its part of P^T.  Loads go from memory to registers through
// resources of one page's tile that end at the sequence's last token.
template <int D, int DT, int NT, int PP, int MT>
__global__ void __launch_bounds__(256, D * MT <= 64 ? 3 : D * MT <= 256 ? 2 : 1)
kv_tree_kernel(TreeArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
               const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int KS = D / 32;   // MFMA steps along a key
  constexpr int VD = D / 64;   // dwords of a token's value a lane holds
  constexpr int OT = D / 16;   // output tiles
  constexpr int ST = 16 * NT;  // tokens of a step
  constexpr int TW = 16 * MT;
  constexpr int LD = D + 4;
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * LD];
  const int lane = lane_id(), wave = scalar(wave_id()), c = lane & 15, b = lane >> 4;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int head = (int)blockIdx.y;

  zero_padding<D>(a, batch, head, group, (int)blockIdx.x, (int)gridDim.x, 256);
  const KvLanes lanes(batch, shift);
  const TreeDeal<TW> deal{a, group};
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
  auto begin_part = [&] {
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
      from[m] = !real ? 0 : pos < 0 ? 0x7fffffff : a.window > 0 ? min(max(max(pos, q.first) + 1 - a.window, 0), max(q.first, 0)) : 0;
      most_from = max(most_from, (uint32_t)from[m]);
#pragma unroll
      for (int i = 0; i < KS; ++i) qf[m][i] = u32x4{0, 0, 0, 0};
      if (real) {
        const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
        for (int i = 0; i < KS; ++i) qf[m][i] = *(const u32x4*)(src + 64 * (i >> 1) + 16 * b + 8 * (i & 1)) ^ a.q_sign;
      }
    }
    lo_all = (int)wave_max_u32_dpp(most_from);
    place(t);
    load_keys(t);
    load_values(t);
    pages_of(t + 4 * ST);
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
    place(t + 4 * ST);
    load_keys(t + 4 * ST);
    pages_of(t + 8 * ST);
    if (t < lo_all || t + ST > q.first) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int token = t + 16 * i + 4 * b, node = token - q.first, at = node >> 5;
          const uint64_t both = (uint64_t)mask_word(bits[m], a.words, at + 1) << 32 | mask_word(bits[m], a.words, at);
          const uint32_t seen = (uint32_t)(both >> (node & 31));
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (token + r < from[m] || token + r >= q.tokens || !(seen >> r & 1)) w[m][i][r] = -__builtin_inff();
        }
    }
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
    load_values(t + 4 * ST);
  };
  // Whether a column sees any token of this part that is there (its sum is NaN).
  auto sees_any = [&](int m) {
    if (any_there(pages, cache.pages, max(from[m], lo), min(max(q.first, 0), hi), shift)) return true;
    if (from[m] == 0x7fffffff) return false;
    for (int t = max(max(q.first, 0), lo); t < hi; ++t) {
      const int node = t - q.first;
      if ((mask_word(bits[m], a.words, node >> 5) >> (node & 31) & 1) && any_there(pages, cache.pages, t, t + 1, shift)) return true;
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
    for (int t = lo + ST * wave; t < hi; t += 4 * ST) step(t);
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
      for (int i = (int)threadIdx.x; i < 16 * (D / 2); i += 256) {
        const int col = i / (D / 2), d = 2 * (i - col * (D / 2));
        const int it = old_tile * TW + 16 * m + col;
        if (it >= old.rows * group) break;
        float most = -__builtin_inff();
#pragma unroll
        for (int v = 0; v < 4; ++v) most = fmaxf(most, lds[(v * 16 + col) * LD + D]);
        const float base = most == -__builtin_inff() ? 0.0f : most;
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
          float* dst = a.part + ((((int64_t)head * a.shares + (int)blockIdx.x) * 2 + (old_within == 0)) * TW + 16 * m + col) * LD;
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

// The parts of split tiles joined in the order of their tokens, one wave per row and query
// head.
template <int D, int DT, int TW>
__global__ void __launch_bounds__(256)
kv_tree_join_kernel(TreeArgs a, KvCache cache, KvBatch batch) {
  constexpr int LD = D + 4, PER = D / 64;
  const int shift = cache.page_shift, group = scalar(a.heads / cache.kv_heads);
  const int at = (int)blockIdx.x * 4 + scalar(wave_id());
  const KvLanes lanes(batch, shift);
  const TreeDeal<TW> deal{a, group};
  const int row = scalar(at / a.heads), qh = at - row * a.heads, head = scalar(qh / group);
  if (row >= batch.rows) return;
  int block = 0;  // blocks of the sequences before s
  const int s = lanes.of_row(row, block, deal);
  if (s < 0) return;
  const KvSeq q = lanes[s];
  const int item = (row - q.row0) * group + (qh - head * group), tile = scalar(item / TW);
  const int run = max(deal.run(lanes), 1), blocks = deal.blocks(q);
  block += tile * blocks;
  // (within the shares also where row bounds that go back make counts wrap)
  const int x0 = min(max(scalar(block / run), 0), a.shares - 1);
  const int chunks = min(max(scalar((block + blocks - 1) / run), x0), a.shares - 1) - x0 + 1;
  if (chunks == 1) return;  // written already
  // part 1 of the run it begins in, then part 0 of those behind
  const float* src = a.part + ((((int64_t)head * a.shares + x0) * 2 + 1) * TW + (item - tile * TW)) * LD;
  auto at_part = [&](int i) { return src + (i == 0 ? 0 : (int64_t)(2 * i - 1) * TW) * LD; };
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

// Tokens up to which one workgroup reads a tile's whole, which saves the second launch.
constexpr int64_t kWhole = 1024;

struct TreePlan {
  int columns;  // tiles of 16 that a wave holds at once
  int shares, block_shift;
  size_t part;  // bytes
};

// From what the host knows: rows and sequences, not their lengths.
static TreePlan tree_plan(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size, int64_t width,
                          int64_t seqs, int64_t window) {
  TreePlan p{};
  const int64_t items = rows * (heads / kv_heads), each = (items + std::max<int64_t>(seqs, 1) - 1) / std::max<int64_t>(seqs, 1);
  p.columns = each <= 16 ? 1 : each <= 32 || dim == 256 ? 2 : 4;
  const int64_t slots = 256 * (dim * p.columns <= 64 ? 3 : dim * p.columns <= 256 ? 2 : 1);
  p.shares = (int)std::max<int64_t>(slots / kv_heads, 1);
  const int64_t tokens = width * page_size, span = window > 0 ? std::min(tokens, window + rows + 64) : tokens;
  p.block_shift = 2;
  const bool whole = span <= kWhole;
  while (whole && (64LL << p.block_shift) < span) ++p.block_shift;  // (no tile in two blocks: they would need `part`)
  if (!whole) p.part = sizeof(float) * (size_t)(p.shares * kv_heads * 2 * 16 * p.columns * (dim + 4));
  return p;
}

template <int D, int DT, int NT, int PP, int MT>
static void launch_columns(const TreeArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  hipLaunchKernelGGL((kv_tree_kernel<D, DT, NT, PP, MT>), dim3((unsigned)a.shares, (unsigned)c.kv_heads), dim3(256), 0, st, a, c,
                     b, b.table, c.k_scale, c.v_scale);
  if (a.part != nullptr)
    hipLaunchKernelGGL((kv_tree_join_kernel<D, DT, 16 * MT>), dim3((unsigned)(((int64_t)b.rows * a.heads + 3) / 4)), dim3(256), 0,
                       st, a, c, b);
}

template <int D, int DT, int NT, int PP>
static void launch_pages(const TreeArgs& a, const TreePlan& p, const KvCache& c, const KvBatch& b, hipStream_t st) {
  if (p.columns == 1)
    launch_columns<D, DT, NT, PP, 1>(a, c, b, st);
  else if (p.columns == 2)
    launch_columns<D, DT, NT, PP, 2>(a, c, b, st);
  else if constexpr (D < 256)
    launch_columns<D, DT, NT, PP, 4>(a, c, b, st);
}

template <int D, int DT>
static void launch_tree(const TreeArgs& a, const TreePlan& p, const KvCache& c, const KvBatch& b, hipStream_t st) {
  constexpr int NT = D == 256 ? 2 : 4;  // (registers)
  const int page = 1 << c.page_shift;
  if (page >= 16 * NT)
    launch_pages<D, DT, NT, 1>(a, p, c, b, st);
  else if (page == 8 * NT)
    launch_pages<D, DT, NT, 2>(a, p, c, b, st);
  else if constexpr (NT == 4)
    launch_pages<D, DT, NT, 4>(a, p, c, b, st);
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
  return tree_plan(rows, heads, kv_heads, dim, page_size, table_width, seqs, 0).part;  // (a window needs no more than none)
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
  const int64_t tiles = empty ? 0 : rows * (heads / kv_heads) / (16 * p.columns) + seqs;
  const int64_t blocks = tiles * ((table_width * page_size + 255) / 256);
  if (rows * heads * 64 >= (1LL << 32) || blocks >= (1LL << 30)) {
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
  a.shares = p.shares, a.block_shift = p.block_shift;
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
