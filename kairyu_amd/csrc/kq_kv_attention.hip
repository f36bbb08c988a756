// Attention over the paged e4m3 cache.
//
// o = sum_t p_t v_t / sum_t p_t with p_t = exp(scale * q . k_t - max) over the tokens
// a row sees, in one pass with a running maximum.  Key codes enter the products as
// they are and the page's scale multiplies the finished dot product; the value scale
// joins the exponent instead, w_t = log2(e) scale k_scale (q . code_t) + log2 v_scale,
// so that exp2(w_t - max w) <= 1 multiplies the value's codes whatever the scales of
// the pages are and keeps 11 bits as fp16; the denominator adds exp2(w_t - max w) /
// v_scale.  Maxima, denominators and outputs are held in fp32.
#include "kq_kv.h"

#include <algorithm>

namespace kq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct AttendArgs {
  const uint16_t* q;
  int64_t q_ld, q_hs;
  uint16_t* out;  // [rows][heads][D]
  float* part;    // partial outputs of split sequences, null: none can be split
  float scale;    // times log2 e
  int heads, causal, window;
  int shares;     // workgroups per kv head that the batch's tokens are dealt to
};

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
// tokens that they see to blocks of 256.  The blocks of all tiles, one after the
// other, are dealt to `shares` workgroups per kv head in equal runs, so that every
// workgroup streams the same number of bytes whatever the lengths are (units cut per
// sequence left a third of the chip idle at the end of a ragged batch: 64 contexts of
// up to 6000 tokens, XX us).  A run covers whole tiles, written at once, and
// at most two parts of tiles: the end of one begun before it (part 0) and the
// beginning of one that goes on behind it (part 1).
struct Deal {
  int64_t run;  // blocks of a workgroup

  // 64-token step of the first token that any row sees
  KQ_DEV static int first(const AttendArgs& a, const KvSeq& q) {
    return a.window > 0 ? max(q.first + 1 - a.window, 0) >> 6 : 0;
  }
  // at least one, so that rows that see nothing are written as well
  KQ_DEV static int blocks(const AttendArgs& a, const KvSeq& q) {
    return (max(((q.tokens + 63) >> 6) - first(a, q), 1) + 3) >> 2;
  }
  KQ_DEV static int tiles(const KvSeq& q, int group) { return (q.rows * group + 15) >> 4; }
};

// The same run in every workgroup.
KQ_DEV Deal deal_of(const AttendArgs& a, const KvBatch& b, int shift, int group) {
  int64_t total = 0;
  for (int s0 = 0; s0 < b.seqs; s0 += 64) {
    const int s = s0 + lane_id();
    int v = 0;
    if (s < b.seqs) {
      const KvSeq q = kv_seq(b, s, shift);
      v = Deal::tiles(q, group) * Deal::blocks(a, q);
    }
    total += __builtin_amdgcn_readlane(wave_scan(v), 63);
  }
  Deal r;
  r.run = (total + a.shares - 1) / a.shares;
  return r;
}

// Keys and values of one step of 16 * NT tokens in registers, and their scales.
template <int D, int NT, int PP>
struct Step {
  u32x4 k[NT][D / 64];
  uint32_t v[NT * 4][D / 64];
  float ks[PP], vs[PP];  // scale times log2 e; value scale (0: no tokens here)
};

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
// read as zero without a branch.
template <int D, int DT, int NT, int PP>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2)
kv_attend_rows_kernel(AttendArgs a, KvCache cache, KvBatch batch, const int32_t* __restrict__ table,
                      const float* __restrict__ k_scale, const float* __restrict__ v_scale) {
  constexpr int KS = D / 32;   // MFMA steps along a key
  constexpr int VD = D / 64;   // dwords of a token's value a lane holds
  constexpr int OT = D / 16;   // output tiles
  constexpr int ST = 16 * NT;  // tokens of a step
  constexpr int LD = D + 4;
  extern __shared__ float lds[];  // [4][16][LD]
  const int lane = lane_id(), wave = wave_id(), c = lane & 15, b = lane >> 4;
  const int shift = cache.page_shift, group = a.heads / cache.kv_heads;
  const int head = (int)blockIdx.y;

  {  // rows of no sequence
    const int last = batch.seqs > 0 ? min(max(batch.cu[batch.seqs], 0), batch.rows) : 0;
    const int first = batch.seqs > 0 ? min(max(batch.cu[0], 0), last) : 0;
    const int words = group * D / 2;
    for (int i = (int)blockIdx.x; i < first + batch.rows - last; i += (int)gridDim.x) {
      const int64_t row = i < first ? i : last + (i - first);
      uint32_t* dst = (uint32_t*)(a.out + (row * a.heads + head * group) * D);
      for (int j = (int)threadIdx.x; j < words; j += 256) dst[j] = 0;
    }
  }

  const Deal deal = deal_of(a, batch, shift, group);
  const int64_t run_end = ((int64_t)blockIdx.x + 1) * deal.run;
  int64_t block = (int64_t)blockIdx.x * deal.run;
  int within = 0;  // blocks of the sequence before `block`
  int s = kv_find(block, batch.seqs, within, [&](int i) {
    const KvSeq q = kv_seq(batch, i, shift);
    return Deal::tiles(q, group) * Deal::blocks(a, q);
  });
  if (s < 0) return;
  KvSeq q = kv_seq(batch, s, shift);
  int blocks = Deal::blocks(a, q), tile = within / blocks;
  within -= tile * blocks;
  const int64_t tile_bytes = (int64_t)D << shift;
  const int in_page = (1 << shift) - 1;
  const int k_lane = c * D + 16 * b, v_lane = 4 * b * D + c * (D / 16);

  while (true) {
  const int item = tile * 16 + c;  // this lane's column: row item / group, head item % group
  const bool real = item < q.rows * group;
  const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
  const int pos = q.first + row;
  // tokens [from, to) of this column; [lo, hi) of the tile; [lo_all, hi_all) of every row
  const int to = a.causal ? min(q.tokens, pos + 1) : q.tokens;
  const int from = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
  const int row_lo = (tile * 16) / group, row_hi = min(q.rows - 1, (tile * 16 + 15) / group);
  int hi = a.causal ? min(q.tokens, q.first + row_hi + 1) : q.tokens;
  int lo = a.window > 0 ? max(q.first + row_lo + 1 - a.window, 0) : 0;
  const int hi_all = a.causal ? min(q.tokens, q.first + row_lo + 1) : q.tokens;
  const int lo_all = a.window > 0 ? max(q.first + row_hi + 1 - a.window, 0) : 0;
  const int part_blocks = (int)min((int64_t)(blocks - within), run_end - block);
  const int begin = Deal::first(a, q) * 64 + within * 256;
  hi = min((int64_t)hi, (int64_t)begin + (int64_t)part_blocks * 256);
  lo = max(lo & ~63, begin);

  u32x4 qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) qf[i] = u32x4{0, 0, 0, 0};
  if (real) {
    const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *(const u32x4*)(src + 64 * (i >> 1) + 16 * b + 8 * (i & 1));
  }

  const int32_t* pages = table + (int64_t)s * batch.table_ld;
  // pages of the step at t (-1 past the tile's last token)
  auto pages_of = [&](int t, int (&id)[PP]) {
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      const int at = t + p * (ST / PP);
      const int got = pages[min(at, max(hi - 1, 0)) >> shift];
      id[p] = at < hi ? got : -1;
    }
  };
  auto load = [&](int t, const int (&id)[PP], Step<D, NT, PP>& x) {
#pragma unroll
    for (int p = 0; p < PP; ++p) {
      const int at = t + p * (ST / PP);
      const int page = __builtin_amdgcn_readfirstlane(id[p]);
      const bool there = page >= 0 && page < cache.pages;
      const int64_t head_tile = (int64_t)(there ? page : 0) * cache.kv_heads + head;
      const int left = min(q.tokens - (at & ~in_page), in_page + 1);
      const uint32_t size = there ? (uint32_t)(left * D) : 0u;
      const i32x4 kr = make_rsrc(cache.k + head_tile * tile_bytes, size);
      const i32x4 vr = make_rsrc(cache.v + head_tile * tile_bytes, size);
      const int off = __builtin_amdgcn_readfirstlane((at & in_page) * D);
#pragma unroll
      for (int i = p * (NT / PP); i < (p + 1) * (NT / PP); ++i) {
        const int so = off + (i - p * (NT / PP)) * 16 * D;
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
          x.k[i][h] = __builtin_bit_cast(u32x4, kq_rbl_v4i32(kr, k_lane + 64 * h, so, 0));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (VD == 1) {
            x.v[4 * i + r][0] = (uint32_t)kq_rbl_i32(vr, v_lane + r * D, so, 0);
          } else if constexpr (VD == 2) {
            const i32x2 w = kq_rbl_v2i32(vr, v_lane + r * D, so, 0);
            x.v[4 * i + r][0] = (uint32_t)w[0];
            x.v[4 * i + r][1] = (uint32_t)w[1];
          } else {
            const i32x4 w = kq_rbl_v4i32(vr, v_lane + r * D, so, 0);
#pragma unroll
            for (int d = 0; d < VD; ++d) x.v[4 * i + r][d] = (uint32_t)w[d];
          }
        }
      }
      x.ks[p] = there ? k_scale[head_tile] * a.scale : 0.0f;
      x.vs[p] = there ? v_scale[head_tile] : 0.0f;
    }
  };

  f32x4 o[OT];
#pragma unroll
  for (int j = 0; j < OT; ++j) o[j] = f32x4{0, 0, 0, 0};
  float top = -__builtin_inff(), sum = 0.0f;
  auto compute = [&](int t, const Step<D, NT, PP>& x) {
    f32x4 w[NT];
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < KS / 2; ++h) {
        acc = mfma16<DT>(widen_codes<DT>(x.k[i][h][0], x.k[i][h][1]), qf[2 * h], acc);
        acc = mfma16<DT>(widen_codes<DT>(x.k[i][h][2], x.k[i][h][3]), qf[2 * h + 1], acc);
      }
      const int p = i / (NT / PP);
      const float shift_v = __builtin_amdgcn_logf(x.vs[p]);  // (-inf where there are no tokens)
#pragma unroll
      for (int r = 0; r < 4; ++r) w[i][r] = fmaf(acc[r], x.ks[p], shift_v);
    }
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
      for (int r = 0; r < 4; ++r) w[i][r] = __builtin_amdgcn_exp2f(w[i][r] - base);
      const float vs = x.vs[i / (NT / PP)];
      sum += (w[i][0] + w[i][1] + w[i][2] + w[i][3]) * (vs > 0.0f ? 1.0f / vs : 0.0f);
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
          for (int r = 0; r < 4; ++r) in[e][r] = x.v[8 * g + 4 * e + r][d];
          transpose4(in[e], out[e]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[4 * d + j] = mfma16<KQ_DTYPE_F16>(widen_codes<KQ_DTYPE_F16>(out[0][j], out[1][j]), p[g], o[4 * d + j]);
      }
  };

  // one step in flight while another is computed, the pages of a third looked up
  int t = lo + ST * wave;
  if (t < hi) {
    int id[PP];
    Step<D, NT, PP> x, y;
    pages_of(t, id);
    load(t, id, x);
    pages_of(t + 4 * ST, id);
    while (true) {
      load(t + 4 * ST, id, y);
      pages_of(t + 8 * ST, id);
      compute(t, x);
      t += 4 * ST;
      if (t >= hi) break;
      load(t + 4 * ST, id, x);
      pages_of(t + 8 * ST, id);
      compute(t, y);
      t += 4 * ST;
      if (t >= hi) break;
    }
  }
  sum = column_sum(sum);

  // the waves' parts meet in LDS, added in wave order
  const bool whole = part_blocks == blocks;
  __syncthreads();  // (the last tile's parts have been read)
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
  __syncthreads();
  for (int i = (int)threadIdx.x; i < 16 * (D / 2); i += 256) {
    const int col = i / (D / 2), d = 2 * (i - col * (D / 2));
    const int it = tile * 16 + col;
    if (it >= q.rows * group) break;
    float m = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < 4; ++v) m = fmaxf(m, lds[(v * 16 + col) * LD + D]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float x = 0.0f, y = 0.0f, l = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float* part = lds + (v * 16 + col) * LD;
      const float f = __builtin_amdgcn_exp2f(part[D] - base);
      x += part[d] * f;
      y += part[d + 1] * f;
      l += part[D + 1] * f;
    }
    if (!whole) {
      float* dst = a.part + ((((int64_t)head * a.shares + (int)blockIdx.x) * 2 + (within == 0)) * 16 + col) * LD;
      *(f32x2_t*)(dst + d) = f32x2_t{x, y};
      if (d == 0) *(f32x2_t*)(dst + D) = f32x2_t{m, l};
      continue;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees no token is zero)
    const int rw = it / group;
    uint32_t* dst = (uint32_t*)(a.out + ((int64_t)(q.row0 + rw) * a.heads + head * group + (it - rw * group)) * D + d);
    *dst = pack_act2(x * inv, y * inv, DT);
  }

  block += part_blocks;
  within = 0;
  if (block >= run_end) return;
  if (++tile >= Deal::tiles(q, group)) {
    tile = 0;
    do {
      if (++s >= batch.seqs) return;
      q = kv_seq(batch, s, shift);
    } while (q.rows == 0);
    blocks = Deal::blocks(a, q);
  }
  }
}

// The parts of split sequences joined in the order of their tokens: one wave per row
// and query head.
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv_attend_join_kernel(AttendArgs a, KvCache cache, KvBatch batch) {
  constexpr int LD = D + 4, PER = D / 64;
  const int shift = cache.page_shift, group = a.heads / cache.kv_heads;
  const int64_t at = (int64_t)blockIdx.x * 4 + wave_id();
  if (at >= (int64_t)batch.rows * a.heads) return;
  const int row = (int)(at / a.heads), qh = (int)(at - (int64_t)row * a.heads);
  const Deal deal = deal_of(a, batch, shift, group);
  int64_t block;
  const int s = kv_of_row(row, batch, shift, block, [&](int i) {
    const KvSeq q = kv_seq(batch, i, shift);
    return Deal::tiles(q, group) * Deal::blocks(a, q);
  });
  if (s < 0) return;
  const KvSeq q = kv_seq(batch, s, shift);
  const int blocks = Deal::blocks(a, q);
  const int head = qh / group, item = (row - q.row0) * group + (qh - head * group);
  block += (int64_t)(item >> 4) * blocks;
  const int x0 = (int)(block / deal.run), chunks = (int)((block + blocks - 1) / deal.run) - x0 + 1;
  if (chunks == 1) return;  // written already
  // part 1 of the run it begins in, then part 0 of those behind
  const float* src = a.part + ((((int64_t)head * a.shares + x0) * 2 + 1) * 16 + (item & 15)) * LD;
  auto at_part = [&](int i) { return src + (int64_t)(i == 0 ? 0 : 2 * i - 1) * 16 * LD; };
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

// Workgroups that fill the chip: 256 CUs times what the registers let a CU hold.
constexpr int rows_slots(int64_t dim) { return 256 * (dim == 64 ? 3 : dim == 128 ? 2 : 1); }

static int rows_shares(int64_t kv_heads, int64_t dim) { return (int)std::max<int64_t>(rows_slots(dim) / kv_heads, 1); }

// Whether a tile can have more than one block, and so be split.
static bool rows_split(int64_t page_size, int64_t width) { return width * page_size > 256; }

template <int D, int DT, int NT, int PP>
static void launch_rows(const AttendArgs& a, bool split, const KvCache& c, const KvBatch& b, hipStream_t st) {
  const size_t lds = sizeof(float) * 4 * 16 * (D + 4);
  hipLaunchKernelGGL((kv_attend_rows_kernel<D, DT, NT, PP>), dim3((unsigned)a.shares, (unsigned)c.kv_heads), dim3(256), lds, st, a,
                     c, b, b.table, c.k_scale, c.v_scale);
  if (split)
    hipLaunchKernelGGL((kv_attend_join_kernel<D, DT>), dim3((unsigned)(((int64_t)b.rows * a.heads + 3) / 4)), dim3(256), 0, st, a,
                       c, b);
}

template <int D, int DT>
static void pick_pages(const AttendArgs& a, bool split, const KvCache& c, const KvBatch& b, hipStream_t st) {
  constexpr int NT = D == 256 ? 2 : 4;  // (registers)
  const int page = 1 << c.page_shift;
  if (page >= 16 * NT)
    launch_rows<D, DT, NT, 1>(a, split, c, b, st);
  else if (page == 8 * NT)
    launch_rows<D, DT, NT, 2>(a, split, c, b, st);
  else if constexpr (NT == 4)
    launch_rows<D, DT, NT, 4>(a, split, c, b, st);
}

template <int D>
static void pick_rows(const AttendArgs& a, bool split, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  if (dtype == KQ_DTYPE_BF16)
    pick_pages<D, KQ_DTYPE_BF16>(a, split, c, b, st);
  else
    pick_pages<D, KQ_DTYPE_F16>(a, split, c, b, st);
}

}  // namespace kq

using namespace kq;

extern "C" size_t kq_kv_attention_workspace_size(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                                 int64_t page_size, int64_t table_width, int64_t seqs) {
  if (rows < 1 || heads < 1 || kv_heads < 1 || dim < 1 || page_size < 1 || table_width < 0 || seqs < 0) return 0;
  return rows_split(page_size, table_width) ? sizeof(float) * (size_t)(rows_shares(kv_heads, dim) * kv_heads * 2 * 16 * (dim + 4)) : 0;
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
  const bool split = !empty && rows_split(page_size, table_width);
  if (split && (workspace == nullptr || workspace_bytes < kq_kv_attention_workspace_size(rows, heads, kv_heads, dim, page_size,
                                                                                           table_width, seqs))) {
    set_error("%s: workspace of %zu bytes is too small", what, workspace_bytes);
    return KQ_EWORKSPACE;
  }
  // threads of one launch, and blocks of all tiles
  if (rows * heads * 64 >= (1LL << 32) ||
      (rows * (heads / kv_heads) / 16 + seqs) * ((table_width * page_size + 255) / 256) >= (1LL << 31)) {
    set_error("%s: %lld rows of %lld heads over up to %lld tokens are past the supported range", what, (long long)rows,
              (long long)heads, (long long)(table_width * page_size));
    return KQ_EINVAL;
  }
  AttendArgs a{};
  a.q = (const uint16_t*)q;
  a.q_ld = q_ld, a.q_hs = q_hs;
  a.out = (uint16_t*)out;
  a.part = (float*)workspace;
  a.scale = scale * 1.44269504088896340736f;
  a.heads = (int)heads, a.causal = causal != 0, a.window = (int)window;
  a.shares = rows_shares(kv_heads, dim);
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  const KvCache c{(uint8_t*)k_cache, (uint8_t*)v_cache, (float*)k_scale, (float*)v_scale, pages, (int)kv_heads, shift};
  // (without pages or table columns no sequence is looked at and all rows are padding)
  const KvBatch b{table, cu, lengths, table_ld, empty ? 0 : (int)seqs, (int)table_width, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  if (dim == 64)
    pick_rows<64>(a, split, c, b, dtype, st);
  else if (dim == 128)
    pick_rows<128>(a, split, c, b, dtype, st);
  else
    pick_rows<256>(a, split, c, b, dtype, st);
  return check_launch(what);
}
