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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct AttendArgs {
  const uint16_t* q;
  int64_t q_ld, q_hs;
  uint16_t* out;  // [rows][heads][D]
  float scale;    // times log2 e
  int heads, causal, window;
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

// max over the four lanes that hold one column (lanes l, l ^ 16, l ^ 32, l ^ 48)
KQ_DEV float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
KQ_DEV float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// One workgroup: 16 rows (new tokens x the group's query heads) of one sequence and
// kv head; its four waves take the sequence's tokens apart, 64 at a step.
//
// Products run transposed, S^T = K Q^T and O^T = V^T P^T, on 16x16x32 MFMAs: lane
// (c, b) = (l % 16, l / 16) then holds scores of query row c for tokens 4b..4b+3 of
// each 16-token tile, which are, for two tiles, just the eight tokens that it has to
// hand over as its part of P^T: no score leaves its lane.  Keys and values go from
// memory to registers; a lane loads D / 16 bytes of each of its 16 tokens' values and
// transposes them by bytes (the order of d within an output tile is free: row c of
// tile j is d = c * D / 16 + j, so a lane ends up with neighbouring elements).
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv_attend_rows_kernel(AttendArgs a, KvCache cache, KvBatch batch) {
  constexpr int KS = D / 32;  // MFMA steps along a key
  constexpr int VD = D / 64;  // dwords of a token's value a lane holds
  constexpr int OT = D / 16;  // output tiles
  extern __shared__ float lds[];  // [4][16][D + 2]
  const int lane = lane_id(), wave = wave_id(), c = lane & 15, b = lane >> 4;
  const int shift = cache.page_shift, group = a.heads / cache.kv_heads;
  const int head = (int)blockIdx.y;
  int tile;
  const int s = kv_find((int)blockIdx.x, batch.seqs, tile, [&](int i) {
    const KvSeq q = kv_seq(batch, i, shift);
    return (q.rows * group + 15) >> 4;
  });
  if (s < 0) return;
  const KvSeq q = kv_seq(batch, s, shift);
  const int item = tile * 16 + c;  // this lane's column: row item / group, head item % group
  const bool real = item < q.rows * group;
  const int row = real ? item / group : 0, qh = real ? item - row * group : 0;
  const int pos = q.first + row;
  // tokens [from, to) of this column, [lo, hi) of the tile
  int to = a.causal ? min(q.tokens, pos + 1) : q.tokens;
  int from = a.window > 0 ? max(pos + 1 - a.window, 0) : 0;
  if (!real) to = from = 0;
  const int row_lo = (tile * 16) / group, row_hi = min(q.rows - 1, (tile * 16 + 15) / group);
  const int hi = a.causal ? min(q.tokens, q.first + row_hi + 1) : q.tokens;
  const int lo = a.window > 0 ? max(q.first + row_lo + 1 - a.window, 0) : 0;

  u32x4 qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) qf[i] = u32x4{0, 0, 0, 0};
  if (real) {
    const uint16_t* src = a.q + (int64_t)(q.row0 + row) * a.q_ld + (int64_t)(head * group + qh) * a.q_hs;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *(const u32x4*)(src + 64 * (i >> 1) + 16 * b + 8 * (i & 1));
  }

  f32x4 o[OT];
#pragma unroll
  for (int j = 0; j < OT; ++j) o[j] = f32x4{0, 0, 0, 0};
  float top = -__builtin_inff(), sum = 0.0f;
  const int64_t tile_bytes = (int64_t)D << shift;
  for (int t0 = (lo & ~63) + 64 * wave; t0 < hi; t0 += 256) {
    f32x4 w[4];
    float inv_v[4];
    u32x2 unused;
    (void)unused;
    uint32_t vr[16][VD];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + 16 * i;
      int page = t < hi ? kv_page(batch, cache, s, t >> shift) : -1;
      page = __builtin_amdgcn_readfirstlane(page);
      const bool there = page >= 0;
      const int64_t at = (int64_t)max(page, 0) * cache.kv_heads + head;
      const int off = (t & ((1 << shift) - 1)) * D;
      const uint8_t* kp = cache.k + at * tile_bytes + off + c * D + 16 * b;
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < KS / 2; ++h) {
        const u32x4 raw = *(const u32x4*)(kp + 64 * h);
        acc = mfma16<DT>(widen_codes<DT>(raw[0], raw[1]), qf[2 * h], acc);
        acc = mfma16<DT>(widen_codes<DT>(raw[2], raw[3]), qf[2 * h + 1], acc);
      }
      const uint8_t* vp = cache.v + at * tile_bytes + off + 4 * b * D + c * (D / 16);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < VD; ++d) {
          const uint32_t x = *(const uint32_t*)(vp + r * D + 4 * d);
          // slots past the end hold whatever was there, NaN perhaps
          vr[4 * i + r][d] = there && t + 4 * b + r < q.tokens ? x : 0u;
        }
      const float ks = there ? cache.k_scale[at] * a.scale : 0.0f;
      const float vs = there ? cache.v_scale[at] : 1.0f;
      inv_v[i] = 1.0f / vs;
      const float shift_v = __builtin_amdgcn_logf(vs);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int token = t + 4 * b + r;
        w[i][r] = there && token >= from && token < to ? acc[r] * ks + shift_v : -__builtin_inff();
      }
    }
    float m = top;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, w[i][r]);
    m = column_max(m);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    top = m;
    sum *= keep;
#pragma unroll
    for (int j = 0; j < OT; ++j) o[j] *= keep;
    u32x4 p[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) w[i][r] = __builtin_amdgcn_exp2f(w[i][r] - base);
      sum += (w[i][0] + w[i][1] + w[i][2] + w[i][3]) * inv_v[i];
      p[i >> 1][2 * (i & 1)] = pack_act2(w[i][0], w[i][1], KQ_DTYPE_F16);
      p[i >> 1][2 * (i & 1) + 1] = pack_act2(w[i][2], w[i][3], KQ_DTYPE_F16);
    }
#pragma unroll
    for (int d = 0; d < VD; ++d)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t in[2][4], out[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int r = 0; r < 4; ++r) in[e][r] = vr[8 * g + 4 * e + r][d];
          transpose4(in[e], out[e]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[4 * d + j] = mfma16<KQ_DTYPE_F16>(widen_codes<KQ_DTYPE_F16>(out[0][j], out[1][j]), p[g], o[4 * d + j]);
      }
  }
  sum = column_sum(sum);

  // the waves' parts meet in LDS, added in wave order
  float* mine = lds + (wave * 16 + c) * (D + 2);
#pragma unroll
  for (int j = 0; j < OT; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) mine[(4 * b + r) * OT + j] = o[j][r];
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
    for (int v = 0; v < 4; ++v) m = fmaxf(m, lds[(v * 16 + col) * (D + 2) + D]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float x = 0.0f, y = 0.0f, l = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float* part = lds + (v * 16 + col) * (D + 2);
      const float f = __builtin_amdgcn_exp2f(part[D] - base);
      x += part[d] * f;
      y += part[d + 1] * f;
      l += part[D + 1] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees no token is zero)
    const int rw = it / group;
    uint32_t* dst = (uint32_t*)(a.out + ((int64_t)(q.row0 + rw) * a.heads + head * group + (it - rw * group)) * D + d);
    *dst = pack_act2(x * inv, y * inv, DT);
  }
}

// Rows past the last sequence are zero.
__global__ void kv_pad_kernel(uint32_t* out, const int32_t* cu, int seqs, int rows, int row_words) {
  const int row = (int)blockIdx.x;
  const int first = seqs > 0 ? cu[0] : rows, last = seqs > 0 ? cu[seqs] : 0;
  if (row >= first && row < last) return;
  for (int i = (int)threadIdx.x; i < row_words; i += (int)blockDim.x) out[(int64_t)row * row_words + i] = 0;
}

template <int D, int DT>
static void launch_rows(const AttendArgs& a, const KvCache& c, const KvBatch& b, hipStream_t st) {
  const int group = a.heads / c.kv_heads;
  const int64_t tiles = std::min<int64_t>((int64_t)b.rows * group, (int64_t)b.rows * group / 16 + b.seqs);
  const size_t lds = sizeof(float) * 4 * 16 * (D + 2);
  hipLaunchKernelGGL((kv_attend_rows_kernel<D, DT>), dim3((unsigned)tiles, (unsigned)c.kv_heads), dim3(256), lds, st, a, c, b);
}

template <int D>
static void pick_rows(const AttendArgs& a, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  if (dtype == KQ_DTYPE_BF16)
    launch_rows<D, KQ_DTYPE_BF16>(a, c, b, st);
  else
    launch_rows<D, KQ_DTYPE_F16>(a, c, b, st);
}

}  // namespace kq

using namespace kq;

extern "C" int kq_kv_attention(const void* q, int64_t q_ld, int64_t q_hs, int dtype, int64_t rows, int64_t heads,
                               int64_t kv_heads, int64_t dim, const uint8_t* k_cache, const uint8_t* v_cache,
                               const float* k_scale, const float* v_scale, int64_t pages, int64_t page_size,
                               const int32_t* table, int64_t table_ld, int64_t table_width, const int32_t* cu,
                               const int32_t* lengths, int64_t seqs, float scale, int causal, int64_t window, void* out,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "kq_kv_attention";
  (void)workspace;
  (void)workspace_bytes;
  int rc = kv_check(what, dtype, rows, heads, kv_heads, dim, page_size, pages, seqs, table_width, table_ld);
  if (rc) return rc;
  if (window < 0 || window > (1 << 30) || (window > 0 && !causal)) {
    set_error("%s: window %lld (a window is of causal attention)", what, (long long)window);
    return KQ_EINVAL;
  }
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) % 16 != 0 || (q_ld | q_hs) % 8 != 0) {
    set_error("%s: tensors need 16-byte aligned rows and heads", what);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  AttendArgs a{(const uint16_t*)q, q_ld, q_hs, (uint16_t*)out, scale * 1.44269504088896340736f, (int)heads, causal != 0,
               (int)window};
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  const KvCache c{(uint8_t*)k_cache, (uint8_t*)v_cache, (float*)k_scale, (float*)v_scale, pages, (int)kv_heads, shift};
  const KvBatch b{table, cu, lengths, table_ld, (int)seqs, (int)table_width, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(kv_pad_kernel, dim3((unsigned)rows), dim3(256), 0, st, (uint32_t*)out, cu, (int)seqs, (int)rows,
                     (int)(heads * dim / 2));
  if (seqs > 0 && pages > 0) {
    if (dim == 64)
      pick_rows<64>(a, c, b, dtype, st);
    else if (dim == 128)
      pick_rows<128>(a, c, b, dtype, st);
    else
      pick_rows<256>(a, c, b, dtype, st);
  }
  return check_launch(what);
}

extern "C" size_t kq_kv_attention_workspace_size(int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
                                                 int64_t page_size, int64_t table_width, int64_t seqs) {
  return 0;
}
