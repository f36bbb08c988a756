// What the attention kernels over the paged e4m3 cache share: products with widened
// codes, reductions over a column's lanes, rows of no sequence.
#pragma once

#include "kq_kv.h"

namespace kq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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
template <int D, typename Args>
KQ_DEV void zero_padding(const Args& a, const KvBatch& batch, int head, int group, int nth, int of, int threads) {
  const int last = batch.seqs > 0 ? min(max(batch.cu[batch.seqs], 0), batch.rows) : 0;
  const int first = batch.seqs > 0 ? min(max(batch.cu[0], 0), last) : 0;
  const int words = group * D / 2;
  for (int i = nth; i < first + batch.rows - last; i += of) {
    const int64_t row = i < first ? i : last + (i - first);
    uint32_t* dst = (uint32_t*)(a.out + (row * a.heads + head * group) * D);
    for (int j = (int)threadIdx.x; j < words; j += threads) dst[j] = 0;
  }
}

}  // namespace kq
