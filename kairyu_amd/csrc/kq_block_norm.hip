// The norms around a decoder block in one pass over its rows:
//
//   b = x / rms(x) * post          (post-norm of the block's output, optional)
//   r = residual + residual_scale * gate * b
//   y = r / rms(r) * weight        (pre-norm of the next block)
//
// with rms(z) = sqrt(mean(z^2) + eps) and, for weights kept as an offset from one,
// 1 + weight.  r goes back to the residual stream in its type and y out in 16 bits or
// as the next projection's quantized rows (per token e4m3 or int8, or 1x128 e4m3
// blocks, scale max(amax, 1e-12) / 448 or / 127).  Everything between the loads and
// those stores is fp32: the second norm and the quantization see r and y unrounded,
// one rounding fewer on each than the separate operations have.
//
// One workgroup per row, the row in registers, each operand read once.  HBM bound on
// many rows (8192 of 4096, gate and fp32 residual, out in blocks: 437 MB in 76-87 us,
// 5.0-5.7 TB/s, the rate of a copy); on few, by the chain load -> sum -> sum -> store
// (48 of 3584: 4.2 us), so the amax joins the second sum (amax(y) = amax(r * weight) /
// rms(r)) instead of following it.
#include "kq_common.h"

#include <algorithm>

namespace kq {

enum { kNormPlain = 0, kNormFp8 = 1, kNormInt8 = 2, kNormBlocks = 3 };

struct NormArgs {
  const uint16_t* x;
  const void* residual;     // null: r = residual_scale * gate * b
  const uint16_t* post;     // null: b = x
  const uint16_t* gate;     // null: 1
  const uint16_t* weight;
  int64_t x_ld, residual_ld, gate_ld;  // gate_ld 0: one row for all
  void* r_out;              // [rows][hidden], of the residual's type
  void* y_out;              // 16 bits, or e4m3 / int8
  float* scales;            // [rows] or [rows][ceil(hidden / 128)]
  int64_t hidden;
  float eps, residual_scale, offset;
};

// Elements [i, i + 8) of a 16-bit row, packed as they are; 0 past its end.
KQ_DEV u32x4 norm_raw(const uint16_t* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 8 <= n) return *(const u32x4*)(p + i);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = i + 2 * j < n ? p[i + 2 * j] : 0u, hi = i + 2 * j + 1 < n ? p[i + 2 * j + 1] : 0u;
    w[j] = lo | hi << 16;
  }
  return u32x4{w[0], w[1], w[2], w[3]};
}
KQ_DEV void norm_widen(u32x4 raw, int dtype, float v[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = act_lo(raw[j], dtype);
    v[2 * j + 1] = act_hi(raw[j], dtype);
  }
}

// Sum of one value and (if asked for) maximum of another over the workgroup.
KQ_DEV void block_sum(float& sum, uint32_t& most, float* red, uint32_t* redm) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
  most = wave_max_u32_dpp(most);
  if (lane_id() == 0) {
    red[wave_id()] = sum;
    redm[wave_id()] = most;
  }
  __syncthreads();
  sum = 0.0f;
  most = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
    sum += red[w];
    most = max(most, redm[w]);
  }
}

// Four quantized elements y / s.  Finite rows take the correctly rounded quotient from
// one reciprocal a row (div_by_recip: s is at least 1e-12 / 448) and the hardware's
// conversions; rows that hold inf or NaN keep IEEE division and NaN codes.
template <bool INT8>
KQ_DEV uint32_t quant4(const float y[4], float s, float rs, bool fast) {
  float t[4];
  uint32_t w = 0;
  if (fast) {
    constexpr float most = INT8 ? 127.0f : 448.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = fminf(fmaxf(div_by_recip(y[e], s, rs), -most), most);
    if (!INT8) return pack4_e4m3(t[0], t[1], t[2], t[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= ((uint32_t)(int32_t)__builtin_rintf(t[e]) & 0xffu) << (8 * e);
    return w;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float q = __fdiv_rn(y[e], s);
    if (INT8)
      w |= ((uint32_t)(int32_t)__builtin_rintf(clamp_keep_nan(q, 127.0f)) & 0xffu) << (8 * e);
    else
      w |= f32_to_e4m3(clamp_keep_nan(q, 448.0f)) << (8 * e);
  }
  return w;
}

template <int NCH, int MODE>
__global__ void __launch_bounds__(1024)
block_norm_kernel(NormArgs a, int dtype, int res_dtype, bool vec) {
  __shared__ float red[2][16];
  __shared__ uint32_t redm[2][16];
  const int64_t row = blockIdx.x, n = a.hidden;
  const int tid = (int)threadIdx.x, threads = (int)blockDim.x;
  float v[NCH][8], r[NCH][8];
  const uint16_t* x = a.x + row * a.x_ld;
  float sum = 0.0f;
  // every operand is on its way before the first sum goes round
  u32x4 xr[NCH], wr[NCH], pr[NCH], gr[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t i = ((int64_t)tid + (int64_t)threads * c) * 8;
    xr[c] = norm_raw(x, i, n, vec);
    if (a.residual == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[c][e] = 0.0f;
    } else if (res_dtype == KQ_DTYPE_F32) {
      const float* p = (const float*)a.residual + row * a.residual_ld;
      if (vec && i + 8 <= n) {
        const f32x4 lo = *(const f32x4*)(p + i), hi = *(const f32x4*)(p + i + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r[c][e] = lo[e];
          r[c][4 + e] = hi[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[c][e] = i + e < n ? p[i + e] : 0.0f;
      }
    } else {
      norm_widen(norm_raw((const uint16_t*)a.residual + row * a.residual_ld, i, n, vec), dtype, r[c]);
    }
    if (a.gate != nullptr) gr[c] = norm_raw(a.gate + row * a.gate_ld, i, n, vec);
    if (a.post != nullptr) pr[c] = norm_raw(a.post, i, n, vec);
    wr[c] = norm_raw(a.weight, i, n, vec);
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    norm_widen(xr[c], dtype, v[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[c][e] * v[c][e];
  }
  float inv = 1.0f;
  uint32_t none = 0;
  if (a.post != nullptr) {
    block_sum(sum, none, red[0], redm[0]);
    inv = 1.0f / sqrtf(sum / (float)n + a.eps);
  }
  float sum2 = 0.0f;
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t i = ((int64_t)tid + (int64_t)threads * c) * 8;
    if (i < n) {
      if (a.post != nullptr) {
        float w[8];
        norm_widen(pr[c], dtype, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * inv * (w[e] + a.offset);
      }
      if (a.gate != nullptr) {
        float g[8];
        norm_widen(gr[c], dtype, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] *= g[e];
      }
      float w[8];
      norm_widen(wr[c], dtype, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = i + e < n ? r[c][e] + a.residual_scale * v[c][e] : 0.0f;
        sum2 += z * z;
        r[c][e] = z;
        v[c][e] = z * (w[e] + a.offset);
        if (MODE == kNormFp8 || MODE == kNormInt8) most = max(most, __float_as_uint(v[c][e]) & 0x7fffffffu);
      }
      // r in the residual's type
      if (res_dtype == KQ_DTYPE_F32) {
        float* p = (float*)a.r_out + row * n;
        if (vec && i + 8 <= n) {
          *(f32x4*)(p + i) = f32x4{r[c][0], r[c][1], r[c][2], r[c][3]};
          *(f32x4*)(p + i + 4) = f32x4{r[c][4], r[c][5], r[c][6], r[c][7]};
        } else {
          for (int e = 0; e < 8 && i + e < n; ++e) p[i + e] = r[c][e];
        }
      } else {
        uint16_t* p = (uint16_t*)a.r_out + row * n;
        if (vec && i + 8 <= n) {
          *(u32x4*)(p + i) = u32x4{pack_act2(r[c][0], r[c][1], dtype), pack_act2(r[c][2], r[c][3], dtype),
                                   pack_act2(r[c][4], r[c][5], dtype), pack_act2(r[c][6], r[c][7], dtype)};
        } else {
          for (int e = 0; e < 8 && i + e < n; ++e) p[i + e] = f32_to_out(r[c][e], dtype);
        }
      }
    }
  }
  block_sum(sum2, most, red[1], redm[1]);
  inv = 1.0f / sqrtf(sum2 / (float)n + a.eps);
  float s = 0.0f;
  bool fast = true;
  if (MODE == kNormFp8 || MODE == kNormInt8) {
    fast = most < 0x7f800000u && inv <= 3.402823466e38f;
    s = __fdiv_rn(max_keep_nan(__uint_as_float(most) * inv, 1e-12f), MODE == kNormFp8 ? 448.0f : 127.0f);
    if (tid == 0) a.scales[row] = s;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t i = ((int64_t)tid + (int64_t)threads * c) * 8;
    float y[8];
    if (MODE == kNormBlocks) {  // 16 neighbouring lanes hold a block of 128
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = i < n ? v[c][e] * inv : 0.0f;
        top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
      }
      top = dpp_max_u32<0xB1>(top);
      top = dpp_max_u32<0x4E>(top);
      top = dpp_max_u32<0x141>(top);
      top = dpp_max_u32<0x140>(top);
      s = __fdiv_rn(max_keep_nan(__uint_as_float(top), 1e-12f), 448.0f);
      fast = __ballot(top >= 0x7f800000u) == 0;
      if (i < n && (tid & 15) == 0) a.scales[row * ((n + 127) / 128) + i / 128] = s;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = i < n ? v[c][e] * inv : 0.0f;
    }
    if (i >= n) continue;
    if (MODE == kNormPlain) {
      uint16_t* p = (uint16_t*)a.y_out + row * n;
      if (vec && i + 8 <= n) {
        *(u32x4*)(p + i) = u32x4{pack_act2(y[0], y[1], dtype), pack_act2(y[2], y[3], dtype), pack_act2(y[4], y[5], dtype),
                                 pack_act2(y[6], y[7], dtype)};
      } else {
        for (int e = 0; e < 8 && i + e < n; ++e) p[i + e] = f32_to_out(y[e], dtype);
      }
      continue;
    }
    const float rs = __fdiv_rn(1.0f, s);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = quant4<MODE == kNormInt8>(y + 4 * h, s, rs, fast);
    uint8_t* p = (uint8_t*)a.y_out + row * n;
    if (vec && i + 8 <= n) {
      *(u32x2*)(p + i) = u32x2{w[0], w[1]};
    } else {
      for (int e = 0; e < 8 && i + e < n; ++e) p[i + e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

template <int NCH>
static void launch_norm(const NormArgs& a, int mode, int dtype, int res_dtype, bool vec, int64_t rows, int threads,
                        hipStream_t st) {
  const dim3 g((unsigned)rows), t((unsigned)threads);
  switch (mode) {
    case kNormPlain: hipLaunchKernelGGL((block_norm_kernel<NCH, kNormPlain>), g, t, 0, st, a, dtype, res_dtype, vec); break;
    case kNormFp8: hipLaunchKernelGGL((block_norm_kernel<NCH, kNormFp8>), g, t, 0, st, a, dtype, res_dtype, vec); break;
    case kNormInt8: hipLaunchKernelGGL((block_norm_kernel<NCH, kNormInt8>), g, t, 0, st, a, dtype, res_dtype, vec); break;
    default: hipLaunchKernelGGL((block_norm_kernel<NCH, kNormBlocks>), g, t, 0, st, a, dtype, res_dtype, vec); break;
  }
}

}  // namespace kq

using namespace kq;

extern "C" int kq_block_norm(const void* x, int dtype, int64_t rows, int64_t hidden, int64_t x_ld, const void* residual,
                             int residual_dtype, int64_t residual_ld, const void* post, const void* gate, int64_t gate_ld,
                             float residual_scale, const void* weight, float offset, float eps, int mode, void* r_out,
                             void* y_out, float* scales, void* stream) {
  if (dtype != KQ_DTYPE_F16 && dtype != KQ_DTYPE_BF16) {
    set_error("kq_block_norm: activation dtype must be fp16 or bf16 (code %d)", dtype);
    return KQ_EUNSUPPORTED;
  }
  if (residual_dtype != dtype && residual_dtype != KQ_DTYPE_F32) {
    set_error("kq_block_norm: residual dtype must be the activations' or fp32 (code %d)", residual_dtype);
    return KQ_EUNSUPPORTED;
  }
  if (rows < 0 || rows > 0x3fffff || hidden < 1 || hidden > 32768 || x_ld < hidden ||
      (residual != nullptr && residual_ld < hidden) || (gate != nullptr && gate_ld != 0 && gate_ld < hidden) || mode < 0 ||
      mode > 3) {
    set_error("kq_block_norm: bad shape rows=%lld hidden=%lld (mode %d)", (long long)rows, (long long)hidden, mode);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  NormArgs a{};
  a.x = (const uint16_t*)x;
  a.residual = residual;
  a.post = (const uint16_t*)post;
  a.gate = (const uint16_t*)gate;
  a.weight = (const uint16_t*)weight;
  a.x_ld = x_ld, a.residual_ld = residual_ld, a.gate_ld = gate_ld;
  a.r_out = r_out, a.y_out = y_out, a.scales = scales;
  a.hidden = hidden;
  a.eps = eps, a.residual_scale = residual_scale, a.offset = offset;
  const uintptr_t at = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)post | (uintptr_t)gate | (uintptr_t)weight |
                       (uintptr_t)r_out | (uintptr_t)y_out;
  const bool vec = at % 16 == 0 && (x_ld | residual_ld | gate_ld | hidden) % 8 == 0;
  // rows that fill the chip keep up to 512 threads each, so that several are in flight on
  // a CU (4096 rows of 8192: 54.6 us, with 256 threads 58.5); fewer spread a row over 1024
  const int64_t chunks = (hidden + 7) / 8;
  const int64_t wide = rows < 256 ? 1024 : 512;
  const int nch = chunks <= wide ? 1 : chunks <= 2 * 1024 ? 2 : 4;
  const int64_t per = (chunks + nch - 1) / nch;
  const int threads = (int)std::min<int64_t>(1024, std::max<int64_t>(64, (per + 63) / 64 * 64));
  hipStream_t st = (hipStream_t)stream;
  switch (nch) {
    case 1: launch_norm<1>(a, mode, dtype, residual_dtype, vec, rows, threads, st); break;
    case 2: launch_norm<2>(a, mode, dtype, residual_dtype, vec, rows, threads, st); break;
    default: launch_norm<4>(a, mode, dtype, residual_dtype, vec, rows, threads, st); break;
  }
  return check_launch("kq_block_norm");
}
