// Rotary positions and the append to a paged e4m3 cache in one launch.
//
// Query and key heads (optionally normed per head, x / rms(x) * weight) turn by
// their position's angles, x1' = x1 cos - x2 sin, x2' = x2 cos + x1 sin, from the
// caller's fp32 table of cos and sin; rotated queries are written in 16 bits, keys
// and values as e4m3 codes of x * 2^-e with one exponent per page and head: the
// smallest e with max |x| <= 448 * 2^e over what the page is given, and never below
// the exponent it has already where it holds earlier tokens.  A page whose exponent
// grows has its earlier codes moved to the new scale.  Powers of two make that move
// exact (but for codes that fall below e4m3's normal range, which round once more),
// and dividing by the scale as well; a floating-point code loses nothing to a scale
// that is up to twice as large as it had to be.
//
// A token whose rotated key or whose value is not finite in a head is stored there
// as a key of NaN codes, and such elements of its value as 0: every row that attends
// to it becomes NaN and no row that does not, since no 0 * NaN enters a sum of values.
#include "kq_kv.h"

#include <algorithm>

namespace kq {

struct AppendArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_ld, k_ld, v_ld;  // elements from one row to the next
  int64_t q_hs, k_hs, v_hs;  // and from one head to the next
  uint16_t* q_out;           // [rows][heads][D]
  const float* cos_sin;      // [positions][rotary]: cos, then sin
  int64_t positions;
  const int32_t* at;         // [rows], or null: a row turns by its slot
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  float eps;
  int heads, rotary, interleaved;  // (rotary 0: no rotation)
  int page_units;  // workgroups of the append (the rest rotate queries)
};

KQ_DEV void widen(u32x4 raw, int dtype, float v[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = act_lo(raw[j], dtype);
    v[2 * j + 1] = act_hi(raw[j], dtype);
  }
}

// What one thread holds of a head's row: two chunks of 8 elements whose rotation needs
// no other thread's, i.e. chunks c and c + rotary / 16 of half-split pairs; what does not
// rotate goes in neighbouring chunks.  D / 16 neighbouring lanes hold a row.
struct Pairing {
  int c0, c1;   // chunks
  int angle;    // first of this thread's angles (half-split: 8 for both; interleaved: 4 each)
  bool turned;
};

template <int D>
KQ_DEV Pairing pairing(int u, const AppendArgs& a) {
  Pairing p;
  const int turning = a.rotary >> 4;  // pairs of chunks that rotate
  p.turned = u < turning;
  if (p.turned && !a.interleaved) {
    p.c0 = u;
    p.c1 = u + turning;
    p.angle = 8 * u;
  } else {
    p.c0 = 2 * u;
    p.c1 = 2 * u + 1;
    p.angle = 8 * u;
  }
  return p;
}

// cos and sin of the thread's 8 angles at a position; NaN before and past the table
struct Angles {
  float co[8], si[8];
};
KQ_DEV Angles angles_at(const Pairing& p, int pos, const AppendArgs& a) {
  Angles g;
  const bool there = pos >= 0 && pos < a.positions;
  const float* at = a.cos_sin + (int64_t)(there ? pos : 0) * a.rotary + p.angle;
  const int half = a.rotary >> 1;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x4 co = there ? *(const f32x4*)(at + 4 * h) : f32x4{0, 0, 0, 0};
    const f32x4 si = there ? *(const f32x4*)(at + half + 4 * h) : f32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g.co[4 * h + e] = there ? co[e] : __builtin_nanf("");
      g.si[4 * h + e] = si[e];
    }
  }
  return g;
}

// Norm over the row's lanes (all of them active).
template <int D>
KQ_DEV void head_norm(const Pairing& p, const uint16_t* norm, float eps, int dtype, float x[2][8]) {
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += x[0][e] * x[0][e];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += x[1][e] * x[1][e];
#pragma unroll
  for (int off = 1; off < D / 16; off <<= 1) sum += __shfl_xor(sum, off, 64);
  const float inv = 1.0f / sqrtf(sum * (1.0f / D) + eps);
  float w[8];
  widen(*(const u32x4*)(norm + 8 * p.c0), dtype, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[0][e] = x[0][e] * inv * w[e];
  widen(*(const u32x4*)(norm + 8 * p.c1), dtype, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[1][e] = x[1][e] * inv * w[e];
}

KQ_DEV void turn(const Pairing& p, const Angles& g, bool interleaved, float x[2][8]) {
  if (!p.turned) return;
  if (interleaved) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float co = g.co[4 * h + e], si = g.si[4 * h + e], y = x[h][2 * e], z = x[h][2 * e + 1];
        x[h][2 * e] = y * co - z * si;
        x[h][2 * e + 1] = z * co + y * si;
      }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = x[0][e], z = x[1][e];
      x[0][e] = y * g.co[e] - z * g.si[e];
      x[1][e] = z * g.co[e] + y * g.si[e];
    }
  }
}

// 2^e, the smallest with amax <= 448 * 2^e (448 = 7 * 2^6); amax at least 1e-12
KQ_DEV float kv_scale_for(float amax) {
  const uint32_t u = __float_as_uint(fmaxf(amax, 1e-12f));
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

KQ_DEV bool finite8(const float v[8]) {
  bool ok = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) ok = ok && fabsf(v[e]) <= 3.402823466e38f;
  return ok;
}

KQ_DEV u32x2 encode8(const float v[8], float inv) {
  u32x2 w;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = fminf(fmaxf(v[4 * h + e] * inv, -448.0f), 448.0f);
    w[h] = pack4_e4m3(t[0], t[1], t[2], t[3]);
  }
  return w;
}

// Workgroups [0, page_units): one page of one sequence and one kv head each, its new
// tokens in registers (NCH pairs of chunks a thread, keys and values), so that the scale
// is known before a code is written and each row is read once.  The others: query rows,
// HPT heads of one row a thread, which share their angles.
//
// Bound by HBM on prompts: 8 of up to 2048 rows, 32 + 8 + 8 heads of 128, 183 MB, 40 us
// (4.6 TB/s; a copy's rate is 5.2).  64 single tokens take 6 us: a launch and the chain
// bounds -> table entry -> page -> scales -> codes, whose rows' loads go first.
template <int D, int NCH, int THREADS, int HPT>
__global__ void __launch_bounds__(THREADS)
kv_append_kernel(AppendArgs a, KvCache cache, KvBatch batch, int dtype) {
  constexpr int TPR = D / 16;          // threads of a head's row
  constexpr int ROWS = THREADS / TPR;  // rows a workgroup holds at once
  const int tid = (int)threadIdx.x, rr = tid / TPR;
  const Pairing p = pairing<D>(tid % TPR, a);
  const int shift = cache.page_shift, page_size = 1 << shift;
  const KvLanes lanes(batch, shift);
  if ((int)blockIdx.x >= a.page_units) {
    const int per_row = (a.heads + HPT - 1) / HPT;  // threads (times TPR) of a query row
    const int64_t unit = (int64_t)(blockIdx.x - a.page_units) * ROWS + rr;
    const int64_t row_ = unit / per_row;
    const int head0 = (int)(unit - row_ * per_row) * HPT;
    const int row = (int)(row_ < batch.rows ? row_ : batch.rows - 1);
    // the sequence of the wave's first row, and from there for rows of another
    int unused;
    const int row0 = scalar(row);
    const int s0 = lanes.of_row(row0, unused, [](const KvSeq&) { return 0; });
    int pos = -1;  // (padding)
    KvSeq q{};
    if (s0 >= 0) q = lanes[s0];
    if (__ballot(row < q.row0 || row >= q.row0 + q.rows) == 0) {
      pos = q.first + row - q.row0;
    } else {
      // (padding does not look through the sequences)
      const int last = batch.seqs > 0 ? batch.cu[batch.seqs] : 0;
      for (int s = max(s0, 0); row < last && s < batch.seqs && batch.cu[s] <= row; ++s) {
        q = kv_seq(batch, s, shift);
        if (row >= q.row0 && row < q.row0 + q.rows) pos = q.first + row - q.row0;
      }
    }
    const uint16_t* src = a.q + (int64_t)row * a.q_ld;
    u32x4 raw[HPT][2];
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      const uint16_t* at = src + (int64_t)min(head0 + i, a.heads - 1) * a.q_hs;
      raw[i][0] = *(const u32x4*)(at + 8 * p.c0);
      raw[i][1] = *(const u32x4*)(at + 8 * p.c1);
    }
    Angles g;
    if (p.turned) g = angles_at(p, a.at != nullptr ? a.at[row] : max(pos, 0), a);
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      float x[2][8];
      widen(raw[i][0], dtype, x[0]);
      widen(raw[i][1], dtype, x[1]);
      if (a.q_norm != nullptr) head_norm<D>(p, a.q_norm, a.eps, dtype, x);
      turn(p, g, a.interleaved, x);
      if (row_ >= batch.rows || head0 + i >= a.heads) continue;
      uint16_t* dst = a.q_out + ((int64_t)row * a.heads + head0 + i) * D;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 w = {0, 0, 0, 0};
        if (pos >= 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack_act2(x[h][2 * j], x[h][2 * j + 1], dtype);
        }
        *(u32x4*)(dst + 8 * (h == 0 ? p.c0 : p.c1)) = w;
      }
    }
    return;
  }

  __shared__ uint32_t red[2][THREADS / 64];
  const int unit = scalar((int)blockIdx.x / cache.kv_heads), head = (int)blockIdx.x - unit * cache.kv_heads;
  int nth;
  const int s = lanes.find(unit, nth, [&](const KvSeq& q) {
    const int lo = max(q.first, 0);
    return q.rows > 0 && lo < q.tokens ? ((q.tokens - 1) >> shift) - (lo >> shift) + 1 : 0;
  });
  if (s < 0) return;
  const KvSeq q = lanes[s];
  const int slot = (max(q.first, 0) >> shift) + nth;
  const int lo = max(max(q.first, 0), slot << shift), hi = min(q.tokens, (slot + 1) << shift);  // positions stored here
  const int kept = lo & (page_size - 1);                                                        // earlier tokens

  // the rows are on their way while the page is looked up and then its scales
  u32x4 raw[NCH][4];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int64_t row = q.row0 + (min(lo + i * ROWS + rr, hi - 1) - q.first);
    const uint16_t* ks = a.k + row * a.k_ld + (int64_t)head * a.k_hs;
    const uint16_t* vs = a.v + row * a.v_ld + (int64_t)head * a.v_hs;
    raw[i][0] = *(const u32x4*)(ks + 8 * p.c0);
    raw[i][1] = *(const u32x4*)(ks + 8 * p.c1);
    raw[i][2] = *(const u32x4*)(vs + 8 * p.c0);
    raw[i][3] = *(const u32x4*)(vs + 8 * p.c1);
  }
  const int page = scalar(batch.table[(int64_t)s * batch.table_ld + slot]);
  if (page < 0 || page >= cache.pages) return;
  const int64_t tile = (int64_t)page * cache.kv_heads + head;
  const float ko = cache.k_scale[tile], vo = cache.v_scale[tile];  // (needed where kept > 0)

  float k[NCH][2][8], v[NCH][2][8];
  uint32_t bad = 0;
  float ka = 0.0f, va = 0.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int pos = lo + i * ROWS + rr;
    if (pos >= hi) continue;  // (whole rows: a row's lanes stay together)
    widen(raw[i][0], dtype, k[i][0]);
    widen(raw[i][1], dtype, k[i][1]);
    widen(raw[i][2], dtype, v[i][0]);
    widen(raw[i][3], dtype, v[i][1]);
    Angles g;
    if (p.turned) g = angles_at(p, a.at != nullptr ? a.at[q.row0 + (pos - q.first)] : pos, a);
    if (a.k_norm != nullptr) head_norm<D>(p, a.k_norm, a.eps, dtype, k[i]);
    turn(p, g, a.interleaved, k[i]);
    int ok = finite8(k[i][0]) && finite8(k[i][1]) && finite8(v[i][0]) && finite8(v[i][1]);
#pragma unroll
    for (int off = 1; off < TPR; off <<= 1) ok &= __shfl_xor(ok, off, 64);
    if (!ok) bad |= 1u << i;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(fabsf(v[i][h][e]) <= 3.402823466e38f)) v[i][h][e] = 0.0f;
        if (ok) ka = fmaxf(ka, fabsf(k[i][h][e]));
        va = fmaxf(va, fabsf(v[i][h][e]));
      }
  }
  const uint32_t kb = wave_max_u32_dpp(__float_as_uint(ka)), vb = wave_max_u32_dpp(__float_as_uint(va));
  if (lane_id() == 0) {
    red[0][wave_id()] = kb;
    red[1][wave_id()] = vb;
  }
  asm volatile("" ::"v"(ko), "v"(vo));  // (every thread has read the scales before one writes them)
  __syncthreads();
  uint32_t kt = 0, vt = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    kt = max(kt, red[0][w]);
    vt = max(vt, red[1][w]);
  }
  uint8_t* kc = cache.k + (tile << shift) * D;
  uint8_t* vc = cache.v + (tile << shift) * D;
  float ks = kv_scale_for(__uint_as_float(kt)), vs = kv_scale_for(__uint_as_float(vt));
  if (kept > 0) {
    const float kn = fmaxf(ks, ko), vn = fmaxf(vs, vo);
    const float kr = ko / kn, vr = vo / vn;
    if (kr < 1.0f || vr < 1.0f) {  // keys and values together: their loads are in flight at once
      const int n = kept * (D / 16);
      for (int i = tid; i < n; i += 2 * THREADS) {
        u32x4 w[4];
        const int j = min(i + THREADS, n - 1);  // (past the end: the last chunk, not stored)
        w[0] = *(const u32x4*)(kc + 16 * i);
        w[1] = *(const u32x4*)(vc + 16 * i);
        w[2] = *(const u32x4*)(kc + 16 * j);
        w[3] = *(const u32x4*)(vc + 16 * j);
        if (kr < 1.0f) *(u32x4*)(kc + 16 * i) = move16(w[0], kr);
        if (vr < 1.0f) *(u32x4*)(vc + 16 * i) = move16(w[1], vr);
        if (i + THREADS < n) {
          if (kr < 1.0f) *(u32x4*)(kc + 16 * j) = move16(w[2], kr);
          if (vr < 1.0f) *(u32x4*)(vc + 16 * j) = move16(w[3], vr);
        }
      }
    }
    ks = kn;
    vs = vn;
  }
  if (tid == 0) {
    cache.k_scale[tile] = ks;
    cache.v_scale[tile] = vs;
  }
  const float ki = 1.0f / ks, vi = 1.0f / vs;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int pos = lo + i * ROWS + rr;
    if (pos >= hi) continue;
    const int at = (pos & (page_size - 1)) * D;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 8 * (h == 0 ? p.c0 : p.c1);
      *(u32x2*)(kc + at + c) = (bad >> i) & 1 ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : encode8(k[i][h], ki);
      *(u32x2*)(vc + at + c) = encode8(v[i][h], vi);
    }
  }
}

int kv_check(const char* what, int dtype, int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim,
             int64_t page_size, int64_t pages, int64_t seqs, int64_t table_width, int64_t table_ld) {
  if (dtype != KQ_DTYPE_F16 && dtype != KQ_DTYPE_BF16) {
    set_error("%s: activation dtype must be fp16 or bf16 (code %d)", what, dtype);
    return KQ_EUNSUPPORTED;
  }
  if (dim != 64 && dim != 128 && dim != 256) {
    set_error("%s: head dim must be 64, 128 or 256, got %lld", what, (long long)dim);
    return KQ_EINVAL;
  }
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) {
    set_error("%s: page size must be 16, 32, 64 or 128 tokens, got %lld", what, (long long)page_size);
    return KQ_EINVAL;
  }
  if (rows < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || pages < 0 || seqs < 0 || table_width < 0 ||
      table_ld < table_width) {
    set_error("%s: bad shape rows=%lld heads=%lld kv_heads=%lld pages=%lld seqs=%lld table=[%lld, pitch %lld]", what,
              (long long)rows, (long long)heads, (long long)kv_heads, (long long)pages, (long long)seqs,
              (long long)table_width, (long long)table_ld);
    return KQ_EINVAL;
  }
  // 32-bit row, page and unit counts inside the kernels
  if (rows > (1 << 24) || heads > 1024 || pages * kv_heads >= (1LL << 29) || seqs > (1 << 24) || table_width > (1 << 24) / page_size * 64) {
    set_error("%s: rows=%lld, heads=%lld, pages=%lld, seqs=%lld or table width %lld past the supported range", what,
              (long long)rows, (long long)heads, (long long)pages, (long long)seqs, (long long)table_width);
    return KQ_EINVAL;
  }
  return KQ_OK;
}

template <int D, int NCH, int THREADS, int HPT>
static void launch_append(const AppendArgs& a, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  const int rows = THREADS / (D / 16);
  const int64_t query = ((int64_t)b.rows * ((a.heads + HPT - 1) / HPT) + rows - 1) / rows;
  hipLaunchKernelGGL((kv_append_kernel<D, NCH, THREADS, HPT>), dim3((unsigned)(a.page_units + query)), dim3(THREADS), 0, st, a, c, b,
                     dtype);
}

// A page's tokens in registers: 256 threads hold 4096 elements a pair of chunks.  Pages of
// 8192 go to 512 threads where the rows are few and the chain is what takes the time (64
// single tokens 6.1 us, with 256 threads 6.7; the prompts 43.3 and 41.6), pages of 16384
// to 512 with two pairs (the prompts 42.2 us, with 1024 and one pair 47.9; 6.2 and 7.7), larger ones to 1024
// with two (heads of 256: 49 us, with 512 and four 54).
template <int D, int HPT>
static void pick_append(const AppendArgs& a, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  const int elements = D << c.page_shift;
  if (elements <= 4096)
    launch_append<D, 1, 256, HPT>(a, c, b, dtype, st);
  else if (elements <= 8192)
    launch_append<D, HPT == 4 ? 2 : 1, HPT == 4 ? 256 : 512, HPT>(a, c, b, dtype, st);
  else if (elements <= 16384)
    launch_append<D, 2, 512, HPT>(a, c, b, dtype, st);
  else
    launch_append<D, 2, 1024, HPT>(a, c, b, dtype, st);
}

// Four heads a thread, which share their angles' loads, once that still fills the chip;
// one where the rows are few (the prompts above 41 us with four and 48 with one, the 64
// single tokens with it 8.7 and 6.8).
template <int D>
static void pick_heads(const AppendArgs& a, const KvCache& c, const KvBatch& b, int dtype, hipStream_t st) {
  if ((int64_t)b.rows * a.heads * D >= 4 * 256 * 4096)
    pick_append<D, 4>(a, c, b, dtype, st);
  else
    pick_append<D, 1>(a, c, b, dtype, st);
}

}  // namespace kq

using namespace kq;

extern "C" int kq_kv_rotate_append_at(const int32_t* at, const void* q, int64_t q_ld, int64_t q_hs, const void* k,
                                      int64_t k_ld, int64_t k_hs, const void* v, int64_t v_ld, int64_t v_hs, int dtype,
                                      int64_t rows, int64_t heads, int64_t kv_heads, int64_t dim, uint8_t* k_cache,
                                      uint8_t* v_cache, float* k_scale, float* v_scale, int64_t pages, int64_t page_size,
                                      const int32_t* table, int64_t table_ld, int64_t table_width, const int32_t* cu,
                                      const int32_t* lengths, int64_t seqs, const float* cos_sin, int64_t positions,
                                      int64_t rotary, int interleaved, const void* q_norm, const void* k_norm, float eps,
                                      void* q_out, void* stream) {
  const char* what = at != nullptr ? "kq_kv_rotate_append_at" : "kq_kv_rotate_append";
  int rc = kv_check(what, dtype, rows, heads, kv_heads, dim, page_size, pages, seqs, table_width, table_ld);
  if (rc) return rc;
  // (a table without positions has no address, but turns: every position is past it)
  const bool turns = cos_sin != nullptr || (rotary > 0 && positions == 0);
  if (turns && (rotary < 16 || rotary > dim || rotary % 16 != 0 || positions < 0)) {
    set_error("%s: rotary width must be a multiple of 16 up to the head dim, got %lld", what, (long long)rotary);
    return KQ_EINVAL;
  }
  const uintptr_t align = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache |
                          (uintptr_t)cos_sin | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)q_out;
  if (align % 16 != 0 || (q_ld | q_hs | k_ld | k_hs | v_ld | v_hs) % 8 != 0) {
    set_error("%s: tensors need 16-byte aligned rows and heads", what);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  AppendArgs a{};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_ld = q_ld, a.q_hs = q_hs, a.k_ld = k_ld, a.k_hs = k_hs, a.v_ld = v_ld, a.v_hs = v_hs;
  a.q_out = (uint16_t*)q_out;
  a.cos_sin = cos_sin;
  a.positions = positions;
  a.at = at;
  a.rotary = turns ? (int)rotary : 0;
  a.interleaved = interleaved;
  a.q_norm = (const uint16_t*)q_norm;
  a.k_norm = (const uint16_t*)k_norm;
  a.eps = eps;
  a.heads = (int)heads;
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  // a sequence of n rows touches at most 1 + ceil((n - 1) / page) pages, and a row at most one
  const int64_t units = seqs == 0 || pages == 0 ? 0 : std::min<int64_t>(rows, 2 * seqs + rows / page_size);
  if ((units * kv_heads + rows * heads * dim / 4096 + 1) * 1024 >= (1LL << 32)) {  // threads of one launch
    set_error("%s: %lld rows of %lld heads are past the supported range", what, (long long)rows, (long long)heads);
    return KQ_EINVAL;
  }
  a.page_units = (int)(units * kv_heads);
  const KvCache c{k_cache, v_cache, k_scale, v_scale, pages, (int)kv_heads, shift};
  const KvBatch b{table, cu, lengths, table_ld, (int)seqs, (int)table_width, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  if (dim == 64)
    pick_heads<64>(a, c, b, dtype, st);
  else if (dim == 128)
    pick_heads<128>(a, c, b, dtype, st);
  else
    pick_heads<256>(a, c, b, dtype, st);
  return check_launch(what);
}

extern "C" int kq_kv_rotate_append(const void* q, int64_t q_ld, int64_t q_hs, const void* k, int64_t k_ld, int64_t k_hs,
                                   const void* v, int64_t v_ld, int64_t v_hs, int dtype, int64_t rows, int64_t heads,
                                   int64_t kv_heads, int64_t dim, uint8_t* k_cache, uint8_t* v_cache, float* k_scale,
                                   float* v_scale, int64_t pages, int64_t page_size, const int32_t* table, int64_t table_ld,
                                   int64_t table_width, const int32_t* cu, const int32_t* lengths, int64_t seqs,
                                   const float* cos_sin, int64_t positions, int64_t rotary, int interleaved,
                                   const void* q_norm, const void* k_norm, float eps, void* q_out, void* stream) {
  return kq_kv_rotate_append_at(nullptr, q, q_ld, q_hs, k, k_ld, k_hs, v, v_ld, v_hs, dtype, rows, heads, kv_heads, dim,
                                k_cache, v_cache, k_scale, v_scale, pages, page_size, table, table_ld, table_width, cu,
                                lengths, seqs, cos_sin, positions, rotary, interleaved, q_norm, k_norm, eps, q_out,
                                stream);
}
