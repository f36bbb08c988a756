// Pages of the paged e4m3 cache that sequences share, and tokens that move in it: copies
// of pages, forks of sequences, and the move of kept drafts behind their context.
//
// A page is the same in every layer, so a launch takes all layers' caches (up to
// kMostLayers; their addresses are kernel arguments, and more take more launches).
#include "kq_kv.h"

#include <algorithm>

namespace kq {

constexpr int kMostLayers = 64;

struct KvLayer {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
};
struct KvLayers {
  KvLayer at[kMostLayers];
  int64_t pages;
  int kv_heads, page_shift, dim_shift;  // head dim: 1 << dim_shift
};

KQ_DEV bool is_page(int p, int64_t pages) { return p >= 0 && p < pages; }

// ---------------------------------------------------------------- copies
// Bytes of `src` to `dst` by a workgroup or a wave, both 16-byte aligned, `bytes` a multiple
// of 16: four chunks a thread in flight.
template <int THREADS>
KQ_DEV void copy_bytes(const uint8_t* src, uint8_t* dst, int bytes) {
  constexpr int STEP = 16 * THREADS;
  for (int at = (int)(threadIdx.x % THREADS) * 16; at < bytes; at += 4 * STEP) {
    u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * STEP < bytes) w[i] = *(const u32x4*)(src + at + i * STEP);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * STEP < bytes) *(u32x4*)(dst + at + i * STEP) = w[i];
  }
}

constexpr int kCopyBytes = 16384;  // of a page, by one workgroup

// One workgroup: 16 KiB of a pair's page, of keys or values of one layer.  HBM: 512 pages of 64
// tokens, 8 heads of 128, in 16 layers (2.1 GB to and fro) in 405 us, 5.3 TB/s; four pages in 32
// layers 6.1 us (from the caches of the chip).
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(KvLayers c, const int32_t* __restrict__ sources, const int32_t* __restrict__ targets, int parts) {
  const int pair = (int)blockIdx.x / parts, part = (int)blockIdx.x - pair * parts;
  const int from = sources[pair], to = targets[pair];
  if (!is_page(from, c.pages) || !is_page(to, c.pages) || from == to) return;
  const KvLayer& layer = c.at[blockIdx.z];
  const bool values = blockIdx.y != 0;
  uint8_t* codes = values ? layer.v : layer.k;
  const int64_t bytes = (int64_t)c.kv_heads << (c.page_shift + c.dim_shift);
  const int64_t at = (int64_t)part * kCopyBytes;
  copy_bytes<256>(codes + from * bytes + at, codes + to * bytes + at, (int)min((int64_t)kCopyBytes, bytes - at));
  if (part == 0) {
    float* scales = values ? layer.v_scale : layer.k_scale;
    for (int h = (int)threadIdx.x; h < c.kv_heads; h += 256)
      scales[(int64_t)to * c.kv_heads + h] = scales[(int64_t)from * c.kv_heads + h];
  }
}

// ---------------------------------------------------------------- forks
struct ForkArgs {
  const int32_t* table;  // [seqs][width], row pitch table_ld
  int64_t table_ld;
  const int32_t* lengths;
  const int32_t* parents;
  int32_t* holders;  // [pages]
  int32_t* new_table;  // [rows][width]
  int32_t* new_lengths;
  int32_t* missing;
  int32_t* eldest;  // scratch: [seqs], the first new row of each old one
  int32_t* free;    // [rows * slots], the lowest free pages
  int32_t* copies;  // [rows][2], the pages that a half-filled one is copied from and to (-1: none)
  int seqs, rows, width;
  int room, slots;  // slots: pages that a row's next `room` tokens can touch
};

KQ_DEV int fork_parent(const ForkArgs& a, int j) {
  const int p = a.parents[j];
  return p >= 0 && p < a.seqs ? p : -1;
}
// First slot behind the pages of `length` tokens and `room` more.
KQ_DEV int64_t slots_end(int length, int room, int shift) { return ((int64_t)length + room + (1 << shift) - 1) >> shift; }

// Prefix sums over a workgroup of 1024: `mine` of each wave is uniform.
struct WaveSums {
  int before, all;
};
KQ_DEV WaveSums wave_sums(int mine, int* lds) {
  __syncthreads();
  if (lane_id() == 0) lds[wave_id()] = mine;
  __syncthreads();
  WaveSums s{0, 0};
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const int n = lds[w];
    s.before += w < wave_id() ? n : 0;
    s.all += n;
  }
  return s;
}

// One workgroup: which pages are free, and which rows get them.  Pages are numbered in the
// order of rows and slots and free pages in their own, so that the result does not depend
// on any order of threads.  Only reads the holders, which the second launch changes.
//
// Latency, some five trips to memory and as many barriers: 4.4 us for 8 new rows, 5 for 128.
// One workgroup needs no order among several, but reads 4096 holders a step: where the first free
// pages are the last of 65536, a whole call takes 24 us in a graph (9 with free pages in front), of a million
// 298 (231 with eight loads a thread, which cost 0.5 us in small pools).
__global__ void __launch_bounds__(1024) kv_fork_plan_kernel(ForkArgs a, int64_t pages, int shift) {
  __shared__ int lds[16];
  const int tid = (int)threadIdx.x, wave = scalar(wave_id());
  for (int s = tid; s < a.seqs; s += 1024) a.eldest[s] = 0x7fffffff;
  const int items = a.rows * a.slots;
  int found = 0;
  constexpr int K = 4, SPAN = 1024 * K;
  for (int64_t base = 0; base < pages && found < items; base += SPAN) {
    uint64_t free[K];
    int n = 0, held[K];  // (all on their way at once)
    const int64_t first = base + wave * 64 * K + lane_id();
#pragma unroll
    for (int k = 0; k < K; ++k) held[k] = a.holders[min(first + 64 * k, pages - 1)];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      free[k] = __ballot(first + 64 * k < pages && held[k] == 0);
      n += __popcll(free[k]);
    }
    const WaveSums sums = wave_sums(n, lds);
    int at = found + sums.before;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int mine = at + __popcll(free[k] & ((1ull << lane_id()) - 1));
      if ((free[k] >> lane_id() & 1) && mine < items) a.free[mine] = (int)base + (wave * K + k) * 64 + lane_id();
      at += __popcll(free[k]);
    }
    found += sums.all;
  }
  found = min(found, items);
  __syncthreads();  // (eldest is cleared, the free pages are listed)
  for (int j = tid; j < a.rows; j += 1024) {
    const int p = fork_parent(a, j);
    if (p >= 0) atomicMin(&a.eldest[p], j);
    a.new_lengths[j] = p >= 0 ? max(a.lengths[p], 0) : 0;
    a.copies[2 * j] = -1;
  }
  __syncthreads();
  int given = 0;
  for (int base = 0; base < items; base += 1024) {
    const int item = base + tid, j = item / a.slots, u = item - j * a.slots;
    const int p = item < items ? fork_parent(a, j) : -1;
    bool need = false;
    int old = -1, length = 0, slot = 0;
    if (p >= 0) {
      length = max(a.lengths[p], 0);
      slot = (length >> shift) + u;
      if (slot < a.width && slot < slots_end(length, a.room, shift)) {
        old = a.table[p * a.table_ld + slot];
        if (!is_page(old, pages)) old = -1;
        need = !(old >= 0 && a.eldest[p] == j && a.holders[old] == 1);
        if (!need) a.new_table[(int64_t)j * a.width + slot] = old;
      }
    }
    const uint64_t needs = __ballot(need);
    const WaveSums sums = wave_sums(__popcll(needs), lds);
    if (need) {
      const int rank = given + sums.before + __popcll(needs & ((1ull << lane_id()) - 1));
      const int page = rank < found ? a.free[rank] : -1;
      a.new_table[(int64_t)j * a.width + slot] = page;
      if (u == 0 && old >= 0 && page >= 0 && (length & ((1 << shift) - 1)) != 0) {
        a.copies[2 * j] = old;
        a.copies[2 * j + 1] = page;
      }
    }
    given += sums.all;
  }
  if (tid == 0) *a.missing = max(given - found, 0);
}

// The first `tables` workgroups: the other entries of the new table, and the holders (sums
// of whole numbers, in any order).  The others: half-filled pages, keys or values of one layer each.
// Latency for few rows (8 in 32 layers 5.8 us), then HBM: 128 rows in 16 layers 12.9 us.  These, and the
// plan's above, are one kernel's times under the profiler; both launches in a graph take 9.0 and 20.
__global__ void __launch_bounds__(256) kv_fork_kernel(ForkArgs a, KvLayers c, int tables, int layers) {
  const int shift = c.page_shift;
  if ((int)blockIdx.x < tables) {
    const int64_t entry = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(entry / a.width), slot = (int)(entry - (int64_t)row * a.width);
    if (row < a.rows) {
      const int p = fork_parent(a, row);
      int page = -1;
      if (p >= 0) {
        const int length = max(a.lengths[p], 0);
        const int old_ = a.table[p * a.table_ld + slot], old = is_page(old_, c.pages) ? old_ : -1;
        const bool eldest = a.eldest[p] == row;
        // with no room a half-filled page is shared as well
        const int64_t shared = a.room > 0 ? length >> shift : slots_end(length, 0, shift);
        if (slot < shared) {
          page = old;
          if (old >= 0 && !eldest) atomicAdd(&a.holders[old], 1);
        } else {
          if (slot < slots_end(length, a.room, shift)) page = a.new_table[entry];
          if (page != old) {  // (the eldest row takes over what its parent holds)
            if (page >= 0) atomicAdd(&a.holders[page], 1);
            if (old >= 0 && eldest) atomicAdd(&a.holders[old], -1);
          } else if (old >= 0 && !eldest) {
            atomicAdd(&a.holders[old], 1);
          }
        }
      }
      a.new_table[entry] = page;
    }
    if (row < a.seqs && a.eldest[row] == 0x7fffffff) {  // nobody goes on from it
      const int old = a.table[row * a.table_ld + slot];
      if (is_page(old, c.pages)) atomicAdd(&a.holders[old], -1);
    }
    return;
  }
  // (row, layer, keys or values); a wave copies every fourth head's tokens
  int unit = (int)blockIdx.x - tables;
  const int values = unit & 1;
  unit >>= 1;
  const int row = unit / layers;
  const int from = a.copies[2 * row];
  if (from < 0) return;
  const int to = a.copies[2 * row + 1];
  const KvLayer& layer = c.at[unit - row * layers];
  const int bytes = (a.new_lengths[row] & ((1 << shift) - 1)) << c.dim_shift;
  uint8_t* codes = values ? layer.v : layer.k;
  float* scales = values ? layer.v_scale : layer.k_scale;
  const int64_t src = (int64_t)from * c.kv_heads, dst = (int64_t)to * c.kv_heads;
  for (int h = (int)threadIdx.x; h < c.kv_heads; h += 256) scales[dst + h] = scales[src + h];
  for (int h = scalar(wave_id()); h < c.kv_heads; h += 4)
    copy_bytes<64>(codes + ((src + h) << (shift + c.dim_shift)), codes + ((dst + h) << (shift + c.dim_shift)), bytes);
}

// ------------------------------------------------- kept tokens behind their context
struct KeepArgs {
  const int32_t* kept;  // [seqs][most]
  const int32_t* counts;
  int32_t* new_lengths;
  int most;
};

constexpr int kMostNodes = 1024;
constexpr int kScales = 1024;  // of a sequence's pages that a workgroup holds in LDS

// One workgroup a sequence and layer.  Token first + kept[i] goes to slot first + i, i in
// steps of what the workgroup's threads hold: a step's codes are all in registers before
// one is written, and what later steps read lies behind what this one writes (kept[i] >= i).
//
// A page's new scale is the largest of its tokens' old ones, so code * (old / new) is
// rounded once, and is exact between powers of two but for codes that fall below e4m3's
// normal range.  Which old pages a page's tokens come from is found once for all heads
// (`sources`, a bit for each page behind the first); scales are held in LDS where they fit (64
// pages of 8 heads), else read by those who need them, and written last.
//
// Latency: bounds, kept tokens and pages, checks and scales, codes, one after the other.  One
// sequence in 32 layers 6.3 us, 64 in 28 layers 9.3, where bytes alone would take 2.4 (with scales
// read where they are needed, four times in turn, 7.2 and 10.2), in a graph.
template <int DS>
__global__ void __launch_bounds__(256) kv_keep_kernel(KeepArgs a, KvLayers c, KvBatch batch) {
  constexpr int CH = 1 << (DS - 4);  // 16-byte chunks of a token
  constexpr int U = 4;               // chunks a thread holds
  constexpr int SPAN = kMostNodes / 16 + 1;
  __shared__ int kept[kMostNodes];
  __shared__ int pages[SPAN];
  __shared__ uint32_t sources[SPAN][3];
  __shared__ float olds[kScales], growns[kScales];  // [page][head][keys, values], where they fit
  __shared__ int stop;
  const int tid = (int)threadIdx.x, s = (int)blockIdx.x, shift = c.page_shift, in_page = (1 << shift) - 1;
  const KvSeq q = kv_seq_uniform(batch, s, shift);
  const int n = min(q.rows, kMostNodes), first = q.first;
  const int count = first < 0 ? 0 : min(max(a.counts[s], 0), a.most);
  const int slot0 = max(first, 0) >> shift;
  const int32_t* table = batch.table + (int64_t)s * batch.table_ld;
  if (tid == 0) stop = count;
  for (int i = tid; i < count; i += 256) kept[i] = a.kept[(int64_t)s * a.most + i];
  for (int i = tid; i < SPAN; i += 256) {
    const int p = slot0 + i < batch.table_width ? table[slot0 + i] : -1;
    pages[i] = is_page(p, c.pages) ? p : -1;
    sources[i][0] = sources[i][1] = sources[i][2] = 0;
  }
  __syncthreads();
  auto slot_of = [&](int node) { return ((first + node) >> shift) - slot0; };
  const KvLayer& layer = c.at[blockIdx.y];
  const int heads = c.kv_heads, span = count > 0 && n > 0 ? slot_of(n - 1) + 1 : 0;
  const bool fits = (int64_t)span * 2 * heads <= kScales;
  if (fits)
    for (int i = tid; i < span * 2 * heads; i += 256) {
      const int page = pages[i / (2 * heads)], u = i % (2 * heads);
      olds[i] = page < 0 ? 0.0f : (u & 1 ? layer.v_scale : layer.k_scale)[(int64_t)page * heads + (u >> 1)];
    }
  for (int i = tid; i < count; i += 256) {
    const int node = kept[i];
    const bool good = node >= 0 && node < n && (i == 0 || kept[i - 1] < node) && i < n && pages[slot_of(node)] >= 0 && pages[slot_of(i)] >= 0;
    if (!good) atomicMin(&stop, i);
  }
  __syncthreads();
  const int keep = scalar(stop);
  if (tid == 0 && blockIdx.y == 0) a.new_lengths[s] = max(first, 0) + keep;
  if (keep == 0) return;
  for (int i = tid; i < keep; i += 256) {
    const int from = slot_of(kept[i]);
    atomicOr(&sources[slot_of(i)][from >> 5], 1u << (from & 31));
  }
  const int before = first & in_page, last_slot = slot_of(keep - 1);
  if (tid == 0 && before > 0) atomicOr(&sources[0][0], 1u);  // (its own earlier tokens)
  __syncthreads();

  // u: 2 head, or 2 head + 1 for values.  The scale that a page has, and the one it gets.
  auto old_of = [&](int slot, int u) {
    if (fits) return olds[slot * 2 * heads + u];
    return (u & 1 ? layer.v_scale : layer.k_scale)[(int64_t)pages[slot] * heads + (u >> 1)];
  };
  auto largest = [&](int to, int u) {
    float m = 0.0f;
#pragma unroll
    for (int w = 0; w < 3; ++w)
      for (uint32_t bits = sources[to][w]; bits != 0; bits &= bits - 1) m = fmaxf(m, old_of(32 * w + __builtin_ctz(bits), u));
    return m;
  };
  if (fits) {
    for (int i = tid; i < (last_slot + 1) * 2 * heads; i += 256) growns[i] = largest(i / (2 * heads), i % (2 * heads));
    __syncthreads();
  }
  auto grown_of = [&](int slot, int u) { return fits ? growns[slot * 2 * heads + u] : largest(slot, u); };
  // earlier tokens of the first page, where its scale grows
  if (before > 0) {
    for (int u = wave_id(); u < 2 * heads; u += 4) {
      const int64_t tile = (int64_t)pages[0] * heads + (u >> 1);
      const float old = old_of(0, u), grown = grown_of(0, u);
      if (old == grown) continue;
      uint8_t* codes = (u & 1 ? layer.v : layer.k) + (tile << (shift + DS));
      for (int i = lane_id(); i < before * CH; i += 64) *(u32x4*)(codes + 16 * i) = move16(*(const u32x4*)(codes + 16 * i), old / grown);
    }
  }
  const int units = keep * 2 * heads * CH;  // by tokens, then heads, keys and values, chunks
  for (int base = 0; base < units; base += 256 * U) {
    u32x4 w[U];
    uint8_t* dst[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      dst[k] = nullptr;
      const int unit = base + k * 256 + tid;
      if (unit >= units) continue;
      const int chunk = unit & (CH - 1), which = (unit >> (DS - 4)) & 1, rest = unit >> (DS - 3);
      const int i = rest / heads, head = rest - i * heads;
      const int node = kept[i], from = slot_of(node), to = slot_of(i);
      const int64_t src = (int64_t)pages[from] * heads + head, to_tile = (int64_t)pages[to] * heads + head;
      const float old = old_of(from, 2 * head + which), grown = grown_of(to, 2 * head + which);
      if (node == i && old == grown) continue;
      uint8_t* codes = which ? layer.v : layer.k;
      w[k] = *(const u32x4*)(codes + (src << (shift + DS)) + ((((first + node) & in_page) << DS) + 16 * chunk));
      if (old != grown) w[k] = move16(w[k], old / grown);
      dst[k] = codes + (to_tile << (shift + DS)) + ((((first + i) & in_page) << DS) + 16 * chunk);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (codes and scales are here before any is written)
    __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (dst[k] != nullptr) *(u32x4*)dst[k] = w[k];
    __syncthreads();
  }
  // scales, a head's by one thread and page after page: a page's comes from pages at or behind it
  for (int u = tid; u < 2 * heads; u += 256) {
    float* scales = u & 1 ? layer.v_scale : layer.k_scale;
    for (int to = 0; to <= last_slot; ++to) {
      const float grown = grown_of(to, u);
      scales[(int64_t)pages[to] * heads + (u >> 1)] = grown;
    }
  }
}

static int check_layers(const char* what, const uint64_t* caches, int64_t layers, int64_t pages, int64_t kv_heads,
                        int64_t page_size, int64_t dim, int64_t seqs, int64_t table_width, int64_t table_ld) {
  if (int rc = kv_check(what, KQ_DTYPE_F16, 0, kv_heads, kv_heads, dim, page_size, pages, seqs, table_width, table_ld)) return rc;
  if (layers < 1 || layers > 4096 || caches == nullptr) {
    set_error("%s: %lld caches, 1 to 4096 are supported", what, (long long)layers);
    return KQ_EINVAL;
  }
  for (int64_t i = 0; i < layers; ++i)
    if ((caches[4 * i] | caches[4 * i + 1]) % 16 != 0) {
      set_error("%s: cache codes must be 16-byte aligned", what);
      return KQ_EINVAL;
    }
  return KQ_OK;
}

// Caches [begin, begin + kMostLayers) of a call.
static KvLayers some_layers(const uint64_t* caches, int64_t layers, int64_t begin, int64_t pages, int64_t kv_heads,
                            int64_t page_size, int64_t dim) {
  KvLayers c{};
  for (int64_t i = begin; i < std::min(layers, begin + kMostLayers); ++i)
    c.at[i - begin] = KvLayer{(uint8_t*)caches[4 * i], (uint8_t*)caches[4 * i + 1], (float*)caches[4 * i + 2], (float*)caches[4 * i + 3]};
  c.pages = pages;
  c.kv_heads = (int)kv_heads;
  c.page_shift = 4;
  while ((1 << c.page_shift) < page_size) ++c.page_shift;
  c.dim_shift = dim == 64 ? 6 : dim == 128 ? 7 : 8;
  return c;
}

// Pages that `room` tokens can touch.
static int64_t fork_slots(int64_t page_size, int64_t room) { return room == 0 ? 0 : (room + page_size - 2) / page_size + 1; }

}  // namespace kq

using namespace kq;

extern "C" int kq_kv_copy_pages(const uint64_t* caches, int64_t layers, int64_t pages, int64_t kv_heads, int64_t page_size,
                                int64_t dim, const int32_t* sources, const int32_t* targets, int64_t count, void* stream) {
  const char* what = "kq_kv_copy_pages";
  if (int rc = check_layers(what, caches, layers, pages, kv_heads, page_size, dim, 0, 0, 0)) return rc;
  const int64_t parts = (kv_heads * page_size * dim + kCopyBytes - 1) / kCopyBytes;
  if (count < 0 || count * parts >= (1LL << 24)) {
    set_error("%s: %lld pairs of pages are past the supported range", what, (long long)count);
    return KQ_EINVAL;
  }
  if (count == 0 || pages == 0) return KQ_OK;
  for (int64_t begin = 0; begin < layers; begin += kMostLayers) {
    const KvLayers c = some_layers(caches, layers, begin, pages, kv_heads, page_size, dim);
    const unsigned z = (unsigned)std::min<int64_t>(kMostLayers, layers - begin);
    hipLaunchKernelGGL(kv_copy_pages_kernel, dim3((unsigned)(count * parts), 2, z), dim3(256), 0, (hipStream_t)stream, c, sources,
                       targets, (int)parts);
  }
  return check_launch(what);
}

extern "C" size_t kq_kv_fork_workspace_size(int64_t seqs, int64_t rows, int64_t table_width, int64_t page_size, int64_t room) {
  if (seqs < 0 || rows < 0 || table_width < 0 || page_size < 1 || room < 0) return 0;
  const int64_t slots = std::min(fork_slots(page_size, room), table_width);
  return sizeof(int32_t) * (size_t)(seqs + rows * slots + 2 * rows);
}

extern "C" int kq_kv_fork_sequences(const uint64_t* caches, int64_t layers, int64_t pages, int64_t kv_heads, int64_t page_size,
                                    int64_t dim, int32_t* holders, const int32_t* table, int64_t table_ld, int64_t table_width,
                                    const int32_t* lengths, int64_t seqs, const int32_t* parents, int64_t rows, int64_t room,
                                    int32_t* new_table, int32_t* new_lengths, int32_t* missing, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* what = "kq_kv_fork_sequences";
  if (int rc = check_layers(what, caches, layers, pages, kv_heads, page_size, dim, seqs, table_width, table_ld)) return rc;
  const int64_t slots = std::min(fork_slots(page_size, room), table_width);
  const int64_t tables = (std::max(seqs, rows) * table_width + 255) / 256;
  if (rows < 0 || room < 0 || room > (1 << 24) || rows * slots >= (1LL << 30) || tables >= (1LL << 23) ||
      rows * 2 * std::min<int64_t>(layers, kMostLayers) >= (1LL << 23)) {
    set_error("%s: %lld rows of %lld pages, room for %lld tokens are past the supported range", what, (long long)rows,
              (long long)table_width, (long long)room);
    return KQ_EINVAL;
  }
  if (workspace_bytes < kq_kv_fork_workspace_size(seqs, rows, table_width, page_size, room)) {
    set_error("%s: workspace of %zu bytes is too small", what, workspace_bytes);
    return KQ_EWORKSPACE;
  }
  ForkArgs a{};
  a.table = table, a.table_ld = table_ld, a.lengths = lengths, a.parents = parents, a.holders = holders;
  a.new_table = new_table, a.new_lengths = new_lengths, a.missing = missing;
  a.eldest = (int32_t*)workspace;
  a.free = a.eldest + seqs;
  a.copies = a.free + rows * slots;
  a.seqs = (int)seqs, a.rows = (int)rows, a.width = (int)table_width, a.room = (int)room, a.slots = (int)slots;
  hipStream_t st = (hipStream_t)stream;
  for (int64_t begin = 0; begin < layers; begin += kMostLayers) {
    const KvLayers c = some_layers(caches, layers, begin, pages, kv_heads, page_size, dim);
    const int n = (int)std::min<int64_t>(kMostLayers, layers - begin);
    const int64_t own = begin == 0 ? tables : 0, blocks = own + (slots > 0 ? rows * 2 * n : 0);
    if (begin == 0) hipLaunchKernelGGL(kv_fork_plan_kernel, dim3(1), dim3(1024), 0, st, a, pages, c.page_shift);
    if (blocks > 0) hipLaunchKernelGGL(kv_fork_kernel, dim3((unsigned)blocks), dim3(256), 0, st, a, c, (int)own, n);
  }
  return check_launch(what);
}

extern "C" int kq_kv_keep_tokens(const uint64_t* caches, int64_t layers, int64_t pages, int64_t kv_heads, int64_t page_size,
                                 int64_t dim, const int32_t* table, int64_t table_ld, int64_t table_width, const int32_t* cu,
                                 const int32_t* lengths, int64_t seqs, const int32_t* kept, int64_t most, const int32_t* counts,
                                 int32_t* new_lengths, void* stream) {
  const char* what = "kq_kv_keep_tokens";
  if (int rc = check_layers(what, caches, layers, pages, kv_heads, page_size, dim, seqs, table_width, table_ld)) return rc;
  if (most < 0 || most > kMostNodes || seqs * std::min<int64_t>(layers, kMostLayers) >= (1LL << 24)) {
    set_error("%s: %lld sequences of up to %lld kept tokens are past the supported range", what, (long long)seqs, (long long)most);
    return KQ_EINVAL;
  }
  if (seqs == 0) return KQ_OK;
  const KeepArgs a{kept, counts, new_lengths, (int)most};
  const KvBatch b{table, cu, lengths, table_ld, (int)seqs, (int)table_width, 1 << 24};
  hipStream_t st = (hipStream_t)stream;
  for (int64_t begin = 0; begin < layers; begin += kMostLayers) {
    const KvLayers c = some_layers(caches, layers, begin, pages, kv_heads, page_size, dim);
    const dim3 grid((unsigned)seqs, (unsigned)std::min<int64_t>(kMostLayers, layers - begin));
    if (dim == 64)
      hipLaunchKernelGGL((kv_keep_kernel<6>), grid, dim3(256), 0, st, a, c, b);
    else if (dim == 128)
      hipLaunchKernelGGL((kv_keep_kernel<7>), grid, dim3(256), 0, st, a, c, b);
    else
      hipLaunchKernelGGL((kv_keep_kernel<8>), grid, dim3(256), 0, st, a, c, b);
  }
  return check_launch(what);
}
