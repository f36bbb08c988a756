// Trees of drafted tokens: positions and masks of ancestors from the parents, and the walk
// along the tokens that the model agrees with.
#include "kq_kv.h"

#include <algorithm>

namespace kq {

constexpr int kMostNodes = 1024;

// One workgroup a sequence.  A node's parent lies before it, so a walk upwards ends, and
// meets the words of its mask from the last to the first: each is written once.  What a node
// has above it among the 32 nodes of its own word is found first, with the node that it leaves
// the word to; then each row goes from word to word, which makes 64 steps of 1024.
//
// Latency: bounds, parents, LDS, and a step of some 200 cycles for each level: one tree of 8 rows
// 2.2 us, a chain of 1024 21 (every row from node to node 281).
__global__ void __launch_bounds__(kMostNodes)
draft_tree_kernel(KvBatch batch, const int32_t* __restrict__ parents, int most, int window, uint32_t* __restrict__ mask,
                  int32_t* __restrict__ positions) {
  __shared__ int16_t parent[kMostNodes], leaves_to[kMostNodes];
  __shared__ uint32_t inside[kMostNodes];
  const int tid = (int)threadIdx.x, threads = (int)blockDim.x, words = (most + 31) >> 5;
  auto none = [&](int64_t row, int from_word) {
    for (int w = from_word; w >= 0; --w) mask[row * words + w] = 0;
  };
  // rows of no sequence, dealt to the workgroups (up to 2^32 threads, past what an int counts)
  const int last = batch.seqs > 0 ? min(max(batch.cu[batch.seqs], 0), batch.rows) : 0;
  const int begin = batch.seqs > 0 ? min(max(batch.cu[0], 0), last) : 0;
  for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < begin + batch.rows - last; i += (int64_t)gridDim.x * threads) {
    const int64_t row = i < begin ? i : last + (i - begin);
    none(row, words - 1);
    positions[row] = -1;
  }
  if ((int)blockIdx.x >= batch.seqs) return;
  const KvSeq q = kv_seq(batch, (int)blockIdx.x, 4);
  const int n = min(q.rows, most);
  for (int i = tid; i < n; i += threads) {
    const int p = parents[q.row0 + i];
    parent[i] = (int16_t)(p >= 0 && p < i ? p : -1);
  }
  __syncthreads();
  for (int i = tid; i < n; i += threads) {
    uint32_t bits = 0;
    int at = i;
    do {
      bits |= 1u << (at & 31);
      at = parent[at];
    } while (at >= (i & ~31));
    inside[i] = bits;
    leaves_to[i] = (int16_t)at;
  }
  __syncthreads();
  for (int i = tid; i < q.rows; i += threads) {
    const int64_t row = q.row0 + i;
    int nodes = 0, word = words - 1;
    if (i < n && q.first + i >= 0) {
      for (int at = i; at >= 0; at = leaves_to[at]) {
        uint32_t bits = inside[at];
        const int here = __popc(bits);
        // (the nearest are the highest)
        for (int far = window > 0 ? min(nodes + here - window, here) : 0; far > 0; --far) bits &= bits - 1;
        nodes += here;
        for (; word > at >> 5; --word) mask[row * words + word] = 0;
        mask[row * words + word--] = bits;
      }
    }
    none(row, word);
    const int position = q.first + nodes - 1;
    if (nodes > 0 && position < 0) none(row, words - 1);
    positions[row] = nodes > 0 && position >= 0 ? position : -1;
  }
}

// One workgroup a sequence: the lowest child of each row that has the token that the model says
// there (a minimum in LDS, the same in any order), then the walk from child to child.
//
// Latency, as above: one tree of 8 rows 1.9 us, a chain of 1024 that is kept whole 56 (with a look at
// all rows for each step 236).
template <typename T>
__global__ void __launch_bounds__(256)
draft_accept_kernel(KvBatch batch, const T* __restrict__ tokens, const T* __restrict__ targets,
                    const int32_t* __restrict__ parents, int most, int32_t* __restrict__ kept, int32_t* __restrict__ counts,
                    T* __restrict__ following) {
  __shared__ T target[kMostNodes];
  __shared__ int child[kMostNodes], path[kMostNodes];
  __shared__ int length;
  constexpr int kNone = 0x7fffffff, U = kMostNodes / 256;
  const int s = (int)blockIdx.x, tid = (int)threadIdx.x, threads = (int)blockDim.x;
  const int lo = min(max(batch.cu[s], 0), batch.rows), hi = min(max(batch.cu[s + 1], lo), batch.rows);
  const int n = scalar(min(hi - lo, most));
  T token[U];
  int parent[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = tid + u * threads;
    if (i >= n) break;
    parent[u] = parents[lo + i];
    token[u] = tokens[lo + i];
    target[i] = targets[lo + i];
    child[i] = kNone;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = tid + u * threads;
    if (i >= n) break;
    if (parent[u] >= 0 && parent[u] < i && token[u] == target[parent[u]]) atomicMin(&child[parent[u]], i);
  }
  __syncthreads();
  if (tid == 0) {
    int count = 0;
    for (int at = 0; at < n; at = child[at]) path[count++] = at;
    length = count;
    counts[s] = count;
    following[s] = count > 0 ? target[path[count - 1]] : (T)-1;
  }
  __syncthreads();
  const int count = length;
  for (int i = tid; i < most; i += threads) kept[(int64_t)s * most + i] = i < count ? path[i] : -1;
}

static int check_drafts(const char* what, int64_t rows, int64_t seqs, int64_t most) {
  if (rows < 0 || seqs < 0 || rows > (1 << 24) || seqs >= (1 << 24)) {
    set_error("%s: bad shape rows=%lld seqs=%lld", what, (long long)rows, (long long)seqs);
    return KQ_EINVAL;
  }
  if (most < 1 || most > kMostNodes) {
    set_error("%s: 1 to %d new rows of a sequence are supported, got %lld", what, kMostNodes, (long long)most);
    return KQ_EINVAL;
  }
  return KQ_OK;
}

}  // namespace kq

using namespace kq;

extern "C" int kq_draft_tree(const int32_t* parents, int64_t rows, const int32_t* cu, const int32_t* lengths, int64_t seqs,
                             int64_t most, int64_t window, int32_t* mask, int32_t* positions, void* stream) {
  const char* what = "kq_draft_tree";
  if (int rc = check_drafts(what, rows, seqs, most)) return rc;
  if (window < 0 || window > (1 << 30)) {
    set_error("%s: window %lld", what, (long long)window);
    return KQ_EINVAL;
  }
  if (rows == 0) return KQ_OK;
  const KvBatch b{nullptr, cu, lengths, 0, (int)seqs, 0, (int)rows};
  // (a thread a row, and fewer than 2^32 of them)
  const int64_t threads = std::min<int64_t>((most + 63) / 64 * 64, seqs < (1 << 22) ? kMostNodes : 128);
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)std::max<int64_t>(seqs, 1)), dim3((unsigned)threads), 0, (hipStream_t)stream, b,
                     parents, (int)most, (int)window, (uint32_t*)mask, positions);
  return check_launch(what);
}

extern "C" int kq_draft_accept(const void* tokens, const void* targets, int wide, const int32_t* parents, int64_t rows,
                               const int32_t* cu, int64_t seqs, int64_t most, int32_t* kept, int32_t* counts, void* following,
                               void* stream) {
  const char* what = "kq_draft_accept";
  if (int rc = check_drafts(what, rows, seqs, most)) return rc;
  if (seqs == 0) return KQ_OK;
  const KvBatch b{nullptr, cu, nullptr, 0, (int)seqs, 0, (int)rows};
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)seqs), block((unsigned)std::min<int64_t>((most + 63) / 64 * 64, 256));
  if (wide)
    hipLaunchKernelGGL((draft_accept_kernel<int64_t>), grid, block, 0, st, b, (const int64_t*)tokens,
                       (const int64_t*)targets, parents, (int)most, kept, counts, (int64_t*)following);
  else
    hipLaunchKernelGGL((draft_accept_kernel<int32_t>), grid, block, 0, st, b, (const int32_t*)tokens,
                       (const int32_t*)targets, parents, (int)most, kept, counts, (int32_t*)following);
  return check_launch(what);
}
