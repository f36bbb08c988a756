// Trees of drafted tokens: positions and masks of ancestors from the parents, and the walk
// along the tokens that the model agrees with.
#include "kq_kv.h"

#include <algorithm>

namespace kq {

constexpr int kMostNodes = 1024;

// One workgroup a sequence.  A node's parent lies before it, so a walk upwards ends, and
// meets the words of its mask from the last to the first: each is written once.
//
// Latency: bounds, parents, LDS, and a step of some 100 cycles for each level.
__global__ void __launch_bounds__(256)
draft_tree_kernel(KvBatch batch, const int32_t* __restrict__ parents, int most, int window, uint32_t* __restrict__ mask,
                  int32_t* __restrict__ positions) {
  __shared__ int16_t parent[kMostNodes];
  const int tid = (int)threadIdx.x, words = (most + 31) >> 5;
  auto none = [&](int64_t row, int from_word) {
    for (int w = from_word; w >= 0; --w) mask[row * words + w] = 0;
  };
  // rows of no sequence, dealt to the workgroups
  const int last = batch.seqs > 0 ? min(max(batch.cu[batch.seqs], 0), batch.rows) : 0;
  const int begin = batch.seqs > 0 ? min(max(batch.cu[0], 0), last) : 0;
  for (int i = (int)blockIdx.x * 256 + tid; i < begin + batch.rows - last; i += (int)gridDim.x * 256) {
    const int row = i < begin ? i : last + (i - begin);
    none(row, words - 1);
    positions[row] = -1;
  }
  if ((int)blockIdx.x >= batch.seqs) return;
  const KvSeq q = kv_seq(batch, (int)blockIdx.x, 4);
  const int n = min(q.rows, most);
  for (int i = tid; i < n; i += 256) {
    const int p = parents[q.row0 + i];
    parent[i] = (int16_t)(p >= 0 && p < i ? p : -1);
  }
  __syncthreads();
  for (int i = tid; i < q.rows; i += 256) {
    const int64_t row = q.row0 + i;
    int depth = -1, at = i < n ? i : -1, word = words - 1;
    uint32_t bits = 0;
    // the levels above; whether the row has a token is known when its depth is
    for (; at >= 0; at = parent[at]) {
      ++depth;
      if (window > 0 && depth >= window) continue;
      for (; word > at >> 5; --word, bits = 0) mask[row * words + word] = bits;
      bits |= 1u << (at & 31);
    }
    for (; word >= 0; --word, bits = 0) mask[row * words + word] = bits;
    const int position = q.first + depth;
    const bool there = i < n && q.first + i >= 0 && position >= 0;
    if (!there) none(row, words - 1);
    positions[row] = there ? position : -1;
  }
}

// One wave a sequence: its rows' parents and tokens in LDS, then step by step the lowest
// child that has the token that the model says, 64 rows at a look.
template <typename T>
__global__ void __launch_bounds__(64)
draft_accept_kernel(KvBatch batch, const T* __restrict__ tokens, const T* __restrict__ targets,
                    const int32_t* __restrict__ parents, int most, int32_t* __restrict__ kept, int32_t* __restrict__ counts,
                    T* __restrict__ following) {
  __shared__ T token[kMostNodes], target[kMostNodes];
  __shared__ int16_t parent[kMostNodes];
  const int s = (int)blockIdx.x, lane = lane_id();
  const int lo = min(max(batch.cu[s], 0), batch.rows), hi = min(max(batch.cu[s + 1], lo), batch.rows);
  const int n = scalar(min(hi - lo, most));
  for (int i = lane; i < n; i += 64) {
    const int p = parents[lo + i];
    parent[i] = (int16_t)(p >= 0 && p < i ? p : -1);
    token[i] = tokens[lo + i];
    target[i] = targets[lo + i];
  }
  __syncthreads();
  int count = 0, at = n > 0 ? 0 : -1;
  T said = (T)-1;
  int32_t* out = kept + (int64_t)s * most;
  while (at >= 0) {
    if (lane == 0) out[count] = at;
    ++count;
    said = target[at];
    int next = -1;
    for (int base = (at + 1) & ~63; base < n && next < 0; base += 64) {
      const int i = base + lane;
      const uint64_t right = __ballot(i < n && parent[i < n ? i : 0] == at && token[i < n ? i : 0] == said);
      if (right != 0) next = base + (int)__builtin_ctzll(right);
    }
    at = scalar(next);
  }
  for (int i = count + lane; i < most; i += 64) out[i] = -1;
  if (lane == 0) {
    counts[s] = count;
    following[s] = said;
  }
}

static int check_drafts(const char* what, int64_t rows, int64_t seqs, int64_t most) {
  if (rows < 0 || seqs < 0 || rows > (1 << 24) || seqs > (1 << 24)) {
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
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)std::max<int64_t>(seqs, 1)), dim3(256), 0, (hipStream_t)stream, b, parents,
                     (int)most, (int)window, (uint32_t*)mask, positions);
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
  if (wide)
    hipLaunchKernelGGL((draft_accept_kernel<int64_t>), dim3((unsigned)seqs), dim3(64), 0, st, b, (const int64_t*)tokens,
                       (const int64_t*)targets, parents, (int)most, kept, counts, (int64_t*)following);
  else
    hipLaunchKernelGGL((draft_accept_kernel<int32_t>), dim3((unsigned)seqs), dim3(64), 0, st, b, (const int32_t*)tokens,
                       (const int32_t*)targets, parents, (int)most, kept, counts, (int32_t*)following);
  return check_launch(what);
}
