// The accepted path of a draft tree (fta_accept_path, include/fta.h).
//
// One workgroup per sequence. In parallel over the nodes: node i matches if its token is what the model picked
// after its parent; the lowest matching child of every parent is kept with an integer minimum in LDS (the same
// result in any order). Then the first wave follows root -> first[root] -> ... through LDS, the walk the same in all
// of its lanes, and lane k keeps the k-th node. Parents precede children, so the walk ends. What bounds it: launch
// latency, and on long paths the walk, one LDS round trip per accepted node: 2.2 us for a tree of 26 nodes, 5.0 us for 256
// of 256, the kernel alone.
#include <hip/hip_runtime.h>

#include "fta_device.h"

namespace fta {
namespace {

constexpr int kMaxTree = 16384;   // nodes whose `first` entries fit 64 KB of LDS

struct AcceptParams {
  const void* tokens;
  const void* targets;
  const void* parents;
  int32_t* idx;
  void* len;
  void* next;
  int32_t q_len, max_accept, token_is_i64, target_is_i64, parent_is_i64, len_is_i64;
  int64_t token_stride[2], target_stride[2], parent_stride[2];
};

__device__ __forceinline__ int64_t load_int(const void* base, int is_i64, int64_t at) {
  return is_i64 ? static_cast<const int64_t*>(base)[at] : static_cast<int64_t>(static_cast<const int32_t*>(base)[at]);
}

__global__ void __launch_bounds__(256) accept_path_kernel(const AcceptParams p) {
  FTA_DYNAMIC_LDS(smem);
  int* first = reinterpret_cast<int*>(smem);   // [q_len]: lowest matching child of a node, q_len = none
  const int b = blockIdx.x, n = p.q_len, threads = blockDim.x;
  for (int i = threadIdx.x; i < n; i += threads) first[i] = n;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += threads) {
    const int64_t parent = load_int(p.parents, p.parent_is_i64, b * p.parent_stride[0] + i * p.parent_stride[1]);
    if (parent < 0 || parent >= i) continue;
    const int64_t token = load_int(p.tokens, p.token_is_i64, b * p.token_stride[0] + i * p.token_stride[1]);
    const int64_t target = load_int(p.targets, p.target_is_i64, b * p.target_stride[0] + parent * p.target_stride[1]);
    if (token == target) atomicMin(&first[parent], i);
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  int32_t* out = p.idx + static_cast<int64_t>(b) * p.max_accept;
  const int lane = threadIdx.x;
  int node = 0, last = 0, count = 0;   // the walk is the same in every lane
  for (int base = 0; base < p.max_accept; base += 64) {
    int mine = 0;
    for (int k = 0; k < 64 && node < n && count < p.max_accept; ++k) {
      last = node;
      ++count;
      if (lane == k) mine = node;
      node = first[node];
    }
    if (base + lane < p.max_accept) out[base + lane] = mine;
  }
  if (lane == 0) {
    if (p.len_is_i64) static_cast<int64_t*>(p.len)[b] = count; else static_cast<int32_t*>(p.len)[b] = count;
    const int64_t token = load_int(p.targets, p.target_is_i64, b * p.target_stride[0] + last * p.target_stride[1]);
    if (p.target_is_i64) static_cast<int64_t*>(p.next)[b] = token; else static_cast<int32_t*>(p.next)[b] = static_cast<int32_t>(token);
  }
}

}  // namespace
}  // namespace fta

extern "C" int fta_accept_path(const fta_accept_args* args, void* hip_stream) {
  using namespace fta;
  if (!args) return FTA_ERR_NULL_POINTER;
  const fta_accept_args& a = *args;
  if (!a.tree_tokens || !a.target_tokens || !a.parents || !a.accept_idx || !a.accept_len || !a.next_token) return FTA_ERR_NULL_POINTER;
  for (int32_t t : {a.token_dtype, a.target_dtype, a.parent_dtype, a.len_dtype})
    if (t != FTA_I32 && t != FTA_I64) return FTA_ERR_DTYPE;
  if (a.bsz <= 0 || a.q_len <= 0 || a.max_accept <= 0) return FTA_ERR_SHAPE;
  if (a.q_len > kMaxTree || a.max_accept > 1 << 30) return FTA_ERR_UNSUPPORTED;   // (the walk's counter is 32 bits)
  for (int i = 0; i < 2; ++i)
    if (a.token_stride[i] < 0 || a.target_stride[i] < 0 || a.parent_stride[i] < 0) return FTA_ERR_STRIDE;
  AcceptParams p{};
  p.tokens = a.tree_tokens; p.targets = a.target_tokens; p.parents = a.parents;
  p.idx = a.accept_idx; p.len = a.accept_len; p.next = a.next_token;
  p.q_len = a.q_len; p.max_accept = a.max_accept;
  p.token_is_i64 = a.token_dtype == FTA_I64; p.target_is_i64 = a.target_dtype == FTA_I64;
  p.parent_is_i64 = a.parent_dtype == FTA_I64; p.len_is_i64 = a.len_dtype == FTA_I64;
  for (int i = 0; i < 2; ++i) {
    p.token_stride[i] = a.token_stride[i]; p.target_stride[i] = a.target_stride[i]; p.parent_stride[i] = a.parent_stride[i];
  }
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
  return launch_checked(accept_path_kernel, dim3(static_cast<unsigned>(a.bsz)), dim3(a.q_len <= 64 ? 64 : 256),
                        static_cast<unsigned>(a.q_len * sizeof(int)), static_cast<hipStream_t>(hip_stream), p);
}
