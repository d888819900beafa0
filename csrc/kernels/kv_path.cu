// Keeps the accepted path of a drafted tree in the paged KV cache.
//
// A tree's node i has its K/V rows at position base + i while it is verified.
// Once a path 0 = p_0 < p_1 < ... is accepted, node p_i is the sequence's token
// at position base + i, so rows base + p_i move to base + i in every layer.
// Since p is increasing, p_i >= i: a thread that moves one element column of
// one (layer, tensor, KV head) in order i = 1, 2, ... never overwrites a row
// it has still to read, in batches of UN loads in flight: rows written before a
// batch lie below its first, so below its sources.
//
// Bound by the moved bytes where they are many (32 layers of 32 heads of 128,
// 8 lanes, 85 MB read and written: 20 us in the kernel, 4.2 TB/s of rows of
// 1 KB; CTAs that take several tensors in turn: 20 us as well) and by the
// chain path -> page -> row -> store where they are few (80 layers of 8 heads,
// one lane: 7.8 us; one load in flight: 9.5).
#include "../common/tree.h"
#include "common.cuh"

namespace kp {

constexpr int NT = 128, UN = 4;

// grid (columns of 2 int64 over n_kv * dh / NT, tensors, lanes)
__global__ void __launch_bounds__(NT) k_keep_path(int64_t* const* __restrict__ planes, int n_pages, int n_kv, int dh,
                                                  const int* __restrict__ pt, int64_t pt_stride, int width,
                                                  const int* __restrict__ base, const int* __restrict__ path,
                                                  const int* __restrict__ n_path, int n, int* __restrict__ err) {
  pdl_wait_dep();
  pdl_allow_next();
  const int lane = blockIdx.z;
  path += (size_t)lane * n;
  pt += lane * pt_stride;
  // independent loads first
  int64_t* plane = planes[blockIdx.y];
  const int p = threadIdx.x < n ? path[threadIdx.x] : 0;
  const int np = n_path[lane], b = base[lane];
  if (np <= 1) return;
  __shared__ int64_t src[tree::MAX_NODES], dst[tree::MAX_NODES];  // row numbers, page * 16 + slot
  __shared__ int bad;
  if (threadIdx.x == 0) bad = np > n || b < 0;
  __syncthreads();
  if (threadIdx.x < np && threadIdx.x < n && b >= 0) {
    const int i = threadIdx.x;
    const bool ok = tree::path_ok(path, i, n, b, width);
    int sp = -1, dp = -1;
    if (ok) sp = pt[(b + p) / tree::PAGE], dp = pt[(b + i) / tree::PAGE];
    if (ok && tree::page_ok(sp, n_pages) && tree::page_ok(dp, n_pages)) {
      src[i] = (int64_t)sp * tree::PAGE + (b + p) % tree::PAGE;
      dst[i] = (int64_t)dp * tree::PAGE + (b + i) % tree::PAGE;
    } else {
      bad = 1;
    }
  }
  __syncthreads();
  if (bad) {  // nothing of this lane moves
    if (threadIdx.x == 0) set_error(err, ARCB_ERR_BOUNDS);
    return;
  }
  const int col = (blockIdx.x * NT + threadIdx.x) * 2;
  if (col >= n_kv * dh) return;
  const int head = col / dh, e = col - head * dh;
  plane += (size_t)head * tree::PAGE * dh + e;
  const size_t page_elems = (size_t)n_kv * tree::PAGE * dh;
  auto at = [&](int64_t r) { return (longlong2*)(plane + (size_t)(r / tree::PAGE) * page_elems + (r % tree::PAGE) * dh); };
  for (int i0 = 1; i0 < np; i0 += UN) {
    longlong2 v[UN];
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (i0 + k < np && src[i0 + k] != dst[i0 + k]) v[k] = *at(src[i0 + k]);
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (i0 + k < np && src[i0 + k] != dst[i0 + k]) *at(dst[i0 + k]) = v[k];
  }
}

}  // namespace kp

// planes: device array of n_planes tensors [n_pages, n_kv, 16, dh] int64 (dh
// even).  Sets ARCB_ERR_BOUNDS and moves nothing of a lane whose path is not
// increasing from 0 or leaves the tree, the table or the cache.
extern "C" int arcb_kv_keep_path(int64_t* const* planes, int n_planes, int n_pages, int n_kv, int dh, const int* pt,
                                 int64_t pt_stride, int width, const int* base, const int* path, const int* n_path,
                                 int lanes, int n, int* err, void* stream) {
  if (n_planes < 1 || n_planes > 65535 || lanes < 1 || lanes > 65535 || n < 1 || n > tree::MAX_NODES || n_kv < 1 ||
      dh < 2 || dh % 2 || width < 1)
    return -2;
  const dim3 grid((n_kv * dh / 2 + kp::NT - 1) / kp::NT, n_planes, lanes);
  return launch_k(kp::k_keep_path, grid, dim3(kp::NT), 0, (cudaStream_t)stream, planes, n_pages, n_kv, dh, pt,
                  pt_stride, width, base, path, n_path, n, err);
}
