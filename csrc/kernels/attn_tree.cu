// Exact attention of drafted-tree nodes over a paged cache.
//
// A lane (request) has `base` cached tokens and n_tree <= 64 drafted nodes
// whose K/V rows follow them at positions base + i.  Query i of the lane sees
// every key below base and those nodes whose bit its 64-bit mask has set (its
// own ancestors and itself).  Per (query, head), with the decode kernels'
// integer semantics (crates/arc-inference/src/cached_integer_model.rs:
// 1448-1476, softmax_i64 integer_lut.rs:78-100) over the visible keys:
// score_j = ((q.k_j >> 16) * attn_scale) >> 16 with a wrapping i64 dot,
// e_j = integer_exp(score_j - max), w_j = (e_j * ONE) / sum e,
// o = sum_j (w_j * v_j) >> 16, each term rounded down by itself.  A node's
// output therefore equals a plain decode's along its path.  A query that sees
// no key gets zeros.
#include "../common/tree.h"
#include "common.cuh"
#include "lut.cuh"

using namespace q16;

namespace at {

constexpr int NT = 128;
constexpr int PAGE = tree::PAGE;

// One CTA per (head, query): scores of every key to scratch, then the exact
// max, sum and weights, then the values.
__global__ void __launch_bounds__(NT) k_attn_tree(const int64_t* __restrict__ q, const int64_t* __restrict__ Kc,
                                                  const int64_t* __restrict__ Vc, int n_pages,
                                                  const int* __restrict__ pt, int64_t pt_stride, int width,
                                                  const int* __restrict__ base, const int* __restrict__ n_tree,
                                                  const int64_t* __restrict__ mask, int nq, int n_heads, int n_kv,
                                                  int dh, int64_t attn_scale, int t_lim, int B,
                                                  int64_t* __restrict__ scores, int8_t* __restrict__ X,
                                                  int* __restrict__ lmax, int64_t* __restrict__ o_out,
                                                  int* __restrict__ err) {
  pdl_wait_dep();
  pdl_allow_next();
  __shared__ int64_t lut[EXP_LUT_N];
  __shared__ int64_t red[NT / 32];
  const int tid = threadIdx.x, ln = tid & 31, w = tid >> 5;
  const int slot = blockIdx.y, head = blockIdx.x, lane = slot / nq, kvh = head / (n_heads / n_kv);
  for (int i = tid; i < EXP_LUT_N; i += NT) lut[i] = g_exp_lut.v[i];
  const int b = base[lane], nt = n_tree[lane];
  int T = tree::lane_keys(b, nt, t_lim, width);
  pt += lane * pt_stride;
  bool bad = T < 0;
  for (int i = tid; !bad && i < (T + PAGE - 1) / PAGE; i += NT) bad |= !tree::page_ok(pt[i], n_pages);
  bad = __syncthreads_or(bad);
  if (bad) {
    if (tid == 0) set_error(err, T < 0 ? ARCB_ERR_SEQ_OVERFLOW : ARCB_ERR_BOUNDS);
    T = 0;
  }
  const uint64_t m = (uint64_t)mask[slot];
  const int64_t* qr = q + ((size_t)slot * n_heads + head) * dh;
  int64_t* sc = scores + ((size_t)slot * n_heads + head) * t_lim;
  auto row = [&](const int64_t* c, int j) {
    return c + (((size_t)pt[j / PAGE] * n_kv + kvh) * PAGE + j % PAGE) * dh;
  };
  int64_t mx = INT64_MIN;
  for (int j = w; j < T; j += NT / 32) {
    if (!tree::visible(j, b, nt, m)) continue;
    const int64_t* kr = row(Kc, j);
    uint64_t d = 0;
    for (int e = ln; e < dh; e += 32) d += (uint64_t)wmul(qr[e], kr[e]);
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) d += (uint64_t)shfl_xor_i64((int64_t)d, s);
    const int64_t x = attn_score((int64_t)d, attn_scale);
    if (ln == 0) sc[j] = x;
    mx = x > mx ? x : mx;
  }
  if (ln == 0) red[w] = mx;
  __syncthreads();
  for (int i = 0; i < NT / 32; ++i) mx = red[i] > mx ? red[i] : mx;
  __syncthreads();
  int64_t su = 0;
  for (int j = tid; j < T; j += NT) {
    const int64_t e = tree::visible(j, b, nt, m) ? integer_exp(wsub(sc[j], mx), lut) : 0;
    sc[j] = e;
    su += e;
  }
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) su += shfl_xor_i64(su, s);
  if (ln == 0) red[w] = su;
  __syncthreads();
  su = 0;
  for (int i = 0; i < NT / 32; ++i) su += red[i];
  int need = 0;
  for (int e = tid; e < dh; e += NT) {
    uint64_t o = 0;
    for (int j = 0; j < T; ++j)
      if (sc[j] != 0) o += (uint64_t)mulshr(udiv_small(sc[j] * ONE, su), row(Vc, j)[e]);
    const size_t col = (size_t)head * dh + e;
    if (o_out) o_out[(size_t)slot * n_heads * dh + col] = (int64_t)o;
    if (X) {
      int8_t dg[8];
      const int nl = limb_split8((int64_t)o, dg);
      need = nl > need ? nl : need;
      for (int l = 0; l < 8; ++l) X[limb_row(l, slot, B) * n_heads * dh + col] = dg[l];
    }
  }
  if (need && lmax) atomicMax(lmax, need);
}

}  // namespace at

extern "C" {

int64_t arcb_attn_tree_ws(int lanes, int nq, int n_heads, int n_kv, int dh, int t_lim) {
  (void)n_kv;
  (void)dh;
  return (int64_t)lanes * nq * n_heads * t_lim * 8;
}

int arcb_attn_tree(const int64_t* q, const int64_t* Kc, const int64_t* Vc, int n_pages, const int* pt,
                   int64_t pt_stride, int width, const int* base, const int* n_tree, const int64_t* mask, int nq,
                   int n_heads, int n_kv, int dh, int64_t attn_scale, int t_lim, int lanes, void* ws, int8_t* X,
                   int* lmax, int64_t* o_out, int* err, void* stream) {
  if (lanes < 1 || nq < 1 || n_kv < 1 || n_heads < 1 || n_heads % n_kv || dh < 1 || t_lim < 1) return -2;
  return launch_k(at::k_attn_tree, dim3(n_heads, lanes * nq), dim3(at::NT), 0, (cudaStream_t)stream, q, Kc, Vc,
                  n_pages, pt, pt_stride, width, base, n_tree, mask, nq, n_heads, n_kv, dh, attn_scale, t_lim,
                  lanes * nq, (int64_t*)ws, X, lmax, o_out, err);
}

}  // extern "C"
