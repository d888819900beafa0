// Drawing tokens and verifying drafted ones with given random numbers, in
// exact integers.
//
// A row of Q16 logits becomes weights as follows.  Each logit is clamped to
// +-2^40 (so a masked logit of any size neither wraps nor wins), the newest
// 64 ids behind the row's node are penalised, compounding, as the greedy
// step does (crates/arc-inference/src/cached_integer_model.rs:1533-1548) with
// the same clamp after each step, z = (x * inv_temp) >> 16, and
// e = integer_exp(z - max z) (integer_lut.rs:56-74), a 17-bit integer.  An
// inverse temperature of 0 or less is greedy: e = ONE at the first maximum,
// 0 elsewhere.  Sums of e are exact 64-bit integers, so nothing here depends
// on the order of a sum.
//
// Random numbers are 31-bit integers u, standing for u / 2^31.
//
//  * draw: t = floor(u * S / 2^31) with S = sum e; the token is the first v
//    whose running sum exceeds t.  A second draw of the same row sees e_v = 0
//    (without replacement); a row with nothing left gives -1.
//  * verify: P_v = floor(e_v * 2^31 / S) from the target's row and Q_v from the
//    draft's.  A child with token d is accepted iff floor(u * Q_d / 2^31) <
//    P_d; a rejected one leaves P_v <- floor(max(P_v - Q_v, 0) * 2^31 / sum)
//    (unchanged where that sum is 0), removes d from the draft's weights, and
//    the next child is asked.  Where no child is accepted the following token
//    is drawn from P as it then stands.
//
// One cluster serves one row (draw) or one node (verify): each CTA holds a
// contiguous part of the vocabulary in shared memory, and the sums and the
// single elements that all of them need cross through distributed shared
// memory.  Every node of every tree is decided at once, whether or not the
// accepted path reaches it; a second small kernel follows the decisions from
// the root.
#include <climits>

#include "../common/tree.h"
#include "common.cuh"
#include "lut.cuh"

using namespace q16;

namespace dr {

constexpr int NT = 512, NW = NT / 32;
constexpr int64_t CLAMP = int64_t(1) << 40;
constexpr int64_t MAX_INV_T = int64_t(1) << 20;
constexpr int HIST = 64;
constexpr int MAX_CS = 16;
constexpr size_t SMEM_MAX = 200 * 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  return ra;
}
__device__ __forceinline__ uint64_t peer_u64(const void* local, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peer_u32(const void* local, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(local, rank)) : "memory");
  return v;
}

__device__ __forceinline__ int64_t clamp40(int64_t x) { return x > CLAMP ? CLAMP : (x < -CLAMP ? -CLAMP : x); }

// floor(num / den) for num <= 2^62 and a quotient of at most 2^31: the double
// estimate is within 1 (three roundings of 2^-53 each), the remainder decides.
__device__ __forceinline__ uint32_t div31(uint64_t num, uint64_t den, double rcp) {
  uint64_t q = (uint64_t)((double)num * rcp);
  const int64_t r = (int64_t)(num - q * den);
  if (r < 0) --q;
  else if ((uint64_t)r >= den) ++q;
  return (uint32_t)q;
}

// What the CTAs of a cluster exchange.
struct Shared {
  int64_t lut[EXP_LUT_N];
  int64_t redv[NW];
  int redi[NW];
  uint64_t wsum[NW];
  int64_t xmax;      // this CTA's largest value and its first index
  int xidx;
  uint64_t xsum[2];  // this CTA's sum, two phases
  int ids[HIST];     // newest first; -1: none
  int n_ids;
};

// The newest 64 ids behind `node`: its path up to (not including) the root,
// then the lane's ring.  The whole CTA calls it.
__device__ void gather_ids(Shared& sh, const int* hist, int count, const int* tokens, const int* parent, int node) {
  __shared__ int n_path;
  if (threadIdx.x == 0) {
    int k = 0;
    for (int i = node; i > 0 && k < HIST; i = tree::parent_of(parent, i)) sh.ids[k++] = tokens[i];
    n_path = k;
  }
  __syncthreads();
  const int np = n_path, c = count < 0 ? 0 : count;
  const int n = np + (c < HIST - np ? c : HIST - np);
  if (threadIdx.x >= np && threadIdx.x < n)
    sh.ids[threadIdx.x] = hist[(unsigned)(c - 1 - ((int)threadIdx.x - np)) & (HIST - 1)];
  if (threadIdx.x == 0) sh.n_ids = n;
  __syncthreads();
}

// Loads this CTA's part [v0, v0 + len) of a row into z (int64, temperature
// applied) and agrees on the cluster's largest value; then e of each element
// into the low words of z and the cluster's sum.  inv <= 0: the one-hot row.
// `ph` is the phase of the exchange cells (the caller alternates it).
__device__ uint64_t row_weights(Shared& sh, const int64_t* __restrict__ row, int v0, int len, int V, int64_t inv,
                                int64_t* z, uint32_t cs) {
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  inv = inv > MAX_INV_T ? MAX_INV_T : inv;
  const bool greedy = inv <= 0;
  for (int i = tid; i < len; i += NT) z[i] = clamp40(__ldcg((const long long*)row + v0 + i));
  __syncthreads();
  if (tid < sh.n_ids) {  // the first entry of an id applies its penalties
    const int t = sh.ids[tid] - v0;
    bool first = sh.ids[tid] >= 0 && sh.ids[tid] < V && t >= 0 && t < len;
    int c = 0;
    for (int j = 0; j < sh.n_ids; ++j) {
      c += sh.ids[j] == sh.ids[tid];
      first &= !(j < tid && sh.ids[j] == sh.ids[tid]);
    }
    if (first) {
      int64_t v = z[t];
      for (int r = 0; r < c; ++r) v = clamp40(penalize(v));
      z[t] = v;
    }
  }
  __syncthreads();
  int64_t bv = INT64_MIN;
  int bi = INT_MAX;
  for (int i = tid; i < len; i += NT) {
    int64_t x = z[i];
    if (!greedy) {
      x = (x * inv) >> FRAC_BITS;
      z[i] = x;
    }
    if (x > bv) bv = x, bi = v0 + i;
  }
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    const int64_t ov = shfl_xor_i64(bv, m);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, m);
    if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
  }
  if (lane == 0) sh.redv[w] = bv, sh.redi[w] = bi;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < NW; ++k)
      if (sh.redv[k] > bv || (sh.redv[k] == bv && sh.redi[k] < bi)) bv = sh.redv[k], bi = sh.redi[k];
    sh.xmax = bv;
    sh.xidx = bi;
  }
  cluster_sync();
  bv = INT64_MIN;
  bi = INT_MAX;
  for (uint32_t r = 0; r < cs; ++r) {
    const int64_t ov = (int64_t)peer_u64(&sh.xmax, r);
    const int oi = (int)peer_u32(&sh.xidx, r);
    if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
  }
  uint64_t s = 0;
  for (int i = tid; i < len; i += NT) {
    const uint32_t e = greedy ? (v0 + i == bi ? (uint32_t)ONE : 0u) : (uint32_t)integer_exp(z[i] - bv, sh.lut);
    ((uint32_t*)z)[2 * i] = e;
    s += e;
  }
  return s;  // this thread's part
}

// Sum over the CTA; every thread gets it.
__device__ uint64_t block_sum(Shared& sh, uint64_t s) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) s += (uint64_t)shfl_xor_i64((int64_t)s, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int k = 0; k < NW; ++k) s += sh.wsum[k];
  return s;
}

// Sum over the cluster, and the sum of the CTAs before this one.
__device__ uint64_t cluster_sum(Shared& sh, uint64_t cta, int ph, uint32_t rank, uint32_t cs, uint64_t& before) {
  if (threadIdx.x == 0) sh.xsum[ph] = cta;
  cluster_sync();
  uint64_t total = 0;
  before = 0;
  for (uint32_t r = 0; r < cs; ++r) {
    const uint64_t x = peer_u64(&sh.xsum[ph], r);
    if (r < rank) before += x;
    total += x;
  }
  return total;
}

// The first element of this CTA's part whose running sum exceeds t (which is
// below the part's sum); val(i) is element i.  The whole CTA calls it.
template <class F>
__device__ int find(Shared& sh, int len, uint64_t t, F val) {
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int per = (len + NW * 32 - 1) / (NW * 32) * 32;  // elements per warp
  const int a = w * per, b = min(len, a + per);
  uint64_t s = 0;
  for (int i = a + lane; i < b; i += 32) s += val(i);
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) s += (uint64_t)shfl_xor_i64((int64_t)s, m);
  __syncthreads();
  if (lane == 0) sh.wsum[w] = s;
  __syncthreads();
  uint64_t before = 0;
  for (int k = 0; k < w; ++k) before += sh.wsum[k];
  if (before <= t && t < before + s) {  // this warp's elements hold it
    for (int i0 = a; i0 < b; i0 += 32) {
      const int i = i0 + lane;
      uint64_t x = i < b ? val(i) : 0;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const uint64_t y = (uint64_t)__shfl_up_sync(0xffffffffu, (unsigned long long)x, m);
        if (lane >= m) x += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + x > t);
      if (hit) {
        if (lane == 0) found = i0 + __ffs(hit) - 1;
        break;
      }
      before += (uint64_t)__shfl_sync(0xffffffffu, (unsigned long long)x, 31);
    }
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ uint64_t scale31(uint32_t u, uint64_t s) {  // floor((u mod 2^31) * s / 2^31), s < 2^63
  return __umul64hi((uint64_t)(u & 0x7fffffffu) << 33, s);
}

__global__ void __launch_bounds__(NT) k_draw(const int64_t* __restrict__ logits, int64_t ldl, int V, int nr, int n,
                                             int node0, int m, const int64_t* __restrict__ inv_temp,
                                             const int* __restrict__ u, const int* __restrict__ hist,
                                             const int* __restrict__ count, const int* __restrict__ tokens,
                                             const int* __restrict__ parent, int seg, int* __restrict__ out) {
  pdl_wait_dep();
  pdl_allow_next();
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Shared sh;
  const uint32_t rank = cluster_rank(), cs = cluster_size();
  const int lane = blockIdx.z, row = lane * nr + blockIdx.y;
  const int v0 = min(V, (int)rank * seg), len = min(V - v0, seg);
  int64_t* z = (int64_t*)dsm;
  uint32_t* e = (uint32_t*)dsm;  // element i at e[2 * i]
  for (int i = threadIdx.x; i < EXP_LUT_N; i += NT) sh.lut[i] = g_exp_lut.v[i];
  gather_ids(sh, hist + lane * HIST, count[lane], tokens + (size_t)lane * n, parent + (size_t)lane * n,
             node0 + blockIdx.y);
  uint64_t mine = block_sum(sh, row_weights(sh, logits + (size_t)row * ldl, v0, len, V, inv_temp[lane], z, cs));
  for (int k = 0; k < m; ++k) {
    uint64_t before;
    const uint64_t total = cluster_sum(sh, mine, k & 1, rank, cs, before);
    const uint64_t t = scale31((uint32_t)u[(size_t)row * m + k], total);
    if (total == 0) {
      if (rank == 0 && threadIdx.x == 0) out[(size_t)row * m + k] = -1;
    } else if (before <= t && t < before + mine) {
      const int i = find(sh, len, t - before, [&](int j) { return (uint64_t)e[2 * j]; });
      mine -= e[2 * i];
      __syncthreads();
      if (threadIdx.x == 0) {
        e[2 * i] = 0;
        out[(size_t)row * m + k] = v0 + i;
      }
      __syncthreads();
    }
  }
  cluster_sync();  // no CTA may exit while a peer still reads its shared memory
}

// One node of one tree: choice = the accepted child or -1, drawn = the token
// that follows the node when no child is accepted.
__global__ void __launch_bounds__(NT) k_verify_node(const int64_t* __restrict__ logits, int64_t ldl,
                                                    const int64_t* __restrict__ dlogits, int64_t ldd, int V, int n,
                                                    const int* __restrict__ tokens, const int* __restrict__ parent,
                                                    const int* __restrict__ n_tree,
                                                    const int64_t* __restrict__ inv_temp,
                                                    const int64_t* __restrict__ d_inv_temp, const int* __restrict__ u,
                                                    const int* __restrict__ hist, const int* __restrict__ count,
                                                    int seg, int* __restrict__ choice, int* __restrict__ drawn) {
  pdl_wait_dep();
  pdl_allow_next();
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Shared sh;
  const uint32_t rank = cluster_rank(), cs = cluster_size();
  const int lane = blockIdx.z, node = blockIdx.y, tid = threadIdx.x;
  const int live = min(n_tree[lane], n);
  if (node >= live) return;  // the whole cluster
  const size_t row = (size_t)lane * n + node;
  tokens += (size_t)lane * n;
  parent += (size_t)lane * n;
  u += (size_t)lane * n * 2;
  const int v0 = min(V, (int)rank * seg), len = min(V - v0, seg);
  int64_t* z = (int64_t*)dsm;              // a row's values; then the draft's weights (low) and max(P - Q, 0) (high)
  uint32_t* eq = (uint32_t*)dsm;
  uint32_t* P = (uint32_t*)(z + seg);
  for (int i = tid; i < EXP_LUT_N; i += NT) sh.lut[i] = g_exp_lut.v[i];
  gather_ids(sh, hist + lane * HIST, count[lane], tokens, parent, node);
  int ph = 0;
  uint64_t before;
  uint64_t mine = block_sum(sh, row_weights(sh, logits + row * ldl, v0, len, V, inv_temp[lane], z, cs));
  uint64_t S = cluster_sum(sh, mine, ph ^= 1, rank, cs, before);
  double rcp = 1.0 / (double)S;
  for (int i = tid; i < len; i += NT) P[i] = div31((uint64_t)eq[2 * i] << 31, S, rcp);
  int first = node + 1;
  while (first < live && tree::parent_of(parent, first) != node) ++first;
  int taken = -1;
  if (first < live) {
    __syncthreads();
    mine = block_sum(sh, row_weights(sh, dlogits + row * ldd, v0, len, V, d_inv_temp[lane], z, cs));
    uint64_t sq = cluster_sum(sh, mine, ph ^= 1, rank, cs, before);
    for (int c = first; c < live; ++c) {
      if (tree::parent_of(parent, c) != node) continue;
      const int d = tokens[c];
      if (d < 0 || d >= V || sq == 0) continue;
      const uint32_t owner = (uint32_t)(d / seg);
      const int at = d - (int)owner * seg;
      const uint32_t pd = peer_u32(&P[at], owner), ed = peer_u32(&eq[2 * at], owner);
      rcp = 1.0 / (double)sq;
      if (scale31((uint32_t)u[2 * c], div31((uint64_t)ed << 31, sq, rcp)) < pd) {
        taken = c;
        break;
      }
      uint64_t s = 0;
      for (int i = tid; i < len; i += NT) {
        const uint32_t p = P[i], q = div31((uint64_t)eq[2 * i] << 31, sq, rcp);
        const uint32_t r = p > q ? p - q : 0;
        eq[2 * i + 1] = r;
        s += r;
      }
      S = cluster_sum(sh, block_sum(sh, s), ph ^= 1, rank, cs, before);
      if (S > 0) {
        rcp = 1.0 / (double)S;
        for (int i = tid; i < len; i += NT) P[i] = div31((uint64_t)eq[2 * i + 1] << 31, S, rcp);
      }
      if (rank == owner && tid == 0) eq[2 * at] = 0;
      sq -= ed;
      cluster_sync();  // the new P and eq before the next child's reads
    }
  }
  if (taken < 0) {
    uint64_t s = 0;
    for (int i = tid; i < len; i += NT) s += P[i];
    mine = block_sum(sh, s);
    S = cluster_sum(sh, mine, ph ^= 1, rank, cs, before);
    const uint64_t t = scale31((uint32_t)u[2 * node + 1], S);
    if (before <= t && t < before + mine) {
      const int i = find(sh, len, t - before, [&](int j) { return (uint64_t)P[j]; });
      if (tid == 0) drawn[row] = v0 + i;
    }
  }
  if (rank == 0 && tid == 0) choice[row] = taken;
  cluster_sync();  // no CTA may exit while a peer still reads its shared memory
}

// Follows the decisions from each lane's root.  One thread per lane.
__global__ void k_verify_path(int lanes, int n, const int* __restrict__ n_tree, const int* __restrict__ choice,
                              const int* __restrict__ drawn, int* __restrict__ path, int* __restrict__ n_path,
                              int* __restrict__ next) {
  pdl_wait_dep();
  pdl_allow_next();
  const int lane = blockIdx.x * blockDim.x + threadIdx.x;
  if (lane >= lanes) return;
  const size_t r0 = (size_t)lane * n;
  int k = 0, node = 0, tok = -1;
  if (min(n_tree[lane], n) > 0)
    for (;;) {  // children come after their parent, so this ends
      path[r0 + k++] = node;
      const int c = choice[r0 + node];
      if (c <= node || c >= n) {
        tok = drawn[r0 + node];
        break;
      }
      node = c;
    }
  n_path[lane] = k;
  next[lane] = tok;
  for (; k < n; ++k) path[r0 + k] = -1;
}

// CTAs per row: enough of them that a part of the vocabulary fits in shared
// memory (`per` bytes an element).
static int cluster_for(int V, int per, int& seg) {
  for (int cs = 8; cs <= MAX_CS; cs *= 2) {
    seg = ((V + cs - 1) / cs + 31) / 32 * 32;
    if ((size_t)seg * per <= SMEM_MAX) return cs;
  }
  return 0;
}

template <typename... KArgs, typename... Args>
static int launch_cluster(void (*k)(KArgs...), int cs, dim3 grid, size_t smem, cudaStream_t st,
                          Args... args) {
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX);
  if (e == cudaSuccess && cs > 8) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = arcb_pdl_enabled();
  cfg.attrs = at;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, k, ((KArgs)args)...);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace dr

extern "C" {

// Largest vocabulary the two entry points below take.
int arcb_draw_max_vocab() { return (int)(dr::SMEM_MAX / 12) / 32 * 32 * dr::MAX_CS; }

// m tokens of each row lane * nr + i (node node0 + i of the lane's tree) into
// out [lanes * nr, m].
int arcb_draw_tokens(const int64_t* logits, int64_t ldl, int V, int lanes, int nr, int n, int node0, int m,
                     const int64_t* inv_temp, const int* u, const int* hist, const int* count, const int* tokens,
                     const int* parent, int* out, void* stream) {
  if (V < 1 || lanes < 1 || nr < 1 || m < 1 || node0 < 0 || node0 + nr > n || n > tree::MAX_NODES || lanes > 65535)
    return -2;
  int seg = 0;
  const int cs = dr::cluster_for(V, 8, seg);
  if (!cs) return -2;
  return dr::launch_cluster(dr::k_draw, cs, dim3(cs, nr, lanes), (size_t)seg * 8, (cudaStream_t)stream, logits,
                            ldl, V, nr, n, node0, m, inv_temp, u, hist, count, tokens, parent, seg, out);
}

// scratch: 2 * lanes * n ints.
int arcb_verify_tree(const int64_t* logits, int64_t ldl, const int64_t* dlogits, int64_t ldd, int V, int lanes, int n,
                     const int* tokens, const int* parent, const int* n_tree, const int64_t* inv_temp,
                     const int64_t* d_inv_temp, const int* u, const int* hist, const int* count, int* scratch,
                     int* path, int* n_path, int* next, void* stream) {
  if (V < 1 || lanes < 1 || n < 1 || n > tree::MAX_NODES || lanes > 65535) return -2;
  int seg = 0;
  const int cs = dr::cluster_for(V, 12, seg);
  if (!cs) return -2;
  int* drawn = scratch + (size_t)lanes * n;
  const int rc = dr::launch_cluster(dr::k_verify_node, cs, dim3(cs, n, lanes), (size_t)seg * 12,
                                    (cudaStream_t)stream, logits, ldl, dlogits, ldd, V, n, tokens, parent, n_tree,
                                    inv_temp, d_inv_temp, u, hist, count, seg, scratch, drawn);
  if (rc) return rc;
  return launch_k(dr::k_verify_path, dim3((lanes + 63) / 64), dim3(64), 0, (cudaStream_t)stream, lanes, n, n_tree,
                  scratch, drawn, path, n_path, next);
}

}  // extern "C"
