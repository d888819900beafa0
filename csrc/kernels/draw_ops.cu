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
// A cluster serves one row (draw) or one node at a time (verify): each CTA
// holds the weights of a contiguous part of the vocabulary in shared memory
// (4 bytes an element; P and Q: 8).  The logits are read once, where 32 bits
// hold the part's (else again for each pass): their low words stand in shared
// memory until they become weights there.  The sums and the single elements
// that all of them need cross through distributed shared memory.
//
// Verification has two schedules.  Where clusters for all nodes cost little more
// than one for the root, every node is decided at once, whether or not the
// accepted path reaches it, and a second small kernel follows the decisions from
// the root: one node's latency.  Larger trees and batches take one cluster per
// lane, which walks from the root and reads only the rows that it meets.
//
// What bounds it is latency: a first touch of DRAM takes one to three
// microseconds (the lane's tree and ring, then the logits, which wait for it), an
// exchange between the CTAs one to one and a half, and a decision needs some
// eight of them in turn.  With nothing left in L2 one row of 32000 takes 9.0 us in
// the kernel (12 to 14 us a call), a drafted chain of 5 of them 20 us a call, 8
// trees of 31 nodes 44 us, 4 trees of 64 nodes of 102400 59 us.  72 rows of
// 102400, three tokens of each, take 55 us: 59 MB, 1 TB/s, in two waves of
// clusters of 8, since half of a row's weights pass SMEM_MAX.  In a row of calls:
// 13, 21, 37 to 45, 50 to 57 and 48 us.
#include <atomic>
#include <climits>

#include "../common/tree.h"
#include "common.cuh"
#include "exp32.cuh"

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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  return ra;
}
__device__ __forceinline__ void push_u64(void* local, uint32_t rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer_addr(local, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void push_u32(void* local, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(local, rank)), "r"(v) : "memory");
}

__device__ __forceinline__ int64_t clamp40(int64_t x) { return x > CLAMP ? CLAMP : (x < -CLAMP ? -CLAMP : x); }

// floor(num / den) for num <= 2^62 and a quotient of at most 2^31: the double
// estimate is within 1 (three roundings of 2^-53 each), the remainder decides.
__device__ __forceinline__ uint32_t div31(uint64_t num, uint64_t den, double rcp) {
  const uint64_t q = (uint64_t)((double)num * rcp);
  const int64_t r = (int64_t)(num - q * den);
  return (uint32_t)q + (r < 0 ? -1 : (uint64_t)r >= den ? 1 : 0);
}

// Scratch, and what the CTAs of a cluster exchange: every CTA stores its value
// into all of them before a cluster barrier and reads its own copies after
// (reading sixteen peers one after another cost 2 us an exchange).  Sums come
// in two phases, so that the next exchange may start while a peer still reads.
// No CTA stores to a peer after its last barrier: any may exit then.  (Stores
// that count their bytes at a barrier of the receiver in place of the cluster
// barriers: one row 8.3 us in the kernel against 9.0, wide trees 57 against 56.)
struct Shared {
  int2 lut[EXP_TABLE_N];
  int64_t redv[NW];  // the first row's warps, then the second's
  int redi[NW];
  uint64_t wsum[NW];
  int64_t xmax[2][MAX_CS];      // largest values (target, draft) and their first indexes
  int xidx[2][MAX_CS];
  uint64_t xsum[2][2][MAX_CS];  // [phase][target, draft]
  uint32_t xchild[2][3];        // [phase] at a child's token: P or its weight, max(P - Q, 0), draft weight
  int ids[HIST];                // newest first
  int met[HIST];                // times that an id is penalised; 0: not its first entry, or not an id
  int parent[tree::MAX_NODES], token[tree::MAX_NODES], hist[HIST];
  int wide[2];                  // the part of the target's, the draft's row has a logit beyond 32 bits
  int count, n_ids, n_path;
};

// The lane's tree (each node's token and parent, -1 where that is no earlier
// node), its ring, and the table of exps: all loads at once.
__device__ __forceinline__ void load_lane(Shared& sh, const int* tokens, const int* parent, int n, const int* hist,
                                          const int* count) {
  static_assert(EXP_LUT_N <= NT && tree::MAX_NODES + HIST < NT, "one element a thread");
  const int tid = threadIdx.x, i = min(tid, n - 1), h = tid & (HIST - 1);
  const int token = __ldg(tokens + i), up = tree::parent_of(parent, i), id = __ldg(hist + h), c = __ldg(count);
  if (tid < EXP_LUT_N) sh.lut[tid] = exp_entry(tid);
  if (tid < n) sh.token[tid] = token, sh.parent[tid] = up;
  if (tid < HIST) sh.hist[tid] = id;
  if (tid == 0) sh.count = max(c, 0);
  __syncthreads();
}

// The newest 64 ids behind `node` (its path up to, not including, the root,
// then the lane's ring), and `skip`: a bit for each of them in this CTA's part
// [v0, v0 + len) of the vocabulary.  The whole CTA calls it.
__device__ void gather_ids(Shared& sh, uint32_t* skip, int node, int V, int v0, int len) {
  const int tid = threadIdx.x;
  for (int i = tid; i < (len + 31) / 32; i += NT) skip[i] = 0;
  if (tid < 2) sh.wide[tid] = 0;
  if (tid == 0) {
    int k = 0;
    for (int i = node; i > 0 && k < HIST; i = sh.parent[i]) sh.ids[k++] = sh.token[i];
    sh.n_path = k;
  }
  __syncthreads();
  const int np = sh.n_path, c = sh.count, n = np + min(c, HIST - np);
  if (tid >= np && tid < n) sh.ids[tid] = sh.hist[(unsigned)(c - 1 - (tid - np)) & (HIST - 1)];
  if (tid == 0) sh.n_ids = n;
  __syncthreads();
  {  // eight threads an id
    const int i = tid >> 3, t = i < n ? sh.ids[i] : -1;
    int m = 0, before = 0;
#pragma unroll
    for (int j = tid & 7; j < HIST; j += 8) {
      const int same = j < n && sh.ids[j] == t;
      m += same;
      before += j < i ? same : 0;
    }
    m |= before << 16;
#pragma unroll
    for (int k = 4; k >= 1; k >>= 1) m += __shfl_xor_sync(0xffffffffu, m, k);
    const bool first = t >= 0 && t < V && m >> 16 == 0;
    if ((tid & 7) == 0 && i < n) {
      sh.met[i] = first ? m : 0;
      if (first && t >= v0 && t < v0 + len) atomicOr(&skip[(t - v0) >> 5], 1u << ((t - v0) & 31));
    }
  }
  __syncthreads();
}

// The threads that share a row: all of the CTA, or half of them a row.
struct Team {
  int k, t, n;  // which row, this thread's place, threads
};

// f(i, x, y) for this thread's pairs of elements i, i + 1 of the part (i even),
// f(i, x) for single ones; x and y are the logits, the skipped ones too.
// 16-byte loads, several in flight, where the row allows them.
template <class F>
__device__ __forceinline__ void each(const int64_t* __restrict__ part, int len, const Team& tm, F f) {
  if (((uintptr_t)part & 15) == 0) {
    const longlong2* p = (const longlong2*)part;
    const int n2 = len / 2;
    for (int i = tm.t; i < n2; i += 4 * tm.n) {
      longlong2 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = i + k * tm.n < n2 ? __ldg(p + i + k * tm.n) : make_longlong2(0, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k * tm.n < n2) f(2 * (i + k * tm.n), (int64_t)x[k].x, (int64_t)x[k].y);
    }
    if ((len & 1) && tm.t == 0) f(len - 1, (int64_t)__ldg((const long long*)part + len - 1));
  } else {
#pragma unroll 1
    for (int i = tm.t; i < len; i += tm.n) f(i, (int64_t)__ldg((const long long*)part + i));
  }
}

// A row's part as it is used.  Clamping and scaling keep the order, so the
// maximum is found before them.
struct Row {
  const int64_t* part;
  int64_t inv;
  __device__ Row(const int64_t* row, int v0, int64_t inv_temp)
      : part(row + v0), inv(inv_temp > MAX_INV_T ? MAX_INV_T : inv_temp) {}
  __device__ bool greedy() const { return inv <= 0; }
  __device__ int64_t value(int64_t x) const { return (clamp40(x) * inv) >> FRAC_BITS; }
  __device__ int64_t penalised(int64_t x, int times) const {  // not scaled
    x = clamp40(x);
    for (int r = 0; r < times; ++r) x = clamp40(penalize(x));
    return x;
  }
};

// Where in the part this thread's id of the row's team stands, or -1.
__device__ __forceinline__ int own_id(const Shared& sh, int v0, int len, const Team& tm) {
  if (tm.t >= sh.n_ids || !sh.met[tm.t]) return -1;
  const int t = sh.ids[tm.t] - v0;
  return t >= 0 && t < len ? t : -1;
}

__device__ __forceinline__ void better(int64_t& v, int& i, int64_t ov, int oi) {
  if (ov > v || (ov == v && oi < i)) v = ov, i = oi;
}

// What row r's logit i of the part becomes, not scaled: the long way.
__device__ int64_t exact(const Shared& sh, const uint32_t* skip, const Row& r, int v0, int i) {
  int times = 0;
  if (skip[i >> 5] >> (i & 31) & 1)
    for (int j = 0; j < sh.n_ids; ++j)
      if (sh.ids[j] == v0 + i) times |= sh.met[j];  // 0 but for the first entry
  return r.penalised(__ldg((const long long*)r.part + i), times);
}

struct Low {  // low words of the logits, and whether those are all
  int* e;
  int high = 0;
  __device__ void operator()(int i, int64_t x) {
    e[i] = (int)x;
    high |= (int)(x >> 32) ^ (int)x >> 31;
  }
  __device__ void operator()(int i, int64_t x, int64_t y) {
    *(int2*)(e + i) = make_int2((int)x, (int)y);
    high |= (int)(x >> 32) ^ (int)x >> 31;
    high |= (int)(y >> 32) ^ (int)y >> 31;
  }
};

// The part's logits, penalised, in 32 bits into e (sh.wide: some do not fit, e
// is void), and the largest clamped one and (of a greedy row) its first index
// by warps into redv / redi.  The whole CTA calls it.
__device__ void warp_max(Shared& sh, const uint32_t* skip, const Row& r, int v0, int len, const Team& tm, uint32_t* e) {
  Low low{(int*)e};
  each(r.part, len, tm, [&](auto... a) { low(a...); });
  if (low.high) sh.wide[tm.k] = 1;
  __syncthreads();
  const int t = own_id(sh, v0, len, tm);
  if (t >= 0) {
    const int64_t x = r.penalised((int)e[t], sh.met[tm.t]);
    e[t] = (uint32_t)x;
    if (x != (int)x) sh.wide[tm.k] = 1;
  }
  __syncthreads();
  int64_t bv = INT64_MIN;
  int bi = INT_MAX;
  if (sh.wide[tm.k]) {
#pragma unroll 1
    for (int i = tm.t; i < len; i += tm.n) {
      const int64_t x = exact(sh, skip, r, v0, i);
      if (x > bv) bv = x, bi = v0 + i;  // a thread meets rising indexes
    }
  } else if (r.greedy()) {
    int m = INT_MIN;
#pragma unroll 2
    for (int i = tm.t; i < len; i += tm.n) {
      const int x = (int)e[i];
      if (x > m || bi == INT_MAX) m = x, bi = v0 + i;
    }
    if (bi != INT_MAX) bv = m;
  } else {
    int m = INT_MIN;
#pragma unroll 4
    for (int i = tm.t * 2; i < len; i += 2 * tm.n) {  // e has an even number of elements
      const int2 x = *(const int2*)(e + i);
      m = max(m, i + 1 < len ? max(x.x, x.y) : x.x);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (len > 0) bv = m, bi = 0;
  }
  if (sh.wide[tm.k] || r.greedy())
#pragma unroll 1
    for (int m = 16; m >= 1; m >>= 1) better(bv, bi, shfl_xor_i64(bv, m), __shfl_xor_sync(0xffffffffu, bi, m));
  if ((threadIdx.x & 31) == 0) sh.redv[threadIdx.x >> 5] = bv, sh.redi[threadIdx.x >> 5] = bi;
}

// The cluster's largest value and first index of n <= 2 rows.
__device__ void cluster_max(Shared& sh, int n, uint32_t rank, uint32_t cs, int64_t* v, int* i) {
  __syncthreads();
  const int k = threadIdx.x >> 5, l = threadIdx.x & 31;
  if (k < n) {  // warp k: row k
    const int nw = NW / n;
    int64_t bv = l < nw ? sh.redv[k * nw + l] : INT64_MIN;
    int bi = l < nw ? sh.redi[k * nw + l] : INT_MAX;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) better(bv, bi, shfl_xor_i64(bv, m), __shfl_xor_sync(0xffffffffu, bi, m));
    if (l < (int)cs) {
      push_u64(&sh.xmax[k][rank], l, (uint64_t)bv);
      push_u32(&sh.xidx[k][rank], l, (uint32_t)bi);
    }
  }
  cluster_sync();
#pragma unroll 1
  for (int c = 0; c < n; ++c) {
    int64_t bv = l < (int)cs ? sh.xmax[c][l] : INT64_MIN;
    int bi = l < (int)cs ? sh.xidx[c][l] : INT_MAX;
#pragma unroll
    for (int m = MAX_CS / 2; m >= 1; m >>= 1) better(bv, bi, shfl_xor_i64(bv, m), __shfl_xor_sync(0xffffffffu, bi, m));
    // lanes 16 and up hold nothing: from the lower half
    bv = __shfl_sync(0xffffffffu, bv, 0), bi = __shfl_sync(0xffffffffu, bi, 0);
    if (c == 0) v[0] = bv, i[0] = bi;
    else v[1] = bv, i[1] = bi;
  }
}

// Weights of the CTA's part into e, from what warp_max left there; this
// thread's part of their sum, in 32 bits: fewer than 2^10 elements of at most
// 2^16 (and 2^15 in a warp).  `top` is the row's largest clamped logit, `first`
// its index.
//
// With zt the scaled top, z - zt + EXP_AT comes of one product and sum,
// x * inv - ((zt - EXP_AT) << 16), shifted; no x is above the top.
__device__ uint32_t weights(Shared& sh, const uint32_t* skip, const Row& r, int v0, int len, int64_t top, int first,
                            const Team& tm, uint32_t* e) {
  const int64_t zt = r.value(top), c = -((zt - EXP_AT) << FRAC_BITS);
  const int inv = (int)r.inv;
  auto weight = [&](int64_t y) {  // y = x * inv + c
    const int at = (int)__funnelshift_r((uint32_t)y, (uint32_t)max((int)(y >> 32), -32768), FRAC_BITS);
    return exp_at(max(at, 2047), sh.lut);
  };
  uint32_t sum = 0;
  if (r.greedy()) {
    for (int i = tm.t; i < len; i += tm.n) e[i] = v0 + i == first ? (uint32_t)ONE : 0u;
    if (tm.t == 0 && first >= v0 && first < v0 + len) sum = (uint32_t)ONE;
  } else if (!sh.wide[tm.k]) {
#pragma unroll 4
    for (int i = tm.t * 2; i < len; i += 2 * tm.n) {  // e has an even number of elements
      const int2 x = *(const int2*)(e + i);
      const uint32_t wx = weight((int64_t)x.x * inv + c), wy = weight((int64_t)x.y * inv + c);
      const uint2 w = make_uint2(wx, i + 1 < len ? wy : 0);
      *(uint2*)(e + i) = w;
      sum += w.x + w.y;
    }
  } else {
#pragma unroll 1
    for (int i = tm.t; i < len; i += tm.n) {
      e[i] = weight(exact(sh, skip, r, v0, i) * inv + c);
      sum += e[i];
    }
  }
  return sum;
}

// Sums over the CTA's teams of what weights returned; every thread gets them.
template <int N>
__device__ __forceinline__ void team_sums(Shared& sh, int n, uint32_t s, uint64_t* out) {
  s = __reduce_add_sync(0xffffffffu, s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = s;
  __syncthreads();
  uint64_t a = 0, b = 0;
#pragma unroll
  for (int w = 0; w < NW / 2; ++w) a += sh.wsum[w], b += sh.wsum[w + NW / 2];
  out[0] = N == 1 || n == 1 ? a + b : a;
  if (N == 2) out[1] = n == 1 ? 0 : b;
}

// The sum over the CTA; every thread gets it.
__device__ __forceinline__ void block_sum(Shared& sh, uint64_t& s) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) s += (uint64_t)shfl_xor_i64((int64_t)s, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += sh.wsum[w];
}

// Exchange of the CTAs' sums mine[0 .. N); total over the cluster, and the
// first one's sum over the CTAs before this one.
template <int N>
__device__ __forceinline__ uint64_t cluster_sum(Shared& sh, const uint64_t* mine, int ph, uint32_t rank, uint32_t cs,
                                                uint64_t* total) {
  if (threadIdx.x < cs)
#pragma unroll
    for (int k = 0; k < N; ++k) push_u64(&sh.xsum[ph][k][rank], threadIdx.x, mine[k]);
  cluster_sync();
  uint64_t before = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) total[k] = 0;
#pragma unroll 4
  for (uint32_t r = 0; r < cs; ++r) {
    if (r < rank) before += sh.xsum[ph][0][r];
#pragma unroll
    for (int k = 0; k < N; ++k) total[k] += sh.xsum[ph][k][r];
  }
  return before;
}

// The first element of this CTA's part whose running sum exceeds t (which is
// below the part's sum); val(i) is element i.  Every thread sums its own
// stretch (an odd number of elements: no bank conflicts), the one whose
// stretch holds t walks through it.  The whole CTA calls it.
template <class F>
__device__ int find(Shared& sh, int len, uint64_t t, F val) {
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int per = (len + NT - 1) / NT | 1, a = min(len, tid * per), b = min(len, a + per);
  uint64_t s = 0;
  for (int i = a; i < b; ++i) s += val(i);
  uint64_t incl = s;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const uint64_t y = (uint64_t)__shfl_up_sync(0xffffffffu, (unsigned long long)incl, m);
    if (lane >= m) incl += y;
  }
  __syncthreads();
  if (lane == 31) sh.wsum[w] = incl;
  __syncthreads();
  uint64_t before = incl - s;
  for (int k = 0; k < w; ++k) before += sh.wsum[k];
  if (before <= t && t < before + s) {
    int i = a;
    for (before += val(i); before <= t; before += val(i)) ++i;
    found = i;
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ uint64_t scale31(uint32_t u, uint64_t s) {  // floor((u mod 2^31) * s / 2^31), s < 2^63
  return __umul64hi((uint64_t)(u & 0x7fffffffu) << 33, s);
}

__global__ void __launch_bounds__(NT, 3) k_draw(const int64_t* __restrict__ logits, int64_t ldl, int V, int nr, int n,
                                             int node0, int m, const int64_t* __restrict__ inv_temp,
                                             const int* __restrict__ u, const int* __restrict__ hist,
                                             const int* __restrict__ count, const int* __restrict__ tokens,
                                             const int* __restrict__ parent, int seg, int* __restrict__ out) {
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Shared sh;
  const uint32_t rank = cluster_rank(), cs = cluster_size();
  const int lane = blockIdx.z, row = lane * nr + blockIdx.y;
  const int v0 = min(V, (int)rank * seg), len = min(V - v0, seg);
  uint32_t* e = (uint32_t*)dsm;
  uint32_t* skip = e + seg;
  cluster_arrive();  // waited for before the first store to a peer: it runs by then
  pdl_wait_dep();
  pdl_allow_next();
  const Row r(logits + (size_t)row * ldl, v0, inv_temp[lane]);
  load_lane(sh, tokens + (size_t)lane * n, parent + (size_t)lane * n, n, hist + lane * HIST, count + lane);
  gather_ids(sh, skip, node0 + blockIdx.y, V, v0, len);
  int64_t top[2];
  int first[2];
  const Team tm{0, (int)threadIdx.x, NT};
  warp_max(sh, skip, r, v0, len, tm, e);
  cluster_wait();
  cluster_max(sh, 1, rank, cs, top, first);
  uint64_t mine;
  team_sums<1>(sh, 1, weights(sh, skip, r, v0, len, top[0], first[0], tm, e), &mine);
  for (int k = 0; k < m; ++k) {
    uint64_t total;
    const uint64_t before = cluster_sum<1>(sh, &mine, k & 1, rank, cs, &total);
    const uint64_t t = scale31((uint32_t)u[(size_t)row * m + k], total);
    if (total == 0) {
      if (rank == 0 && threadIdx.x == 0) out[(size_t)row * m + k] = -1;
    } else if (before <= t && t < before + mine) {
      const int i = find(sh, len, t - before, [&](int j) { return (uint64_t)e[j]; });
      mine -= e[i];
      __syncthreads();
      if (threadIdx.x == 0) {
        e[i] = 0;
        out[(size_t)row * m + k] = v0 + i;
      }
      __syncthreads();
    }
  }
}

// grid (cluster, nodes, lanes): every node's decision into path: the accepted
// child c, or -1 - t for the token t that follows the node when none is.  WALK,
// grid (cluster, 1, lanes): the lane's path.
template <bool WALK>
__global__ void __launch_bounds__(NT, 2) k_verify(const int64_t* __restrict__ logits, int64_t ldl,
                                               const int64_t* __restrict__ dlogits, int64_t ldd, int V, int n,
                                               const int* __restrict__ tokens, const int* __restrict__ parent,
                                               const int* __restrict__ n_tree, const int64_t* __restrict__ inv_temp,
                                               const int64_t* __restrict__ d_inv_temp, const int* __restrict__ u,
                                               const int* __restrict__ hist, const int* __restrict__ count, int seg,
                                               int* __restrict__ path, int* __restrict__ n_path,
                                               int* __restrict__ next) {
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ Shared sh;
  const uint32_t rank = cluster_rank(), cs = cluster_size();
  const int lane = blockIdx.z, tid = threadIdx.x;
  const int v0 = min(V, (int)rank * seg), len = min(V - v0, seg);
  uint32_t* P = (uint32_t*)dsm;
  uint32_t* eq = P + seg;
  uint32_t* skip = eq + seg;
  cluster_arrive();  // waited for before the first store to a peer: it runs by then
  pdl_wait_dep();
  pdl_allow_next();
  const int live = min(n_tree[lane], n);
  int node = WALK ? 0 : blockIdx.y;
  const size_t lane0 = (size_t)lane * n;
  if (node >= live) {  // the whole cluster
    cluster_wait();
    if (WALK && rank == 0) {
      for (int i = tid; i < n; i += NT) path[lane0 + i] = -1;
      if (tid == 0) n_path[lane] = 0, next[lane] = -1;
    }
    return;
  }
  load_lane(sh, tokens + lane0, parent + lane0, n, hist + lane * HIST, count + lane);
  u += lane0 * 2;
  int ph = 0, length = 0;
  bool first_node = true;
  uint64_t kids = 0;  // the node's children whose token is one, not asked yet
  auto next_child = [&]() {
    const int c = kids ? __ffsll((long long)kids) - 1 : live;
    kids &= kids - 1;
    return c;
  };
  for (;;) {
    const size_t row = lane0 + node;
    kids = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 32 * h + (tid & 31);
      const bool kid = i < live && sh.parent[i] == node && sh.token[i] >= 0 && sh.token[i] < V;
      kids |= (uint64_t)__ballot_sync(0xffffffffu, kid) << 32 * h;
    }
    int c = next_child();
    const bool inner = c < live;
    gather_ids(sh, skip, node, V, v0, len);
    // half of the warps for each of the two rows: one latency, and one copy of
    // the code (instructions come from DRAM too)
    const int n_rows = inner ? 2 : 1, tn = NT / n_rows;
    const Team tm{tid / tn, tid % tn, tn};
    const Row r(tm.k ? dlogits + row * ldd : logits + row * ldl, v0, (tm.k ? d_inv_temp : inv_temp)[lane]);
    uint32_t* e = tm.k ? eq : P;
    warp_max(sh, skip, r, v0, len, tm, e);
    if (first_node) cluster_wait();
    first_node = false;
    int64_t top[2];
    int first[2];
    cluster_max(sh, n_rows, rank, cs, top, first);
    // one CTA stores what child c's test needs into all of them, with the sums of phase ph
    auto push_child = [&](uint32_t a, uint32_t b, uint32_t e) {
      if (tid < cs) {
        push_u32(&sh.xchild[ph][0], tid, a);
        push_u32(&sh.xchild[ph][1], tid, b);
        push_u32(&sh.xchild[ph][2], tid, e);
      }
    };
    uint64_t mine[2], S[2], before;
    const uint32_t sum =
        weights(sh, skip, r, v0, len, tm.k ? top[1] : top[0], tm.k ? first[1] : first[0], tm, e);
    team_sums<2>(sh, n_rows, sum, mine);
    ph ^= 1;
    if (inner && sh.token[c] / seg == (int)rank) push_child(P[sh.token[c] - v0], 0, eq[sh.token[c] - v0]);
    before = cluster_sum<2>(sh, mine, ph, rank, cs, S);
    // P = floor(e * 2^31 / S), made of the weights in place once it is needed as a whole
    const double rp = 1.0 / (double)S[0];
    auto normalise = [&]() {
#pragma unroll 4
      for (int i = tid; i < len; i += NT) P[i] = div31((uint64_t)P[i] << 31, S[0], rp);
    };
    int taken = -1;
    bool whole = false;
    uint32_t pd = inner ? div31((uint64_t)sh.xchild[ph][0] << 31, S[0], rp) : 0, ed = sh.xchild[ph][2];
    uint64_t sq = S[1];
    while (c < live && sq > 0) {
      const int d = sh.token[c];
      const double rq = 1.0 / (double)sq;
      if (scale31((uint32_t)u[2 * c], div31((uint64_t)ed << 31, sq, rq)) < pd) {
        taken = c;
        break;
      }
      if (!whole) {
        normalise();
        __syncthreads();
        whole = true;
      }
      auto rest = [&](int i) -> uint32_t {
        const uint32_t p = P[i], q = div31((uint64_t)eq[i] << 31, sq, rq);
        return p > q ? p - q : 0;
      };
      uint64_t s = 0, left;
#pragma unroll 4
      for (int i = tid; i < len; i += NT) s += rest(i);
      block_sum(sh, s);
      const int c2 = next_child(), d2 = c2 < live ? sh.token[c2] : 0;
      ph ^= 1;
      if (c2 < live && d2 / seg == (int)rank) push_child(P[d2 - v0], rest(d2 - v0), d2 == d ? 0 : eq[d2 - v0]);
      cluster_sum<1>(sh, &s, ph, rank, cs, &left);
      if (left > 0) {
        const double rl = 1.0 / (double)left;
#pragma unroll 4
        for (int i = tid; i < len; i += NT) P[i] = div31((uint64_t)rest(i) << 31, left, rl);
        pd = div31((uint64_t)sh.xchild[ph][1] << 31, left, rl);
      } else {
        pd = sh.xchild[ph][0];
      }
      __syncthreads();
      if (d / seg == (int)rank && tid == 0) eq[d - v0] = 0;
      __syncthreads();
      sq -= ed;
      ed = sh.xchild[ph][2];
      c = c2;
    }
    if (taken < 0) {
      if (!whole) {
        normalise();
        __syncthreads();
      }
      uint64_t s = 0, all;
      for (int i = tid; i < len; i += NT) s += P[i];
      block_sum(sh, s);
      ph ^= 1;
      before = cluster_sum<1>(sh, &s, ph, rank, cs, &all);
      const uint64_t t = scale31((uint32_t)u[2 * node + 1], all);
      if (before <= t && t < before + s) {
        const int i = find(sh, len, t - before, [&](int j) { return (uint64_t)P[j]; });
        if (tid == 0) {
          if (WALK) next[lane] = v0 + i;
          else path[row] = -1 - (v0 + i);
        }
      }
    }
    if (!WALK) {
      if (rank == 0 && tid == 0 && taken >= 0) path[row] = taken;
      break;
    }
    if (rank == 0 && tid == 0) path[lane0 + length] = node;
    ++length;
    if (taken < 0) {
      if (rank == 0) {
        for (int i = length + tid; i < n; i += NT) path[lane0 + i] = -1;
        if (tid == 0) n_path[lane] = length;
      }
      break;
    }
    node = taken;  // a later node: the walk ends
  }
}

// Follows the decisions, in place, from each lane's root: the k-th node of a
// path is k or a later one, whose decision is read before entry k is written.
// One thread per lane.
__global__ void k_verify_path(int lanes, int n, const int* __restrict__ n_tree, int* path, int* __restrict__ n_path,
                              int* __restrict__ next) {
  pdl_wait_dep();
  pdl_allow_next();
  const int lane = blockIdx.x * blockDim.x + threadIdx.x;
  if (lane >= lanes) return;
  path += (size_t)lane * n;
  int k = 0, node = 0, tok = -1;
  if (min(n_tree[lane], n) > 0)
    for (;;) {  // children come after their parent, so this ends
      const int c = path[node];
      path[k++] = node;
      if (c <= node || c >= n) {
        tok = -1 - c;
        break;
      }
      node = c;
    }
  n_path[lane] = k;
  next[lane] = tok;
  for (; k < n; ++k) path[k] = -1;
}

// Part of the vocabulary per CTA of a cluster of cs, and its shared memory
// (`per` bytes an element and a bit for the penalised ids).
static size_t part_of(int V, int cs, int per, int& seg) {
  seg = ((V + cs - 1) / cs + 31) / 32 * 32;
  return (size_t)seg * per + seg / 8;
}

// CTAs per SM: `most` by their registers.
static int per_sm(size_t smem, int most) {
  const int by_smem = (int)((224 * 1024) / (smem + sizeof(Shared) + 1024));
  return by_smem < most ? by_smem : most;
}

// How `rows` rows are divided over clusters.
struct Split {
  int cs, seg;
  size_t smem;
  int64_t cost;
};

// The cluster size whose clusters finish first: the number that run one after
// another times what one takes: a fixed part (exchanges and loads: as long as
// FIXED elements, and EACH for every CTA) and its elements, `per` / 4 words of
// each, the longer the more CTAs share an SM.  Measured for three draws of each
// row, with clusters of 16 / 8 / 4 / 2 CTAs: V = 32000, one row 16.4 / 16.4 /
// 20.5 / 24.6 us, 24 rows 31 / 21 / 21 / 27, 128 rows 100 / 53 / 43 / 35;
// V = 102400, one row 21 / 25 / 31 / (no room), 32 rows 43 / 31 / 35, 128 rows
// 133 / 86 / 82.
static Split split_of(int64_t rows, int V, int per, int most) {
  constexpr int FIXED = 28000, EACH = 60;
  constexpr int AT_ONCE[4] = {7, 16, 35, 74};  // clusters of 16, 8, 4, 2 CTAs that the GPU's SM groups hold, one CTA per SM
  Split best = {};
  for (int i = 0; i < 4; ++i) {
    Split x = {};
    x.cs = 16 >> i;
    x.smem = part_of(V, x.cs, per, x.seg);
    if (i > 0 && x.smem > SMEM_MAX) break;
    const int64_t held = per_sm(x.smem, most), at_once = AT_ONCE[i] * held, share = (rows * x.cs + 147) / 148;
    const int64_t waves = (rows + at_once - 1) / at_once;
    x.cost = waves * (FIXED + EACH * x.cs + x.seg * (per / 4) * (share < held ? share : held));
    if (i == 0 || x.cost < best.cost) best = x;
  }
  return best;
}

template <typename... KArgs, typename... Args>
static int launch_cluster(void (*k)(KArgs...), std::atomic<uint64_t>& ready, int cs, dim3 grid, size_t smem,
                          cudaStream_t st, Args... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready.load() >> (dev & 63) & 1)) {  // the kernel's attributes, once per device
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  }
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
int arcb_draw_max_vocab() { return (int)(dr::SMEM_MAX * 8 / 65) / 32 * 32 * dr::MAX_CS; }

// m tokens of each row lane * nr + i (node node0 + i of the lane's tree) into
// out [lanes * nr, m].
int arcb_draw_tokens(const int64_t* logits, int64_t ldl, int V, int lanes, int nr, int n, int node0, int m,
                     const int64_t* inv_temp, const int* u, const int* hist, const int* count, const int* tokens,
                     const int* parent, int* out, void* stream) {
  if (V < 1 || V > arcb_draw_max_vocab() || lanes < 1 || nr < 1 || m < 1 || node0 < 0 || node0 + nr > n ||
      n > tree::MAX_NODES || lanes > 65535)
    return -2;
  const dr::Split x = dr::split_of((int64_t)lanes * nr, V, 4, 3);
  static std::atomic<uint64_t> ready{0};
  return dr::launch_cluster(dr::k_draw, ready, x.cs, dim3(x.cs, nr, lanes), x.smem, (cudaStream_t)stream, logits, ldl, V,
                            nr, n, node0, m, inv_temp, u, hist, count, tokens, parent, x.seg, out);
}

int arcb_verify_tree(const int64_t* logits, int64_t ldl, const int64_t* dlogits, int64_t ldd, int V, int lanes, int n,
                     const int* tokens, const int* parent, const int* n_tree, const int64_t* inv_temp,
                     const int64_t* d_inv_temp, const int* u, const int* hist, const int* count, int* path,
                     int* n_path, int* next, void* stream) {
  if (V < 1 || V > arcb_draw_max_vocab() || lanes < 1 || n < 1 || n > tree::MAX_NODES || lanes > 65535) return -2;
  static std::atomic<uint64_t> walk{0}, all{0};
  cudaStream_t st = (cudaStream_t)stream;
  const dr::Split each = dr::split_of((int64_t)lanes * n, V, 8, 2), walk_of = dr::split_of(lanes, V, 8, 2);
  // A path is a few nodes long, so all nodes at once may take the time of 1.7.  Measured, at
  // once / along the path, V = 32000: 16 nodes of a lane 25 / 38 us, 31 nodes 28 / 38, 64 nodes
  // 47 / 37, 8 lanes of 31 nodes 90 / 45; V = 102400: 13 nodes 37 / 44, 31 nodes 49 / 39.
  if (each.cost * 10 > walk_of.cost * 17)
    return dr::launch_cluster(dr::k_verify<true>, walk, walk_of.cs, dim3(walk_of.cs, 1, lanes), walk_of.smem, st, logits,
                              ldl, dlogits, ldd, V, n, tokens, parent, n_tree, inv_temp, d_inv_temp, u, hist, count,
                              walk_of.seg, path, n_path, next);
  const int rc = dr::launch_cluster(dr::k_verify<false>, all, each.cs, dim3(each.cs, n, lanes), each.smem, st, logits,
                                    ldl, dlogits, ldd, V, n, tokens, parent, n_tree, inv_temp, d_inv_temp, u, hist,
                                    count, each.seg, path, n_path, next);
  if (rc) return rc;
  return launch_k(dr::k_verify_path, dim3((lanes + 63) / 64), dim3(64), 0, st, lanes, n, n_tree, path, n_path, next);
}

}  // extern "C"
