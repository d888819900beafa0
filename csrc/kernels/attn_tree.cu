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
//
// The queries of a KV head (nq nodes x G query heads: R rows) share its K and
// V.  Exact weights need the global max and sum before the first value, so
// there are four kernels (for few rows and keys, two: k_scores makes the query
// digits itself, and each value CTA the maxima and sums of its lane's rows):
//
//  0. k_queries: the query rows' digits (see 1) in groups of 32 rows.
//  1. k_scores, one CTA per 128 keys.  K's int64 elements become signed
//     radix-256 digits (byte l of (x + 0x80..80) ^ 0x80..80, int8), one
//     128-byte-swizzled plane of 128 keys x dh per digit, read once from DRAM;
//     the query rows' planes come by bulk copies, 32 rows at a time.  q.k =
//     sum_s D_s << 8s with D_s = sum_{a+b=s} K_a.Q_b^T: tcgen05 kind::i8
//     products of M = 128 keys, N = 32 rows into one TMEM accumulator per s
//     (exact in int32: at most 4 * 128 * 2^14).  3 digits (|x| < 2^23) are
//     usual; up to 4 (|x| < 2^31) run this way, wider tiles take 64-bit
//     products.  Scores are stored relative to their tile's max (differences
//     below -2^30 clamped: their exp is 0 either way) or, where 32 bits hold
//     them, as they are; the rows' maxima join by atomics.
//  2. k_sums: each row's sum of exps, split over key chunks.
//  3. k_values: w.v for up to 128 rows and a range of keys.  The floor of each
//     term rules out a matrix product, but one single-precision FMA rounding
//     toward minus infinity is exact: acc <- rd(acc + w * (v / 2^16)) with acc
//     an integer in [2^23, 2^24), where floats are the integers, adds
//     floor(w * v / 2^16).  acc starts at 1.5 * 2^23 and moves by at most
//     max|v| + (number of keys) < 2^22, since the weights sum to at most ONE.
//     Chunks with wider values take 64-bit terms.
//     CTAs that share a lane add their sums with atomics (integers: any order
//     gives the same), two int32 in one 64-bit word; the last to arrive writes.
//
// Measured with nothing left in L2 and t_lim at the longest lane's keys, a call
// (in brackets: one of a row of calls) and its kernels 0 to 3 by themselves: 4
// lanes of 64 nodes, 64 heads over 8 KV heads, up to 1552 keys 314 us [309] (9,
// 88, 31, 198); 9 nodes, 30 thousand keys 362 us [354] (5, 118, 38, 210: K and V,
// 493 MB, at 1.4 TB/s); 8 lanes of 31 nodes, 32 heads, up to 528 keys 122 us [116]
// (6, 41, 13, 64); 16 nodes, 402 keys 37 us [32]; 5 nodes, 42 keys, 4 heads 24 us
// [17].  A larger t_lim costs score CTAs that find no keys, workspace, and the
// form of two kernels: at 2048, in a row of calls, 312, 135, 39 and 21 us.
// Values of 62.0 and more, or keys and queries of more than 32 bits, take 64-bit
// products: 31 nodes a lane 1390 or 1580 us, 30 thousand keys 5.6 or 8.7 ms; rows
// whose exps sum to 2^30 (flat scores over 16 thousand keys) 64-bit divisions:
// 30 thousand keys 489 us.
#include <atomic>

#include "../common/tree.h"
#include "common.cuh"
#include "exp32.cuh"

using namespace q16;

namespace at {

constexpr int PAGE = tree::PAGE;
constexpr int TILE = 128;           // keys per score CTA
constexpr int RQ = 32;              // query rows per MMA group
constexpr int PLANES = 4;           // digits that take the tensor path
constexpr int NT_S = 256;           // k_scores threads
constexpr int NT_V = 256;           // k_sums and k_values threads, at most
constexpr int MAX_RG = 128;         // rows per k_values CTA
constexpr int SMALL = 1 << 29;      // bound of scores stored as they are
constexpr int FAR = -(1 << 30);     // a score whose exp is 0
constexpr int64_t NONE = -(int64_t(1) << 62);  // max of no keys
constexpr int VMAX = (1 << 22) - (1 << 17);    // values of the single-precision form
constexpr int SMEM_V = 2 * (32 * (128 * 8 + MAX_RG * 4) + MAX_RG * 8);  // k_values shared memory, at most
// Rows * keys of a lane and KV head up to which two kernels do the work of four (FEW).
// Measured, two against four: 32 heads of 128, one lane, 16 rows, 250 keys 34 / 37 us, 506 keys
// 40 / 44, 1018 keys 54 / 51; 31 rows of 250 keys 40 / 42; 4 lanes of 31 rows 65 / 64; 16 lanes
// of 8 rows, 250 keys 116 / 119; 64 heads over 8, 4 nodes, 250 keys 38 / 39, 506 keys 42 / 41.
constexpr int FEW_MOST = 1 << 13;
constexpr int MAX_RANGE = 1 << 16;             // keys per k_values CTA: VMAX + MAX_RANGE < 2^22

struct Args {
  const int64_t* q;
  const int64_t* Kc;
  const int64_t* Vc;
  const int* pt;
  const int* base;
  const int* n_tree;
  const int64_t* mask;
  int64_t pt_stride, attn_scale;
  int n_pages, width, nq, n_heads, n_kv, dh, t_lim, B, lane0, lanes;
  int R, Rp, G, tiles, chunks, groups, RG, splits, rows_s, qgroups;
  // workspace
  int* S;              // [lanes][n_kv][tiles][groups][TILE][RG] scores less ref
  int64_t* ref;        // [lanes][n_kv][tiles][Rp]: 0, or the tile's max where scores are not small
  int64_t* M;          // [lanes][n_kv][tiles][Rp]: the tile's max (FEW)
  uint8_t* planes;     // [lanes][n_kv][qgroups][PLANES][RQ][128] query digits, swizzled
  uint4* qinfo;        // [lanes][n_kv][qgroups] ors of low and high digit words, largest magnitude
  int64_t* wide;       // [n_kv][groups][splits + lanes][RG][dh]: 64-bit terms of a segment
  // set to NONE and to zero by k_queries:
  int64_t* gmax;       // [lanes][n_kv][Rp] rows' largest scores
  uint64_t* sums;      // [lanes][n_kv][Rp] of exps
  uint64_t* acc;       // [lanes][n_kv][groups][RG][dh / 2]: two int32 sums each
  int* arrived;        // [lanes][n_kv][groups]
  int* bad;            // [lanes]
  int* is_wide;        // [n_kv][groups][splits + lanes]
  int8_t* X;
  int* lmax;
  int64_t* o_out;
  int* err;
};

// What a tile's stored scores need added to be relative to the row's max.  A
// score that is not seen is stored as FAR; both clamps leave its exp 0 and
// the sum within int32.  EXP_AT more: exp32's second argument.
__device__ __forceinline__ int rebase(int64_t ref, int64_t row_max) {
  const int64_t d = ref - row_max;
  return (d < FAR ? FAR : (d > SMALL ? SMALL : (int)d)) + EXP_AT;
}

// Four int64 -> digit words: plane l's word in p[l]; the low and high digit
// words are or-ed into lo / hi.
__device__ __forceinline__ void digits4(const int64_t* x, uint32_t* p, uint32_t& lo, uint32_t& hi) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t y = ((uint64_t)x[i] + 0x8080808080808080ull) ^ 0x8080808080808080ull;
    w[i] = (uint32_t)y;
    lo |= w[i];
    hi |= (uint32_t)(y >> 32);
  }
  const uint32_t t0 = __byte_perm(w[0], w[1], 0x5140), t1 = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t t2 = __byte_perm(w[0], w[1], 0x7362), t3 = __byte_perm(w[2], w[3], 0x7362);
  p[0] = __byte_perm(t0, t1, 0x5410);
  p[1] = __byte_perm(t0, t1, 0x7632);
  p[2] = __byte_perm(t2, t3, 0x5410);
  p[3] = __byte_perm(t2, t3, 0x7632);
}
// The largest |x| of four values that fit in 32 bits (one less for a negative x).
__device__ __forceinline__ uint32_t magnitude4(const int64_t* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, (uint32_t)(x[i] ^ (x[i] >> 63)));
  return m;
}
// Digit planes that an or of low digit words needs.
__device__ __forceinline__ int planes_of(uint32_t lo) { return lo >> 24 ? 4 : lo >> 16 ? 3 : lo >> 8 ? 2 : 1; }

__device__ __forceinline__ void load4(int64_t* x, const int64_t* src) {
  const longlong2 a = __ldg((const longlong2*)src), b = __ldg((const longlong2*)src + 1);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// ----------------------------------------------------------------- 0. queries
// Digit planes of query rows r0 .. r0 + RQ - 1 into out, and into info (zero
// before) the ors of their low and high digit words and the largest magnitude.
// All NT_S threads call it.
template <int DHP>
__device__ __forceinline__ void query_planes(const Args& A, int lane, int kvh, int r0, uint8_t* out, uint32_t* info) {
  constexpr int TPR = DHP / 4, QN = RQ * TPR / NT_S;
  const int tid = threadIdx.x, col = (tid % TPR) * 4;
  int64_t x[QN][4];
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int rr = r0 + tid / TPR + i * (NT_S / TPR);
    if (rr < A.R && col < A.dh)
      load4(x[i], A.q + ((size_t)(lane * A.nq + rr / A.G) * A.n_heads + kvh * A.G + rr % A.G) * A.dh + col);
    else
      x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0;
  }
  uint32_t lo = 0, hi = 0, mag = 0;
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int r = tid / TPR + i * (NT_S / TPR);
    uint32_t d[4];
    digits4(x[i], d, lo, hi);
    mag = max(mag, magnitude4(x[i]));
    const uint32_t at = r * 128 + (((col >> 4) ^ (r & 7)) << 4) + (col & 15);
#pragma unroll
    for (int l = 0; l < PLANES; ++l) *(uint32_t*)(out + l * (RQ * 128) + at) = d[l];
  }
  lo = __reduce_or_sync(0xffffffffu, lo);
  hi = __reduce_or_sync(0xffffffffu, hi);
  mag = __reduce_max_sync(0xffffffffu, mag);
  if ((tid & 31) == 0) {
    atomicOr(&info[0], lo);
    atomicOr(&info[1], hi);
    atomicMax(&info[2], mag);
  }
}

// Start values of what the later kernels add to, for lane z of the launch and
// KV head kvh; CTA i of n writes its part.
__device__ __forceinline__ void start_values(const Args& A, int z, int kvh, int i, int n) {
  const int tid = threadIdx.x;
  const size_t lk = (size_t)z * A.n_kv + kvh;
  ulonglong2* acc = (ulonglong2*)(A.acc + lk * A.groups * A.RG * (A.dh / 2));
  for (int k = i * NT_S + tid; k < A.groups * A.RG * (A.dh / 4); k += n * NT_S) acc[k] = make_ulonglong2(0, 0);
  for (int k = i * NT_S + tid; k < A.Rp; k += n * NT_S) {
    A.sums[lk * A.Rp + k] = 0;
    A.gmax[lk * A.Rp + k] = NONE;
  }
  if (i == 0) {
    for (int k = tid; k < A.groups; k += NT_S) A.arrived[lk * A.groups + k] = 0;
    if (kvh == 0 && tid == 0) A.bad[z] = 0;
    if (z == 0)
      for (int k = tid; k < A.groups * (A.splits + A.lanes); k += NT_S)
        A.is_wide[(size_t)kvh * A.groups * (A.splits + A.lanes) + k] = 0;
  }
}

// grid (qgroups, n_kv, lanes): query digits in the layout that k_scores
// copies, and the start values.
template <int DHP>
__global__ void __launch_bounds__(NT_S) k_queries(const __grid_constant__ Args A) {
  __shared__ uint32_t info[3];
  const int tid = threadIdx.x, g = blockIdx.x, kvh = blockIdx.y;
  const size_t at = ((size_t)blockIdx.z * A.n_kv + kvh) * A.qgroups + g;
  if (tid < 3) info[tid] = 0;
  __syncthreads();
  pdl_wait_dep();
  pdl_allow_next();
  start_values(A, blockIdx.z, kvh, g, A.qgroups);
  query_planes<DHP>(A, A.lane0 + blockIdx.z, kvh, g * RQ, A.planes + at * (PLANES * RQ * 128), info);
  __syncthreads();
  if (tid == 0) A.qinfo[at] = make_uint4(info[0], info[1], info[2], 0);
}

// ------------------------------------------------------------------ 1. scores
__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// grid (tiles, n_kv * row blocks of rows_s, lanes).
// Two CTAs an SM take turns at the tensor cores, the loads of K (two rounds of
// 64 KB a CTA) and the epilogues, of which each group of 32 rows costs about 2300
// cycles, its products 1300 and the steps between them 1500; a ninth warp that
// issues the products a group ahead took the same time (wide trees 84 us against
// 88, long ones 122 against 119), and so did K's second round fetched ahead.
// DHP: row pitch class of the planes (64 or 128 >= dh).
// FEW: at most RQ rows, whose digits each CTA makes itself; the tiles' maxima
// are stored for k_values, which does k_sums' work too: two launches.
template <int DHP, bool FEW>
__global__ void __launch_bounds__(NT_S, 2) k_scores(const __grid_constant__ Args A) {
  constexpr int KP = TILE * 128, QP = RQ * 128;  // bytes per plane
  constexpr int TPR = DHP / 4;                   // threads per row
  constexpr int TMEM_COLS = 256;                 // (2 * PLANES - 1) * RQ = 224 used
  extern __shared__ __align__(1024) uint8_t dsm[];
  __shared__ int64_t wmax[2][4][RQ];
  __shared__ uint64_t qmask[2][RQ];
  __shared__ int pages[TILE / PAGE];
  __shared__ uint32_t or_k[3], or_q[3];  // ors of the keys' (queries') low and high digit words, largest magnitude
  __shared__ uint32_t tslot;
  __shared__ __align__(8) uint64_t done, qfull[2];
  __shared__ int s_abort;
  const int tid = threadIdx.x, ln = tid & 31, w = tid >> 5;
  const int rbs = (A.R + A.rows_s - 1) / A.rows_s;
  const int tile = blockIdx.x, kvh = blockIdx.y / rbs, lane = A.lane0 + blockIdx.z;
  const int r_lo = (blockIdx.y % rbs) * A.rows_s, r_hi = min(A.R, r_lo + A.rows_s);
  const size_t lk = (size_t)blockIdx.z * A.n_kv + kvh;
  const uint32_t kbase = (smem_u32(dsm) + 1023u) & ~1023u, qbase = kbase + PLANES * KP;
  uint8_t* kp = dsm + (kbase - smem_u32(dsm));
  if (w == 0) {
    tmem_alloc(smem_u32(&tslot), TMEM_COLS);
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(smem_u32(&done), 1);
    mbar_init(smem_u32(&qfull[0]), 1);
    mbar_init(smem_u32(&qfull[1]), 1);
    fence_barrier_init();
    s_abort = 0;
  }
  if (tid < 3) or_k[tid] = or_q[tid] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  // the dependents start only after every CTA of this grid holds its TMEM
  pdl_wait_dep();
  pdl_allow_next();
  const int base = A.base[lane], nt = A.n_tree[lane];
  const int T = tree::lane_keys(base, nt, A.t_lim, A.width);
  const int j0 = tile * TILE;
  const bool live = j0 < T;
  if (live && tid < TILE / PAGE) {
    const int j = j0 + tid * PAGE;
    const int p = j < T ? A.pt[lane * A.pt_stride + j / PAGE] : -1;
    pages[tid] = tree::page_ok(p, A.n_pages) ? p : -1;
  }
  auto load_q = [&](int r0, int b) {  // one thread: the planes of rows r0 .. r0 + RQ - 1 into buffer b
    const uint32_t bar = smem_u32(&qfull[b]);
    mbar_arrive_expect_tx(bar, PLANES * QP);
    bulk_g2s(qbase + b * PLANES * QP, A.planes + (lk * A.qgroups + r0 / RQ) * (PLANES * QP), PLANES * QP, bar);
  };
  if constexpr (FEW) start_values(A, blockIdx.z, kvh, tile, gridDim.x);
  if (!FEW && live && tid == 0) load_q(r_lo, 0);
  __syncthreads();
  if (live) {
    if constexpr (FEW) query_planes<DHP>(A, lane, kvh, 0, kp + PLANES * KP, or_q);
    const int col = (ln % TPR) * 4;
    // ---- K digit planes: a warp reads 32 / TPR whole rows at a time
    constexpr int RPW = 32 / TPR, STEPS = TILE / (8 * RPW), UN = STEPS < 8 ? STEPS : 8;
    uint32_t lo = 0, hi = 0, mag = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < STEPS; s0 += UN) {
      int64_t x[UN][4];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = ((s0 + u) * 8 + w) * RPW + ln / TPR, p = pages[r / PAGE];
        if (col < A.dh && p >= 0 && j0 + r < T)
          load4(x[u], A.Kc + (((size_t)p * A.n_kv + kvh) * PAGE + r % PAGE) * A.dh + col);
        else
          x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0;
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = ((s0 + u) * 8 + w) * RPW + ln / TPR;
        uint32_t d[4];
        digits4(x[u], d, lo, hi);
        mag = max(mag, magnitude4(x[u]));
        const uint32_t at = r * 128 + (((col >> 4) ^ (r & 7)) << 4) + (col & 15);
#pragma unroll
        for (int l = 0; l < PLANES; ++l) *(uint32_t*)(kp + l * KP + at) = d[l];
      }
    }
    lo = __reduce_or_sync(0xffffffffu, lo);
    hi = __reduce_or_sync(0xffffffffu, hi);
    mag = __reduce_max_sync(0xffffffffu, mag);
    if (ln == 0) {
      atomicOr(&or_k[0], lo);
      atomicOr(&or_k[1], hi);
      atomicMax(&or_k[2], mag);
    }
    const int j = j0 + (w & 3) * 32 + ln;  // this thread's key in the epilogue
    const size_t group_elems = (size_t)TILE * A.RG;
    int* S0 = A.S + (lk * A.tiles + tile) * A.groups * group_elems;
    const int kend = (A.dh + 31) / 32;
    const bool all_seen = j0 + TILE <= base;  // every key of the tile is below the tree
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    const int lk_n = planes_of(or_k[0]);
    uint32_t products = 0;  // groups that took the tensor path
    const uint64_t small_lim = (uint64_t(1) << 47) / A.dh;
    const uint64_t kd = sw128_kmajor_desc(kbase), qd0 = sw128_kmajor_desc(qbase);  // start addresses count in 16 bytes
    const uint4* qinfo = A.qinfo + lk * A.qgroups + r_lo / RQ;
    uint4 q_next = FEW ? make_uint4(or_q[0], or_q[1], or_q[2], 0) : __ldg(qinfo);
    for (int r0 = r_lo, n = 0; r0 < r_hi; r0 += RQ, ++n) {
      const int rows = min(RQ, r_hi - r0), b = n & 1;
      const uint4 qi = q_next;
      if (r0 + RQ < r_hi) q_next = __ldg(qinfo + n + 1);
      const int lq_n = planes_of(qi.x);
      const bool wide = (or_k[1] | qi.y) != 0;
      // |q.k| <= dh * max|k| * max|q| < 2^47 and scale <= ONE / 4: 32 bits hold
      // every step below, and |score| <= 2^29
      const bool small = !wide && A.attn_scale >= 0 && A.attn_scale <= ONE / 4 &&
                         ((uint64_t)or_k[2] + 1) * ((uint64_t)qi.z + 1) < small_lim;
      if (!all_seen && tid < RQ)
        qmask[b][tid] = tid < rows ? (uint64_t)A.mask[(size_t)lane * A.nq + (r0 + tid) / A.G] : 0;
      if (tid == 0) {
        // the other buffer's products are done (waited for by all before the last barrier)
        if (r0 + RQ < r_hi) load_q(r0 + RQ, b ^ 1);
        if (!FEW && !mbar_wait(smem_u32(&qfull[b]), (n >> 1) & 1)) s_abort = 1;
        if (!wide) {
          // K_a times the stacked planes Q_0 | Q_1 | ..: plane b lands in accumulator a + b.
          // At k = 0 the accumulator that a reaches first is overwritten, by a product of its own.
          const uint64_t qd = qd0 + b * (PLANES * QP / 16);
          const uint32_t all = idesc_i8(TILE, lq_n * RQ), most = idesc_i8(TILE, (lq_n - 1) * RQ), one = idesc_i8(TILE, RQ);
          for (int a = 0; a < lk_n; ++a) {
            const uint64_t ka = kd + a * (KP / 16);
            const uint32_t acc = tmem + a * RQ;
            if (a == 0) {
              mma_i8(acc, ka, qd, all, 0u);
            } else {
              if (lq_n > 1) mma_i8(acc, ka, qd, most, 1u);
              mma_i8(acc + (lq_n - 1) * RQ, ka, qd + (lq_n - 1) * (QP / 16), one, 0u);
            }
#pragma unroll
            for (int k = 1; k < DHP / 32; ++k)  // 32 bytes along the planes' rows
              if (k < kend) mma_i8(acc, ka + 2 * k, qd + 2 * k, all, 1u);
          }
          mma_commit(smem_u32(&done));
        }
      }
      if (!all_seen) __syncthreads();  // qmask
      if (!wide) {
        if (!mbar_wait(smem_u32(&done), products & 1)) s_abort = 1;
        ++products;
        tc_fence_after();
      }
      // ---- scores of 16 rows per warp: rows c0 .. c0 + 15 of the group
      const int c0 = (w >> 2) * 16, ns = lk_n + lq_n - 1;
      const uint32_t tcol = tmem + ((uint32_t)(w & 3) << 21) + c0;
      if (c0 < rows) {
        uint32_t seen = 0xffff;  // bit i: row c0 + i sees this key
        if (!all_seen) {
          seen = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (tree::visible(j, base, nt, qmask[b][c0 + i])) seen |= 1u << i;
        }
        int out[16];
        if (small) {
          // dot >> 16 = D_2 + (D_3 << 8) + (D_4 << 16) + .. + ((D_0 + (D_1 << 8)) >> 16): modulo 2^32
          uint32_t r[16], t[16];
          tmem_ld16(tcol, t);
          if (ns > 1) {
            tmem_ld16(tcol + RQ, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) t[i] += r[i] << 8;
          } else {
            tmem_ld_wait();
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = (uint32_t)((int)t[i] >> 16);
#pragma unroll
          for (int s = 2; s < 2 * PLANES - 2; ++s)  // D_6 << 32 is 0
            if (s < ns) {
              tmem_ld16(tcol + s * RQ, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) t[i] += r[i] << (8 * s - 16);
            }
          const int sc = (int)A.attn_scale << 16;  // (x * scale) >> 16 = the high word of x * (scale << 16)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            out[i] = __mulhi((int)t[i], sc);
            if (!all_seen && !(seen >> i & 1)) out[i] = FAR;
          }
        } else {
          int64_t sc[16], m64 = NONE;  // lane i: max of row c0 + i over the warp's keys
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[i] = 0;
          if (!wide) {
#pragma unroll 1
            for (int s = 0; s < ns; ++s) {
              uint32_t r[16];
              tmem_ld16(tcol + s * RQ, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[i] += (int64_t)((uint64_t)(int64_t)(int)r[i] << (8 * s));
            }
          } else {
            const int p = pages[(j - j0) / PAGE];
            const int64_t* kr = A.Kc + (((size_t)(p < 0 ? 0 : p) * A.n_kv + kvh) * PAGE + j % PAGE) * A.dh;
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
              uint64_t d = 0;
              const int rr = r0 + c0 + i;
              if (p >= 0 && j < T && c0 + i < rows) {
                const int64_t* qr =
                    A.q + ((size_t)(lane * A.nq + rr / A.G) * A.n_heads + kvh * A.G + rr % A.G) * A.dh;
                for (int e = 0; e < A.dh; ++e) d += (uint64_t)wmul(qr[e], kr[e]);
              }
#pragma unroll
              for (int m = 0; m < 16; ++m)
                if (m == i) sc[m] = (int64_t)d;
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sc[i] = attn_score(sc[i], A.attn_scale);
            int64_t m = seen >> i & 1 ? sc[i] : NONE;
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) {
              const int64_t o = shfl_xor_i64(m, x);
              m = o > m ? o : m;
            }
            if (ln == i) m64 = m;
          }
          if (ln < 16) wmax[b][w & 3][c0 + ln] = m64;
          asm volatile("bar.sync %0, 128;" ::"r"(1 + (w >> 2)) : "memory");  // the four warps of these rows
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            int64_t m = wmax[b][0][c0 + i];
#pragma unroll
            for (int k = 1; k < 4; ++k) m = wmax[b][k][c0 + i] > m ? wmax[b][k][c0 + i] : m;
            const int64_t d = sc[i] - m;
            out[i] = (seen >> i & 1) && d > FAR ? (int)d : FAR;
          }
        }
        // Four lanes' scores of 16 rows become each lane's of four rows of the four keys, so that
        // a store writes whole 64-byte pieces of a key's rows.
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
          const bool up = ln & x;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (!(q & x))
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                int &lo_ = out[4 * q + i], &hi_ = out[4 * (q + x) + i];
                const int got = __shfl_xor_sync(0xffffffffu, up ? lo_ : hi_, x);
                (up ? lo_ : hi_) = got;
              }
        }
        // 16 rows lie in one group: RG is a multiple of 16, or the only group's 8
        const int c4 = c0 + 4 * (ln & 3);
        int* dst = S0 + (size_t)((r0 + c0) / A.RG) * group_elems + (r0 + c4) % A.RG;
        if (c4 < rows)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *(int4*)(dst + ((w & 3) * 32 + (ln & ~3) + k) * A.RG) =
                make_int4(out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
        if (small) {  // the rows' maxima over the warp's keys
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            int m = max(max(out[i], out[4 + i]), max(out[8 + i], out[12 + i]));
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, x));
            if (ln < 4) wmax[b][w & 3][c4 + i] = m == FAR ? NONE : m;
          }
        }
      }
      tc_fence_before();
      __syncthreads();  // wmax; this group's accumulators and query planes are read
      tc_fence_after();
      if (tid < rows) {
        int64_t m = wmax[b][0][tid];
#pragma unroll
        for (int k = 1; k < 4; ++k) m = wmax[b][k][tid] > m ? wmax[b][k][tid] : m;
        A.ref[(lk * A.tiles + tile) * A.Rp + r0 + tid] = small ? 0 : m;
        if (FEW) A.M[(lk * A.tiles + tile) * A.Rp + r0 + tid] = m;
        else if (m != NONE) atomicMax((long long*)A.gmax + lk * A.Rp + r0 + tid, (long long)m);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s_abort) set_error(A.err, ARCB_ERR_TIMEOUT_DONE);
  if (w == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// -------------------------------------------------------------------- 2. sums
// grid (chunks, n_kv * groups, lanes): a thread takes four rows of every
// (threads / (RG / 4))-th key.  About 20 instructions an exp and a table lookup:
// 19 million exps of 77 MB in 31 us.
__global__ void __launch_bounds__(NT_V) k_sums(const __grid_constant__ Args A) {
  __shared__ int2 lut[EXP_TABLE_N];
  __shared__ int64_t rmax[MAX_RG];
  __shared__ uint32_t rlow[MAX_RG], rhigh[MAX_RG];  // sums of 24-bit words: 64-bit shared atomics are loops
  const int NT = blockDim.x, tid = threadIdx.x, RG = A.RG;
  load_exp(lut, NT);
  pdl_wait_dep();
  pdl_allow_next();
  const int kvh = blockIdx.y / A.groups, grp = blockIdx.y % A.groups, r0 = grp * RG, rows = min(RG, A.R - r0);
  const int lane = A.lane0 + blockIdx.z, T = tree::lane_keys(A.base[lane], A.n_tree[lane], A.t_lim, A.width);
  if (T <= 0) return;
  const size_t lk = (size_t)blockIdx.z * A.n_kv + kvh;
  const int nt = (T + TILE - 1) / TILE, X = min((int)gridDim.x, nt);
  if ((int)blockIdx.x >= X) return;
  const int t0 = (int)((int64_t)blockIdx.x * nt / X), t1 = (int)((int64_t)(blockIdx.x + 1) * nt / X);
  const int64_t* ref = A.ref + lk * A.tiles * A.Rp + r0;
  if (tid < RG) rmax[tid] = tid < rows ? A.gmax[lk * A.Rp + r0 + tid] : NONE, rlow[tid] = rhigh[tid] = 0;
  __syncthreads();
  const int q = tid % (RG / 4) * 4, k0 = tid / (RG / 4), kl = NT / (RG / 4);
  uint64_t s[4] = {0, 0, 0, 0};
  for (int t = t0; t < t1; ++t) {
    int off[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) off[c] = q + c < rows ? rebase(ref[(size_t)t * A.Rp + q + c], rmax[q + c]) : FAR;
    const int* S = A.S + ((lk * A.tiles + t) * A.groups + grp) * (size_t)TILE * RG + q;
    uint32_t p[4] = {0, 0, 0, 0};  // at most TILE exps
#pragma unroll 8
    for (int k = k0; k < TILE; k += kl) {
      const int4 x = *(const int4*)(S + k * RG);
      p[0] += exp32(x.x, off[0], lut);
      p[1] += exp32(x.y, off[1], lut);
      p[2] += exp32(x.z, off[2], lut);
      p[3] += exp32(x.w, off[3], lut);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] += p[c];
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (q + c < rows) {
      atomicAdd(&rlow[q + c], (uint32_t)s[c] & 0xffffff);
      if (s[c] >> 24) atomicAdd(&rhigh[q + c], (uint32_t)(s[c] >> 24));
    }
  __syncthreads();
  if (tid < rows)
    atomicAdd((unsigned long long*)A.sums + lk * A.Rp + r0 + tid, rlow[tid] + ((unsigned long long)rhigh[tid] << 24));
}

// ------------------------------------------------------------------ 3. values
// 8 consecutive digits planes of four int64 outputs, and their limb count.
__device__ __forceinline__ int store_limbs4(int8_t* X, int slot, int B, size_t ldx, size_t col, const int64_t* o) {
  int need = 0;
  uint32_t lo[4], hi[4], l4 = 0, h4 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t y = ((uint64_t)o[i] + 0x8080808080808080ull) ^ 0x8080808080808080ull;
    lo[i] = (uint32_t)y;
    hi[i] = (uint32_t)(y >> 32);
    l4 |= lo[i];
    h4 |= hi[i];
  }
  need = h4 ? 4 + planes_of(h4) : (l4 ? planes_of(l4) : 0);
#pragma unroll
  for (int l = 0; l < 8; ++l) {
    const uint32_t* v = l < 4 ? lo : hi;
    const int s = 8 * (l & 3);
    const uint32_t word = (v[0] >> s & 255u) | (v[1] >> s & 255u) << 8 | (v[2] >> s & 255u) << 16 | (v[3] >> s & 255u) << 24;
    *(uint32_t*)(X + limb_row(l, slot, B) * ldx + col) = word;
  }
  return need;
}

// grid (splits, n_kv * groups).  The lanes' chunks of CK keys, one after
// another, are divided evenly over the splits; a CTA works through its part
// of each lane that it touches (a segment).  V pages and scores come by bulk
// copies, one chunk ahead.  A warp takes UR rows (unit) x all dims, a lane
// the dims 2 ln, 2 ln + 1 (and 64 + those); kparts warps per unit take every
// kparts-th key.
// Bound by the FMAs and what feeds them: of 130 million warp instructions for 4 x
// 64 nodes, 58 % are FMAs (their pipe 49 % busy, issue slots 65 %), the rest the
// weights, the conversion of V and the loads from shared memory.  FMAs of two
// terms run at the same rate and cost moves; warps that only convert and weigh
// while others add were no faster.
// FEW: at most RQ rows (one group) of few keys; each segment finds its rows'
// maxima and sums from all scores of the lane.
template <int DPL, int UR, int CK, bool FEW>
__global__ void __launch_bounds__(NT_V, 2) k_values(const __grid_constant__ Args A) {
  extern __shared__ __align__(1024) uint8_t dsm[];
  constexpr int DHP = 32 * DPL;
  __shared__ int2 lut[EXP_TABLE_N];
  __shared__ int64_t rmax[MAX_RG];
  __shared__ uint64_t rsum[MAX_RG];
  __shared__ __align__(16) float rrcp[MAX_RG];     // ONE / sum
  __shared__ __align__(16) uint32_t rden[MAX_RG];  // sum
  __shared__ __align__(8) uint64_t full[2];
  __shared__ int s_last, s_need, s_long;
  const int NT = blockDim.x, tid = threadIdx.x, ln = tid & 31, w = tid >> 5;
  const int RG = A.RG, units = RG / UR, unit = w % units, kpart = w / units, kparts = NT / 32 / units;
  const int vbytes = CK * A.dh * 8, sbytes = CK * RG * 4;
  uint8_t* vbuf = dsm;                                 // 2 x [CK][dh] int64
  float* wbuf = (float*)(dsm + 2 * vbytes);            // 2 x [CK][RG] scores, then weights in place
  int64_t* rbuf = (int64_t*)(dsm + 2 * (vbytes + sbytes));  // 2 x [RG] what the scores are relative to
  int* osum = (int*)dsm;                               // [RG][DHP] at a segment's end
  load_exp(lut, NT);
  if (tid == 0) {
    s_need = 0;
    mbar_init(smem_u32(&full[0]), 1);
    mbar_init(smem_u32(&full[1]), 1);
    fence_barrier_init();
  }
  pdl_wait_dep();
  pdl_allow_next();
  const int kvh = blockIdx.y / A.groups, grp = blockIdx.y % A.groups, r0 = grp * RG, rows = min(RG, A.R - r0);
  auto chunks_of = [&](int T) { return T > 0 ? (T + CK - 1) / CK : 1; };  // a lane without keys: one, for its zeros
  int64_t N = 0;
  for (int b = 0; b < A.lanes; ++b)
    N += chunks_of(tree::lane_keys(A.base[A.lane0 + b], A.n_tree[A.lane0 + b], A.t_lim, A.width));
  const int64_t x = blockIdx.x, X = N < (int64_t)gridDim.x ? N : (int64_t)gridDim.x;
  if (x >= X) return;
  const int64_t c_lo = x * N / X, c_hi = (x + 1) * N / X;
  // the softmax rows of this thread's quad in the weight stage: NT is a multiple of RG / 4
  const int rq = tid % (RG / 4) * 4, kq = tid / (RG / 4), kq_step = NT / (RG / 4);
  uint32_t issued = 0, used = 0;  // chunks
  int need = 0;
  int64_t off = 0;
  for (int bz = 0; bz < A.lanes && off < c_hi; ++bz) {
    const int lane = A.lane0 + bz;
    int T = tree::lane_keys(A.base[lane], A.n_tree[lane], A.t_lim, A.width);
    const int n = chunks_of(T);
    const int64_t first = off;
    off += n;
    if (off <= c_lo) continue;
    const int a0 = (int)(c_lo > first ? c_lo - first : 0), a1 = (int)(c_hi < off ? c_hi - first : n);
    // CTAs that share the lane
    const int64_t xf = ((first + 1) * X - 1) / N, xl = (off * X - 1) / N;
    const size_t lk = (size_t)bz * A.n_kv + kvh, lkg = lk * A.groups + grp;
    const int* pt = A.pt + lane * A.pt_stride;
    // the segment's slot for 64-bit terms: x + bz differs from any other's
    const size_t slot0 = (size_t)blockIdx.y * (gridDim.x + A.lanes) + bz;
    int64_t* part = A.wide + (slot0 + x) * RG * A.dh;
    bool bad = T < 0;
    for (int i = a0 * (CK / PAGE) + tid; !bad && i < min(a1 * (CK / PAGE), (T + PAGE - 1) / PAGE); i += NT)
      bad |= !tree::page_ok(pt[i], A.n_pages);
    if (tid == 0) s_long = 0;
    bad = __syncthreads_or(bad);
    if (bad && tid == 0) {
      set_error(A.err, T < 0 ? ARCB_ERR_SEQ_OVERFLOW : ARCB_ERR_BOUNDS);
      atomicOr(A.bad + bz, 1);
    }
    const bool live = T > 0 && !bad;
    if (FEW && live) {
      const int nt = (T + TILE - 1) / TILE;
      if (tid < RG) {
        int64_t m = NONE;
        if (tid < rows)
#pragma unroll 4
          for (int t = 0; t < nt; ++t) m = max(m, A.M[(lk * A.tiles + t) * A.Rp + tid]);
        rmax[tid] = m;
        rden[tid] = 0;
      }
      __syncthreads();
      uint32_t s[4] = {0, 0, 0, 0};  // FEW_MOST exps at most
      for (int t = 0; t < nt; ++t) {
        const int64_t* ref = A.ref + (lk * A.tiles + t) * A.Rp + rq;
        const int* S = A.S + (lk * A.tiles + t) * (size_t)TILE * RG + rq;
        int off4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) off4[c] = rq + c < rows ? rebase(ref[c], rmax[rq + c]) : FAR;
        const int k1 = min(TILE, T - t * TILE);  // keys behind are as far as unseen ones
#pragma unroll 4
        for (int k = kq; k < k1; k += kq_step) {
          const int4 v = *(const int4*)(S + k * RG);
          s[0] += exp32(v.x, off4[0], lut);
          s[1] += exp32(v.y, off4[1], lut);
          s[2] += exp32(v.z, off4[2], lut);
          s[3] += exp32(v.w, off4[3], lut);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (rq + c < rows) atomicAdd(&rden[rq + c], s[c]);
      __syncthreads();
    }
    if (live && tid < RG) {
      const bool row = tid < rows;
      const uint64_t s = FEW ? rden[tid] : (row ? A.sums[lk * A.Rp + r0 + tid] : 0);
      if (!FEW) rmax[tid] = row ? A.gmax[lk * A.Rp + r0 + tid] : NONE;
      rsum[tid] = s ? s : 1;  // a row without keys: every exp is 0
      rden[tid] = (uint32_t)rsum[tid];
      rrcp[tid] = 65536.0f * __frcp_rn((float)(int64_t)rsum[tid]);
      if (s >> 30) s_long = 1;
    }
    float acc[DPL][UR];
#pragma unroll
    for (int d = 0; d < DPL; ++d)
#pragma unroll
      for (int i = 0; i < UR; ++i) acc[d][i] = 12582912.0f;
    __syncthreads();
    bool any_wide = false;
    if (live) {
      const bool lng = s_long != 0;
      int ro[4];       // what the tile's scores need added
      int pg[CK / PAGE];  // thread 0: page ids of the chunk to issue next
      auto fetch = [&](int c) {
#pragma unroll
        for (int i = 0; i < CK / PAGE; ++i) {
          const int at = c * (CK / PAGE) + i;
          pg[i] = at < (T + PAGE - 1) / PAGE ? pt[at] : -1;
        }
      };
      auto issue = [&](int c) {  // thread 0
        const uint32_t bar = smem_u32(&full[issued & 1]), buf = issued & 1;
        const uint32_t pbytes = PAGE * A.dh * 8;
        uint32_t bytes = sbytes + RG * 8;
#pragma unroll
        for (int i = 0; i < CK / PAGE; ++i) bytes += pg[i] >= 0 ? pbytes : 0;
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int i = 0; i < CK / PAGE; ++i)
          if (pg[i] >= 0)
            bulk_g2s(smem_u32(vbuf) + buf * vbytes + i * pbytes,
                     A.Vc + ((size_t)pg[i] * A.n_kv + kvh) * PAGE * A.dh, pbytes, bar);
        const int t = c / (TILE / CK);
        bulk_g2s(smem_u32(rbuf + buf * RG), A.ref + (lk * A.tiles + t) * A.Rp + r0, RG * 8, bar);
        bulk_g2s(smem_u32(wbuf) + buf * sbytes,
                 A.S + (((lk * A.tiles + t) * A.groups + grp) * TILE + (c % (TILE / CK)) * CK) * (size_t)RG, sbytes, bar);
      };
      if (tid == 0) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // after the last segment's accesses
        fetch(a0);
        issue(a0);
        fetch(a0 + 1);
      }
      ++issued;
      for (int c = a0; c < a1; ++c) {
        const int j0 = c * CK, keys = min(CK, T - j0);
        if (c + 1 < a1) {
          if (tid == 0) {
            issue(c + 1);
            fetch(c + 2);
          }
          ++issued;
        }
        if (!mbar_wait(smem_u32(&full[used & 1]), (used >> 1) & 1)) set_error(A.err, ARCB_ERR_TIMEOUT_FULL);
        int64_t* vb = (int64_t*)(vbuf + (used & 1) * vbytes);
        float* wb = wbuf + (used & 1) * CK * RG;
        if (c == a0 || c % (TILE / CK) == 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k) ro[k] = rq + k < rows ? rebase(rbuf[(used & 1) * RG + rq + k], rmax[rq + k]) : FAR;
        }
        ++used;
        // values to single precision, v / 2^16, into the first half of each row: a warp holds
        // a whole row meanwhile.  Where they fit, y = v + VMAX is in [0, 2 VMAX]: the low bits
        // of the float 2^23 + y, then exact: (that - 2^23 - VMAX) / 2^16
        uint32_t high = 0, most = 0;
#pragma unroll 2
        for (int k = w; k < keys; k += NT / 32) {
          int64_t* row = vb + k * A.dh;
          float2 f[DPL / 2];
#pragma unroll
          for (int h = 0; h < DPL / 2; ++h) {
            const int e = 2 * ln + 64 * h;
            const longlong2 v = e < A.dh ? *(const longlong2*)(row + e) : make_longlong2(0, 0);
            const uint64_t y0 = (uint64_t)v.x + VMAX, y1 = (uint64_t)v.y + VMAX;
            high |= (uint32_t)(y0 >> 32) | (uint32_t)(y1 >> 32);
            most = max(most, max((uint32_t)y0, (uint32_t)y1));
            const float c = -(float)(8388608 + VMAX) / 65536.0f;
            f[h] = make_float2(__fmaf_rn(__uint_as_float(0x4B000000u + (uint32_t)y0), 1.0f / 65536.0f, c),
                               __fmaf_rn(__uint_as_float(0x4B000000u + (uint32_t)y1), 1.0f / 65536.0f, c));
          }
          __syncwarp();
#pragma unroll
          for (int h = 0; h < DPL / 2; ++h)
            if (2 * ln + 64 * h < A.dh) *(float2*)((float*)row + 2 * ln + 64 * h) = f[h];
        }
        // weights floor(e * ONE / sum), at most ONE, in place: the estimate e * (ONE / sum)
        // in single precision is within 1, the remainder decides (in 32 bits for sums below 2^30)
        float* wq = wb + rq;
        if (!lng) {
#pragma unroll 2
          for (int k = kq; k < CK; k += kq_step) {
            const int4 sc = *(const int4*)(wq + k * RG);
            const float4 rc = *(const float4*)(rrcp + rq);
            const uint4 de = *(const uint4*)(rden + rq);
            const int xs[4] = {sc.x, sc.y, sc.z, sc.w};
            const float rcp[4] = {rc.x, rc.y, rc.z, rc.w};
            const uint32_t den[4] = {de.x, de.y, de.z, de.w};
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t e = exp32(xs[i], ro[i], lut);
              const float qf = __fmaf_rd(__uint_as_float(0x4B000000u + e) - 8388608.0f, rcp[i], 8388608.0f);
              const int rem = (int)((e << 16) - (__float_as_uint(qf) - 0x4B000000u) * den[i]);
              o[i] = qf - (rem < 0 ? 8388609.0f : (rem >= (int)den[i] ? 8388607.0f : 8388608.0f));
            }
            *(float4*)(wq + k * RG) = make_float4(o[0], o[1], o[2], o[3]);
          }
        } else {
          for (int k = kq; k < CK; k += kq_step)
            for (int i = 0; i < 4; ++i) {
              const int64_t e = exp32(__float_as_int(wq[k * RG + i]), ro[i], lut);
              wq[k * RG + i] = (float)(int)(e * ONE / (int64_t)rsum[rq + i]);
            }
        }
        const bool fit = __syncthreads_and(high == 0 && most <= 2 * VMAX);
        if (fit) {
          const float* vrow = (const float*)vb + min(ln * DPL, A.dh - DPL);
          const float* wrow = wb + unit * UR;
#pragma unroll 1
          for (int k = kpart; k < keys; k += kparts) {  // rows behind may hold anything
            float wt[UR];
            float v[DPL];
#pragma unroll
            for (int i = 0; i < UR; i += 4) *(float4*)(wt + i) = *(const float4*)(wrow + k * RG + i);
            if constexpr (DPL == 4) *(float4*)v = *(const float4*)(vrow + k * 2 * A.dh);
            else *(float2*)v = *(const float2*)(vrow + k * 2 * A.dh);
#pragma unroll
            for (int d = 0; d < DPL; ++d)
#pragma unroll
              for (int i = 0; i < UR; ++i) acc[d][i] = __fmaf_rd(wt[i], v[d], acc[d][i]);
          }
        } else {  // 64-bit terms into this CTA's partial sums
          for (int i = tid; i < RG * A.dh; i += NT) {
            const int r = i / A.dh, e = i - r * A.dh;
            uint64_t o = any_wide ? (uint64_t)part[i] : 0;
            for (int k = 0; k < keys; ++k) {
              const int64_t wt = (int64_t)wb[k * RG + r];
              const int64_t* v = A.Vc + (((size_t)pt[(j0 + k) / PAGE] * A.n_kv + kvh) * PAGE + (j0 + k) % PAGE) * A.dh;
              if (wt) o += (uint64_t)mulshr(wt, v[e]);
            }
            part[i] = (int64_t)o;
          }
          any_wide = true;
        }
        __syncthreads();
        if (tid == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copies
      }
      for (int i = tid; i < RG * DHP; i += NT) osum[i] = 0;
      __syncthreads();
#pragma unroll
      for (int d = 0; d < DPL; ++d)
#pragma unroll
        for (int i = 0; i < UR; ++i) {
          int* o = osum + (unit * UR + i) * DHP + ln * DPL + d;
          const int a = __float_as_int(acc[d][i]) - 0x4B400000;
          if (kparts == 1) *o = a;
          else atomicAdd(o, a);
        }
      __syncthreads();
    }
    const int quads = A.dh / 4;
    bool lost = !live, wides = false;  // the lane gives zeros; some segment has 64-bit terms
    unsigned long long* acc2 = (unsigned long long*)A.acc + lkg * RG * (A.dh / 2);
    if (xl > xf) {
      if (live)
        for (int i = tid; i < rows * (A.dh / 2); i += NT) {
          const int r = i / (A.dh / 2), e = i % (A.dh / 2) * 2;
          const int2 v = *(const int2*)(osum + r * DHP + e);
          // both sums and their totals over the lane fit in int32
          atomicAdd(acc2 + i, (unsigned long long)(((int64_t)v.y << 32) + v.x));
        }
      if (any_wide && tid == 0) A.is_wide[slot0 + x] = 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(A.arrived + lkg, 1) == (int)(xl - xf);
      __syncthreads();
      if (!s_last) continue;
      __threadfence();
      lost |= __ldcg(A.bad + bz) != 0;
      for (int64_t s = xf + tid; s <= xl; s += NT) wides |= __ldcg(A.is_wide + slot0 + s) != 0;
      wides = __syncthreads_or(wides);
    }
    const size_t d = (size_t)A.n_heads * A.dh;
    for (int i = tid; i < rows * quads; i += NT) {
      const int r = i / quads, e = i % quads * 4, rr = r0 + r;
      int64_t o[4] = {0, 0, 0, 0};
      if (!lost && xl > xf) {
        const ulonglong2 v = __ldcg((const ulonglong2*)(acc2 + r * (A.dh / 2) + e / 2));
        o[0] = (int)(uint32_t)v.x, o[1] = ((int64_t)v.x - o[0]) >> 32;
        o[2] = (int)(uint32_t)v.y, o[3] = ((int64_t)v.y - o[2]) >> 32;
        for (int64_t s = xf; wides && s <= xl; ++s)
          if (__ldcg(A.is_wide + slot0 + s))
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = wadd(o[c], __ldcg(A.wide + (slot0 + s) * RG * A.dh + r * A.dh + e + c));
      } else if (!lost) {
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = wadd(osum[r * DHP + e + c], any_wide ? part[r * A.dh + e + c] : 0);
      }
      const int slot = lane * A.nq + rr / A.G;
      const size_t col = (size_t)(kvh * A.G + rr % A.G) * A.dh + e;
      if (A.o_out) {
        longlong2* p = (longlong2*)(A.o_out + slot * d + col);
        p[0] = make_longlong2(o[0], o[1]);
        p[1] = make_longlong2(o[2], o[3]);
      }
      if (A.X) need = max(need, store_limbs4(A.X, slot, A.B, d, col, o));
    }
  }
  if (A.X && A.lmax) {
    need = __reduce_max_sync(0xffffffffu, need);
    if (ln == 0 && need) atomicMax(&s_need, need);
    __syncthreads();
    if (tid == 0 && s_need) atomicMax(A.lmax, s_need);
  }
}

// Sizes that follow from the shapes; `lanes` of them per launch.
struct Plan {
  int lanes, R, Rp, G, tiles, chunks, groups, RG, splits, threads, unit, rows_s, qgroups, per_sm;
  bool few;
  size_t oS, oQ, oI, oR, oM, oG, oSum, oW, oAcc, oA, oB, oF, bytes;
};

// Lanes are batched to this many bytes of scores and of workspace in all, but one at least.
// 512 lanes of 64 nodes and 64 keys, 64 heads over 8, take 5.5 GB and 4.68 ms in one batch,
// 5.04 ms in the five that 1.25 GB hold; inputs and outputs are 4 GB and more there.
constexpr size_t WS_SCORES = size_t(1) << 30, WS_MOST = 6 * WS_SCORES;

// Whether no call takes these sizes (plan() divides by some of them, and the grids and
// 32-bit products below hold the others).
static bool refused(int lanes, int nq, int n_heads, int n_kv, int dh, int t_lim) {
  if (lanes < 1 || nq < 1 || n_kv < 1 || n_heads < 1 || n_heads % n_kv || dh < 8 || dh > 128 || dh % 8 || t_lim < 1)
    return true;
  const int64_t R = (int64_t)nq * (n_heads / n_kv);
  return (int64_t)lanes * nq > 65535 || t_lim > 65535 * 16 * TILE || n_kv * ((R + RQ - 1) / RQ) > 65535;
}

static Plan plan(int lanes, int nq, int n_heads, int n_kv, int dh, int t_lim) {
  Plan p;
  p.G = n_heads / n_kv;
  p.R = nq * p.G;
  p.groups = (p.R + MAX_RG - 1) / MAX_RG;
  // rows a warp holds: 16, or the only 8 (8 query heads of one node a lane, 32 lanes of 2000
  // keys: 307 us, padded to 16 358; 4 nodes of 8 lanes, 500 keys: 110 and 128)
  p.unit = p.R <= 8 ? 8 : 16;
  p.RG = ((p.R + p.groups - 1) / p.groups + p.unit - 1) / p.unit * p.unit;
  p.Rp = p.groups * p.RG;
  p.tiles = (t_lim + TILE - 1) / TILE;
  const int units = p.RG / p.unit;
  p.threads = 32 * units * (units >= 5 ? 1 : (units >= 3 ? 2 : (units == 2 ? 4 : 8)));
  // five-warp value CTAs run three to an SM with chunks of one page; the others two, with
  // two pages (64 nodes: 315 us, 325 with one page).  9 nodes, 8 query heads per KV head, three
  // against two, a lane of 100 / 500 / 2000 / 8000 / 30000 keys: 59 / 61 / 78 / 145 / 361 us and
  // 59 / 64 / 80 / 153 / 392; 8 lanes of 100 / 500 / 2000 / 8000 keys: 82 / 121 / 229 / 708 and
  // 70 / 123 / 244 / 762
  p.per_sm = p.threads == 160 ? 3 : 2;
  p.qgroups = (p.R + RQ - 1) / RQ;
  p.few = p.R <= RQ && (int64_t)p.RG * t_lim <= FEW_MOST;
  // the lanes' keys are divided evenly over the CTAs that run at once; a CTA's
  // part of a lane stays below MAX_RANGE keys
  p.splits = p.per_sm * 148 / (n_kv * p.groups);
  if (p.splits < 1) p.splits = 1;
  // workspace of a lane: scores, query digits, maxima and sums, output sums, and the slots of
  // 64-bit terms that it adds (its own, and its share of `least` below); and of any number of lanes
  const size_t per_s = (size_t)n_kv * p.tiles * TILE * p.Rp * 4;
  const size_t slot = (size_t)n_kv * p.groups * ((size_t)p.RG * dh * 8 + 4);
  const size_t per_lane = per_s + (size_t)n_kv * (p.qgroups * (PLANES * RQ * 128 + sizeof(uint4)) +
                                                  (size_t)p.tiles * p.Rp * (p.few ? 16 : 8) + p.Rp * 16 +
                                                  (size_t)p.groups * (p.RG * dh * 4 + 4)) +
                          4 + slot + (size_t)p.tiles * TILE * slot / (MAX_RANGE - 32) + 1;
  const size_t fixed = (p.splits + 1) * slot + 16 * 256;
  const size_t all = fixed < WS_MOST ? (WS_MOST - fixed) / per_lane : 0, scores = WS_SCORES / per_s;
  const size_t fit = all < scores ? all : scores;
  p.lanes = fit < 1 ? 1 : (fit < (size_t)lanes ? (int)fit : lanes);
  const int have = p.lanes * n_kv * p.groups;
  const int64_t least = ((int64_t)p.lanes * p.tiles * TILE + MAX_RANGE - 1) / (MAX_RANGE - 32);
  if (p.splits < least) p.splits = (int)least;
  p.chunks = (12 * 148 + have - 1) / have;  // of the sums: short ones, many loads in flight
  if (p.chunks > p.tiles) p.chunks = p.tiles;
  // score CTAs take all rows of their tile unless that leaves SMs idle (two CTAs each, and
  // tiles without keys): 4 lanes of 64 nodes in two blocks of rows 88 us, in one 103
  const int blocks = p.tiles * n_kv * p.lanes, want = (4 * 148 + blocks - 1) / blocks, most = (p.R + 63) / 64;
  p.rows_s = ((p.R + (want < most ? want : most) - 1) / (want < most ? want : most) + RQ - 1) / RQ * RQ;
  size_t o = 0;
  auto take = [&](size_t n) {
    const size_t at = o;
    o += (n + 255) / 256 * 256;
    return at;
  };
  const size_t lk = (size_t)p.lanes * n_kv;
  p.oS = take((size_t)p.lanes * per_s);
  p.oQ = take(lk * p.qgroups * PLANES * RQ * 128);
  p.oI = take(lk * p.qgroups * sizeof(uint4));
  p.oR = take(lk * p.tiles * p.Rp * 8);
  p.oM = take(p.few ? lk * p.tiles * p.Rp * 8 : 0);
  p.oG = take(lk * p.Rp * 8);
  p.oSum = take(lk * p.Rp * 8);
  const size_t slots = (size_t)n_kv * p.groups * (p.splits + p.lanes);
  p.oW = take(slots * p.RG * dh * 8);
  p.oAcc = take(lk * p.groups * p.RG * dh * 4);
  p.oA = take(lk * p.groups * 4);
  p.oB = take(p.lanes * 4);
  p.oF = take(slots * 4);
  p.bytes = o;
  return p;
}

template <int DHP, int UR, int CK, bool FEW>
static int run(Args A, const Plan& p, int lanes, cudaStream_t st) {
  constexpr int smem_s = 1024 + PLANES * (TILE + 2 * RQ) * 128;
  const int vals = 2 * (CK * (A.dh * 8 + p.RG * 4) + p.RG * 8), sums = p.RG * DHP * 4, smem_v = vals > sums ? vals : sums;
  const auto ks = k_scores<DHP, FEW>;
  const auto kv = k_values<DHP / 32, UR, CK, FEW>;
  static std::atomic<uint64_t> ready{0};  // the kernels' attributes are set, a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(ready.load() >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(ks, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_s);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kv, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_V);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  }
  if (e != cudaSuccess) return (int)e;
  for (int l0 = 0; l0 < lanes; l0 += p.lanes) {
    const int n = lanes - l0 < p.lanes ? lanes - l0 : p.lanes;
    A.lane0 = l0, A.lanes = n;
    int rc = FEW ? 0 : launch_k(k_queries<DHP>, dim3(p.qgroups, A.n_kv, n), dim3(NT_S), 0, st, A);
    if (!rc) rc = launch_k(ks, dim3(p.tiles, A.n_kv * ((p.R + p.rows_s - 1) / p.rows_s), n), dim3(NT_S), smem_s, st, A);
    if (!rc && !FEW) rc = launch_k(k_sums, dim3(p.chunks, A.n_kv * p.groups, n), dim3(p.threads), 0, st, A);
    if (!rc) rc = launch_k(kv, dim3(p.splits, A.n_kv * p.groups), dim3(p.threads), smem_v, st, A);
    if (rc) return rc;
  }
  return 0;
}

template <int DHP>
static int run_dh(const Args& A, const Plan& p, int lanes, cudaStream_t st) {
  if (p.unit == 8) return p.few ? run<DHP, 8, 32, true>(A, p, lanes, st) : run<DHP, 8, 32, false>(A, p, lanes, st);
  if (p.few) return run<DHP, 16, 32, true>(A, p, lanes, st);
  return p.per_sm == 3 ? run<DHP, 16, 16, false>(A, p, lanes, st) : run<DHP, 16, 32, false>(A, p, lanes, st);
}

}  // namespace at

extern "C" {

// Workspace bytes of arcb_attn_tree; -1 for sizes that it refuses.
int64_t arcb_attn_tree_ws(int lanes, int nq, int n_heads, int n_kv, int dh, int t_lim) {
  if (at::refused(lanes, nq, n_heads, n_kv, dh, t_lim)) return -1;
  return (int64_t)at::plan(lanes, nq, n_heads, n_kv, dh, t_lim).bytes;
}

int arcb_attn_tree(const int64_t* q, const int64_t* Kc, const int64_t* Vc, int n_pages, const int* pt,
                   int64_t pt_stride, int width, const int* base, const int* n_tree, const int64_t* mask, int nq,
                   int n_heads, int n_kv, int dh, int64_t attn_scale, int t_lim, int lanes, void* ws, int8_t* X,
                   int* lmax, int64_t* o_out, int* err, void* stream) {
  if (at::refused(lanes, nq, n_heads, n_kv, dh, t_lim) || width < 1) return -2;
  const at::Plan p = at::plan(lanes, nq, n_heads, n_kv, dh, t_lim);
  uint8_t* b = (uint8_t*)ws;
  at::Args A = {};
  A.q = q, A.Kc = Kc, A.Vc = Vc, A.pt = pt, A.base = base, A.n_tree = n_tree, A.mask = mask;
  A.pt_stride = pt_stride, A.attn_scale = attn_scale;
  A.n_pages = n_pages, A.width = width, A.nq = nq, A.n_heads = n_heads, A.n_kv = n_kv, A.dh = dh, A.t_lim = t_lim;
  A.B = lanes * nq;
  A.R = p.R, A.Rp = p.Rp, A.G = p.G, A.tiles = p.tiles, A.chunks = p.chunks, A.groups = p.groups, A.RG = p.RG;
  A.splits = p.splits, A.rows_s = p.rows_s, A.qgroups = p.qgroups;
  A.S = (int*)(b + p.oS), A.planes = b + p.oQ, A.qinfo = (uint4*)(b + p.oI), A.ref = (int64_t*)(b + p.oR);
  A.M = (int64_t*)(b + p.oM), A.gmax = (int64_t*)(b + p.oG);
  A.sums = (uint64_t*)(b + p.oSum), A.wide = (int64_t*)(b + p.oW), A.acc = (uint64_t*)(b + p.oAcc);
  A.arrived = (int*)(b + p.oA), A.bad = (int*)(b + p.oB), A.is_wide = (int*)(b + p.oF);
  A.X = X, A.lmax = lmax, A.o_out = o_out, A.err = err;
  cudaStream_t st = (cudaStream_t)stream;
  if (dh <= 64) return at::run_dh<64>(A, p, lanes, st);
  return at::run_dh<128>(A, p, lanes, st);
}

}  // extern "C"
