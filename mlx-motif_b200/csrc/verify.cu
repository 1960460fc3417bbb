// Verification of drafted tokens against the target's probabilities from given random numbers.
//
// Row 0 of a tree is the last committed token, rows 1 .. T−1 are drafted tokens, parents[i] < i. The
// law of row r is p_r = softmax(p_logits[r] / τ), the draft's is q_r. From row 0 the children c of the
// current row are tested in ascending order: c is accepted with probability min(1, w(x_c) / q(x_c)),
// where w starts as p and becomes max(0, w − q) renormalised after every rejection; an accepted child
// becomes the current row. The next token is drawn from w of the row where the walk ends. Repeating the
// residual step has a closed form: after j rejections w ∝ (p − a_j·q)⁺ with
//   a_0 = 0, S_0 = 1,   a_{j+1} = a_j + S_j,   S_j = Σ_x (p(x) − a_j·q(x))⁺,
// (by induction: w_j = (p − a_j q)⁺ / S_j, and w_j − q = (p − (a_j + S_j) q) / S_j where it is positive),
// so child c is accepted iff u_c·q(x_c)·S < (p(x_c) − a·q(x_c))⁺, and no residual is ever stored.
// Children have larger indices than their row, so one ascending pass over the rows walks the tree.
//
// The drawn token is the first x whose running sum of w exceeds u_0 times the whole. A vocabulary has
// as many borders between tokens as entries: with sums or exponentials in 32 bits (2^-24 relative) some
// 1% of the draws over 2·10^5 entries would fall to the other side of one, so they are in 64 bits.
//
// Two launches:
//   verify_stats_kernel reads every row once at memory speed: per 8192-entry chunk the maximum and Σ exp
//     against it in 32 bits (the walk repeats a test that this cannot decide with sums in 64 bits), or at
//     τ = 0 the largest logit and its first index;
//   verify_walk_kernel walks the tree, one thread-block cluster a sequence. All CTAs of a cluster take the
//     same decisions from the chunks' values; where a child is rejected they sum their parts of the row's
//     S_j in 64 bits and exchange the sums through distributed shared memory (each part added in the same
//     order by everyone, so the CTAs stay in step without another word). The draw finds the CTA, then the
//     warp's range, then the entry.
// The walk is bound by latency, step after step on one cluster: a pass over a row pair of 219520 entries is 439 k
// exponentials of nine 64-bit operations on the cluster's SMs, whose 64-bit pipes are 12 % active over a walk.
// Measured: a tree of 64 over 219520 fp16 entries 28 us (the row sums read 55.8 MB in 13, floor 8.5; the rest is
// the walk), a chain of five 20 (both rows of every rejection summed once more), 16 trees of nine over 32001 bf16
// entries 25, a greedy chain of 17 fp32 rows 8.3 (14.9 MB, floor 2.3).
#include <cooperative_groups.h>

#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "sweep.cuh"

namespace motif {
namespace {

constexpr int kChunk = 8192, kStatThreads = 256;
constexpr int kWalkThreads = 512, kWalkWarps = kWalkThreads / 32;
constexpr int kMaxRows = 1024, kMaxCluster = 16;
// A test in 32 bits that is closer to its border u·q = p than (kMargin + chunks·kMarginChunk)·(p + q) + kMarginTiny is
// repeated with sums in 64 bits, both rows added in the same order. In steps of 2^-24 relative, an exponential 2^x has 5
// roundings of its exponent (l − m, 1/τ, log2 e, their product, the product with l − m), ln 2·|x| each: 409 for
// |x| ≤ 118, and 4 of its own. The row's sum: its exponentials weigh themselves, so that |x| counts by its mean, at most
// log2 of the vocabulary, 30 (104); 23 additions within a chunk; chunks/8 additions and chunks/32 + 4 changes of the
// maximum, 4 each, over the chunks. With the quotient and products less than 600 + chunks/4. Below 2^-118 a
// probability may be anything down to 0 (2^-126 and less is flushed): there kMarginTiny decides.
constexpr float kMargin = 1.f / (1 << 14), kMarginChunk = 1.f / (1 << 26), kMarginTiny = 0x1p-100f;

struct VerifyArgs {
  const void *p, *q;
  int64_t pb, pr, qb, qr;  // element strides of sequence and row
  const int32_t *tokens, *parents;
  int64_t parents_b;
  const float* u;
  int32_t *accepted, *path, *next;
  float2* stats;             // [B][T + R][chunks]: maximum, Σ exp
  unsigned long long* tops;  // τ = 0: [B][T][chunks] keys
  int T, R, V, chunks;
  double inv_t;  // 0: greedy
};

template <typename T>
__device__ __forceinline__ float logit(const T* l, int i) {
  return fmaxf(to_f<T>(l[i]), -INFINITY);  // NaN counts as -inf
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Order-preserving key of (value, index): the larger value, then the smaller index.
__device__ __forceinline__ unsigned long long top_key(float v, int i) {
  uint32_t b = __float_as_uint(v + 0.f);  // −0 ties with 0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }
__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// Larger of two packed pairs; a NaN loses.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, float) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}

// One chunk of one row: [lo, hi), lo on a 16-byte boundary of the row but for the first chunk, whose few entries
// before the boundary are its `head`. Issue-bound before the pairs' maxima and the plain sum were taken apart from
// the rare cases (13.7 instructions an entry: 17 us for 127 rows of 219520; now about 6).
template <typename T, bool GREEDY>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(VerifyArgs a) {
  constexpr int kVec = 16 / (int)sizeof(T), kLoads = kChunk / kVec / kStatThreads;
  __shared__ float sf[8];
  __shared__ unsigned long long sk[8];
  const int row = blockIdx.y, c = blockIdx.x, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  const T* l = row < a.T ? static_cast<const T*>(a.p) + b * a.pb + row * a.pr
                         : static_cast<const T*>(a.q) + b * a.qb + (row - a.T) * a.qr;
  const int shift = min((int)((16 - reinterpret_cast<uintptr_t>(l) % 16) % 16 / sizeof(T)), a.V);
  const int lo = min(c * kChunk + shift, a.V), hi = c + 1 == a.chunks ? a.V : min(lo + kChunk, a.V);
  const int n_vec = (hi - lo) / kVec;
  // a place without a vector holds -inf throughout
  const uint32_t none = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  uint4 raw[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int v = tid + i * kStatThreads;
    raw[i] = v < n_vec ? reinterpret_cast<const uint4*>(l + lo)[v] : make_uint4(none, none, none, none);
  }
  // the entries outside whole vectors: before the first chunk's boundary, and behind the last vector
  const int tail0 = lo + n_vec * kVec;
  int edge = -1;
  if (c == 0 && tid < shift) edge = tid;
  if (tid >= 32 && tail0 + tid - 32 < hi) edge = tail0 + tid - 32;
  const float ev = edge >= 0 ? logit(l, edge) : -INFINITY;
  if constexpr (GREEDY) {
    unsigned long long top = edge >= 0 ? top_key(ev, edge) : 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int v = tid + i * kStatThreads;
      if (v >= n_vec) continue;
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int x = 0; x < kVec; ++x) {
        const unsigned long long k = top_key(logit(e, x), lo + v * kVec + x);
        top = k > top ? k : top;
      }
    }
    top = warp_max_u64(top);
    if (lane == 0) sk[warp] = top;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < 8; ++w) top = sk[w] > top ? sk[w] : top;
      a.tops[((int64_t)b * a.T + row) * a.chunks + c] = top;
    }
    return;
  }
  uint32_t mx = none;
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    mx = max2(mx, max2(max2(raw[i].x, raw[i].y, T{}), max2(raw[i].z, raw[i].w, T{}), T{}), T{});
  const T* pair = reinterpret_cast<const T*>(&mx);
  float m = fmaxf(ev, logit(pair, 0));
  if (sizeof(T) == 2) m = fmaxf(m, logit(pair, sizeof(T) == 2 ? 1 : 0));
  m = warp_max(m);
  if (lane == 0) sf[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sf[w]);
  const float k = (float)a.inv_t * 1.4426950408889634f;
  float z = 0.f;
  if (fabsf(m) < INFINITY) {
    float zs[4] = {edge >= 0 ? ex2((ev - m) * k) : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int x = 0; x < kVec; ++x) zs[x & 3] += ex2((to_f<T>(e[x]) - m) * k);
    }
    z = (zs[0] + zs[1]) + (zs[2] + zs[3]);
  }
  if (m == INFINITY || z != z) {  // infinite entries share the law; a NaN counts as -inf
    auto term = [&](float f) { return m == INFINITY ? (f == m ? 1.f : 0.f) : ex2((f - m) * k); };
    z = edge >= 0 ? term(ev) : 0.f;
#pragma unroll 1
    for (int i = 0; i < kLoads; ++i) {
      const int v = tid + i * kStatThreads;
      if (v >= n_vec) break;
#pragma unroll 1
      for (int x = 0; x < kVec; ++x) z += term(logit(l, lo + v * kVec + x));
    }
  }
  z = warp_sum(z);
  __syncthreads();
  if (lane == 0) sf[warp] = z;
  __syncthreads();
  if (tid == 0) {
    z = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) z += sf[w];
    a.stats[((int64_t)b * (a.T + a.R) + row) * a.chunks + c] = make_float2(m, z);
  }
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Bytes per tree row in shared memory: links, token, uniform, two logits, two probabilities, two laws (or a key).
constexpr int kRowBytes = 4 * 12;

// One cluster per sequence; CTA `rank` owns the vocabulary range [rank·V/C, (rank+1)·V/C), a warp a sixteenth of it.
// CACHE: the range's exponentials of the current row pair fit shared memory and are computed once a row; else
// every sweep computes them again. Most of the code runs once a call, so it is kept short: a line of it that is
// not in the instruction cache costs as much as a load.
template <typename T, bool CACHE>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(VerifyArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ double ws[kWalkWarps], sums[2][kMaxCluster][2];
  __shared__ double scan[kWalkWarps], table[kSweepTable];
  __shared__ int found;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool greedy = a.inv_t == 0.0;
  // Another CTA's shared memory may be written once that CTA has started: everyone arrives here and waits below,
  // behind the row laws.
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed;\n" ::: "memory");
  unsigned long long* top = reinterpret_cast<unsigned long long*>(dyn);  // τ = 0: a row's largest entry; in place of …
  float* pm = reinterpret_cast<float*>(dyn);                             // … the row's target law: maximum, 1 / Σ
  float* pz = pm + a.T;
  float* qm = pz + a.T;  // its draft law
  float* qz = qm + a.T;
  int* par = reinterpret_cast<int*>(qz + a.T);  // parent; -1: the root, or no row that can be accepted
  int* tok = par + a.T;
  int* first = tok + a.T;  // first child, next sibling (-1: none)
  int* next = first + a.T;
  float* u = reinterpret_cast<float*>(next + a.T);
  float* px = u + a.T;  // logits of the row's token in its parent's rows
  float* qx = px + a.T;
  double* cache = reinterpret_cast<double*>(dyn + (((size_t)kRowBytes * a.T + 15) & ~(size_t)15));
  const T* P = static_cast<const T*>(a.p) + b * a.pb;
  const T* Q = static_cast<const T*>(a.q) + b * a.qb;
  for (int i = tid; i < a.T; i += kWalkThreads) {
    int pa = i ? a.parents[b * a.parents_b + i] : -1;
    const int x = a.tokens[(int64_t)b * a.T + i];
    if (pa >= i || x < 0 || x >= a.V || (!greedy && pa >= a.R)) pa = -1;
    par[i] = pa;
    tok[i] = x;
    if (greedy) continue;
    u[i] = a.u[(int64_t)b * a.T + i];
    px[i] = pa >= 0 ? logit(P + pa * a.pr, x) : 0.f;
    qx[i] = pa >= 0 ? logit(Q + pa * a.qr, x) : 0.f;
  }
  if (!greedy && tid < kSweepTable) table[tid] = exp2(tid / (double)kSweepTable);
  __syncthreads();
  // links: a warp finds a row's children, 32 rows a ballot, from the last to the first
#pragma unroll 1
  for (int i = warp; i < a.T; i += kWalkWarps) {
    int after = -1;  // the child that follows those of this ballot
#pragma unroll 1
    for (int j0 = (a.T - 1) & ~31; j0 + 31 > i; j0 -= 32) {
      const int j = j0 + lane;
      const bool mine = j < a.T && par[j] == i;
      const unsigned kids = __ballot_sync(0xffffffffu, mine);
      const unsigned later = lane < 31 ? kids >> (lane + 1) : 0;
      if (mine) next[j] = later ? j + __ffs(later) : after;
      after = kids ? j0 + __ffs(kids) - 1 : after;
      if (j0 == 0) break;
    }
    if (lane == 0) first[i] = after;
  }
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  // the rows' laws (τ = 0: their largest entries) from the chunks: eight lanes a row
  const float kf = (float)a.inv_t * 1.4426950408889634f;
#pragma unroll 1
  for (int r0 = tid / 8; r0 < a.T + a.R; r0 += kWalkThreads / 8) {
    const unsigned mask = 0xFFu << (lane & 24);
    if (greedy) {
      unsigned long long k = 0;
      for (int c = lane & 7; c < a.chunks; c += 8) {
        const unsigned long long v = a.tops[((int64_t)b * a.T + r0) * a.chunks + c];
        k = v > k ? v : k;
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        const unsigned long long v = __shfl_xor_sync(mask, k, o);
        k = v > k ? v : k;
      }
      if ((lane & 7) == 0) top[r0] = k;
      continue;
    }
    const float2* st = a.stats + ((int64_t)b * (a.T + a.R) + r0) * a.chunks;
    float m = -INFINITY, z = 0.f;
    for (int c0 = lane & 7; c0 < a.chunks; c0 += 32) {  // four chunks of a lane at once
      float2 s[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) s[x] = c0 + 8 * x < a.chunks ? st[c0 + 8 * x] : make_float2(-INFINITY, 0.f);
      const float top4 = fmaxf(fmaxf(fmaxf(s[0].x, s[1].x), fmaxf(s[2].x, s[3].x)), m);
      z = m == top4 ? z : z * ex2((m - top4) * kf);
      m = top4;
#pragma unroll
      for (int x = 0; x < 4; ++x) z += s[x].x == m ? s[x].y : s[x].y * ex2((s[x].x - m) * kf);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(mask, m, o), z2 = __shfl_xor_sync(mask, z, o), t = fmaxf(m, m2);
      z = (m == t ? z : z * ex2((m - t) * kf)) + (m2 == t ? z2 : z2 * ex2((m2 - t) * kf));
      m = t;
    }
    if ((lane & 7) == 0) {
      const bool p = r0 < a.T;
      const int r = p ? r0 : r0 - a.T;
      (p ? pm : qm)[r] = m;
      (p ? pz : qz)[r] = m > -INFINITY ? 1.f / z : 0.f;  // a row without a finite logit has no law
    }
  }
  __syncthreads();

  int32_t* path = a.path + (int64_t)b * a.T;
  if (greedy) {
    if (tid == 0) {
      int cur = 0, kept = 1;
      auto best = [&](int r) { return key_value(top[r]) > -INFINITY ? key_index(top[r]) : -1; };
      int want = best(0);
      path[0] = 0;
      for (int i = first[0]; i >= 0;) {
        if (want >= 0 && tok[i] == want) {
          cur = i;
          path[kept++] = i;
          want = best(i);
          i = first[cur];
        } else {
          i = next[i];
        }
      }
      a.accepted[b] = kept - 1;
      a.next[b] = max(want, 0);
      found = kept;
    }
    __syncthreads();
    for (int i = found + tid; i < a.T; i += kWalkThreads) path[i] = -1;
    return;
  }

  const int v0 = (int)((int64_t)rank * a.V / C), v1 = (int)((int64_t)(rank + 1) * a.V / C), span = v1 - v0;
  auto range = [&](int w) { return v0 + (int)((int64_t)w * span / kWalkWarps); };
  const int w0 = range(warp), w1 = range(warp + 1);
  const double k = a.inv_t * 1.4426950408889634074;  // log2 e
  // The current row's laws: maxima, and in `exact` form 1 / Σ in 64 bits; its residual (p − coef·q)⁺ / S.
  float mp = pm[0], mq = 0.f;
  double izp = 1.0, izq = 1.0, coef = 0.0, S = 1.0;
  bool exact = false;
  const float margin = kMargin + a.chunks * kMarginChunk;
  int phase = 0;
  // exp((l − m)/τ); an infinite maximum's entries share the law, a row of -inf has none
  auto entry = [&](float l, float m) {
    const double e = sweep_weight(l, (double)m, k, table);
    return fabsf(m) < INFINITY ? e : m > 0.f && l == m ? 1.0 : 0.0;
  };
  // Sums of two values over the cluster, the same on every CTA; my warps' sums of the first stay in ws.
  auto total = [&](double x, double y, double& sx, double& sy) {
    x = warp_sum_f64(x), y = warp_sum_f64(y);
    __syncthreads();
    if (lane == 0) ws[warp] = x, scan[warp] = y;
    __syncthreads();
    if (tid < C) {  // my CTA's sums into every CTA's slots
      double cx = 0.0, cy = 0.0;
#pragma unroll 4
      for (int w = 0; w < kWalkWarps; ++w) cx += ws[w], cy += scan[w];
      double* dst = cluster.map_shared_rank(&sums[phase][rank][0], tid);
      dst[0] = cx, dst[1] = cy;
    }
    cluster.sync();
    sx = sy = 0.0;
#pragma unroll 4
    for (int c = 0; c < C; ++c) sx += sums[phase][c][0], sy += sums[phase][c][1];
    phase ^= 1;  // the other slots' readers are behind the next sync
  };
  // Exponentials of my warp's range of the row(s) into the cache: the logits first, many loads in flight, then each
  // in place of its logit.
  auto fill = [&](const T* p, const T* q) {
    constexpr int kU = 9;
    for (int e0 = w0 + lane; e0 < w1; e0 += 32 * kU) {
      T x[kU], y[kU];
#pragma unroll
      for (int i = 0; i < kU; ++i) {
        const int e = min(e0 + 32 * i, w1 - 1);
        x[i] = p[e];
        if (q) y[i] = q[e];
      }
#pragma unroll
      for (int i = 0; i < kU; ++i) {
        const int e = min(e0 + 32 * i, w1 - 1);  // the last lanes write one entry more than once, the same value
        *reinterpret_cast<float*>(cache + e - v0) = logit(x, i);
        if (q) *reinterpret_cast<float*>(cache + span + e - v0) = logit(y, i);
      }
    }
    __syncwarp();
#pragma unroll 4
    for (int e = w0 + lane - v0; e < w1 - v0; e += 32) {
      cache[e] = entry(*reinterpret_cast<const float*>(cache + e), mp);
      if (q) cache[span + e] = entry(*reinterpret_cast<const float*>(cache + span + e), mq);
    }
    __syncwarp();
  };
  auto at_p = [&](const T* p, int e) { return CACHE ? cache[e - v0] : entry(logit(p, e), mp); };
  auto at_q = [&](const T* q, int e) { return CACHE ? cache[span + e - v0] : entry(logit(q, e), mq); };
  auto make_exact = [&](const T* p, const T* q) {
    if (CACHE) fill(p, q);
    double x = 0.0, y = 0.0, sx, sy;
#pragma unroll 4
    for (int e = w0 + lane; e < w1; e += 32) x += at_p(p, e), y += at_q(q, e);
    total(x, y, sx, sy);
    izp = sx > 0.0 ? 1.0 / sx : 0.0;
    izq = sy > 0.0 ? 1.0 / sy : 0.0;
    exact = true;
  };

  if (C > 1) asm volatile("barrier.cluster.wait;\n" ::: "memory");  // every CTA of the cluster has started
  int cur = 0, kept = 1;
  if (rank == 0 && tid == 0) path[0] = 0;
  for (int i = first[0]; i >= 0;) {
    const T* p = P + cur * a.pr;
    const T* q = Q + cur * a.qr;
    bool ok = false, sure = false;
    if (!exact) {  // the first child: w = p, in 32 bits where that decides
      mq = qm[cur];
      auto prob = [&](float l, float m, float iz) { return l == m ? iz : ex2((l - m) * kf) * iz; };
      const float pe = prob(px[i], mp, pz[cur]), qe = prob(qx[i], mq, qz[cur]), ue = u[i] * qe;
      ok = ue < pe;
      sure = fabsf(ue - pe) > margin * (pe + qe) + kMarginTiny;
    }
    if (!sure) {
      if (!exact) make_exact(p, q);
      const double pe = entry(px[i], mp) * izp, qe = entry(qx[i], mq) * izq;
      ok = (double)u[i] * qe * S < pe - coef * qe;
    }
    if (ok) {
      if (rank == 0 && tid == 0) path[kept] = i;
      ++kept;
      cur = i;
      i = first[cur];
      coef = 0.0, S = 1.0, exact = false;
      mp = pm[cur];
      continue;
    }
    if (!exact) make_exact(p, q);
    coef += S;
    double s = 0.0, unused;
#pragma unroll 4
    for (int e = w0 + lane; e < w1; e += 32) s += fmax(0.0, at_p(p, e) * izp - coef * (at_q(q, e) * izq));
    total(s, 0.0, S, unused);
    i = next[i];
  }
  // the draw, from (p − coef·q)⁺ or (no rejection, or an empty residual) from p
  const T* p = P + cur * a.pr;
  const T* q = Q + (cur < a.R ? cur : 0) * a.qr;
  double W = S;
  const bool plain = coef == 0.0 || !(S > 0.0);
  if (plain) {
    double s = 0.0, unused;
    if (CACHE && !exact) fill(p, nullptr);
#pragma unroll 4
    for (int e = w0 + lane; e < w1; e += 32) s += at_p(p, e);
    total(s, 0.0, W, unused);
  }
  auto w = [&](int e) { return plain ? at_p(p, e) : fmax(0.0, at_p(p, e) * izp - coef * (at_q(q, e) * izq)); };
  // the CTA, then the warp's range that holds the border; the last one with any weight if none goes beyond it (u_0 ≥ 1,
  // or rounding). `before`: the weights in front of it
  const double target = u[0] < 1.f ? (double)u[0] * W : INFINITY;
  double before = 0.0, upto = 0.0;
  int cta = -1, sub = -1;
  for (int c = 0; c < C; ++c) {
    const double x = sums[phase ^ 1][c][0];
    if (!(x > 0.0)) continue;
    cta = c;
    before = upto;
    upto += x;
    if (upto > target) break;
  }
  if (cta < 0) {  // a row without a finite logit
    if (rank == 0 && tid == 0) a.next[b] = 0;
  } else if (cta == rank) {
    upto = before;
    for (int k = 0; k < kWalkWarps; ++k) {
      const double x = ws[k];
      if (!(x > 0.0)) continue;
      sub = k;
      before = upto;
      upto += x;
      if (upto > target) break;
    }
    const int e0 = range(sub), e1 = range(sub + 1), per = (e1 - e0 + kWalkThreads - 1) / kWalkThreads;
    const int mine0 = min(e0 + tid * per, e1), mine1 = min(mine0 + per, e1);
    double mine = 0.0;
    int last = -1;
    for (int e = mine0; e < mine1; ++e) {
      const double x = w(e);
      mine += x;
      if (x > 0.0) last = e;
    }
    double run = mine;  // inclusive scan over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += x;
    }
    if (tid == 0) found = 0x7fffffff;
    if (lane == 31) scan[warp] = run;
    __syncthreads();
    for (int k = 0; k < warp; ++k) before += scan[k];
    run += before;
    if (mine > 0.0 && run > target) {
      double r = run - mine;
      int at = last;
      for (int e = mine0; e < mine1; ++e) {
        const double x = w(e);
        r += x;
        if (x > 0.0 && r > target) { at = e; break; }
      }
      atomicMin(&found, at);
    }
    __syncthreads();
    const bool none = found == 0x7fffffff;
    __syncthreads();
    if (none) {  // nothing beyond the target: the last entry with weight
      if (tid == 0) found = -1;
      __syncthreads();
      if (last >= 0) atomicMax(&found, last);
      __syncthreads();
    }
    if (tid == 0) a.next[b] = max(found, 0);
  }
  if (rank == 0) {
    if (tid == 0) a.accepted[b] = kept - 1;
    for (int i = kept + tid; i < a.T; i += kWalkThreads) path[i] = -1;
  }
  // every write into another CTA's shared memory was before the last sync: a CTA may end
}

constexpr size_t kRoom = 224 * 1024;  // dynamic shared memory beside the walk's static 2.8 KB

int chunks_of(int64_t V) { return (int)ceil_div(V, kChunk); }

// Clusters of 16 CTAs need a part of the GPU with 16 free SMs where a CTA takes the most shared memory that a call asks
// for (smaller calls share SMs): asked for that size, once per device. The kernel's attributes are set.
template <typename T>
bool clusters_of_16() {
  static std::atomic<int> known[64]{};  // 0: not asked, 1: they fit, 2: they do not
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && known[dev] != 0) return known[dev] == 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(16);
  cfg.blockDim = dim3(kWalkThreads);
  cfg.dynamicSmemBytes = kRoom;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 16;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  int n = 0;
  const bool fit = cudaOccupancyMaxActiveClusters(&n, verify_walk_kernel<T, true>, &cfg) == cudaSuccess && n > 0;
  (void)cudaGetLastError();
  if (dev < 64) known[dev] = fit ? 1 : 2;
  return fit;
}

template <typename T>
int launch_verify(const VerifyArgs& a, int64_t batch, cudaStream_t st) {
  const bool greedy = a.inv_t == 0.0;
  const dim3 chunks((unsigned)a.chunks, (unsigned)(a.T + a.R), (unsigned)batch);
  if (greedy) verify_stats_kernel<T, true><<<chunks, kStatThreads, 0, st>>>(a);
  else verify_stats_kernel<T, false><<<chunks, kStatThreads, 0, st>>>(a);
  const int rc = check_launch("speculative_verify");
  if (rc) return rc;
  // CTAs of a cluster: all SMs together serve the batch, and a CTA has 2048 entries or more
  int C = 1;
  while (!greedy && C < kMaxCluster && 2 * C * batch <= 128 && a.V / (2 * C) >= 2048) C *= 2;
  const size_t rows = ((size_t)kRowBytes * a.T + 15) & ~(size_t)15;
  auto bytes = [&](int c) { return rows + 16 * (size_t)(a.V / c + 1); };
  bool cache = !greedy && bytes(C) <= kRoom;
  auto kern = cache ? verify_walk_kernel<T, true> : verify_walk_kernel<T, false>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = once_per_device(done, [] {
    for (auto f : {verify_walk_kernel<T, true>, verify_walk_kernel<T, false>}) {
      cudaError_t r = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (r == cudaSuccess) r = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRoom);
      if (r != cudaSuccess) return r;
    }
    return cudaSuccess;
  });
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "speculative_verify: cluster attribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * C));
  cfg.blockDim = dim3(kWalkThreads);
  cfg.dynamicSmemBytes = cache ? bytes(C) : rows;
  cfg.stream = st;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)C;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (C > 8 && !clusters_of_16<T>()) {
    C = 8;
    cfg.gridDim = dim3((unsigned)(batch * C));
    at[1].val.clusterDim.x = 8;
    cache = bytes(C) <= kRoom;
    kern = cache ? verify_walk_kernel<T, true> : verify_walk_kernel<T, false>;
    cfg.dynamicSmemBytes = cache ? bytes(C) : rows;
  }
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "speculative_verify: %s", cudaGetErrorString(e));
  return MOTIF_OK;
}

}  // namespace
}  // namespace motif

using namespace motif;

extern "C" {

size_t motif_speculative_verify_workspace_bytes(int64_t batch, int64_t rows, int64_t draft_rows, int64_t vocab) {
  if (batch < 1 || rows < 1 || draft_rows < 0 || vocab < 1) return 0;
  return 8 * (size_t)batch * (size_t)(rows + draft_rows) * (size_t)chunks_of(vocab);
}

int motif_speculative_verify(int dtype, const void* p_logits, int64_t p_batch_stride, int64_t p_row_stride,
                             const void* q_logits, int64_t q_batch_stride, int64_t q_row_stride, int64_t draft_rows,
                             const int32_t* tokens, const int32_t* parents, int64_t parents_batch_stride,
                             const float* uniforms, int64_t batch, int64_t rows, int64_t vocab, double temperature,
                             int32_t* accepted, int32_t* path, int32_t* next_token, void* workspace,
                             size_t workspace_bytes, void* stream) {
  MOTIF_REQUIRE(p_logits && tokens && parents && accepted && path && next_token, MOTIF_ERR_NULL,
                "speculative_verify: null pointer");
  MOTIF_REQUIRE(temperature == 0.0 || (temperature >= 1e-6 && temperature <= 1e6), MOTIF_ERR_BAD_CONTRACT,
                "speculative_verify: temperature %g (0, or 1e-6 .. 1e6)", temperature);
  MOTIF_REQUIRE(temperature == 0.0 || (q_logits && uniforms), MOTIF_ERR_NULL,
                "speculative_verify: q_logits and uniforms are needed at temperature %f", temperature);
  MOTIF_REQUIRE(batch >= 1 && batch < 65536 && rows >= 1 && rows <= kMaxRows && vocab >= 1 && vocab < (1ll << 30),
                MOTIF_ERR_BAD_SHAPE, "speculative_verify: batch=%lld rows=%lld (1..1024) vocab=%lld", (long long)batch,
                (long long)rows, (long long)vocab);
  MOTIF_REQUIRE(temperature == 0.0 || (draft_rows >= 1 && draft_rows <= rows), MOTIF_ERR_BAD_SHAPE,
                "speculative_verify: %lld draft rows (1..%lld)", (long long)draft_rows, (long long)rows);
  MOTIF_REQUIRE(p_row_stride >= 0 && p_batch_stride >= 0 && q_row_stride >= 0 && q_batch_stride >= 0,
                MOTIF_ERR_BAD_SHAPE, "speculative_verify: negative stride");
  MOTIF_REQUIRE(parents_batch_stride == 0 || parents_batch_stride == rows, MOTIF_ERR_BAD_SHAPE,
                "speculative_verify: parents batch stride %lld", (long long)parents_batch_stride);
  const size_t need = motif_speculative_verify_workspace_bytes(batch, rows, temperature > 0.0 ? draft_rows : 0, vocab);
  MOTIF_REQUIRE(workspace && workspace_bytes >= need, MOTIF_ERR_WORKSPACE,
                "speculative_verify: workspace of %zu bytes, needs %zu", workspace_bytes, need);
  VerifyArgs a{};
  a.p = p_logits;
  a.q = temperature == 0.0 ? p_logits : q_logits;
  a.pb = p_batch_stride;
  a.pr = p_row_stride;
  a.qb = q_batch_stride;
  a.qr = q_row_stride;
  a.tokens = tokens;
  a.parents = parents;
  a.parents_b = parents_batch_stride;
  a.u = temperature == 0.0 ? nullptr : uniforms;
  a.accepted = accepted;
  a.path = path;
  a.next = next_token;
  a.T = (int)rows;
  a.R = temperature == 0.0 ? 0 : (int)draft_rows;
  a.V = (int)vocab;
  a.inv_t = temperature > 0.0 ? 1.0 / temperature : 0.0;
  a.chunks = chunks_of(vocab);
  a.stats = static_cast<float2*>(workspace);
  a.tops = static_cast<unsigned long long*>(workspace);
  MOTIF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, MOTIF_ERR_BAD_CONTRACT,
                "speculative_verify: workspace must be 8-byte aligned");
  MOTIF_DISPATCH_FLOAT(dtype, T, return launch_verify<T>(a, batch, as_stream(stream)));
  return MOTIF_OK;
}

}  // extern "C"
