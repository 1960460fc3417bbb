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
#include <cmath>

#include "common.cuh"

namespace motif {
namespace {

constexpr int kVThreads = 1024;

struct VerifyArgs {
  const void *p, *q;
  int64_t pb, pr, qb, qr;  // element strides of sequence and row
  const int32_t *tokens, *parents;
  int64_t parents_b;
  const float* u;
  int32_t *accepted, *path, *next;
  int T, R, V;
  double inv_t;  // 0: greedy
};

template <typename T>
__device__ __forceinline__ float logit(const T* l, int i) {
  const float v = to_f<T>(l[i]);
  return isnan(v) ? -INFINITY : v;
}
// exp((l − m)·inv_t); 1 at the maximum itself (infinite ones included), 0 for a row of −inf
__device__ __forceinline__ double weight(float l, float m, double inv_t) {
  return m == -INFINITY ? 0.0 : l == m ? 1.0 : exp(((double)l - (double)m) * inv_t);
}

__device__ double block_sum_f64(double v, double* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) sm[warp] = v;
  __syncthreads();
  v = sm[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Largest logit of a row and its first index, as one order-preserving key.
template <typename T>
__device__ unsigned long long block_top(const T* l, int V, unsigned long long* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < V; i += kVThreads) {
    uint32_t b = __float_as_uint(logit(l, i) + 0.f);  // −0 ties with 0
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    const unsigned long long k = ((unsigned long long)b << 32) | (0xFFFFFFFFu - (uint32_t)i);
    best = k > best ? k : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, best, o);
    best = w > best ? w : best;
  }
  __syncthreads();
  if (lane == 0) sm[warp] = best;
  __syncthreads();
  best = sm[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, best, o);
    best = w > best ? w : best;
  }
  return best;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

struct Law {
  float m;
  double inv_z;
};
template <typename T>
__device__ Law row_law(const T* l, int V, double inv_t, double* smd, unsigned long long* smk) {
  Law w;
  w.m = key_value(block_top(l, V, smk));
  double z = 0.0;
  for (int i = threadIdx.x; i < V; i += kVThreads) z += weight(logit(l, i), w.m, inv_t);
  z = block_sum_f64(z, smd);
  w.inv_z = z > 0.0 ? 1.0 / z : 0.0;
  return w;
}

template <typename T>
__global__ void __launch_bounds__(kVThreads) verify_kernel(VerifyArgs a) {
  __shared__ double smd[32], part[kVThreads];
  __shared__ unsigned long long smk[32];
  __shared__ int s_token;
  const int b = blockIdx.x, tid = threadIdx.x;
  const T* P = static_cast<const T*>(a.p) + b * a.pb;
  const T* Q = static_cast<const T*>(a.q) + b * a.qb;
  const int32_t* tok = a.tokens + (int64_t)b * a.T;
  const int32_t* par = a.parents + b * a.parents_b;
  const float* u = a.u + (int64_t)b * a.T;
  int32_t* path = a.path + (int64_t)b * a.T;
  const bool greedy = a.inv_t == 0.0;
  int cur = 0, kept = 1;
  double coef = 0.0, S = 1.0;
  bool have_q = false;
  Law lp{}, lq{};
  unsigned long long top = 0;
  auto enter = [&](int r) {
    if (greedy) top = block_top(P + r * a.pr, a.V, smk);
    else lp = row_law(P + r * a.pr, a.V, a.inv_t, smd, smk);
  };
  enter(0);
  for (int i = tid; i < a.T; i += kVThreads) path[i] = i == 0 ? 0 : -1;
  __syncthreads();
  for (int i = 1; i < a.T; ++i) {
    if (par[i] != cur) continue;
    const int x = tok[i];
    if (x < 0 || x >= a.V) continue;  // a padding row
    bool ok;
    if (greedy) {
      ok = key_value(top) > -INFINITY && x == key_index(top);
    } else {
      if (cur >= a.R) continue;  // no draft row: nothing can be tested
      const T* p = P + cur * a.pr;
      const T* q = Q + cur * a.qr;
      if (!have_q) lq = row_law(q, a.V, a.inv_t, smd, smk), have_q = true;
      const double px = weight(logit(p, x), lp.m, a.inv_t) * lp.inv_z;
      const double qx = weight(logit(q, x), lq.m, a.inv_t) * lq.inv_z;
      ok = (double)u[i] * qx * S < px - coef * qx;
      if (!ok) {
        coef += S;
        double s = 0.0;
        for (int e = tid; e < a.V; e += kVThreads)
          s += fmax(0.0, weight(logit(p, e), lp.m, a.inv_t) * lp.inv_z - coef * (weight(logit(q, e), lq.m, a.inv_t) * lq.inv_z));
        S = block_sum_f64(s, smd);
      }
    }
    if (ok) {
      cur = i;
      if (tid == 0) path[kept] = i;
      ++kept;
      coef = 0.0, S = 1.0, have_q = false;
      enter(i);
    }
  }
  if (greedy) {
    if (tid == 0) s_token = key_value(top) > -INFINITY ? key_index(top) : 0;
  } else {
    // contiguous chunks: their sums, then the chunk that holds the border, then the entry
    if (!(S > 0.0)) coef = 0.0;  // an empty residual: the target's own law
    const T* p = P + cur * a.pr;
    const T* q = Q + (cur < a.R ? cur : 0) * a.qr;
    const int per = (a.V + kVThreads - 1) / kVThreads, e0 = min(tid * per, a.V), e1 = min(e0 + per, a.V);
    auto w = [&](int e) {
      const double pe = weight(logit(p, e), lp.m, a.inv_t) * lp.inv_z;
      return coef == 0.0 ? pe : fmax(0.0, pe - coef * (weight(logit(q, e), lq.m, a.inv_t) * lq.inv_z));
    };
    double s = 0.0;
    for (int e = e0; e < e1; ++e) s += w(e);
    part[tid] = s;
    __syncthreads();
    if (tid == 0) {
      double total = 0.0;
      for (int i = 0; i < kVThreads; ++i) total += part[i];
      const double target = (double)u[0] * total;
      double run = 0.0;
      int token = 0;
      bool found = false;
      for (int i = 0; i < kVThreads && !found; ++i) {
        if (part[i] > 0.0 && (run + part[i] > target)) {
          double r = run;
          for (int e = i * per; e < min((i + 1) * per, a.V) && !found; ++e) {
            const double we = w(e);
            if (we > 0.0) token = e;
            r += we;
            found = we > 0.0 && r > target;
          }
        } else if (part[i] > 0.0) {  // kept in case rounding leaves none beyond the target: the last one
          token = -1 - i;
        }
        run += part[i];
      }
      if (token < 0) {
        const int i = -1 - token;
        for (int e = i * per; e < min((i + 1) * per, a.V); ++e)
          if (w(e) > 0.0) token = e;
      }
      s_token = token < 0 ? 0 : token;
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.accepted[b] = kept - 1;
    a.next[b] = s_token;
  }
}

}  // namespace
}  // namespace motif

using namespace motif;

extern "C" {

size_t motif_speculative_verify_workspace_bytes(int64_t batch, int64_t rows, int64_t draft_rows) {
  (void)batch, (void)rows, (void)draft_rows;
  return 16;
}

int motif_speculative_verify(int dtype, const void* p_logits, int64_t p_batch_stride, int64_t p_row_stride,
                             const void* q_logits, int64_t q_batch_stride, int64_t q_row_stride, int64_t draft_rows,
                             const int32_t* tokens, const int32_t* parents, int64_t parents_batch_stride,
                             const float* uniforms, int64_t batch, int64_t rows, int64_t vocab, double temperature,
                             int32_t* accepted, int32_t* path, int32_t* next_token, void* workspace,
                             size_t workspace_bytes, void* stream) {
  MOTIF_REQUIRE(p_logits && tokens && parents && accepted && path && next_token, MOTIF_ERR_NULL,
                "speculative_verify: null pointer");
  MOTIF_REQUIRE(std::isfinite(temperature) && temperature >= 0.0, MOTIF_ERR_BAD_CONTRACT,
                "speculative_verify: temperature %f", temperature);
  MOTIF_REQUIRE(temperature == 0.0 || (q_logits && uniforms), MOTIF_ERR_NULL,
                "speculative_verify: q_logits and uniforms are needed at temperature %f", temperature);
  MOTIF_REQUIRE(batch >= 1 && batch < 65536 && rows >= 1 && rows <= 1024 && vocab >= 1 && vocab < (1ll << 31),
                MOTIF_ERR_BAD_SHAPE, "speculative_verify: batch=%lld rows=%lld (1..1024) vocab=%lld", (long long)batch,
                (long long)rows, (long long)vocab);
  MOTIF_REQUIRE(temperature == 0.0 || (draft_rows >= 1 && draft_rows <= rows), MOTIF_ERR_BAD_SHAPE,
                "speculative_verify: %lld draft rows (1..%lld)", (long long)draft_rows, (long long)rows);
  MOTIF_REQUIRE(p_row_stride >= 0 && p_batch_stride >= 0 && q_row_stride >= 0 && q_batch_stride >= 0,
                MOTIF_ERR_BAD_SHAPE, "speculative_verify: negative stride");
  MOTIF_REQUIRE(parents_batch_stride == 0 || parents_batch_stride == rows, MOTIF_ERR_BAD_SHAPE,
                "speculative_verify: parents batch stride %lld", (long long)parents_batch_stride);
  const size_t need = motif_speculative_verify_workspace_bytes(batch, rows, draft_rows);
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
  a.R = (int)draft_rows;
  a.V = (int)vocab;
  a.inv_t = temperature > 0.0 ? 1.0 / temperature : 0.0;
  MOTIF_DISPATCH_FLOAT(dtype, T, verify_kernel<T><<<(unsigned)batch, kVThreads, 0, as_stream(stream)>>>(a));
  return check_launch("speculative_verify");
}

}  // extern "C"
