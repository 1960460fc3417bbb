// Shared-QK dual-V attention for a tree of drafted tokens over a KV cache.
//
//   o[t] = Σ_c p[t, c]·[v1_c | v2_c],   p[t, ·] = softmax over the visible c of scale·q_t·k_c
//
// for the T rows of a tree whose keys and values are the cache's last T live rows: with n live rows,
// row t sees every cache row c < n − T (the context) and the drafted row c = n − T + j where
// mask[t, j] (causal j ≤ t without a mask). A row that sees nothing gives 0. Rows ≥ n are never
// used, and a drafted row hidden from a query does not reach it, whatever it holds (NaN included).
//
// All GQA heads of a kv head share its rows, so the gqa·T query rows of a kv head are packed
// (head-major) and cut into row tiles; a unit of work is (sequence, kv head, row tile) and its
// key tiles. The tiles of all units form one line that is cut into gridDim.x equal parts
// (Schedule), whatever the sequences' lengths: a CTA may end one unit and start the next. A unit
// that lies in one CTA is normalised and written by it; the others leave fp32 partials (running
// maximum, Σp, unnormalised O) that tree_merge_kernel joins in a fixed order.
#include <cmath>

#include "common.cuh"

namespace motif {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct TreeArgs {
  const void* q;            // (B, HKV·gqa, T, D)
  const void* kv[3];        // k, v1, v2: rows, or packed codes
  const void* sc[3];        // packed: scales, biases (…, D / gs) in the activations' type
  const void* bi[3];
  int64_t sb, sh, sr;       // element strides of batch, head, row of kv (16-bit and fp32 rows)
  const uint8_t* mask;      // (T, T) bytes per sequence, or null: causal
  int64_t mask_b;           // bytes between sequences' masks (0: one for all)
  const int32_t* len_dev;   // live rows, when set; else len
  int len_step;             // 0: one for all sequences
  int len;
  void* y;                  // (B, HKV·gqa, T, 2D)
  float* part_o;            // [2·grid][tile rows][2D]
  float* part_ml;           // [2·grid][tile rows][2]
  int* err;
  int B, HKV, gqa, T, R, row_tiles, cap, gs;
  int tile_rows, tile_keys;
  float scale_log2;
};

__device__ __forceinline__ int live_rows(const TreeArgs& a, int b) {
  const int n = a.len_dev ? a.len_dev[(int64_t)b * a.len_step] : a.len;
  return min(max(n, 0), a.cap);
}
__device__ __forceinline__ int key_tiles(const TreeArgs& a, int n) {
  return max(1, (n + a.tile_keys - 1) / a.tile_keys);  // an empty cache is one tile without a visible key
}

// Line of all units' key tiles, and this CTA's part [x, x1) of it. Every thread of a warp calls it.
struct Schedule {
  int64_t total, x, x1;
  int b;         // sequence of x
  int64_t base;  // its first tile
  int n, nt;     // its live rows and key tiles per unit

  __device__ __forceinline__ Schedule(const TreeArgs& a) {
    const int lane = threadIdx.x & 31;
    const int per_b = a.HKV * a.row_tiles;
    int64_t s = 0;
    for (int i = lane; i < a.B; i += 32) s += key_tiles(a, live_rows(a, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    total = s * per_b;
    x = lo(blockIdx.x, gridDim.x);
    x1 = lo(blockIdx.x + 1, gridDim.x);
    seek(a, x);
  }
  __device__ __forceinline__ int64_t lo(int64_t i, int64_t grid) const { return i * total / grid; }
  // The sequence that holds tile `at` (at < total, or the last one).
  __device__ __forceinline__ void seek(const TreeArgs& a, int64_t at) {
    const int64_t per_b = (int64_t)a.HKV * a.row_tiles;
    b = 0;
    base = 0;
    for (;;) {
      n = live_rows(a, b);
      nt = key_tiles(a, n);
      if (b + 1 >= a.B || at < base + nt * per_b) return;
      base += nt * per_b;
      ++b;
    }
  }
};

// One CTA's share of one unit: key tiles [t0, t1) of row tile rt of kv head g of sequence b.
struct Segment {
  int b, g, rt, n, t0, t1;
  bool whole;   // the unit lies in this CTA
  int64_t slot; // its partial's place otherwise
};

__device__ __forceinline__ bool next_segment(const TreeArgs& a, Schedule& s, Segment& g) {
  if (s.x >= s.x1) return false;
  const int64_t per_b = (int64_t)a.HKV * a.row_tiles;
  if (s.x >= s.base + s.nt * per_b) {
    s.base += s.nt * per_b;
    ++s.b;
    s.n = live_rows(a, s.b);
    s.nt = key_tiles(a, s.n);
  }
  const int64_t in = s.x - s.base;
  const int u = (int)(in / s.nt);
  g.b = s.b;
  g.n = s.n;
  g.g = u / a.row_tiles;
  g.rt = u - g.g * a.row_tiles;
  g.t0 = (int)(in - (int64_t)u * s.nt);
  g.t1 = (int)min((int64_t)s.nt, g.t0 + (s.x1 - s.x));
  g.whole = g.t0 == 0 && g.t1 == s.nt;
  // at most two segments of a CTA are parts: the first (a unit begun before it) and the last
  g.slot = 2 * (int64_t)blockIdx.x + (s.x == s.lo(blockIdx.x, gridDim.x) ? 0 : 1);
  s.x += g.t1 - g.t0;
  return true;
}

// Bit c: row t of sequence b sees cache row p0 + c, c < NB.
template <int NB>
__device__ __forceinline__ uint64_t visible(const TreeArgs& a, int b, int t, int n, int p0) {
  const int ctx = n - a.T;  // negative where fewer than T rows are live
  uint64_t w = 0;
  const uint8_t* m = a.mask ? a.mask + b * a.mask_b + (int64_t)t * a.T : nullptr;
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    const int pos = p0 + c, j = pos - ctx;
    bool v = pos < n;
    if (v && j >= 0) v = m ? m[j] != 0 : j <= t;
    w |= (uint64_t)v << c;
  }
  return w;
}

// Eight consecutive channels [8·c8, 8·c8 + 8) of row `pos` of slot s (kv head g of sequence b) in fp32.
template <typename T, int D, int BITS>
__device__ __forceinline__ void load8(const TreeArgs& a, int s, int b, int g, int pos, int c8, float (&v)[8]) {
  if constexpr (BITS == 16) {
    const T* p = static_cast<const T*>(a.kv[s]) + b * a.sb + g * a.sh + pos * a.sr + c8 * 8;
    load_vec<T, 8>(p, v);
  } else {
    const int64_t row = ((int64_t)b * a.HKV + g) * a.cap + pos;
    const int grp = c8 * 8 / a.gs;
    const float sc = to_f<T>(static_cast<const T*>(a.sc[s])[row * (D / a.gs) + grp]);
    const float bi = to_f<T>(static_cast<const T*>(a.bi[s])[row * (D / a.gs) + grp]);
    if constexpr (BITS == 4) {
      const uint32_t w = static_cast<const uint32_t*>(a.kv[s])[row * (D / 8) + c8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(sc, (float)((w >> (4 * i)) & 15u), bi);
    } else {
      const uint2 w = reinterpret_cast<const uint2*>(a.kv[s])[row * (D / 8) + c8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = fmaf(sc, (float)((w.x >> (8 * i)) & 255u), bi);
        v[4 + i] = fmaf(sc, (float)((w.y >> (8 * i)) & 255u), bi);
      }
    }
  }
}

// ---- CUDA-core form: every type -----------------------------------------------------------------
// 16 query rows × 32 keys per step in fp32. Scores: a lane is a key, a warp two rows, K rows padded
// to D + 4 floats (a quarter-warp's 16-byte reads then fall into different banks). P·V: a thread is
// a channel of [v1 | v2] for all 16 rows (D 128) or for 8 of them (D 64).
constexpr int kSR = 16, kSK = 32, kSThreads = 256;

template <int D>
constexpr int simt_smem() {
  return (int)sizeof(float) * (kSR * D + kSK * (D + 4) + kSK * 2 * D + kSK * kSR + 2 * kSR);
}

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kSThreads, 2) tree_simt_kernel(const __grid_constant__ TreeArgs a) {
  extern __shared__ float sm[];
  float* qs = sm;                     // [kSR][D]
  float* ks = qs + kSR * D;           // [kSK][D + 4]
  float* vs = ks + kSK * (D + 4);     // [kSK][2D]
  float* ps = vs + kSK * 2 * D;       // [kSK][kSR]
  float* alpha = ps + kSK * kSR;      // [kSR]
  float* inv_l = alpha + kSR;         // [kSR]
  constexpr int kAcc = kSR * 2 * D / kSThreads;  // rows of one thread in P·V
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ch = tid % (2 * D), row0 = tid / (2 * D) * kAcc;
  pdl_trigger();

  Schedule sched(a);
  Segment sg;
  while (next_segment(a, sched, sg)) {
    const int64_t qrow = ((int64_t)sg.b * a.HKV + sg.g) * a.R + sg.rt * kSR;  // first packed row of the tile
    const int rows = min(kSR, a.R - sg.rt * kSR);
    __syncthreads();
    for (int i = tid; i < kSR * D / 8; i += kSThreads) {
      const int r = i / (D / 8), c8 = i % (D / 8);
      float v[8] = {};
      if (r < rows) load_vec<T, 8>(static_cast<const T*>(a.q) + (qrow + r) * D + c8 * 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) qs[r * D + c8 * 8 + e] = v[e];
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[kAcc] = {};
    const int t_row[2] = {(sg.rt * kSR + 2 * warp) % a.T, (sg.rt * kSR + 2 * warp + 1) % a.T};
    for (int kt = sg.t0; kt < sg.t1; ++kt) {
      const int p0 = kt * kSK;
      __syncthreads();  // the last tile's readers are done
#pragma unroll
      for (int s = 0; s < 3; ++s)
        for (int i = tid; i < kSK * D / 8; i += kSThreads) {
          const int r = i / (D / 8), c8 = i % (D / 8);
          float v[8] = {};
          if (p0 + r < sg.n) load8<T, D, BITS>(a, s, sg.b, sg.g, p0 + r, c8, v);
          float* dst = s == 0 ? ks + r * (D + 4) + c8 * 8 : vs + r * 2 * D + (s - 1) * D + c8 * 8;
          reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
      __syncthreads();
      float s2[2] = {0.f, 0.f};
      const float4* kr = reinterpret_cast<const float4*>(ks + lane * (D + 4));
      const float4* q0 = reinterpret_cast<const float4*>(qs + 2 * warp * D);
#pragma unroll 8
      for (int d = 0; d < D / 4; ++d) {
        const float4 k4 = kr[d];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 q4 = q0[h * (D / 4) + d];
          s2[h] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s2[h]))));
        }
      }
      const bool tail = p0 + kSK > sg.n - a.T;  // uniform: some key is drafted or past the end
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = s2[h] * a.scale_log2;
        if (tail) {
          const bool live = 2 * warp + h < rows;
          const int pos = p0 + lane, j = pos - (sg.n - a.T);
          bool v = live && pos < sg.n;
          if (v && j >= 0) v = a.mask ? a.mask[sg.b * a.mask_b + (int64_t)t_row[h] * a.T + j] != 0 : j <= t_row[h];
          if (!v) x = -INFINITY;
        }
        const float mt = fmaxf(m[h], warp_max(x));
        const float mb = mt == -INFINITY ? 0.f : mt;
        const float p = exp2f(x - mb);
        const float al = exp2f(m[h] - mb);  // 0 at the first visible key
        l[h] = l[h] * al + warp_sum(p);
        m[h] = mt;
        ps[lane * kSR + 2 * warp + h] = p;
        if (lane == 0) alpha[2 * warp + h] = al;
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kAcc; ++r) acc[r] *= alpha[row0 + r];
      if (!tail) {
#pragma unroll 8
        for (int k = 0; k < kSK; ++k) {
          const float v = vs[k * 2 * D + ch];
#pragma unroll
          for (int r = 0; r < kAcc; ++r) acc[r] = fmaf(ps[k * kSR + row0 + r], v, acc[r]);
        }
      } else {
        // a hidden row's weight is 0, and what it holds may be NaN: it is left out, not multiplied
        for (int k = 0; k < kSK; ++k) {
          const float v = vs[k * 2 * D + ch];
#pragma unroll
          for (int r = 0; r < kAcc; ++r) {
            const float p = ps[k * kSR + row0 + r];
            if (p != 0.f) acc[r] = fmaf(p, v, acc[r]);
          }
        }
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        inv_l[2 * warp + h] = l[h] == 0.f ? 0.f : 1.f / l[h];
        if (!sg.whole && 2 * warp + h < rows) {
          float* ml = a.part_ml + (sg.slot * kSR + 2 * warp + h) * 2;
          ml[0] = m[h];
          ml[1] = l[h];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kAcc; ++r) {
      if (row0 + r >= rows) break;
      if (sg.whole)
        static_cast<T*>(a.y)[(qrow + row0 + r) * 2 * D + ch] = from_f<T>(acc[r] * inv_l[row0 + r]);
      else
        a.part_o[(sg.slot * kSR + row0 + r) * 2 * D + ch] = acc[r];
    }
  }
}

// ---- join of the cut units' partials -----------------------------------------------------------------
// One warp per output row: O = Σ w·O_s / Σ w·l_s, w = 2^(m_s − max m), over the CTAs that held a part
// of the row's unit, in their order. `grid` is the attention kernel's.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ TreeArgs a, int grid) {
  constexpr int V = 2 * D / 32;  // channels of a lane: two (D 128: four) groups of 4, 128 apart
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t rows_b = (int64_t)a.HKV * a.R;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  if (row >= a.B * rows_b) return;
  const int b = (int)(row / rows_b);
  const int pr = (int)(row % a.R), g = (int)(row % rows_b / a.R);
  const int rt = pr / a.tile_rows, r = pr - rt * a.tile_rows;
  const int per_b = a.HKV * a.row_tiles;
  int64_t total = 0, base = 0;
  for (int i = lane; i < a.B; i += 32) {
    const int nt = key_tiles(a, live_rows(a, i));
    total += nt;
    base += i < b ? nt : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    base += __shfl_xor_sync(0xffffffffu, base, o);
  }
  total *= per_b;
  const int nt = key_tiles(a, live_rows(a, b));
  const int64_t s = base * per_b + (int64_t)(g * a.row_tiles + rt) * nt, e = s + nt;
  auto lo = [&](int64_t i) { return i * total / grid; };
  const int64_t i0 = ((s + 1) * grid - 1) / total, i1 = (e * grid - 1) / total;  // CTAs of tiles s and e − 1
  if (i0 == i1) return;  // written by its CTA
  auto slot_row = [&](int64_t i) { return (2 * i + (lo(i) >= s ? 0 : 1)) * a.tile_rows + r; };
  float M = -INFINITY;
  for (int64_t i = i0; i <= i1; ++i)
    if (lo(i) < lo(i + 1)) M = fmaxf(M, a.part_ml[slot_row(i) * 2]);
  float L = 0.f, o[V] = {};
  for (int64_t i = i0; i <= i1; ++i) {
    if (lo(i) >= lo(i + 1)) continue;
    const int64_t sr = slot_row(i);
    const float ms = a.part_ml[sr * 2];
    if (ms == -INFINITY) continue;
    const float w = exp2f(ms - M);
    L = fmaf(w, a.part_ml[sr * 2 + 1], L);
    const float4* p = reinterpret_cast<const float4*>(a.part_o + sr * 2 * D);
#pragma unroll
    for (int v = 0; v < V / 4; ++v) {
      const float4 f = p[v * 32 + lane];
      o[4 * v] = fmaf(w, f.x, o[4 * v]);
      o[4 * v + 1] = fmaf(w, f.y, o[4 * v + 1]);
      o[4 * v + 2] = fmaf(w, f.z, o[4 * v + 2]);
      o[4 * v + 3] = fmaf(w, f.w, o[4 * v + 3]);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int v = 0; v < V / 4; ++v) {
    const float f[4] = {o[4 * v] * inv, o[4 * v + 1] * inv, o[4 * v + 2] * inv, o[4 * v + 3] * inv};
    store_vec<T, 4>(static_cast<T*>(a.y) + row * 2 * D + (v * 32 + lane) * 4, f);
  }
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

// CTAs of the attention launch: as many as run at once, at most one per key tile of the longest lengths.
int64_t grid_of(const TreeArgs& a, int64_t ctas, int64_t len_bound) {
  const int64_t nt = ceil_div(len_bound < 1 ? 1 : len_bound, a.tile_keys);
  const int64_t all = nt * a.B * a.HKV * a.row_tiles;
  return all < ctas ? all : ctas;
}

template <typename T, int D>
int launch_merge(const TreeArgs& a, int64_t grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ceil_div((int64_t)a.B * a.HKV * a.R, 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tree_merge_kernel<T, D>, a, (int)grid);
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: merge launch: %s", cudaGetErrorString(e));
  return MOTIF_OK;
}

template <typename T, int D, int BITS>
int launch_simt(TreeArgs& a, int64_t grid, cudaStream_t st) {
  auto kern = tree_simt_kernel<T, D, BITS>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, simt_smem<D>());
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: smem attribute: %s", cudaGetErrorString(e));
  kern<<<(unsigned)grid, kSThreads, simt_smem<D>(), st>>>(a);
  const int rc = check_launch("sdpa_dual_v_tree");
  return rc ? rc : launch_merge<T, D>(a, grid, st);
}

constexpr int64_t kMaxTreeRows = 256;

struct Plan {
  int tile_rows, tile_keys;
  int64_t ctas;  // CTAs that run at once
};

Plan plan_of() { return Plan{kSR, kSK, 2 * (int64_t)sm_count()}; }

size_t workspace_of(const Plan& p, int64_t D) {
  return sizeof(float) * 2 * (size_t)p.ctas * (size_t)p.tile_rows * (size_t)(2 * D + 2);
}

}  // namespace
}  // namespace motif

using namespace motif;

extern "C" {

size_t motif_sdpa_dual_v_tree_workspace_bytes(int64_t head_dim) {
  return workspace_of(plan_of(), head_dim);
}

int motif_sdpa_dual_v_tree(int dtype, int bits, int group_size, const void* q, const motif_tree_kv* kv,
                           const uint8_t* tree_mask, int64_t mask_batch_stride, float scale, int64_t batch, int64_t h_q,
                           int64_t h_kv, int64_t tree_rows, int64_t kv_cap, int64_t head_dim, int64_t kv_len,
                           const int32_t* kv_len_dev, int64_t kv_len_stride, void* y, void* workspace,
                           size_t workspace_bytes, int* err, void* stream) {
  MOTIF_REQUIRE(q && kv && y, MOTIF_ERR_NULL, "sdpa_dual_v_tree: null pointer");
  MOTIF_REQUIRE(dtype == MOTIF_F16 || dtype == MOTIF_BF16 || dtype == MOTIF_F32, MOTIF_ERR_DTYPE,
                "sdpa_dual_v_tree: unsupported dtype code %d", dtype);
  MOTIF_REQUIRE(bits == 16 || bits == 4 || bits == 8, MOTIF_ERR_DTYPE, "sdpa_dual_v_tree: bits %d (4, 8 or 16)", bits);
  MOTIF_REQUIRE(batch > 0 && h_q > 0 && h_kv > 0 && kv_cap > 0 && kv_cap < (1ll << 30) && batch < (1 << 20) &&
                    h_q < (1 << 16),
                MOTIF_ERR_BAD_SHAPE, "sdpa_dual_v_tree: bad shape B=%lld H_q=%lld H_kv=%lld cap=%lld", (long long)batch,
                (long long)h_q, (long long)h_kv, (long long)kv_cap);
  MOTIF_REQUIRE(tree_rows >= 1 && tree_rows <= kMaxTreeRows, MOTIF_ERR_BAD_CONTRACT,
                "sdpa_dual_v_tree: %lld tree rows (1..%lld)", (long long)tree_rows, (long long)kMaxTreeRows);
  MOTIF_REQUIRE(head_dim == 64 || head_dim == 128, MOTIF_ERR_BAD_CONTRACT,
                "sdpa_dual_v_tree: head_dim %lld not built (64 and 128 are)", (long long)head_dim);
  MOTIF_REQUIRE(h_q % h_kv == 0, MOTIF_ERR_BAD_CONTRACT, "sdpa_dual_v_tree: H_q=%lld must be a multiple of H_kv=%lld",
                (long long)h_q, (long long)h_kv);
  MOTIF_REQUIRE(kv_len_dev || (kv_len >= tree_rows && kv_len <= kv_cap), MOTIF_ERR_BAD_SHAPE,
                "sdpa_dual_v_tree: kv_len=%lld must be in [%lld, %lld]", (long long)kv_len, (long long)tree_rows,
                (long long)kv_cap);
  MOTIF_REQUIRE(!kv_len_dev || kv_len_stride == 0 || kv_len_stride == 1, MOTIF_ERR_BAD_SHAPE,
                "sdpa_dual_v_tree: kv_len_stride %lld (0 or 1)", (long long)kv_len_stride);
  MOTIF_REQUIRE(!tree_mask || mask_batch_stride == 0 || mask_batch_stride == tree_rows * tree_rows, MOTIF_ERR_BAD_SHAPE,
                "sdpa_dual_v_tree: mask batch stride %lld", (long long)mask_batch_stride);
  const int esz = dtype == MOTIF_F32 ? 4 : 2;
  uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(y);
  for (int i = 0; i < 3; ++i) {
    MOTIF_REQUIRE(kv->data[i], MOTIF_ERR_NULL, "sdpa_dual_v_tree: slot %d null", i);
    al |= reinterpret_cast<uintptr_t>(kv->data[i]);
    if (bits != 16) {
      MOTIF_REQUIRE(kv->scales[i] && kv->biases[i], MOTIF_ERR_NULL, "sdpa_dual_v_tree: slot %d scales/biases null", i);
      MOTIF_REQUIRE((reinterpret_cast<uintptr_t>(kv->scales[i]) | reinterpret_cast<uintptr_t>(kv->biases[i])) % esz == 0,
                    MOTIF_ERR_BAD_CONTRACT, "sdpa_dual_v_tree: misaligned scales/biases");
    }
  }
  MOTIF_REQUIRE(al % 16 == 0, MOTIF_ERR_BAD_CONTRACT, "sdpa_dual_v_tree: operands must be 16-byte aligned");
  TreeArgs a{};
  if (bits == 16) {
    a.sb = kv->stride[0];
    a.sh = kv->stride[1];
    a.sr = kv->stride[2];
    MOTIF_REQUIRE(a.sr >= head_dim && a.sh > 0 && a.sb > 0 && (a.sb * esz) % 16 == 0 && (a.sh * esz) % 16 == 0 &&
                      (a.sr * esz) % 16 == 0,
                  MOTIF_ERR_BAD_CONTRACT, "sdpa_dual_v_tree: row strides (%lld, %lld, %lld) must be multiples of 16 bytes",
                  (long long)a.sb, (long long)a.sh, (long long)a.sr);
  } else {
    MOTIF_REQUIRE(group_size >= 8 && group_size % 8 == 0 && head_dim % group_size == 0, MOTIF_ERR_BAD_CONTRACT,
                  "sdpa_dual_v_tree: group_size %d must be a multiple of 8 that divides head_dim", group_size);
  }
  a.q = q;
  for (int i = 0; i < 3; ++i) {
    a.kv[i] = kv->data[i];
    a.sc[i] = kv->scales[i];
    a.bi[i] = kv->biases[i];
  }
  a.mask = tree_mask;
  a.mask_b = mask_batch_stride;
  a.len_dev = kv_len_dev;
  a.len_step = (int)kv_len_stride;
  a.len = (int)kv_len;
  a.y = y;
  a.err = err;
  a.B = (int)batch;
  a.HKV = (int)h_kv;
  a.gqa = (int)(h_q / h_kv);
  a.T = (int)tree_rows;
  a.R = a.gqa * a.T;
  a.cap = (int)kv_cap;
  a.gs = group_size;
  a.scale_log2 = scale * kLog2e;
  const Plan p = plan_of();
  a.tile_rows = p.tile_rows;
  a.tile_keys = p.tile_keys;
  a.row_tiles = (int)ceil_div(a.R, p.tile_rows);
  MOTIF_REQUIRE(workspace && workspace_bytes >= workspace_of(p, head_dim), MOTIF_ERR_WORKSPACE,
                "sdpa_dual_v_tree: workspace of %zu bytes, needs %zu", workspace_bytes, workspace_of(p, head_dim));
  MOTIF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MOTIF_ERR_BAD_CONTRACT,
                "sdpa_dual_v_tree: workspace must be 16-byte aligned");
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + 2 * p.ctas * p.tile_rows * 2 * head_dim;
  const int64_t grid = grid_of(a, p.ctas, kv_len_dev ? kv_cap : kv_len);
  cudaStream_t st = as_stream(stream);
  MOTIF_DISPATCH_FLOAT(dtype, T, {
    if (head_dim == 64) {
      if (bits == 16) return launch_simt<T, 64, 16>(a, grid, st);
      if (bits == 4) return launch_simt<T, 64, 4>(a, grid, st);
      return launch_simt<T, 64, 8>(a, grid, st);
    }
    if (bits == 16) return launch_simt<T, 128, 16>(a, grid, st);
    if (bits == 4) return launch_simt<T, 128, 4>(a, grid, st);
    return launch_simt<T, 128, 8>(a, grid, st);
  });
  return MOTIF_OK;
}

}  // extern "C"
