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
// (Line, Schedule), whatever the sequences' lengths: a CTA may end one unit and start the next. A unit
// that lies in one CTA is normalised and written by it; the others leave fp32 partials (running
// maximum, Σp, unnormalised O) that tree_merge_kernel joins in a fixed order, or, where a unit is short,
// its CTAs are one cluster and join through shared memory.
//
// Bound by the rows of k, v1 and v2, each read once (the packed rows share them), until gqa·T is some hundred:
// 98.7 MB for a tree of 64 over 16064 fp16 rows, 8 kv heads, D 128 (15 us at the copy rate of 6.57 TB/s). Measured
// there: 42 us, some 27 of it in the tiles (a TMA read of the same rows alone 17.6), 8 start and output, 6 the join;
// a tree of 17 over 16017 q4 rows 36 us, bound by the warps that rebuild its tiles (28 MB; floor 4.3); eight
// ragged requests of 31 rows, 263 MB, 85 us (47 % of the copy rate); a chain of five over 164 rows 8.6 us, latency.
#include <cooperative_groups.h>
#include <cuda.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tma.cuh"

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
  float* part_o;            // [parts][2D / 8][slot_rows][8]
  float* part_ml;           // [parts][slot_rows][2]
  int slot_rows;            // rows of a partial: min(tile_rows, R)
  int* err;
  int B, HKV, gqa, T, R, row_tiles, cap, gs;
  int tile_rows, tile_keys;
  int cuts;                 // > 0: every unit is cut into so many parts, grid (cuts, HKV·row_tiles, B)
  int cluster;              // the parts of a unit are one thread-block cluster, which joins them itself
  float scale_log2;
};

__device__ __forceinline__ int live_rows(const TreeArgs& a, int b) {
  const int n = a.len_dev ? a.len_dev[(int64_t)b * a.len_step] : a.len;
  return min(max(n, 0), a.cap);
}
__device__ __forceinline__ int key_tiles(const TreeArgs& a, int n) {
  return max(1, (n + a.tile_keys - 1) / a.tile_keys);  // an empty cache is one tile without a visible key
}

// Sequences of one length: every unit is cut into `cuts` parts, one CTA each. Otherwise the units' key tiles
// form one line that is cut into `grid` parts of equal length; where a CTA has many tiles every unit counts
// `lead` more than it has, since a CTA that ends one unit and begins the next pays for two loads of
// queries and two outputs.
constexpr int kLead = 8, kLeadTiles = 8;

struct Line {
  int total, per, rem, grid, lead;
  __device__ __forceinline__ void init(int tiles, int units, int parts) {  // tiles + kLead·units < 2^31: checked by the host
    grid = parts;
    lead = tiles >= kLeadTiles * grid ? kLead : 0;
    total = tiles + units * lead;
    per = total / grid;
    rem = total - per * grid;
  }
  __device__ __forceinline__ int lo(int i) const { return i * per + i * rem / grid; }  // ⌊i·total / grid⌋
  __device__ __forceinline__ int owner(int x) const {                                  // the part that holds place x
    int i = (int)((float)x * (float)grid / (float)total);
    i = min(max(i, 0), grid - 1);
    while (i > 0 && lo(i) > x) --i;
    while (i + 1 < grid && lo(i + 1) <= x) ++i;
    return i;
  }
};

__device__ __forceinline__ int cut_at(int k, int nt, int cuts) { return (int)((unsigned)k * (unsigned)nt / (unsigned)cuts); }

// This CTA's share of one unit: key tiles [t0, t1) of row tile rt of kv head g of sequence b.
struct Segment {
  int b, g, rt, n, t0, t1;
  int slot;  // its partial's place; -1: the whole unit
};

// Walks this CTA's part of the line. Every thread of a warp constructs it.
struct Schedule {
  int x0, x1;     // the part
  int at, nt, n;  // the current unit's place, key tiles, live rows
  int b, g, rt, lead;

  __device__ __forceinline__ Schedule(const TreeArgs& a) {
    if (a.cuts) {
      n = live_rows(a, 0);
      nt = key_tiles(a, n);
      b = blockIdx.z;
      g = blockIdx.y / a.row_tiles;
      rt = blockIdx.y - g * a.row_tiles;
      at = 0;
      x0 = cut_at(blockIdx.x, nt, a.cuts);
      x1 = cut_at(blockIdx.x + 1, nt, a.cuts);
      return;
    }
    const int per_b = a.HKV * a.row_tiles;
    int tiles = 0;
    for (int i = threadIdx.x & 31; i < a.B; i += 32) tiles += key_tiles(a, live_rows(a, i));
    tiles = (int)__reduce_add_sync(0xffffffffu, (unsigned)tiles) * per_b;
    Line line;
    line.init(tiles, a.B * per_b, gridDim.x);
    lead = line.lead;
    x0 = line.lo(blockIdx.x);
    x1 = line.lo(blockIdx.x + 1);
    b = 0, at = 0;
    for (;;) {  // the sequence and unit of place x0
      n = live_rows(a, b);
      nt = key_tiles(a, n);
      const int len = (nt + lead) * per_b;
      if (b + 1 >= a.B || x0 < at + len) break;
      at += len;
      ++b;
    }
    const int u = (x0 - at) / (nt + lead);
    at += u * (nt + lead);
    g = u / a.row_tiles;
    rt = u - g * a.row_tiles;
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, Segment& s) {
    if (a.cuts) {
      if (at || x0 >= x1) return false;
      at = 1;
      s.b = b, s.g = g, s.rt = rt, s.n = n;
      s.t0 = x0, s.t1 = x1;
      s.slot = x0 == 0 && x1 == nt && !a.cluster ? -1 : (int)((blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x);
      return true;
    }
    for (;;) {
      if (at >= x1 || b >= a.B) return false;
      s.t0 = max(x0 - at - lead, 0);
      s.t1 = min(x1 - at - lead, nt);
      s.b = b, s.g = g, s.rt = rt, s.n = n;
      // at most two segments of a CTA are parts of units: one begun before it, and its last
      s.slot = s.t0 == 0 && s.t1 == nt ? -1 : 2 * (int)blockIdx.x + (s.t0 > 0 ? 0 : 1);
      at += nt + lead;
      if (++rt == a.row_tiles) {
        rt = 0;
        if (++g == a.HKV) {
          g = 0;
          if (++b < a.B) {
            n = live_rows(a, b);
            nt = key_tiles(a, n);
          }
        }
      }
      if (s.t1 > s.t0) return true;
    }
  }
};

// Place of eight channels (chunk c8) of a partial's row: a warp of rows writes whole lines.
template <int D>
__device__ __forceinline__ int64_t part_at(const TreeArgs& a, int slot, int c8, int row) {
  return (((int64_t)slot * (2 * D / 8) + c8) * a.slot_rows + row) * 8;
}

// Tree rows that row t of sequence b sees, j0 ≤ j < j0 + 64, as bits.
__device__ __forceinline__ uint64_t mask_bits(const TreeArgs& a, int b, int t, int j0) {
  if (!a.mask) return t < j0 ? 0 : t - j0 >= 63 ? ~0ull : (2ull << (t - j0)) - 1;
  const uint8_t* m = a.mask + b * a.mask_b + (int64_t)t * a.T;
  uint64_t w = 0;
  if ((((reinterpret_cast<uintptr_t>(m) + j0) | (a.T - j0)) & 7) == 0) {  // whole 8-byte words
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint64_t x = j0 + 8 * i < a.T ? *reinterpret_cast<const uint64_t*>(m + j0 + 8 * i) : 0;
      x |= x >> 4, x |= x >> 2, x |= x >> 1;  // bit 0 of a byte: the byte is not 0 …
      w |= ((x & 0x0101010101010101ull) * 0x0102040810204080ull >> 56) << (8 * i);  // … eight of them side by side
    }
    return w;
  }
#pragma unroll 16
  for (int c = 0; c < 64; ++c)
    if (j0 + c < a.T) w |= (uint64_t)(m[j0 + c] != 0) << c;
  return w;
}

// Bit c: the row sees cache row p0 + c, c < 64, of n live ones; row: its mask_bits from 0 (used where T ≤ 64).
__device__ __forceinline__ uint64_t visible(const TreeArgs& a, uint64_t row, int b, int t, int ctx, int p0) {
  const int j0 = p0 - ctx;  // tree row of cache row p0
  if (j0 <= -64) return ~0ull;
  if (a.T > 64) row = mask_bits(a, b, t, max(j0, 0));
  else if (j0 > 0) row = j0 > 63 ? 0 : row >> j0;
  return j0 < 0 ? row << -j0 | ((1ull << -j0) - 1) : row;  // the context, then the tree
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

  Schedule sched(a);
  Segment sg;
  while (sched.next(a, sg)) {
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
        if (sg.slot >= 0 && 2 * warp + h < rows) {
          float* ml = a.part_ml + ((int64_t)sg.slot * a.slot_rows + 2 * warp + h) * 2;
          ml[0] = m[h];
          ml[1] = l[h];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kAcc; ++r) {
      if (row0 + r >= rows) break;
      if (sg.slot < 0)
        static_cast<T*>(a.y)[(qrow + row0 + r) * 2 * D + ch] = from_f<T>(acc[r] * inv_l[row0 + r]);
      else
        a.part_o[part_at<D>(a, sg.slot, ch >> 3, row0 + r) + (ch & 7)] = acc[r];
    }
  }
}

// ---- tensor-core form: 16-bit rows and packed caches of 16-bit models --------------------------------
// One CTA per SM takes 128 packed query rows (rows past the unit's are zero) and 64-key tiles:
//   S = Q·Kᵀ (M 128, N 64, K D) and O += P·[V1 | V2] (M 128, N 2D, K 64) run as tcgen05.mma into tensor
// memory (S: kSBufs × 64 columns, O: 2D columns); Q and K are K-major and V is MN-major
// as the cache rows lie, in the 128-byte swizzle; P replaces its S in tensor memory.
//   warp 0       TMA: K and V tiles straight from the cache into rings of kStages (16-bit rows), or the
//                packed rows, scales and biases into a ring of raw tiles;
//   warp 1       one lane issues the MMAs, S up to kSBufs tiles ahead of P·V within a segment, so that the
//                softmax groups find their tiles ready (16-bit rows: S from warp 1, P·V from warp 10);
//   warps 2..9   two softmax groups of four warps that take the tiles in turn (one warp alone on a
//                scheduler waits out every latency of its 64-column row: tensor-memory reads, the maximum,
//                the exponentials). A thread is a query row: it takes S from tensor memory and writes P in
//                the type. The groups share the row's reference maximum, handed from tile to tile; it is
//                raised, and O rescaled in tensor memory, only when a row's maximum grew by more than 2^8
//                (weights stay ≤ 256, and the result is exact). Each group sums its own tiles' weights; at
//                the end group A writes the V1 half of the rows and group B the V2 half. Warps without a
//                row only keep the barriers.
//   warps 10..15 (packed) rebuild K and V tiles from the codes with packed 16-bit arithmetic: the code is
//                exact in the type (exponent trick), scale·code + bias one fused rounding.
// Where the tile holds drafted rows or the cache's end, the softmax warps clear V rows that no query may
// use (rows ≥ n, whatever the buffer holds) and drafted rows with a non-finite value: a zero weight times
// NaN would reach queries the row is hidden from. The queries that do see such a row add it at the end
// from the cache itself.
// Every wait is bounded; one that runs out sets the abort flag, rows not finished become NaN and the
// error word is set, and the CTA drains its copies and MMAs before it frees tensor memory.
constexpr int kTR = 128, kTK = 64;

template <int BITS>
struct TcCfg {
  // K and V operand tiles. V is held until P·V, K free after S; packed caches also need room for raw tiles
  // (8-bit ones are twice as large).
  static constexpr int kStages = BITS == 8 ? 2 : 3;
  static constexpr int kVStages = BITS == 16 ? 4 : BITS == 4 ? 3 : 2;
  static constexpr int kThreads = BITS == 16 ? 352 : 512;
  static constexpr int kFill = BITS == 16 ? 1 : 6;  // arrivals that fill a K or V tile
};
constexpr int kRawMax = 4;
constexpr int kSBufs = 4;  // S tiles in tensor memory
constexpr int kMaxCluster = 8;

struct TcArgs {
  TreeArgs t;
  CUtensorMap tm[3];  // k, v1, v2 rows
  int raw_stages, code_bytes, group_bytes;  // packed: ring depth, bytes of a row's codes and of its scales
};

struct Cleared {
  int seg;           // the segment the bits belong to
  uint32_t bits[8];  // tree rows
};

template <int D, int BITS>
struct TcMap {  // shared memory, bytes from a 1024-byte boundary
  static constexpr int kHalves = D / 64;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kHalves * kTR * 128;
  static constexpr int kKBytes = kHalves * kTK * 128;
  static constexpr int kV = kK + TcCfg<BITS>::kStages * kKBytes;
  static constexpr int kVBytes = 2 * kKBytes;
  static constexpr int kBar = kV + TcCfg<BITS>::kVStages * kVBytes;
  static constexpr int kNumBars = 1 + 2 * TcCfg<BITS>::kStages + 2 * TcCfg<BITS>::kVStages + 3 * kSBufs + 1 + 2 * kRawMax + 13;
  static constexpr int kState = kBar + kNumBars * 8 + 16;  // [128] reference maxima, [2][128] sums of the groups
  static constexpr int kJoin = kState + 3 * kTR * 4;       // [128] (maximum, sum) of this CTA's part, its rows' weights
  static constexpr int kBad = kJoin + kTR * 8 + (kTR + 2 * kMaxCluster) * 4;        // drafted rows cleared: [2 segments][8 warps] Cleared
  static constexpr int kRaw = (kBad + 2 * 8 * (int)sizeof(Cleared) + 127) / 128 * 128;
};

// Eight floats as one 32-byte sector: two 16-byte halves would each make L2 fetch the rest of it from memory.
__device__ __forceinline__ void store_sector(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Bounded mbarrier wait: about half a second of polls, far above any pipeline stage.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 16); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

constexpr int kTestPolls = 1 << 23;  // of two or three tests each: about half a second too
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Cluster join: channels [4·c4, 4·c4 + 4) of a row of the CTA's unnormalised O, in place of the K and V tiles. Eight rows
// (lanes that write) and eight chunks of a row (lanes that read) fall into different banks.
template <int D>
__device__ __forceinline__ int join_at(int row, int c4) {
  return row * 2 * D * 4 + ((c4 ^ (row & 7)) << 4);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D[tmem] (+)= A·B of kind::f16, the two shared-memory descriptors given by their lower words and the common upper one.
__device__ __forceinline__ void mma_words(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
      " setp.ne.b32 p, %5, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// The same with A (rows in lanes, two 16-bit values of K a column) in tensor memory.
__device__ __forceinline__ void mma_tmem_a(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Any of the two 16-bit values of w is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool nonfinite2(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// Channel held at position i of an 8-channel chunk of the operand tiles: q4 words give the channel pairs
// (j, j + 4) in one instruction, so K, V and Q keep that order and the output undoes it.
template <int BITS>
__host__ __device__ constexpr int chunk_channel(int i) {
  return BITS == 4 ? (i & 1) * 4 + (i >> 1) : i;
}

// Eight codes (q4: one word; q8: two) -> eight values scale·code + bias of the type, chunk order. One rounding to the
// type (half a step, 2^-11 or 2^-8), since the tensor cores take 16-bit operands: the values that motif_dequantize
// gives. Over a long context it adds to a result's error what rounding P does (4·10^-4 against 3·10^-4, fp16).
template <typename T, int BITS>
__device__ __forceinline__ uint4 dequant8(uint32_t w0, uint32_t w1, T sc, T bi) {
  uint32_t r[4];
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 s2 = __half2half2(sc), b2 = __half2half2(bi);
    auto code = [](uint32_t x) { return *reinterpret_cast<__half2*>(&x); };
    __half2 q[4];
    if constexpr (BITS == 4) {
      const __half2 k1024 = __float2half2_rn(1024.f), k16 = __float2half2_rn(0.0625f), k64 = __float2half2_rn(-64.f);
      const uint32_t hi = w0 >> 8;
      q[0] = __hsub2(code((w0 & 0x000F000Fu) | 0x64006400u), k1024);
      q[1] = __hfma2(code((w0 & 0x00F000F0u) | 0x64006400u), k16, k64);
      q[2] = __hsub2(code((hi & 0x000F000Fu) | 0x64006400u), k1024);
      q[3] = __hfma2(code((hi & 0x00F000F0u) | 0x64006400u), k16, k64);
    } else {
      const __half2 k1024 = __float2half2_rn(1024.f);
      q[0] = __hsub2(code(__byte_perm(w0, 0x64646464u, 0x4140)), k1024);
      q[1] = __hsub2(code(__byte_perm(w0, 0x64646464u, 0x4342)), k1024);
      q[2] = __hsub2(code(__byte_perm(w1, 0x64646464u, 0x4140)), k1024);
      q[3] = __hsub2(code(__byte_perm(w1, 0x64646464u, 0x4342)), k1024);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 v = __hfma2(q[i], s2, b2);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else if constexpr (BITS == 4) {
    const __nv_bfloat162 s2 = __bfloat162bfloat162(sc), b2 = __bfloat162bfloat162(bi);
    const __nv_bfloat162 k128 = __float2bfloat162_rn(128.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x = ((w0 >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 v = __hfma2(__hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), k128), s2, b2);
      r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {  // eight bits do not fit bf16's exponent trick: through fp32
    const float s = to_f<T>(sc), b = to_f<T>(bi);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaf(s, (float)(((i < 4 ? w0 : w1) >> (8 * (i & 3))) & 255u), b);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Adds Σ p_j·v_j over the cleared drafted rows j that packed row pr (tree row t) sees to half `grp` of its output
// (yrow, normalised by inv) or partial (slot, row), read from the cache. Their V holds an infinity or NaN, so this
// runs for broken inputs only; the finite channels of such an output row are rounded once more per row added.
template <typename T, int D, int BITS>
__device__ __forceinline__ void add_cleared(const TreeArgs& a, int b, int g, const Cleared* bad, int seg, int pr, int t,
                                            int ctx, float m_ref, float inv, int grp, T* yrow, int slot, int row,
                                            uint8_t* joined) {
  const T* q = static_cast<const T*>(a.q) + (((int64_t)b * a.HKV + g) * a.R + pr) * D;
#pragma unroll 1
  for (int j = 0; j < a.T; ++j) {
    uint32_t w = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) w |= bad[i].seg == seg ? bad[i].bits[j >> 5] : 0u;
    if (!((w >> (j & 31)) & 1)) continue;
    if (!(a.mask ? a.mask[b * a.mask_b + (int64_t)t * a.T + j] != 0 : j <= t)) continue;
    float s = 0.f, v[8];
#pragma unroll 1
    for (int c8 = 0; c8 < D / 8; ++c8) {
      load8<T, D, BITS>(a, 0, b, g, ctx + j, c8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(to_f<T>(q[c8 * 8 + e]), v[e], s);
    }
    const float p = exp2f(fmaf(s, a.scale_log2, m_ref == -INFINITY ? 0.f : -m_ref));
#pragma unroll 1
    for (int c8 = 0; c8 < D / 8; ++c8) {
      load8<T, D, BITS>(a, 1 + grp, b, g, ctx + j, c8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = grp * D + c8 * 8 + e;
        if (yrow) {
          yrow[c] = from_f<T>(fmaf(p * inv, v[e], to_f<T>(yrow[c])));
        } else {
          float& o = a.cluster ? reinterpret_cast<float*>(joined + join_at<D>(row, c >> 2))[c & 3]
                               : a.part_o[part_at<D>(a, slot, c >> 3, row) + e];
          o = fmaf(p, v[e], o);
        }
      }
    }
  }
}

// The parts of a unit meet in distributed shared memory: CTA `rank` of the cluster joins the rows rank, rank + C, …
// of all CTAs, O = Σ w·O_s / Σ w·l_s with w = 2^(m_s − max m), in the order of the parts.
template <typename T, int D>
__device__ __forceinline__ void join_cluster(const TreeArgs& a, uint8_t* part, float2* ml, float* weights) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  cluster.sync();  // every part is in place
  const int rt = blockIdx.y % a.row_tiles, g = blockIdx.y / a.row_tiles;
  const int rows = min(kTR, a.R - rt * kTR), mine = rank < rows ? (rows - rank + C - 1) / C : 0;
  T* y = static_cast<T*>(a.y) + (((int64_t)blockIdx.z * a.HKV + g) * a.R + rt * kTR) * 2 * D;
  // a row's weights, already over its sum: 16 lanes a row, a lane a part
  for (int i = threadIdx.x >> 4; i < (mine + 1) / 2 * 2; i += blockDim.x >> 4) {
    const int s = threadIdx.x & 15;
    float2 v = make_float2(-INFINITY, 0.f);
    if (i < mine && s < C) v = *cluster.map_shared_rank(ml + rank + i * C, s);
    float top = v.x;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float w = v.x == -INFINITY ? 0.f : exp2f(v.x - top), den = v.x == -INFINITY ? v.y : w * v.y;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    if (i < mine && s < C) weights[i * C + s] = den == 0.f ? 0.f : den == den ? w / den : NAN;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < mine * (2 * D / 4); i += blockDim.x) {
    const int k = i / (2 * D / 4), c4 = i % (2 * D / 4), row = rank + k * C;
    float o[4] = {};
#pragma unroll 4
    for (int s = 0; s < C; ++s) {
      const float w = weights[k * C + s];
      if (w == 0.f) continue;  // an empty part, or one that saw no key of this row
      const float4 f = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part, s) + join_at<D>(row, c4));
      o[0] = fmaf(w, f.x, o[0]), o[1] = fmaf(w, f.y, o[1]), o[2] = fmaf(w, f.z, o[2]), o[3] = fmaf(w, f.w, o[3]);
    }
    store_vec<T, 4>(y + (int64_t)row * 2 * D + c4 * 4, o);
  }
  cluster.sync();  // the others may still read this CTA's part
}

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(TcCfg<BITS>::kThreads, 1) tree_tc_kernel(const __grid_constant__ TcArgs ta) {
  using Cfg = TcCfg<BITS>;
  using Map = TcMap<D, BITS>;
  constexpr int NS = Cfg::kStages, NV = Cfg::kVStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kColS = 0, kColO = kSBufs * kTK, kCols = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const TreeArgs& a = ta.t;
  const uint32_t sb = tc::smem_addr(smem);
  const uint32_t bar = sb + Map::kBar;
  const uint32_t q_full = bar;
  auto k_full = [&](int s) { return bar + 8u * (1 + s); };
  auto k_empty = [&](int s) { return bar + 8u * (1 + NS + s); };
  constexpr int kB0 = 1 + 2 * NS, kB1 = kB0 + 2 * NV, kB2 = kB1 + kSBufs, kB3 = kB2 + 2 * kSBufs + 1, kB4 = kB3 + 2 * kRawMax;
  auto v_full = [&](int s) { return bar + 8u * (kB0 + s); };
  auto v_empty = [&](int s) { return bar + 8u * (kB0 + NV + s); };
  auto s_full = [&](int s) { return bar + 8u * (kB1 + s); };
  auto p_full = [&](int s) { return bar + 8u * (kB2 + s); };  // P, and P·V done, by the S buffer that holds P
  auto o_done = [&](int s) { return bar + 8u * (kB2 + kSBufs + s); };
  const uint32_t drain = bar + 8u * (kB2 + 2 * kSBufs);
  auto raw_full = [&](int s) { return bar + 8u * (kB3 + s); };
  auto raw_empty = [&](int s) { return bar + 8u * (kB3 + kRawMax + s); };
  auto m_next = [&](int g, int q) { return bar + 8u * (kB4 + 4 * g + q); };  // maxima handed on by group g
  auto l_both = [&](int q) { return bar + 8u * (kB4 + 8 + q); };
  const uint32_t o_read = bar + 8u * (kB4 + 12);  // every softmax warp has read its part of a segment's O and sums
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Map::kBar + Map::kNumBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  Schedule sched(a);
  Segment sg;
  bool more = sched.next(a, sg);
  const bool softmax = warp >= 2 && warp < 10;
  const int grp = warp >= 6, q = warp & 3;  // softmax: a warp reads tensor-memory lanes 32·(warp mod 4) ..
  const int r = q * 32 + lane;
  // A query row's half (group A the first channels, B the second), issued before the first copies fill the memory
  // system's queues: straight to its swizzled place, or (q4: the channels change places) through registers.
  constexpr int kQRegs = BITS == 4 ? D / 16 : 1;
  uint4 qv[kQRegs];
  auto q_place = [&](int i) {
    const int c8 = grp * (D / 16) + i;
    return Map::kQ + (c8 >> 3) * kTR * 128 + r * 128 + (((c8 & 7) ^ (r & 7)) << 4);
  };
  auto fetch_q = [&](const Segment& g) {
    const int pr = g.rt * kTR + r;
    const bool live = pr < a.R;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                      (((int64_t)g.b * a.HKV + g.g) * a.R + (live ? pr : 0)) * D) + grp * (D / 16);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      if constexpr (BITS == 4)
        qv[i] = live ? src[i] : make_uint4(0, 0, 0, 0);
      else
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sb + q_place(i)), "l"(src + i), "r"(live ? 16 : 0)
                     : "memory");
    }
  };
  if (softmax && more) fetch_q(sg);
  if (threadIdx.x < Map::kNumBars) {  // a barrier a thread: one thread's loop over all takes 1 us
    const int i = threadIdx.x;
    int count = 1;
    if (i == 0) count = 8;                                                                  // q_full
    if ((i >= 1 && i < 1 + NS) || (i >= kB0 && i < kB0 + NV)) count = Cfg::kFill;           // k_full, v_full
    if (i >= kB2 && i < kB2 + kSBufs) count = 4;                                            // p_full
    if (i >= kB3 + kRawMax && i < kB4) count = Cfg::kFill;                                  // raw_empty
    if (i >= kB4 + 8 && i < kB4 + 12) count = 2;                                            // l_both
    if (i == kB4 + 12) count = 8;                                                           // o_read
    if (i == kB2 + 2 * kSBufs) count = BITS == 16 ? 2 : 1;                                  // drain
    tc::mbar_init(bar + 8u * i, count);
    if (i < 16) reinterpret_cast<Cleared*>(smem + Map::kBad)[i].seg = -1;
    if (i == 0) *abort_flag = 0;
    tc::mbar_fence_init();
  }
  float2* join_ml = reinterpret_cast<float2*>(smem + Map::kJoin);
  if (softmax && grp == 0) join_ml[r] = make_float2(-INFINITY, 0.f);  // a part without a tile
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_addr(tmem_slot), kCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Below, `it` counts this CTA's key tiles over all its segments: ring stages and barrier parities follow it.
  if (warp == 0) {
    if (lane == 0) {  // ---- copies ----
      int it = 0, k_iss = 0, v_iss = 0;
      bool ok = true;
      for (; ok && more; more = sched.next(a, sg)) {
        for (int kt = sg.t0; kt < sg.t1; ++kt, ++it) {
          const int p0 = kt * kTK;
          if (*abort_flag) { ok = false; break; }
          if constexpr (BITS == 16) {
            const int s = it % NS, sv = it % NV;
            if (it >= NS && !bar_wait(k_empty(s), (it / NS - 1) & 1)) { ok = false; break; }
            const uint32_t kb = sb + Map::kK + s * Map::kKBytes;
            tc::mbar_expect_tx(k_full(s), Map::kKBytes);
#pragma unroll
            for (int h = 0; h < Map::kHalves; ++h)
              tc::tma_load_4d(kb + h * kTK * 128, &ta.tm[0], h * 128, p0, sg.g, sg.b, k_full(s));
            k_iss = it + 1;
            if (it >= NV && !bar_wait(v_empty(sv), (it / NV - 1) & 1)) { ok = false; break; }
            const uint32_t vb = sb + Map::kV + sv * Map::kVBytes;
            tc::mbar_expect_tx(v_full(sv), Map::kVBytes);
#pragma unroll
            for (int h = 0; h < 2 * Map::kHalves; ++h)
              tc::tma_load_4d(vb + h * kTK * 128, &ta.tm[1 + h / Map::kHalves], (h % Map::kHalves) * 128, p0, sg.g, sg.b,
                              v_full(sv));
            v_iss = it + 1;
          } else {
            const int s = it % ta.raw_stages;
            if (it >= ta.raw_stages && !bar_wait(raw_empty(s), (it / ta.raw_stages - 1) & 1)) { ok = false; break; }
            const int rows = min(kTK, a.cap - p0);
            const int64_t row = ((int64_t)sg.b * a.HKV + sg.g) * a.cap + p0;
            const uint32_t cb = rows * ta.code_bytes, gb = rows * ta.group_bytes;
            uint32_t dst = sb + Map::kRaw + s * (3 * kTK * ta.code_bytes + 6 * kTK * ta.group_bytes);
            tc::mbar_expect_tx(raw_full(s), 3 * cb + 6 * gb);
#pragma unroll
            for (int i = 0; i < 3; ++i, dst += kTK * ta.code_bytes)
              tc::bulk_load(dst, static_cast<const char*>(a.kv[i]) + row * ta.code_bytes, cb, raw_full(s));
#pragma unroll
            for (int i = 0; i < 3; ++i, dst += 2 * kTK * ta.group_bytes) {
              tc::bulk_load(dst, static_cast<const char*>(a.sc[i]) + row * ta.group_bytes, gb, raw_full(s));
              tc::bulk_load(dst + kTK * ta.group_bytes, static_cast<const char*>(a.bi[i]) + row * ta.group_bytes, gb,
                            raw_full(s));
            }
            k_iss = it + 1;
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // the copies issued last on each stage have landed before the CTA may exit
      const int ring = BITS == 16 ? NS : ta.raw_stages;
      for (int j = max(0, k_iss - ring); j < k_iss; ++j)
        if (!bar_wait(BITS == 16 ? k_full(j % ring) : raw_full(j % ring), (j / ring) & 1)) *abort_flag = 1;
      for (int j = max(0, v_iss - NV); j < v_iss; ++j)
        if (!bar_wait(v_full(j % NV), (j / NV) & 1)) *abort_flag = 1;
    }
  } else if (warp == 1 || (BITS == 16 && warp == 10)) {
    if (lane == 0) {  // ---- MMAs ----
      constexpr uint32_t idesc_qk = tc::idesc_f16_f32(kTR, kTK, false, false, kBf16);
      constexpr uint32_t idesc_pv = tc::idesc_f16_f32(kTR, 2 * D, true, false, kBf16);
      // Descriptors as words: the upper ones are one constant (1024-byte atoms, 128-byte swizzle) and the lower
      // ones advance by constants, so that a product costs one addition.
      constexpr uint32_t hi = 1024 >> 4 | 1u << 14 | 2u << 29;
      // in a cluster, shared addresses carry the CTA's rank above the 18 bits that a descriptor holds
      auto lower = [&](int at, uint32_t lbo) { return ((sb + at) >> 4 & 0x3FFF) | lbo << 16; };
      const uint32_t q_lo = lower(Map::kQ, 1), k_lo = lower(Map::kK, 1), v_lo = lower(Map::kV, kTK * 128 >> 4);
      auto issue_qk = [&](int j) {
        const int s = j % NS;
        tc::tc_fence_after();
        const uint32_t kl = k_lo + s * (Map::kKBytes >> 4), d = tmem + kColS + kTK * (j % kSBufs);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_words(d, q_lo + (kk >> 2) * (kTR * 128 >> 4) + (kk & 3) * 2, kl + (kk >> 2) * (kTK * 128 >> 4) + (kk & 3) * 2, hi,
                    idesc_qk, kk > 0);
        tc::mma_commit(s_full(j % kSBufs));
        tc::mma_commit(k_empty(s));
      };
      auto issue_pv = [&](int j, bool accumulate) {
        tc::tc_fence_after();
        const uint32_t pt = tmem + kColS + kTK * (j % kSBufs), vl = v_lo + (j % NV) * (Map::kVBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kTK / 16; ++kk)
          mma_tmem_a(tmem + kColO, pt + kk * 8, vl + kk * (2048 >> 4), hi, idesc_pv, accumulate || kk > 0);
        tc::mma_commit(o_done(j % kSBufs));
        tc::mma_commit(v_empty(j % NV));
      };
      bool ok = true;
      if constexpr (BITS == 16) {
        // Two issuers: products of one thread wait for its own polls and issue slots (0.36 us an S, 0.19 us a P·V and
        // as much again between them: 1.15 us a tile from one thread).
        int it = 0, seg = 0;
        for (; ok && more; more = sched.next(a, sg), ++seg) {
          // A segment's first P·V overwrites O, which both groups read after they met in l_both.
          if (warp == 1 || seg) ok = bar_wait(warp == 1 ? q_full : o_read, (warp == 1 ? seg : seg + 1) & 1);
          for (int kt = sg.t0; ok && kt < sg.t1; ++kt, ++it) {
            if (warp == 1) {  // S: its buffer is free once the P·V of kSBufs tiles before has read P there
              ok = (it < kSBufs || bar_wait(o_done(it % kSBufs), (it / kSBufs - 1) & 1)) && bar_wait(k_full(it % NS), (it / NS) & 1);
              if (ok) issue_qk(it);
            } else {
              ok = bar_wait(p_full(it % kSBufs), (it / kSBufs) & 1) && bar_wait(v_full(it % NV), (it / NV) & 1);
              if (ok) issue_pv(it, kt > sg.t0);
            }
            if (*abort_flag) ok = false;
          }
        }
      } else {
        int it = 0, qn = 0, seg = 0;  // the next P·V, the next S
        for (; ok && more; more = sched.next(a, sg), ++seg) {
          ok = bar_wait(q_full, seg & 1);
          const int end = it + sg.t1 - sg.t0, begin = it;
          // S runs up to kSBufs tiles ahead of P·V; its buffer is free once the P·V of kSBufs tiles before has read P there.
          for (int polls = 0; ok && it < end;) {
            const bool s_ahead = qn < end && qn < it + kSBufs &&
                                 (qn < kSBufs || bar_test(o_done(qn % kSBufs), (qn / kSBufs - 1) & 1));
            if (s_ahead && (qn <= it + 1 || !bar_test(p_full(it % kSBufs), (it / kSBufs) & 1)) &&
                bar_test(k_full(qn % NS), (qn / NS) & 1)) {
              issue_qk(qn++);
              polls = 0;
            } else if (qn > it && (it > begin || bar_test(o_read, (seg + 1) & 1)) &&  // O as above; before the first phase the parity of a finished one
                       bar_test(p_full(it % kSBufs), (it / kSBufs) & 1) && bar_test(v_full(it % NV), (it / NV) & 1)) {
              issue_pv(it, it > begin);
              ++it;
              polls = 0;
            } else if (++polls > kTestPolls || *abort_flag) {
              ok = false;
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // every MMA this thread issued completes before tensor memory can be freed
      tc::mma_commit(drain);
      if (!bar_wait(drain, 0)) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp < 10) {  // ---- softmax: one thread per query row, two groups ----
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16);
    const float mult = fabsf(a.scale_log2);
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80000000u : 0u;  // scale < 0: −S with |scale|
    float* m_row = reinterpret_cast<float*>(smem + Map::kState) + r;
    float* l_row = m_row + kTR;  // group g's sum at l_row[g * kTR]
    Cleared* bad_all = reinterpret_cast<Cleared*>(smem + Map::kBad);
    auto store_q = [&]() {
      if constexpr (BITS == 4) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {  // (0,1)(2,3)(4,5)(6,7) -> (0,4)(1,5)(2,6)(3,7)
          const uint4 v = qv[i];
          *reinterpret_cast<uint4*>(smem + q_place(i)) =
              make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                         __byte_perm(v.y, v.w, 0x7632));
        }
      } else {
        asm volatile("cp.async.wait_all;\n" ::: "memory");
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
    };
    // Bounded wait of the whole warp; false once anything has run out.
    auto wait = [&](uint32_t b, int phase) {
      const bool got = bar_wait(b, phase & 1);
      return !__any_sync(0xffffffffu, !got || *abort_flag);
    };
    bool alive = true;
    int it = 0, seg = 0;
    int handed = 0, joined = 0;  // phases of m_next and l_both: a warp without a row takes no part in a segment's
    if (more) store_q();
    while (more) {
      const int pr = sg.rt * kTR + r;
      const bool live = pr < a.R;
      const bool work = sg.rt * kTR + q * 32 < a.R;  // this warp has a row
      const int t = live ? pr % a.T : 0;
      const int ctx = sg.n - a.T;
      // read before the first tile arrives
      const uint64_t mrow = live && a.T <= 64 && sg.t1 * kTK > ctx ? mask_bits(a, sg.b, t, 0) : 0;
      float m_mine = -INFINITY, l = 0.f;  // the maximum that l refers to
      for (int kt = sg.t0; kt < sg.t1; ++kt, ++it) {
        if ((it & 1) != grp || !alive) continue;
        const int p0 = kt * kTK;
        const bool tail = p0 + kTK > ctx;  // drafted rows or the cache's end in this tile
        const uint64_t vis = tail && live ? visible(a, mrow, sg.b, t, ctx, p0) : 0;
        if (!(alive = wait(s_full(it % kSBufs), it / kSBufs))) continue;
        tc::tc_fence_after();
        const uint32_t ts = trow + kColS + kTK * (it % kSBufs);
        bool need = false;
        float factor = 1.f, mb = 0.f, mul = mult;
        constexpr bool kKeep = BITS == 16;  // registers for all 64 columns; else they are read twice, in one loop's code
        float sv[kKeep ? 2 : 1][32];
        auto load_s = [&](int h, float (&x)[32]) {
          uint32_t u[32];
          tc::tmem_ld32(ts + 32 * h, u);
          tc::tmem_ld_wait();
          if (flip) {
#pragma unroll
            for (int c = 0; c < 32; ++c) u[c] ^= flip;
          }
          if (tail) {
            const uint32_t v = (uint32_t)(vis >> (32 * h));
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = (v >> c) & 1 ? __uint_as_float(u[c]) * mult : -INFINITY;
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(u[c]);
          }
        };
        if (work) {
          if (tail) mul = 1.f;
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll(kKeep ? 2 : 1)
          for (int h = 0; h < 2; ++h) {
            load_s(h, sv[kKeep ? h : 0]);
#pragma unroll
            for (int c = 0; c < 32; ++c) mx[c & 3] = fmaxf(mx[c & 3], sv[kKeep ? h : 0][c]);
          }
          float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          m_tile = m_tile == -INFINITY ? -INFINITY : m_tile * mul;
          float m_prev = -INFINITY;
          if (kt > sg.t0) {
            if (!(alive = wait(m_next(grp ^ 1, q), handed++))) continue;
            m_prev = *m_row;
          }
          need = m_tile > m_prev + 8.f;
          const float m_new = need ? m_tile : m_prev;
          *m_row = m_new;
          if (kt + 1 < sg.t1) {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(m_next(grp, q));
          }
          if (need) factor = ex2(m_prev - m_new);  // 0 at the first visible key
          if (m_new != m_mine) l *= ex2(m_mine - m_new);
          m_mine = m_new;
          mb = m_new == -INFINITY ? 0.f : m_new;
        }
        if (tail) {  // clear the V rows a zero weight may not meet
          const int st = it % NV;
          if (!(alive = wait(v_full(st), it / NV))) continue;
          const int vr = q * 16 + (lane >> 1), pos = p0 + vr;
          bool clear = pos >= sg.n;
          uint8_t* vrow = smem + Map::kV + st * Map::kVBytes + (lane & 1) * Map::kHalves * kTK * 128 + vr * 128;
          if (!clear && pos >= ctx) {
            bool nf = false;
#pragma unroll
            for (int h = 0; h < Map::kHalves; ++h)
#pragma unroll 4
              for (int c = 0; c < 8; ++c) {
                const uint4 v = *reinterpret_cast<const uint4*>(vrow + h * kTK * 128 + ((c + vr) & 7) * 16);
                nf |= nonfinite2<T>(v.x) | nonfinite2<T>(v.y) | nonfinite2<T>(v.z) | nonfinite2<T>(v.w);
              }
            clear = nf;
          }
          clear |= __shfl_xor_sync(0xffffffffu, clear, 1);
          if (clear) {
#pragma unroll
            for (int h = 0; h < Map::kHalves; ++h)
#pragma unroll 4
              for (int c = 0; c < 8; ++c)
                *reinterpret_cast<uint4*>(vrow + h * kTK * 128 + ((c + vr) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          const bool drafted = clear && pos < sg.n;
          if (__any_sync(0xffffffffu, drafted)) {
            // The slot was last read two segments ago; this segment's first S, which needs every warp's Q of
            // it, came after that.
            Cleared* mine = bad_all + (seg & 1) * 8 + grp * 4 + q;
            if (mine->seg != seg && lane < 8) mine->bits[lane] = 0;
            __syncwarp();
            if (lane == 0) mine->seg = seg;
            if (drafted && (lane & 1) == 0) atomicOr(&mine->bits[(pos - ctx) >> 5], 1u << ((pos - ctx) & 31));
          }
        }
        if (work) {  // P in the type (one rounding of each weight), over the first half of its S
          float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll(kKeep ? 2 : 1)
          for (int h = 0; h < 2; ++h) {
            float(&x)[32] = sv[kKeep ? h : 0];
            if constexpr (!kKeep) load_s(h, x);
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float e0 = ex2(fmaf(x[2 * c], mul, -mb)), e1 = ex2(fmaf(x[2 * c + 1], mul, -mb));
              ps[c & 3] += e0 + e1;
              pk[c] = pack2<T>(e0, e1);
            }
            tc::tmem_st16(ts + 16 * h, pk);
          }
          tc::tmem_st_wait();
          l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        }
        // O takes a raised maximum once the last tile's P·V has completed
        if (kt > sg.t0 && __any_sync(0xffffffffu, need)) {
          if (!(alive = wait(o_done((it - 1) % kSBufs), (it - 1) / kSBufs))) continue;
          tc::tc_fence_after();
#pragma unroll 1
          for (int cb = 0; cb < 2 * D / 32; ++cb) {
            uint32_t ov[32];
            tc::tmem_ld32(trow + kColO + cb * 32, ov);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * factor);
            tc::tmem_st32(trow + kColO + cb * 32, ov);
          }
          tc::tmem_st_wait();
        }
        if (tail) tc::fence_proxy_async_smem();  // the cleared rows
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(it % kSBufs));
      }
      Segment nx;
      more = sched.next(a, nx);
      if (BITS == 4 && more) fetch_q(nx);
      const int e = it - 1;  // the segment's last tile
      if (alive) alive = wait(s_full(e % kSBufs), e / kSBufs);
      // its S is complete: Q is free, and the next segment's first product can start
      if (more && alive) {
        if (BITS != 4) fetch_q(nx);
        store_q();
      }
      if (alive) alive = wait(o_done(e % kSBufs), e / kSBufs);
      tc::tc_fence_after();
      if (work) {
        float m_ref = -INFINITY;
        if (alive) {  // both groups' sums at the last maximum
          m_ref = *m_row;
          if (m_ref != m_mine) l *= ex2(m_mine - m_ref);
          l_row[grp * kTR] = l;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(l_both(q));
          alive = wait(l_both(q), joined++);
          l = l_row[0] + l_row[kTR];
        }
        const float inv = !alive ? NAN : l == 0.f ? 0.f : 1.f / l;
        const int64_t row = ((int64_t)sg.b * a.HKV + sg.g) * a.R + pr;
        const Cleared* bad = bad_all + (seg & 1) * 8;
        bool any_bad = false;
#pragma unroll
        for (int w = 0; w < 8; ++w) any_bad |= bad[w].seg == seg;
        if (a.cluster && grp == 0) join_ml[r] = make_float2(m_ref, alive ? l : NAN);
        else if (sg.slot >= 0 && live && grp == 0)
          *reinterpret_cast<float2*>(a.part_ml + ((int64_t)sg.slot * a.slot_rows + r) * 2) = make_float2(m_ref, alive ? l : NAN);
        // a thread writes whole 32-byte sectors of its row
#pragma unroll 1
        for (int cb = grp * (D / 32); cb < (grp + 1) * (D / 32); ++cb) {
          uint32_t ov[32];
          tc::tmem_ld32(trow + kColO + cb * 32, ov);
          tc::tmem_ld_wait();
          if (!live) continue;
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[(i & ~7) + chunk_channel<BITS>(i & 7)] = alive ? __uint_as_float(ov[i]) : NAN;
          if (sg.slot < 0) {
            T* dst = static_cast<T*>(a.y) + row * 2 * D + cb * 32;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              *reinterpret_cast<uint4*>(dst + 8 * c) =
                  make_uint4(pack2<T>(o[8 * c] * inv, o[8 * c + 1] * inv), pack2<T>(o[8 * c + 2] * inv, o[8 * c + 3] * inv),
                             pack2<T>(o[8 * c + 4] * inv, o[8 * c + 5] * inv), pack2<T>(o[8 * c + 6] * inv, o[8 * c + 7] * inv));
          } else if (a.cluster) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<float4*>(smem + Map::kK + join_at<D>(r, cb * 8 + c)) =
                  make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          } else {
            float* dst = a.part_o + part_at<D>(a, sg.slot, cb * 4, r);
#pragma unroll
            for (int c = 0; c < 4; ++c) store_sector(dst + (int64_t)c * a.slot_rows * 8, o + 8 * c);
          }
        }
        if (any_bad && alive && live)
          add_cleared<T, D, BITS>(a, sg.b, sg.g, bad, seg, pr, t, ctx, m_ref, inv, grp,
                                  sg.slot < 0 ? static_cast<T*>(a.y) + row * 2 * D : nullptr, sg.slot, r, smem + Map::kK);
      }
      // This warp's last read of the segment's O (and of l_row: the next sums are written after the next segment's
      // P·V) is over. Every softmax warp arrives, with a row or without.
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(o_read);
      if (!alive) *abort_flag = 1;
      sg = nx;
      ++seg;
    }
  } else if constexpr (BITS != 16) {  // ---- operand tiles from packed rows ----
    const int tid = threadIdx.x - 320;
    constexpr int kUnits = kTK * D / 32;  // 32 channels of one row
    constexpr int kFillThreads = Cfg::kThreads - 320, kPer = 3 * kUnits / kFillThreads;
    static_assert(kPer * kFillThreads == 3 * kUnits, "whole units per thread");
    const int gs_log = 31 - __clz(a.gs);  // the group size divides 64 or 128
    // A thread's units lie in one 32-channel column, in rows that are equal mod 8: its four chunks' places in a row
    // are fixed. Their order differs between a row's halves so that eight lanes write to eight bank groups.
    static_assert(kFillThreads % (8 * (D / 32)) == 0 && kUnits % (8 * (D / 32)) == 0, "one column, one swizzle a thread");
    const int c32 = tid % (D / 32), flip = D == 128 ? (c32 >> 1) << 1 : 0, bias_at = kTK * (D >> gs_log);
    const int g_off = (c32 * 32 >> gs_log) * (int)sizeof(T);
    int off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c8 = c32 * 4 + (k ^ flip);
      off[k] = (c8 >> 3) * kTK * 128 + (((c8 & 7) ^ (tid / (D / 32) & 7)) << 4);
    }
    int it = 0;
    bool alive = true;
    for (; alive && more; more = sched.next(a, sg)) {
      for (int kt = sg.t0; kt < sg.t1; ++kt, ++it) {
        const int rs = it % ta.raw_stages, s = it % NS;
        const uint32_t par = (it / NS - 1) & 1;
        const bool ok = bar_wait(raw_full(rs), (it / ta.raw_stages) & 1) &&
                        (it < NS || (bar_wait(k_empty(s), par) && bar_wait(v_empty(s), par)));  // NV is NS here
        if (__any_sync(0xffffffffu, !ok || *abort_flag)) { alive = false; break; }
        const uint8_t* raw = smem + Map::kRaw + rs * (3 * kTK * ta.code_bytes + 6 * kTK * ta.group_bytes);
        uint8_t* kt_ = smem + Map::kK + s * Map::kKBytes;
        uint8_t* vt_ = smem + Map::kV + s * Map::kVBytes - Map::kKBytes;  // slot 1 and 2: V1, V2
        const uint8_t* groups = raw + 3 * kTK * ta.code_bytes + g_off;
        // one short loop: several roles' code shares the instruction caches
#pragma unroll 1
        for (int x = 0; x < kPer; ++x) {
          const int u = tid + x * kFillThreads, slot = u / kUnits, row = u % kUnits / (D / 32);
          uint32_t w[BITS];
#pragma unroll
          for (int i = 0; i < BITS / 4; ++i) *reinterpret_cast<uint4*>(w + 4 * i) = reinterpret_cast<const uint4*>(raw)[u * (BITS / 4) + i];
          const T* sc = reinterpret_cast<const T*>(groups + (slot * 2 * kTK + row) * ta.group_bytes);
          uint8_t* tile = (slot == 0 ? kt_ : vt_ + slot * Map::kKBytes) + row * 128;
          T s8 = sc[0], b8 = sc[bias_at];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w0, w1 = 0;
            if constexpr (BITS == 4) {
              w0 = flip ? w[k ^ 2] : w[k];
            } else {
              w0 = flip ? w[2 * (k ^ 2)] : w[2 * k];
              w1 = flip ? w[2 * (k ^ 2) + 1] : w[2 * k + 1];
            }
            if (gs_log < 5) s8 = sc[((k ^ flip) * 8) >> gs_log], b8 = sc[(((k ^ flip) * 8) >> gs_log) + bias_at];  // groups inside the unit
            *reinterpret_cast<uint4*>(tile + off[k]) = dequant8<T, BITS>(w0, w1, s8, b8);
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(k_full(s));
          tc::mbar_arrive(v_full(s));
          tc::mbar_arrive(raw_empty(rs));
        }
      }
    }
    if (!alive) *abort_flag = 1;
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kCols);
  }
  if (a.cluster) join_cluster<T, D>(a, smem + Map::kK, join_ml, reinterpret_cast<float*>(join_ml + kTR));
  if (threadIdx.x == 0 && *abort_flag && a.err) *reinterpret_cast<volatile int*>(a.err) = 1;  // may be host memory
}

// ---- join of the cut units' partials -----------------------------------------------------------------
// O = Σ w·O_s / Σ w·l_s, w = 2^(m_s − max m), over the parts of the row's unit in their order. Four warps
// take every fourth part of one output row and add up through shared memory; a lane holds eight channels
// (one sector of a part; D 64: two parts at a time).
constexpr int kMergeWarps = 4, kMergeRows = 2;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kMergeWarps * kMergeRows) tree_merge_kernel(const __grid_constant__ TreeArgs a, int grid) {
  constexpr int kChunks = 2 * D / 8;         // lanes of one part
  constexpr int kSub = 32 / kChunks;         // parts of one warp step
  constexpr int kStep = kMergeWarps * kSub;  // parts of one step of the row's warps
  __shared__ __align__(16) float so[kMergeRows][kStep][2 * D];
  __shared__ float2 sml[kMergeRows][kStep];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slot_row = warp / kMergeWarps, w = warp % kMergeWarps;
  const int64_t row = (int64_t)blockIdx.x * kMergeRows + slot_row;
  const int rows_b = a.HKV * a.R;
  const bool valid = row < (int64_t)a.B * rows_b;
  const int b = valid ? (int)(row / rows_b) : 0, in_b = valid ? (int)(row - (int64_t)b * rows_b) : 0;
  const int g = in_b / a.R, pr = in_b - g * a.R;
  const int rt = pr / a.tile_rows, r = pr - rt * a.tile_rows;
  const int per_b = a.HKV * a.row_tiles, u = g * a.row_tiles + rt;
  // parts first .. first + parts − 1 of the unit; part k's place, -1 for an empty one
  int parts, first = 0, at = 0;
  Line line;
  const int nt = key_tiles(a, live_rows(a, b));
  if (a.cuts) {
    parts = nt > 1 ? a.cuts : 1;
    first = (b * per_b + u) * a.cuts;
  } else {
    int tiles = 0, before = 0;
    for (int i = lane; i < a.B; i += 32) {
      const int x = key_tiles(a, live_rows(a, i));
      tiles += x;
      before += i < b ? x : 0;
    }
    tiles = (int)__reduce_add_sync(0xffffffffu, (unsigned)tiles) * per_b;
    before = (int)__reduce_add_sync(0xffffffffu, (unsigned)before) * per_b;
    line.init(tiles, a.B * per_b, grid);
    at = before + b * per_b * line.lead + u * (nt + line.lead) + line.lead;  // the unit's first key tile
    first = line.owner(at);
    parts = line.owner(at + nt - 1) - first + 1;
  }
  auto place = [&](int k) -> int {
    if (a.cuts) return cut_at(k, nt, a.cuts) < cut_at(k + 1, nt, a.cuts) ? first + k : -1;
    const int from = line.lo(first + k);
    return from >= line.lo(first + k + 1) ? -1 : 2 * (first + k) + (from > at ? 0 : 1);
  };
  const bool join = valid && parts > 1;  // else written by its CTA
  const int sub = lane / kChunks, chunk = lane % kChunks;
  float M = -INFINITY, L = 0.f, o[8] = {};
  if (join) {
    constexpr int kU = 5;  // parts in flight
    for (int k0 = w * kSub + sub; k0 < parts; k0 += kStep * kU) {
      float m[kU], l[kU];
      float4 f[kU][2];
#pragma unroll
      for (int x = 0; x < kU; ++x) {
        const int k = k0 + x * kStep, at_ = k < parts ? place(k) : -1;
        m[x] = -INFINITY, l[x] = 0.f;
        if (at_ < 0) continue;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + ((int64_t)at_ * a.slot_rows + r) * 2);
        const float4* p = reinterpret_cast<const float4*>(a.part_o + part_at<D>(a, at_, chunk, r));
        m[x] = ml.x, l[x] = ml.y;
        f[x][0] = p[0], f[x][1] = p[1];
      }
      float top = M;
#pragma unroll
      for (int x = 0; x < kU; ++x) top = fmaxf(top, m[x]);
      const float c0 = top == M ? 1.f : exp2f(M - top);
      M = top, L *= c0;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= c0;
#pragma unroll
      for (int x = 0; x < kU; ++x) {
        if (m[x] == -INFINITY) {  // empty, or a part that saw no key of this row: its O is not used
          L += l[x] == l[x] ? 0.f : l[x];
          continue;
        }
        const float c = exp2f(m[x] - M);
        L = fmaf(c, l[x], L);
        o[0] = fmaf(c, f[x][0].x, o[0]), o[1] = fmaf(c, f[x][0].y, o[1]);
        o[2] = fmaf(c, f[x][0].z, o[2]), o[3] = fmaf(c, f[x][0].w, o[3]);
        o[4] = fmaf(c, f[x][1].x, o[4]), o[5] = fmaf(c, f[x][1].y, o[5]);
        o[6] = fmaf(c, f[x][1].z, o[6]), o[7] = fmaf(c, f[x][1].w, o[7]);
      }
    }
    const int ps = w * kSub + sub;
    reinterpret_cast<float4*>(&so[slot_row][ps][chunk * 8])[0] = make_float4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<float4*>(&so[slot_row][ps][chunk * 8])[1] = make_float4(o[4], o[5], o[6], o[7]);
    if (chunk == 0) sml[slot_row][ps] = make_float2(M, L);
  }
  __syncthreads();
  if (!join) return;
  float top = -INFINITY, den = 0.f, c[kStep];
#pragma unroll
  for (int i = 0; i < kStep; ++i) top = fmaxf(top, sml[slot_row][i].x);
#pragma unroll
  for (int i = 0; i < kStep; ++i) {
    const float2 ml = sml[slot_row][i];
    c[i] = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    den += ml.x == -INFINITY ? ml.y : c[i] * ml.y;
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  for (int ch = threadIdx.x % (32 * kMergeWarps); ch < D; ch += 32 * kMergeWarps) {  // two channels a thread
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      if (c[i] == 0.f) continue;
      const float2 p = *reinterpret_cast<const float2*>(&so[slot_row][i][2 * ch]);
      v.x = fmaf(c[i], p.x, v.x), v.y = fmaf(c[i], p.y, v.y);
    }
    T* dst = static_cast<T*>(a.y) + row * 2 * D + 2 * ch;
    dst[0] = from_f<T>(v.x * inv), dst[1] = from_f<T>(v.y * inv);
  }
}

int sm_count() {  // of the first device asked for: a machine's GPUs are alike
  static std::atomic<int> known{0};
  int n = known;
  if (n > 0) return n;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      n < 1) {
    (void)cudaGetLastError();
    return 148;
  }
  known = n;
  return n;
}

constexpr int64_t kMaxTreeRows = 256, kMaxCap = 1 << 30, kMaxBatch = 1 << 20, kMaxHeads = 1 << 16;

// Shared memory of the K and V tiles, which a cluster's join takes over.
int join_room(int bits, int64_t D) {
  const int k = bits == 16 ? TcMap<128, 16>::kBar - TcMap<128, 16>::kK
                : bits == 4 ? TcMap<128, 4>::kBar - TcMap<128, 4>::kK
                            : TcMap<128, 8>::kBar - TcMap<128, 8>::kK;
  return D == 128 ? k : k / 2;
}

// Which kernel serves a call, and its launch shape.
struct Plan {
  bool tc;
  int tile_rows, tile_keys, row_tiles, slot_rows;
  int cuts;       // parts of every unit, or 0: the line
  bool cluster;   // joined by the cluster of a unit's CTAs, without a second launch
  int64_t tiles;  // key tiles of all units at the longest lengths
  int64_t line;   // length of the line at most
  int64_t grid;   // CTAs: at most as many as run at once
  size_t ml_offset, bytes;
};

// The tensor-core form takes 16-bit types; packed rows need tiles that start on 16-byte boundaries in the
// scales too (any capacity that is a multiple of 8 does). The rest runs on the CUDA cores.
// Units of one length are cut evenly unless that would leave more than an eighth of the CTAs idle.
Plan make_plan(int dtype, int bits, int gs, int64_t B, int64_t HKV, int64_t R, int64_t D, int64_t cap, int64_t len_bound,
               bool one_length) {
  Plan p{};
  p.tc = dtype != MOTIF_F32 && (bits == 16 || (cap * (D / gs)) % 8 == 0);
  p.tile_rows = p.tc ? kTR : kSR;
  p.tile_keys = p.tc ? kTK : kSK;
  p.row_tiles = (int)ceil_div(R, p.tile_rows);
  p.slot_rows = (int)(R < p.tile_rows ? R : p.tile_rows);
  const int64_t ctas = (p.tc ? 1 : 2) * (int64_t)sm_count();
  const int64_t nt = ceil_div(len_bound < 1 ? 1 : len_bound, p.tile_keys), units = B * HKV * p.row_tiles;
  p.tiles = nt * units;
  p.line = p.tiles + kLead * units;
  p.grid = p.tiles < ctas ? p.tiles : ctas;
  int64_t parts = 2 * p.grid;
  if ((one_length || B == 1) && units <= ctas && B < 65536 && HKV * p.row_tiles < 65536) {
    // Parts of a unit, in us: a tile of a part about 0.9; a join in the cluster 3.5; one by a second launch 5 (with
    // the host's share) and 0.1 a part. With one CTA an SM only some 64 CTAs run at once as clusters of eight
    // (16 units of 8 parts took two rounds, 24 us against 14 with a second launch).
    const int64_t most = ctas / units < nt ? ctas / units : nt;
    const bool room = p.tc && p.slot_rows * 2 * D * 4 <= join_room(bits, D);
    int64_t c = 1;
    double best = 0.9 * nt;
    for (int64_t k = 2; k <= most; ++k) {
      const double t = 0.9 * ceil_div(nt, k) + 5.0 + 0.1 * k;
      if (t < best) best = t, c = k;
    }
    if (room)
      for (int64_t k = 2; k <= kMaxCluster && k <= nt && k * units <= 64; ++k) {
        const double t = 0.9 * ceil_div(nt, k) + 3.5;
        if (t < best) best = t, c = k, p.cluster = true;
      }
    // cut_at multiplies in 32 bits: a longer cache is a line
    if (c * nt < (1ll << 32) && (p.cluster || c < most || most == nt || 8 * c * units >= 7 * ctas)) {
      p.cuts = (int)c;
      parts = p.cluster || c == 1 ? 0 : c * units;
    }
  }
  p.ml_offset = sizeof(float) * (size_t)parts * p.slot_rows * 2 * (size_t)D;
  p.bytes = p.ml_offset + sizeof(float) * (size_t)parts * p.slot_rows * 2;
  return p;
}

dim3 grid_of(const TreeArgs& a, const Plan& p) {
  return a.cuts ? dim3((unsigned)a.cuts, (unsigned)(a.HKV * a.row_tiles), (unsigned)a.B) : dim3((unsigned)p.grid);
}

// A plain launch: started early (programmatic dependent launch), the join's waiting CTAs cost the attention kernel
// more than the launch saves (41 against 37 us for a tree of 42 over 16064 rows).
template <typename T, int D>
int launch_merge(const TreeArgs& a, const Plan& p, cudaStream_t st) {
  if (a.cuts == 1 || a.cluster) return MOTIF_OK;  // every unit in one part, or joined already
  const int64_t rows = (int64_t)a.B * a.HKV * a.R;
  tree_merge_kernel<T, D><<<(unsigned)ceil_div(rows, kMergeRows), 32 * kMergeWarps * kMergeRows, 0, st>>>(a, (int)p.grid);
  return check_launch("sdpa_dual_v_tree join");
}

template <typename T, int D, int BITS>
int launch_simt(const TreeArgs& a, const Plan& p, cudaStream_t st) {
  auto kern = tree_simt_kernel<T, D, BITS>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = once_per_device(
      done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, simt_smem<D>()); });
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: smem attribute: %s", cudaGetErrorString(e));
  kern<<<grid_of(a, p), kSThreads, simt_smem<D>(), st>>>(a);
  const int rc = check_launch("sdpa_dual_v_tree");
  return rc ? rc : launch_merge<T, D>(a, p, st);
}

template <typename T, int D, int BITS>
int launch_tc(const TreeArgs& a, const Plan& p, cudaStream_t st) {
  using Map = TcMap<D, BITS>;
  TcArgs ta{};
  ta.t = a;
  int smem = 1024 + Map::kRaw;
  if constexpr (BITS == 16) {
    const uint64_t dims[3] = {(uint64_t)a.cap, (uint64_t)a.HKV, (uint64_t)a.B};
    const uint64_t strides[3] = {(uint64_t)a.sr * 2, (uint64_t)a.sh * 2, (uint64_t)a.sb * 2};
    for (int i = 0; i < 3; ++i)
      if (!encode_tma_heads(&ta.tm[i], a.kv[i], D * 2, dims, strides, 128, kTK))
        return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: tensor map encoding failed");
  } else {
    ta.code_bytes = D * BITS / 8;
    ta.group_bytes = D / a.gs * 2;
    const int raw = 3 * kTK * ta.code_bytes + 6 * kTK * ta.group_bytes;
    const int room = 227 * 1024 - smem;
    ta.raw_stages = room / raw < kRawMax ? room / raw : kRawMax;
    if (ta.raw_stages < 1) return fail(MOTIF_ERR_BAD_CONTRACT, "sdpa_dual_v_tree: group_size %d too small", a.gs);
    smem += ta.raw_stages * raw;
  }
  auto kern = tree_tc_kernel<T, D, BITS>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = once_per_device(done, [&] {  // the most that any group size takes
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  });
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: attribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid_of(a, p);
  cfg.blockDim = dim3(TcCfg<BITS>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)a.cuts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = a.cluster ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kern, ta);
  if (e != cudaSuccess) return fail(MOTIF_ERR_CUDA, "sdpa_dual_v_tree: %s", cudaGetErrorString(e));
  const int rc = check_launch("sdpa_dual_v_tree");
  return rc ? rc : launch_merge<T, D>(a, p, st);
}

template <typename T, int D, int BITS>
int launch(const TreeArgs& a, const Plan& p, cudaStream_t st) {
  if constexpr (!std::is_same<T, float>::value)
    if (p.tc) return launch_tc<T, D, BITS>(a, p, st);
  return launch_simt<T, D, BITS>(a, p, st);
}

}  // namespace
}  // namespace motif

using namespace motif;

extern "C" {

size_t motif_sdpa_dual_v_tree_workspace_bytes(int dtype, int bits, int group_size, int64_t batch, int64_t h_q,
                                              int64_t h_kv, int64_t tree_rows, int64_t kv_cap, int64_t head_dim,
                                              int64_t kv_len_bound, int one_length) {
  // a call of other sizes is refused
  if (batch < 1 || batch >= kMaxBatch || h_q < 1 || h_q >= kMaxHeads || h_kv < 1 || h_q % h_kv != 0 || tree_rows < 1 ||
      tree_rows > kMaxTreeRows || kv_cap < 1 || kv_cap >= kMaxCap || head_dim < 1 || head_dim > 128 || group_size < 1 ||
      head_dim < group_size)
    return 0;
  return make_plan(dtype, bits, group_size, batch, h_kv, h_q / h_kv * tree_rows, head_dim, kv_cap,
                   kv_len_bound < kv_cap ? kv_len_bound : kv_cap, one_length != 0).bytes;
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
  MOTIF_REQUIRE(batch > 0 && h_q > 0 && h_kv > 0 && kv_cap > 0 && kv_cap < kMaxCap && batch < kMaxBatch &&
                    h_q < kMaxHeads,
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
      al |= reinterpret_cast<uintptr_t>(kv->scales[i]) | reinterpret_cast<uintptr_t>(kv->biases[i]);
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
  const Plan p = make_plan(dtype, bits, bits == 16 ? 64 : group_size, batch, h_kv, a.R, head_dim, kv_cap,
                           kv_len_dev ? kv_cap : kv_len, !kv_len_dev || kv_len_stride == 0);
  a.tile_rows = p.tile_rows;
  a.tile_keys = p.tile_keys;
  a.row_tiles = p.row_tiles;
  a.slot_rows = p.slot_rows;
  a.cuts = p.cuts;
  a.cluster = p.cluster;
  MOTIF_REQUIRE(p.tiles < (1ll << 28) && p.line < (1ll << 31), MOTIF_ERR_BAD_SHAPE,
                "sdpa_dual_v_tree: %lld key tiles in one call", (long long)p.tiles);
  MOTIF_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes), MOTIF_ERR_WORKSPACE,
                "sdpa_dual_v_tree: workspace of %zu bytes, needs %zu", workspace_bytes, p.bytes);
  MOTIF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MOTIF_ERR_BAD_CONTRACT,
                "sdpa_dual_v_tree: workspace must be 16-byte aligned");
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.ml_offset);
  cudaStream_t st = as_stream(stream);
  MOTIF_DISPATCH_FLOAT(dtype, T, {
    if (head_dim == 64) {
      if (bits == 16) return launch<T, 64, 16>(a, p, st);
      if (bits == 4) return launch<T, 64, 4>(a, p, st);
      return launch<T, 64, 8>(a, p, st);
    }
    if (bits == 16) return launch<T, 128, 16>(a, p, st);
    if (bits == 4) return launch<T, 128, 4>(a, p, st);
    return launch<T, 128, 8>(a, p, st);
  });
  return MOTIF_OK;
}

}  // extern "C"
