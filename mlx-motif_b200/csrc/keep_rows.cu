// The accepted path's rows of a verified tree become the cache's next rows.
//
// After a tree of T rows was appended at cache rows [base, base + T), row base + path[j] moves to row
// base + j for j = 1 .. accepted, in all four slots of every layer. path ascends from path[0] = 0, so
// path[j] ≥ j and the moves run in ascending j without a buffer: rows are taken in groups, each group
// read before it is written, and a later group reads rows ≥ its own j, which no earlier one has written.
//
// One launch serves up to kLayers caches: their pointers travel in the kernel's parameters.
// Bound by the launch: 3 rows of 48 fp16 layers (8 heads, D 128; 2.4 MB read and written) take 3.2 us, 8 rows of 48 q4
// layers 4.9 us; the bytes alone would be 0.4. A CTA moves one buffer of a slot's head (codes, scales and biases one
// after the other: 1.1 us more); packed rows are short, and CTAs of 64 threads all run at once there (of 128: 1.0 us more).
#include "common.cuh"

namespace motif {
namespace {

constexpr int kLayers = 64;
constexpr int kKeepThreads = 128;

struct KeepArgs {
  void* ptr[kLayers][4][3];  // codes or rows, scales, biases
  int32_t row_bytes[3];      // bytes of one row of each (0: absent)
  int32_t unit[3];           // bytes of one access
  int32_t parts;
  int64_t heads;             // batch * heads rows of `cap` rows each
  int64_t cap;
  int64_t limit;             // rows at or beyond it are not touched
  int32_t heads_per_b;
  const int32_t* path;
  int64_t path_b;
  const int32_t* accepted;
  const int32_t* base_dev;
  int32_t base_step;
  int64_t base;
  int32_t T;
};

template <typename U>
__device__ __forceinline__ void move_rows(U* rows, int per_row, const int32_t* path, int n, int64_t cap_left, int T) {
  const int tid = threadIdx.x;
  // units of rows 1..n in order, one per thread and group
  for (int i0 = 0; i0 < n * per_row; i0 += blockDim.x) {
    const int i = i0 + tid;
    const int j = 1 + i / per_row, c = i % per_row;
    U v{};
    bool go = i < n * per_row;
    if (go) {
      const int from = path[j];
      go = from > j && from < T && from < cap_left;  // from == j stays; anything else outside the tree is left alone
      if (go) v = rows[(int64_t)from * per_row + c];
    }
    __syncthreads();
    if (go) rows[(int64_t)j * per_row + c] = v;
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kKeepThreads) keep_rows_kernel(const __grid_constant__ KeepArgs a) {
  const int layer = blockIdx.x >> 2, slot = blockIdx.x & 3;
  const int head = blockIdx.y, b = head / a.heads_per_b;
  const int n = min(a.accepted[b], a.T - 1);
  const int64_t base = a.base_dev ? a.base_dev[(int64_t)b * a.base_step] : a.base;
  if (n <= 0 || base < 0 || base >= a.limit) return;
  const int64_t left = a.limit - base;  // rows of the tree that the cache holds
  const int32_t* path = a.path + b * a.path_b;
  const int k = blockIdx.z;
  char* p = static_cast<char*>(a.ptr[layer][slot][k]) + ((int64_t)head * a.cap + base) * a.row_bytes[k];
  const int per = a.row_bytes[k] / a.unit[k];
  const int m = (int)min((int64_t)n, left - 1);
  switch (a.unit[k]) {
    case 16: move_rows(reinterpret_cast<uint4*>(p), per, path, m, left, a.T); break;
    case 8: move_rows(reinterpret_cast<uint2*>(p), per, path, m, left, a.T); break;
    case 4: move_rows(reinterpret_cast<uint32_t*>(p), per, path, m, left, a.T); break;
    default: move_rows(reinterpret_cast<uint16_t*>(p), per, path, m, left, a.T); break;
  }
}

}  // namespace
}  // namespace motif

using namespace motif;

extern "C" {

int motif_kv4_keep_rows(int dtype, const motif_kv4_slots* caches, int64_t n_caches, const int32_t* path,
                        int64_t path_batch_stride, const int32_t* accepted, int64_t tree_rows, int64_t base,
                        const int32_t* base_dev, int64_t base_stride, int64_t row_limit, void* stream) {
  MOTIF_REQUIRE(caches && path && accepted, MOTIF_ERR_NULL, "keep_rows: null pointer");
  MOTIF_REQUIRE(n_caches >= 1, MOTIF_ERR_BAD_SHAPE, "keep_rows: %lld caches", (long long)n_caches);
  MOTIF_REQUIRE(dtype == MOTIF_F16 || dtype == MOTIF_BF16 || dtype == MOTIF_F32, MOTIF_ERR_DTYPE,
                "keep_rows: unsupported dtype code %d", dtype);
  const motif_kv4_slots& c0 = caches[0];
  MOTIF_REQUIRE(c0.bits == 16 || c0.bits == 4 || c0.bits == 8, MOTIF_ERR_DTYPE, "keep_rows: bits %d", c0.bits);
  MOTIF_REQUIRE(c0.batch >= 1 && c0.batch < 65536 && c0.heads >= 1 && c0.heads < 65536 && c0.capacity >= 1 &&
                    c0.head_dim >= 1 && c0.head_dim <= 65536 && c0.batch * c0.heads < 65536,
                MOTIF_ERR_BAD_SHAPE, "keep_rows: batch=%lld heads=%lld capacity=%lld head_dim=%lld", (long long)c0.batch,
                (long long)c0.heads, (long long)c0.capacity, (long long)c0.head_dim);
  MOTIF_REQUIRE(row_limit >= 1 && row_limit <= c0.capacity, MOTIF_ERR_BAD_SHAPE,
                "keep_rows: row limit %lld outside capacity %lld", (long long)row_limit, (long long)c0.capacity);
  MOTIF_REQUIRE(tree_rows >= 1 && tree_rows <= (1 << 20) && (base_dev || (base >= 0 && base + tree_rows <= row_limit)),
                MOTIF_ERR_BAD_SHAPE, "keep_rows: rows [%lld, %lld) outside capacity %lld", (long long)base,
                (long long)(base + tree_rows), (long long)row_limit);
  MOTIF_REQUIRE(path_batch_stride == tree_rows || (path_batch_stride == 0 && c0.batch == 1), MOTIF_ERR_BAD_SHAPE,
                "keep_rows: path batch stride %lld", (long long)path_batch_stride);
  MOTIF_REQUIRE(!base_dev || base_stride == 0 || base_stride == 1, MOTIF_ERR_BAD_SHAPE, "keep_rows: base stride %lld (0 or 1)",
                (long long)base_stride);
  const int64_t esz = dtype == MOTIF_F32 ? 4 : 2;
  MOTIF_REQUIRE(tree_rows * c0.head_dim * esz < (1ll << 31), MOTIF_ERR_BAD_SHAPE,  // units of the rows, in 32 bits
                "keep_rows: %lld rows of %lld channels", (long long)tree_rows, (long long)c0.head_dim);
  KeepArgs a{};
  a.parts = c0.bits == 16 ? 1 : 3;
  if (c0.bits == 16) {
    a.row_bytes[0] = (int32_t)(c0.head_dim * esz);
  } else {
    MOTIF_REQUIRE(c0.group_size >= 1 && c0.head_dim % c0.group_size == 0 && c0.head_dim * c0.bits % 32 == 0,
                  MOTIF_ERR_BAD_CONTRACT, "keep_rows: head_dim %lld, group_size %d", (long long)c0.head_dim, c0.group_size);
    a.row_bytes[0] = (int32_t)(c0.head_dim * c0.bits / 8);
    a.row_bytes[1] = a.row_bytes[2] = (int32_t)(c0.head_dim / c0.group_size * esz);
  }
  a.heads = c0.batch * c0.heads;
  a.heads_per_b = (int32_t)c0.heads;
  a.cap = c0.capacity;
  a.limit = row_limit;
  a.path = path;
  a.path_b = path_batch_stride;
  a.accepted = accepted;
  a.base_dev = base_dev;
  a.base_step = (int32_t)base_stride;
  a.base = base;
  a.T = (int32_t)tree_rows;
  uintptr_t al[3] = {0, 0, 0};
  for (int64_t l = 0; l < n_caches; ++l) {  // all of them before the first launch: a refused call moves nothing
    const motif_kv4_slots& c = caches[l];
    MOTIF_REQUIRE(c.bits == c0.bits && c.group_size == c0.group_size && c.batch == c0.batch && c.heads == c0.heads &&
                      c.capacity == c0.capacity && c.head_dim == c0.head_dim,
                  MOTIF_ERR_BAD_SHAPE, "keep_rows: cache %lld differs from the first", (long long)l);
    for (int s = 0; s < 4; ++s) {
      const void* p[3] = {c.data[s], c.scales[s], c.biases[s]};
      for (int k = 0; k < a.parts; ++k) {
        MOTIF_REQUIRE(p[k], MOTIF_ERR_NULL, "keep_rows: cache %lld slot %d null", (long long)l, s);
        al[k] |= reinterpret_cast<uintptr_t>(p[k]);
      }
    }
  }
  for (int k = 0; k < a.parts; ++k) {
    const uintptr_t bits = al[k] | (uintptr_t)a.row_bytes[k];
    a.unit[k] = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
    MOTIF_REQUIRE(bits % 2 == 0, MOTIF_ERR_BAD_CONTRACT, "keep_rows: misaligned cache");
  }
  for (int64_t l0 = 0; l0 < n_caches; l0 += kLayers) {
    const int n = (int)(n_caches - l0 < kLayers ? n_caches - l0 : kLayers);
    for (int l = 0; l < n; ++l) {
      const motif_kv4_slots& c = caches[l0 + l];
      for (int s = 0; s < 4; ++s) {
        void* p[3] = {c.data[s], c.scales[s], c.biases[s]};
        for (int k = 0; k < a.parts; ++k) a.ptr[l][s][k] = p[k];
      }
    }
    keep_rows_kernel<<<dim3((unsigned)(4 * n), (unsigned)a.heads, (unsigned)a.parts), a.parts == 1 ? kKeepThreads : kKeepThreads / 2, 0, as_stream(stream)>>>(a);
    const int rc = check_launch("keep_rows");
    if (rc) return rc;
  }
  return MOTIF_OK;
}

}  // extern "C"
