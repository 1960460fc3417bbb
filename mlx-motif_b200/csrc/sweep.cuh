// exp((l − m)/τ) in 64 bits for the verification's sweeps over a row. Plain C++ too, so that it can be compared with
// exp on the host.
#pragma once

#include <cmath>
#include <cstdint>
#include <cstring>

#ifdef __CUDACC__
#define MOTIF_HD __host__ __device__ __forceinline__
#else
#define MOTIF_HD inline
#endif

namespace motif {

constexpr int kSweepTable = 256;

// A table of 2^(j/256) (Tang, "Table-driven implementation of the exponential function in IEEE floating-point
// arithmetic", ACM TOMS 15, 1989): y = (l − m)·k = n/256 + f, |f| ≤ 2^-9, and 2^f by its series to f⁴ (the next term is
// 4·10^-17); k = log2 e / τ. The difference is taken first, so that y ≤ 0 for l ≤ m and 0 at l = m whatever their size
// (m finite). Nine 64-bit operations. Roundings: of l − m (none for logits of one magnitude), of k (1/τ, log2 e and their
// product), each by 2^-53 of y; of 2^f, its table entry and their product, three of 2^-53 at most: within
// (2.8·|y| + 3)·2^-53 of exp((l − m)/τ), 2^-45 at |y| = 60. Below 2^-1022: 0.
MOTIF_HD double sweep_weight(float l, double m, double k, const double* table) {
  constexpr double kMagic = 6755399441055744.0 / kSweepTable;  // 1.5·2^52 / 256: a sum with it is rounded to 1/256
  const double d = (double)l - m;
  const double t = fma(d, k, kMagic), r = t - kMagic;
  const double f = fma(d, k, -r);
  int64_t bits;
  memcpy(&bits, &t, 8);
  const int n = (int)(uint32_t)bits;
  double q = fma(f, 0.0096181291076284772, 0.055504108664821580);  // (ln 2)^i / i!
  q = fma(f, q, 0.24022650695910071);
  q = fma(f, q, 0.69314718055994531);
  const double s = table[n & (kSweepTable - 1)];
  const double e = fma(s * f, q, s);
  memcpy(&bits, &e, 8);
  bits += (int64_t)(((uint64_t)(uint32_t)(n >> 8)) << 52);  // the exponent: the upper word alone changes
  double w;
  memcpy(&w, &bits, 8);
  return r > -1022.0 ? w : 0.0;
}

}  // namespace motif
