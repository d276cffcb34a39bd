// Shared parts of the linear cross entropy's kernels for many rows: operands as panels of fp16 pairs and their products.
//
// A panel holds 256 rows of an operand [rows, k], k cut into blocks of 32: per block 256 lines of 128 bytes (32 hi, 32 lo of one
// row; the eight 16-byte pieces swizzled by the row), so that one block of one panel is 32 KiB of consecutive memory and the LDS
// image that the product kernel reads. k is padded with zeros to a whole block.
#pragma once
#include "common.h"
#include "fp16_pairs.h"

namespace lce {

constexpr int kPanel = 256, kBlock = 32;
constexpr int64_t kBlockBytes = kPanel * 128;

inline int64_t panel_bytes(int64_t rows, int64_t k) { return ceil_div64(rows, kPanel) * ceil_div64(k, kBlock) * kBlockBytes; }

__device__ __forceinline__ char* line_at(char* panels, int64_t row, int64_t kb, int64_t kblocks) {
  return panels + ((row / kPanel) * kblocks + kb) * kBlockBytes + (row % kPanel) * 128;
}

// g / count = m 2^e (0 without a row that counts). A result is put together as ldexp(sum * m, e - shifts): the powers of two that
// scales take off, and a small cotangent, would leave fp32's range as a factor of their own though the result does not.
struct Mean {
  float m;
  int e;
};
__device__ __forceinline__ Mean mean_of(const float* g, const float* count) {
  const float c = g[0], n = count[0];
  if (!(n > 0.f)) return {0.f, 0};
  return {__builtin_amdgcn_frexp_mantf(c) / n, __builtin_amdgcn_frexp_expf(c)};  // (infinities and NaN: themselves, 0)
}

// Source of an operand [rows, k]: element (r, k) at x[r * ld + k], or transposed at x[k * ld + r]. `left_out` (null or one target
// per index along x's first axis): indices with a negative target are zeros. amax: per row the largest finite magnitude.
int32_t pack(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, char* panels, float* amax,
             bool known, hipStream_t s);  // known: amax is there already

// z = W x^T piece: A = W rows (classes v0 .. v0 + cols), B = x rows. stats: per 256 classes and row the maximum and the sum of
// exp(z - maximum); zt: the target's logit, where it lies in the piece.
struct Logits {
  const char *w, *x;
  const float *w_amax, *x_amax, *target;
  int64_t N, cols, v0, D;
  float* stats;  // forward: [tiles of classes][N][2]
  float* zt;
  const float* lse;    // backward
  char *p, *pt;        // dz as panels [rows, classes] and [classes, rows]; either may be null
  int *p_shift, *pt_shift;  // [tiles of classes][N padded], [tiles of rows][cols padded]
};
int32_t logits_stats(const Logits& a, hipStream_t s);
int32_t logits_dz(const Logits& a, hipStream_t s);

// out (+)= c * B A^T: A [rows_a, k] with one scale per row, B [rows_b, k] with one shift per row and 256 of k.
// element (b, a) at out[b * ld + a], or with by_a at out[a * ld + b]. parts: the walk along k cut into that many; part s goes to
// out + s * part_stride. c: the Mean of g and count.
struct Gradient {
  const char *a, *b;
  const float* a_amax;
  const int* b_shift;
  int64_t b_shift_ld;  // rows of b, padded
  int64_t rows_a, rows_b, k;
  float* out;
  int64_t ld;
  int by_a, accumulate, parts, vec;  // (vec: set by gradient())
  int64_t part_stride;
  const float *g, *count;
  const float* left_out;  // null, or per row of b a target: where it is negative the result is 0, whatever a holds
};
int32_t gradient(const Gradient& a, hipStream_t s);
int product_tile(int64_t a, int64_t b);  // edge of the tiles that a product of a x b rows is cut into: 256 or 128

// The largest finite magnitude of every row of an operand (as pack takes it).
int32_t row_amax(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, float* amax, hipStream_t s);

// ---- few rows (lce_direct.hip): the streamed operand [rows, k] in fp32 against N columns held as planes
// Up to here operands are bf16 triples, beyond them fp16 pairs, which take amax. Measured at 100 rows, 50000 classes x 1024: pairs 421 and
// 479 us a step against 447 and 517 (by class, by width), though the forward pass alone reads the weight once more.
constexpr int64_t kTripleRows = 64;
inline int64_t plane_bytes(int64_t rows, int64_t k) { return ceil_div64(rows, 32) * ceil_div64(k, 16) * (3 * 1024); }
int32_t planes(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, const float* amax, char* to, hipStream_t s);
int64_t direct_rows(int64_t N, int64_t rows);  // rows of the streamed operand that share an entry of the statistics

struct Direct {
  const float* a;
  int64_t lda, rows, k;
  const char* planes;
  int64_t N, v0;
  int parts;  // the walk along k cut into that many (x's gradient)
  const float *target, *lse;
  const float *a_amax, *x_amax;  // pairs: of the streamed operand's rows, of the columns
  float *stats, *zt;   // statistics: per direct_rows(N, rows) classes and row
  float* dz;           // cotangents [N, rows], row stride dz_ld, or null
  int64_t dz_ld;
  char* dz_planes;     // or null
  float* out;          // x's gradient: [parts][N][rows]
  int accumulate;
  const float *g, *count;
};
// kcontig: a lies contiguous along k
int32_t direct_stats(const Direct& p, bool kcontig, hipStream_t s);
int32_t direct_dz(const Direct& p, bool kcontig, hipStream_t s);
int32_t direct_dx(const Direct& p, bool kcontig, hipStream_t s);

// out (by_d: [d * ld + v], else [v * ld + d]) = g / count * sum_n x[n, d] dz[n, v]; planes: x's columns along k = n
struct Outer {
  const char* planes;
  const float* x_amax;  // of x's columns (pairs), or null (triples)
  const float* dz;
  int64_t dz_ld, N, D, cols;
  float* out;
  int64_t ld;
  int groups;  // of 128 (pairs: 256) of x's columns per work-group (set by direct_dw)
  const float *g, *count;
};
int32_t direct_dw(const Outer& p, bool by_d, hipStream_t s);

}  // namespace lce
