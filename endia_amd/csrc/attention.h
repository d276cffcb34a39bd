// Shared parts of the attention kernels: what a launch takes, the position buckets, and the tile images of split operands.
#pragma once
#include "common.h"
#include "fp16_pairs.h"

namespace attention {

constexpr int kMaxSide = 128;  // buckets of one side
constexpr int kTile = 32;      // positions of one tile image
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// bucket of n steps: n itself below `exact`, then the largest i with start[i] <= n; `near`: from here on the last bucket
struct Buckets {
  int side, exact, both, near;
  int start[kMaxSide];
};

__device__ __forceinline__ int bucket_of(const Buckets& t, int rel) {
  int base = 0, n = -rel;
  if (t.both) {
    if (rel > 0) {
      base = t.side;
      n = rel;
    }
  } else if (n < 0) {
    n = 0;
  }
  int i = t.exact;
  for (int j = t.exact + 1; j < t.side; ++j) i += t.start[j] <= n;  // (a uniform index: the starts come through the scalar cache)
  return base + (n < t.exact ? n : i);
}

// Of one tile of 32 positions: its shift, and a bit for each position that holds an infinity or NaN.
struct TileInfo {
  int shift;
  unsigned bad;
};

struct Args {
  int64_t B, Q, K, H, Hk, D, G;
  int64_t qs[3], ks[3], vs[3];
  int64_t off;
  int64_t seen;  // keys that any query sees: K, or with causal those before Q + off. What a cache holds behind them takes no part in
                 // a tile's scale, in a product or in a gradient.
  float scale;
  int causal;
  int vec;  // q, k, v (and o, go, which are contiguous) can be read 16 bytes at a time
  const float *q, *k, *v, *lengths, *table;
  const float *out, *go;  // backward
  float *o, *lse;
  float *dq, *dk, *dv;
  // tile images of split operands (see tiles_kernel) and what is known of their tiles
  char *k_rows, *k_cols, *v_rows, *v_cols, *q_rows, *q_cols, *g_rows, *g_cols;
  TileInfo *k_info, *v_info, *q_info, *g_info;
  float* meta;       // per query tile: 32 x lse (base 2), 32 x delta
  float* part;       // partial results of a split walk
  float* part_ml;    // forward: running maximum (base 2) and sum of each partial result
  float* part_table; // per work-group sums of ds by position difference
  float* part_rows;  // per row and part: sums of ds and of p in the two last buckets, of p and of ds over all (8 floats)
  int splits;
  int stages;  // tiles that dq_kernel's LDS holds
  Buckets bk;
};

__device__ __forceinline__ int key_count(const Args& a, int64_t b) {
  if (!a.lengths) return (int)a.seen;
  const float n = a.lengths[b];
  return n > 0.f ? (n < (float)a.seen ? (int)n : (int)a.seen) : 0;
}

// Work-groups are dealt round-robin to the 8 XCDs, each with an L2 of its own: give every XCD a contiguous range of ids, so
// that the work-groups that walk over the same keys (or queries) share an L2.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t id, uint32_t n) { return n & 7 ? id : (id & 7) * (n >> 3) + (id >> 3); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ float pow2i(int e) { return __builtin_ldexpf(1.f, e); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// Four consecutive elements d .. d + 3 of a row of D, zeros behind its end and, without `in`, everywhere. The row has to be
// readable either way: the loads go out unconditionally (clamped to the row), so that many are in flight together.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int d, int D, bool in) {
  float4 f;
  if (VEC) {
    f = *reinterpret_cast<const float4*>(row + min(d, D - 4));
  } else {
    f.x = row[min(d, D - 1)];
    f.y = row[min(d + 1, D - 1)];
    f.z = row[min(d + 2, D - 1)];
    f.w = row[min(d + 3, D - 1)];
  }
  f.x = in && d < D ? f.x : 0.f;
  f.y = in && d + 1 < D ? f.y : 0.f;
  f.z = in && d + 2 < D ? f.z : 0.f;
  f.w = in && d + 3 < D ? f.w : 0.f;
  return f;
}

template <int DP, bool VEC>
__device__ __forceinline__ void load_row(const float* row, bool in, int D, int h, float (&x)[DP / 16][8]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 f = load4<VEC>(row, 16 * s + 8 * h + 4 * j, D, in);
      x[s][4 * j] = f.x;
      x[s][4 * j + 1] = f.y;
      x[s][4 * j + 2] = f.z;
      x[s][4 * j + 3] = f.w;
    }
}

// A row (without `in`: zeros) as B operands of v_mfma_f32_32x32x16_f16, one per 16 elements: the lane with half h of the wave
// holds elements 16 s + 8 h .. + 7. Returns the shift both halves agree on.
template <int DP>
__device__ __forceinline__ int load_fragments(const float* row, bool in, int D, int vec, int h, pairs::half8 (&hi)[DP / 16],
                                              pairs::half8 (&lo)[DP / 16]) {
  float x[DP / 16][8];
  if (vec) load_row<DP, true>(row, in, D, h, x);
  else load_row<DP, false>(row, in, D, h, x);
  float amax = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, pairs::finite_abs(x[s][i]));
  amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
  const int shift = pairs::shift_of(amax);
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[s][i] = pairs::scaled(x[s][i], shift);
    pairs::split8(x[s], hi[s], lo[s]);
  }
  return shift;
}

// The two 16-byte pieces (hi, lo) of step s in line `line` (128 bytes: 32 hi, 32 lo, pieces swizzled by the line number so
// that eight lanes that read eight lines side by side touch all LDS banks).
__device__ __forceinline__ void read_line(const char* lines, int line, int s, int h, pairs::half8& hi, pairs::half8& lo) {
  const char* at = lines + line * 128;
  hi = *reinterpret_cast<const pairs::half8*>(at + (((2 * s + h) ^ (line & 7)) << 4));
  lo = *reinterpret_cast<const pairs::half8*>(at + (((4 + 2 * s + h) ^ (line & 7)) << 4));
}

// An infinity or NaN in v (or do) has to reach the rows that see it, but in a product with p = 0 it would also reach those of its tile
// that do not. So the column images hold zeros in its place, and where a tile has any, they are put into the results behind the walk:
// what `row` holds of them makes the lane's part of `out` NaN. (k and q need this not: they make ds NaN where they are seen.)
__device__ __forceinline__ void put_bad(const float* row, int D, int half, float* out) {
  for (int d = 4 * half; d < D; d += 8)
    for (int at = d; at < min(d + 4, D); ++at)
      if (!(__builtin_fabsf(row[at]) < INFINITY)) out[at] = NAN;
}

// score bias of one head by position difference, -near .. near, in LDS, base 2
__device__ __forceinline__ void load_bias(const Args& a, int h, float* lds, int tid, int threads) {
  for (int i = tid; i <= 2 * a.bk.near; i += threads) lds[i] = a.table[bucket_of(a.bk, i - a.bk.near) * a.H + h] * kLog2e;
}
__device__ __forceinline__ int near_index(int rel, int near) { return min(max(rel, -near), near) + near; }

// host side
int32_t launch_tiles(const Args& a, int DP, bool backward, hipStream_t s);
int32_t launch_rows(const Args& a, int R, hipStream_t s);
int32_t launch_forward(const Args& a, int DP, hipStream_t s);
int32_t launch_combine(const Args& a, hipStream_t s);
int32_t launch_dq(const Args& a, int DP, hipStream_t s);
int32_t launch_dkv(const Args& a, int DP, hipStream_t s);
int64_t table_groups(const Args& a);
int32_t launch_table_grad(const Args& a, double* diff, float* dtable, hipStream_t s);

}  // namespace attention
