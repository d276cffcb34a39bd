// The linear cross entropy for few rows (up to a few hundred): the weight is what there is to read, so it is read as it lies, in
// fp32 and in either storage order, straight into matrix operands; no copy of it in another form is made.
//
// Up to 64 rows an fp32 number is held as three bf16 (hi, mid, lo: 8 + 8 + 8 bits, with fp32's exponent, so nothing has to be
// scaled and no pass over the weight has to find a maximum first). A product is six bf16 products,
//   x y = hi hi + hi mid + mid hi + hi lo + mid mid + lo hi   (the rest is below 2^-24 of it),
// accumulated in fp32: HBM is the bound, the matrix pipe has the time. Beyond 64 rows it has not, and the operands are pairs of
// fp16 (fp16_pairs.h: three products), scaled by the largest magnitude of each class's weights, which the forward pass finds in a
// pass of its own and leaves for the backward pass. The cotangents as an operand of x's gradient stay bf16 triples: a row that is
// nearly right has cotangents far below 1, and no one scale fits all of its classes.
// The small operand (x, or the cotangents) is brought into operand order once ("planes").
//
// stream_kernel: 128 rows of the streamed operand a work-group, 32 per wave, against up to 128 columns, whose planes the waves
// share through LDS; the next chunk of both operands travels while this one is multiplied. stream_few_kernel, for few rows of x
// and few classes: 32 rows a work-group, its four waves share k out among them without a barrier and add up in LDS (2 rows, 9138
// classes x 2315: 37 us against 72 on 72 work-groups of 128; 16 rows, 131072 x 4096: 567 us against 457, so only for few classes).
//
// Bound: HBM up to about 100 columns, the matrix pipe beyond. Measured: 16 rows, 131072 x 4096 (2.1 GB): statistics 455 to 490 us = 4.4 to
// 4.7 TB/s, cotangents 457 us, x's gradient 440 us, the weight's 510 us; 256 rows, 65536 x 4096: statistics 550 us = 250 TFLOP/s of fp32
// products (pairs), x's gradient 770 us = 178 (triples).
#include "linear_cross_entropy.h"

#include <type_traits>

namespace lce {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
using pairs::floatx16;

constexpr int TPB = 256;
constexpr float kLog2e = 1.4426950408889634f;
// Cotangents, at most 1, are held times 2^40, so that the lower parts of hardly likely classes stay in bf16's normal range.
constexpr int kUp = 40;
// planes of 32 columns x 16 of k: 1 KiB for each part
template <typename Op>
constexpr int step_bytes() { return Op::PARTS * 1024; }

struct Triple {
  static constexpr int PARTS = 3;
  typedef bf16x8 Vec;
  bf16x8 p[3];
};
struct Pair {
  static constexpr int PARTS = 2;
  typedef pairs::half8 Vec;
  pairs::half8 p[2];
};

__device__ __forceinline__ void split(const float (&x)[8], int, Triple& t) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float2v r = {x[i], x[i + 1]};
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const bf16x2 h = __builtin_convertvector(r, bf16x2);
      t.p[j][i] = h[0];
      t.p[j][i + 1] = h[1];
      r[0] -= (float)h[0];
      r[1] -= (float)h[1];
    }
  }
}
__device__ __forceinline__ void split(const float (&x)[8], int shift, Pair& t) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = pairs::scaled(x[e], shift);
  pairs::split8(y, t.p[0], t.p[1]);
}

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ floatx16 multiply(const Pair& a, const Pair& b, floatx16 c) { return pairs::mfma_pairs(a.p[0], a.p[1], b.p[0], b.p[1], c); }
__device__ __forceinline__ floatx16 multiply(const Triple& a, const Triple& b, floatx16 c) {
  c = mfma(a.p[2], b.p[0], c);
  c = mfma(a.p[1], b.p[1], c);
  c = mfma(a.p[0], b.p[2], c);
  c = mfma(a.p[1], b.p[0], c);
  c = mfma(a.p[0], b.p[1], c);
  return mfma(a.p[0], b.p[0], c);
}

// Order of k within a step of 16: the lanes of half h hold 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3, the order in which an
// accumulator holds its rows, so that cotangents become operands as they lie.
__device__ __forceinline__ int k_of(int half, int e) { return 8 * (e >> 2) + 4 * half + (e & 3); }

// Elements k0 + k_of(half, e) of row r of an operand that lies contiguous along k (x[r * ld + k]: 16 bytes at a time, which global
// memory gives from any multiple of 4) or along r (x[k * ld + r]). Rows behind the operand's end read its last one; what lies
// behind the end of k becomes zero.
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
template <bool KCONTIG>
__device__ __forceinline__ void load_step(const float* __restrict__ x, int64_t ld, int64_t r, int64_t rows, int64_t k0, int64_t k, int half, float (&v)[8]) {
  r = min(r, rows - 1);
  if (KCONTIG && k0 + 16 <= k) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4u f = *reinterpret_cast<const float4u*>(x + r * ld + k0 + 8 * j + 4 * half);
      v[4 * j] = f[0]; v[4 * j + 1] = f[1]; v[4 * j + 2] = f[2]; v[4 * j + 3] = f[3];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t at = min(k0 + k_of(half, e), k - 1);
    v[e] = KCONTIG ? x[r * ld + at] : x[at * ld + r];
  }
  if (k0 + 16 > k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k0 + k_of(half, e) < k ? v[e] : 0.f;
  }
}

// Planes of an operand [rows, k]: per 32 rows and step of 16 the parts, each 64 lanes x 16 bytes. One wave per step.
template <bool KCONTIG, typename Op>
__global__ __launch_bounds__(TPB) void planes_kernel(const float* __restrict__ x, int64_t ld, int64_t rows, int64_t k, const float* __restrict__ left_out,
                                                     const float* __restrict__ amax, char* __restrict__ planes) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int64_t steps = (k + 15) / 16, step_groups = (steps + 3) / 4;
  const int64_t step = blockIdx.x % step_groups * 4 + (threadIdx.x >> 6), block = blockIdx.x / step_groups, r = block * 32 + (lane & 31);
  if (step >= steps) return;
  float v[8];
  load_step<KCONTIG>(x, ld, r, rows, step * 16, k, half, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t i = KCONTIG ? r : step * 16 + k_of(half, e);  // index along x's first axis
    const bool skip = r >= rows || (left_out && i < (KCONTIG ? rows : k) && left_out[i] < 0.f);
    v[e] = skip ? 0.f : v[e];
  }
  Op t;
  split(v, amax ? pairs::shift_of(amax[min(r, rows - 1)]) : 0, t);
  char* to = planes + (block * steps + step) * step_bytes<Op>() + lane * 16;
#pragma unroll
  for (int j = 0; j < Op::PARTS; ++j) *reinterpret_cast<typename Op::Vec*>(to + j * 1024) = t.p[j];
}

enum { STATS, DZ, DX };

template <typename Op>
__device__ __forceinline__ Op read_planes(const char* from, int lane) {
  Op x;
#pragma unroll
  for (int j = 0; j < Op::PARTS; ++j) x.p[j] = *reinterpret_cast<const typename Op::Vec*>(from + j * 1024 + lane * 16);
  return x;
}

// What becomes of 32 rows of the streamed operand (from r0, `left` of them there) against 32 rows n of x: z of the lane's n in acc.
// Maximum and sum of exp over the rows:
__device__ __forceinline__ void stats_block(const Direct& p, floatx16& acc, int64_t r0, int left, int n, int half, float& m, float& sum) {
  m = -INFINITY;
  sum = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int i = k_of(half, v & 7) + 16 * (v >> 3);
    acc[v] = i < left ? acc[v] : -INFINITY;
    m = fmaxf(m, acc[v]);
  }
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  const float top = m * kLog2e;
  const float t = n < p.N ? p.target[n] : -1.f, local = t - (float)(p.v0 + r0);
  const int hot = local >= 0.f && local < 32.f ? (int)local : -1;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const float z = acc[v];
    if (hot == k_of(half, v & 7) + 16 * (v >> 3) && hot < left) p.zt[n] = z;
    sum += z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -top));
  }
  sum += __shfl_xor(sum, 32, 64);
}

// Cotangents: fp32 [N, rows] for the weight's gradient, and as planes (columns: rows of x, k: classes) for x's.
__device__ __forceinline__ void dz_block(const Direct& p, const floatx16& acc, int64_t r0, int left, int n, int block, int lane, int half) {
  const int64_t zsteps = (p.rows + 15) / 16;
  const float t = n < p.N ? p.target[n] : -1.f, e = p.lse[min((int64_t)n, p.N - 1)] * kLog2e - (float)kUp, local = t - (float)(p.v0 + r0);
  const int hot = local >= 0.f && local < 32.f ? (int)local : -1;
  float d[2][8];
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int i = k_of(half, v & 7) + 16 * (v >> 3);
    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v], kLog2e, -e)) - (i == hot ? (float)(1ll << kUp) : 0.f);
    d[v >> 3][v & 7] = i < left && !(t < 0.f) ? y : 0.f;
  }
  if (p.dz && n < p.N) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int i = k_of(half, v & 7) + 16 * (v >> 3);
      if (i < left) p.dz[(int64_t)n * p.dz_ld + r0 + i] = d[v >> 3][v & 7];
    }
  }
  if (p.dz_planes && block * 32 < p.N)
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (16 * s < left) {
        Triple y;
        split(d[s], 0, y);
        char* to = p.dz_planes + ((int64_t)block * zsteps + r0 / 16 + s) * step_bytes<Triple>() + lane * 16;
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(to + j * 1024) = y.p[j];
      }
}

// sum 2^-kUp g / count as sum * a * b, neither of which leaves fp32's range
struct Down {
  float a, b;
  __device__ __forceinline__ explicit Down(const Mean& c) {
    const int e = c.e - kUp, h = e / 2;
    a = __builtin_ldexpf(c.m, h);
    b = __builtin_ldexpf(1.f, e - h);
  }
  __device__ __forceinline__ float operator()(float sum) const { return sum * a * b; }
};

__device__ __forceinline__ void dx_block(const Direct& p, const floatx16& acc, int64_t r0, int left, int n, int half, int part) {
  if (n >= p.N) return;
  const Down down(mean_of(p.g, p.count));
  const bool skip = p.target[n] < 0.f;  // (its cotangents are 0, but 0 times what the weight holds need not be)
  float* out = p.out + ((int64_t)part * p.N + n) * p.rows + r0;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int i = k_of(half, v & 7) + 16 * (v >> 3);
    const float y = skip ? 0.f : down(acc[v]);
    if (i < left) out[i] = p.accumulate ? out[i] + y : y;
  }
}

// Up to 32 rows of x. Waves take chunks of 4 steps in turn; nothing is shared until the end.
template <bool KCONTIG, int MODE>
__global__ __launch_bounds__(TPB, 2) void stream_few_kernel(Direct p) {
  constexpr int CS = 4;
  __shared__ float red[4][16][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * 32;
  const int part = blockIdx.z;
  const int steps = (int)((p.k + 15) / 16), chunks = (steps + CS - 1) / CS, per = (chunks + p.parts - 1) / p.parts;
  const int c0 = min(part * per, chunks), c1 = min(c0 + per, chunks);
  float next[CS][8], now[CS][8];
  Triple xn[CS], x[CS];
  auto fetch = [&](int c) {
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      load_step<KCONTIG>(p.a, p.lda, r0 + col, p.rows, (int64_t)(c * CS + s) * 16, p.k, half, next[s]);
      xn[s] = read_planes<Triple>(p.planes + (int64_t)min(c * CS + s, steps - 1) * step_bytes<Triple>(), lane);
    }
  };
  floatx16 acc = {};
  int c = c0 + wave;
  if (c < c1) fetch(c);
  for (; c < c1; c += 4) {
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      x[s] = xn[s];
#pragma unroll
      for (int e = 0; e < 8; ++e) now[s][e] = next[s][e];
    }
    if (c + 4 < c1) fetch(c + 4);
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      Triple a;
      split(now[s], 0, a);
      acc = multiply(a, x[s], acc);
    }
  }
#pragma unroll
  for (int v = 0; v < 16; ++v) red[wave][v][lane] = acc[v];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int v = 0; v < 16; ++v) acc[v] = (red[0][v][lane] + red[1][v][lane]) + (red[2][v][lane] + red[3][v][lane]);
  const int left = (int)min(p.rows - r0, (int64_t)32);
  if (MODE == STATS) {
    float m, sum;
    stats_block(p, acc, r0, left, col, half, m, sum);
    if (half == 0 && col < p.N) *reinterpret_cast<float2*>(p.stats + ((int64_t)blockIdx.x * p.N + col) * 2) = make_float2(m, sum);
  } else if (MODE == DZ) {
    dz_block(p, acc, r0, left, col, 0, lane, half);
  } else {
    dx_block(p, acc, r0, left, col, half, part);
  }
}

template <int NB, typename Op, bool KCONTIG, int MODE>
__global__ __launch_bounds__(TPB, 2) void stream_kernel(Direct p) {
  constexpr int CS = NB > 2 ? 2 : 4;  // steps per chunk
  constexpr int STAGE = CS * NB * step_bytes<Op>(), P = Op::PARTS;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  // Work-groups are dealt round-robin to the 8 XCDs: those that read the same 128 rows for different columns follow each other on
  // one XCD, so that the rows come from memory once and then from its L2.
  const uint32_t ntiles = (uint32_t)((p.N + NB * 32 - 1) / (NB * 32)), turn = blockIdx.x >> 3;
  const uint32_t unit = turn / ntiles * 8 + (blockIdx.x & 7);  // of rows and part
  const int64_t group = unit / (uint32_t)p.parts;
  if (group * 128 >= p.rows) return;
  const int64_t r0 = group * 128 + wave * 32;
  const int n0 = (int)(turn % ntiles) * NB * 32, part = (int)(unit % (uint32_t)p.parts);
  const int steps = (int)((p.k + 15) / 16), chunks = (steps + CS - 1) / CS, per = (chunks + p.parts - 1) / p.parts;
  const int c0 = min(part * per, chunks), c1 = min(c0 + per, chunks);
  const int blocks = (int)((p.N + 31) / 32), first_block = n0 / 32;
  const int shift = P == 2 ? pairs::shift_of(p.a_amax[min(r0 + col, p.rows - 1)]) : 0;

  // planes of chunk c: NB blocks of columns, CS steps each (clamped: a step or block behind the end is read again and not used)
  auto request = [&](int c, char* to) {
    constexpr int LINES = CS * NB * P;  // of 1 KiB
#pragma unroll
    for (int i = 0; i < (LINES + 3) / 4; ++i) {
      const int line = i * 4 + wave;
      if (LINES % 4 == 0 || line < LINES) {
        const int b = line / (CS * P), s = line / P % CS, j = line % P;
        const int64_t from = ((int64_t)min(first_block + b, blocks - 1) * steps + min(c * CS + s, steps - 1)) * step_bytes<Op>() + j * 1024;
        pairs::load_to_lds(p.planes + from + lane * 16, to + line * 1024);
      }
    }
  };
  float next[CS][8], now[CS][8];
  auto fetch = [&](int c) {
#pragma unroll
    for (int s = 0; s < CS; ++s) load_step<KCONTIG>(p.a, p.lda, r0 + col, p.rows, (int64_t)(c * CS + s) * 16, p.k, half, next[s]);
  };
  floatx16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = floatx16{};
  if (c0 < c1) {
    request(c0, smem);
    fetch(c0);
  }
  pairs::wait_loads();
  __syncthreads();
  for (int c = c0; c < c1; ++c) {
    const char* stage = smem + ((c - c0) & 1) * STAGE;
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) now[s][e] = next[s][e];
    if (c + 1 < c1) {
      request(c + 1, smem + ((c + 1 - c0) & 1) * STAGE);
      fetch(c + 1);
    }
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      Op a;
      split(now[s], shift, a);
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = multiply(a, read_planes<Op>(stage + (b * CS + s) * step_bytes<Op>(), lane), acc[b]);
    }
    pairs::wait_loads();
    __syncthreads();
  }
  if (P == 2) {  // the scales come off: of the columns per lane, of the rows per register
    float* down = reinterpret_cast<float*>(smem) + wave * 32;
    if (half == 0) down[col] = __builtin_ldexpf(1.f, -shift);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float cx = __builtin_ldexpf(1.f, -pairs::shift_of(p.x_amax[min((int64_t)n0 + b * 32 + col, p.N - 1)]));
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[b][v] = acc[b][v] * cx * down[k_of(half, v & 7) + 16 * (v >> 3)];
    }
    __syncthreads();
  }

  const int left = (int)min(p.rows - r0, (int64_t)32);  // rows of this wave (can be none)
  if (MODE == STATS) {
    float* red = reinterpret_cast<float*>(smem);  // [4 waves][NB * 32][2]
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float m, sum;
      stats_block(p, acc[b], r0, left, n0 + b * 32 + col, half, m, sum);
      if (half == 0) *reinterpret_cast<float2*>(red + (wave * NB * 32 + b * 32 + col) * 2) = make_float2(m, sum);
    }
    __syncthreads();
    if (tid < NB * 32 && n0 + tid < p.N) {
      float m = -INFINITY, sum = 0.f;
      for (int w = 0; w < 4; ++w) m = fmaxf(m, red[(w * NB * 32 + tid) * 2]);
      for (int w = 0; w < 4; ++w) {
        const float mw = red[(w * NB * 32 + tid) * 2], lw = red[(w * NB * 32 + tid) * 2 + 1];
        sum += lw == 0.f ? 0.f : lw * __builtin_amdgcn_exp2f((mw - m) * kLog2e);
      }
      *reinterpret_cast<float2*>(p.stats + (group * p.N + n0 + tid) * 2) = make_float2(m, sum);
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (MODE == DZ) dz_block(p, acc[b], r0, left, n0 + b * 32 + col, first_block + b, lane, half);
      else dx_block(p, acc[b], r0, left, n0 + b * 32 + col, half, part);
    }
  }
}

// dW[d, v] = c sum_n x[n, d] dz[n, v]: a wave takes 32 classes against 4 x 32 (pairs: 8 x 32) of x's columns at a time, whose planes
// the four waves share through LDS. Bound: HBM (the gradient is written once) up to about 128 rows.
template <bool BY_D, typename Op>
__global__ __launch_bounds__(TPB, 2) void outer_kernel(Outer p) {
  constexpr int P = Op::PARTS, DB = P == 2 ? 8 : 4, CS = 2, STAGE = DB * CS * step_bytes<Op>();
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int64_t v0 = (int64_t)blockIdx.x * 128 + wave * 32, v = v0 + col;
  const int steps = (int)((p.N + 15) / 16), chunks = (steps + CS - 1) / CS, blocks = (int)((p.D + 31) / 32);
  const int groups = (blocks + DB - 1) / DB, g0 = blockIdx.y * p.groups, g1 = min(g0 + p.groups, groups);
  const Mean c = mean_of(p.g, p.count);
  const Down down(c);
  const int turns = (g1 - g0) * chunks;
  auto request = [&](int turn, char* to) {
    const int g = g0 + turn / chunks, ch = turn % chunks;
#pragma unroll
    for (int i = 0; i < DB * CS * P / 4; ++i) {
      const int line = i * 4 + wave, b = line / (CS * P), s = line / P % CS, j = line % P;
      const int64_t from = ((int64_t)min(g * DB + b, blocks - 1) * steps + min(ch * CS + s, steps - 1)) * step_bytes<Op>() + j * 1024;
      pairs::load_to_lds(p.planes + from + lane * 16, to + line * 1024);
    }
  };
  int shift = 0;
  if (P == 2) {  // the scale of the class's cotangents over the rows
    float amax = 0.f;
    const float* z = p.dz + min(v, p.cols - 1);
#pragma unroll 8
    for (int64_t n = half; n < p.N; n += 2) amax = fmaxf(amax, pairs::finite_abs(z[n * p.dz_ld]));
    shift = pairs::shift_of(fmaxf(amax, __shfl_xor(amax, 32, 64)));
  }
  float next[CS][8], now[CS][8];
  auto fetch = [&](int turn) {
    const int ch = turn % chunks;
#pragma unroll
    for (int s = 0; s < CS; ++s) load_step<false>(p.dz, p.dz_ld, v, p.cols, (int64_t)(ch * CS + s) * 16, p.N, half, next[s]);
  };
  floatx16 acc[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) acc[b] = floatx16{};
  if (turns > 0) {
    request(0, smem);
    fetch(0);
  }
  pairs::wait_loads();
  __syncthreads();
  for (int turn = 0; turn < turns; ++turn) {
    const char* stage = smem + (turn & 1) * STAGE;
#pragma unroll
    for (int s = 0; s < CS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) now[s][e] = next[s][e];
    if (turn + 1 < turns) {
      request(turn + 1, smem + ((turn + 1) & 1) * STAGE);
      fetch(turn + 1);
    }
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      if ((turn % chunks) * CS + s >= steps) break;
      Op z;
      split(now[s], shift, z);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const Op x = read_planes<Op>(stage + (b * CS + s) * step_bytes<Op>(), lane);
        acc[b] = BY_D ? multiply(x, z, acc[b]) : multiply(z, x, acc[b]);
      }
    }
    if (turn % chunks == chunks - 1) {
      const int d0 = (g0 + turn / chunks) * DB * 32;
      // The axis that lies contiguous in the output is the one along the lanes. (Pairs: the scales come off, of the lane's class and
      // of x's columns, the latter with 2^-kUp; with classes along the registers, lane k has those of class k.)
      const float down_v = __builtin_ldexpf(c.m, c.e - shift);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const float down_lane = P == 2 && !BY_D ? __builtin_ldexpf(1.f, -pairs::shift_of(p.x_amax[min(d0 + b * 32 + col, (int)p.D - 1)]) - kUp) : 1.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = k_of(half, i & 7) + 16 * (i >> 3);
          if (BY_D) {
            const int d = d0 + b * 32 + k;
            const float down_d = P == 2 ? __builtin_ldexpf(1.f, -pairs::shift_of(p.x_amax[min(d, (int)p.D - 1)]) - kUp) : 1.f;
            if (v < p.cols && d < p.D) p.out[(int64_t)d * p.ld + v] = P == 2 ? acc[b][i] * down_v * down_d : down(acc[b][i]);
          } else {
            const int d = d0 + b * 32 + col;
            const float down_k = P == 2 ? __shfl(down_v, k, 64) : 1.f;
            if (d < p.D && v0 + k < p.cols) p.out[(v0 + k) * p.ld + d] = P == 2 ? acc[b][i] * down_k * down_lane : down(acc[b][i]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int b = 0; b < DB; ++b) acc[b] = floatx16{};
    }
    pairs::wait_loads();
    __syncthreads();
  }
}

template <int NB, typename Op, int MODE>
int32_t stream_tiles(const Direct& p, bool kcontig, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div64(ceil_div64(p.rows, 128) * p.parts, 8) * 8 * ceil_div64(p.N, NB * 32)));
  if (kcontig) hipLaunchKernelGGL((stream_kernel<NB, Op, true, MODE>), grid, dim3(TPB), 0, s, p);
  else hipLaunchKernelGGL((stream_kernel<NB, Op, false, MODE>), grid, dim3(TPB), 0, s, p);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

// Up to 32 rows of x and so few classes that groups of 128 would leave half of the CUs idle: groups of 32.
int64_t rows_per_group(int64_t N, int64_t rows) { return N <= 32 && ceil_div64(rows, 128) * 2 < endia::ctx().cu_count ? 32 : 128; }

// Op: operands of statistics and cotangents beyond kTripleRows rows of x are pairs, all others triples
template <int MODE>
int32_t stream(const Direct& p, bool kcontig, hipStream_t s) {
  using Op = typename std::conditional<MODE == DX, Triple, Pair>::type;
  if (MODE != DX && rows_per_group(p.N, p.rows) == 32) {
    const dim3 grid((unsigned)ceil_div64(p.rows, 32), 1, (unsigned)p.parts);
    if (kcontig) hipLaunchKernelGGL((stream_few_kernel<true, MODE>), grid, dim3(TPB), 0, s, p);
    else hipLaunchKernelGGL((stream_few_kernel<false, MODE>), grid, dim3(TPB), 0, s, p);
    ENDIA_LAUNCH_CHECK();
    return ENDIA_HIP_OK;
  }
  if (p.N <= 32) return stream_tiles<1, Triple, MODE>(p, kcontig, s);
  if (p.N <= kTripleRows) return stream_tiles<2, Triple, MODE>(p, kcontig, s);
  // 96 or 128 columns at a time, whichever leaves fewer of them empty
  const int64_t blocks = ceil_div64(p.N, 32);
  return ceil_div64(blocks, 3) * 3 < ceil_div64(blocks, 4) * 4 ? stream_tiles<3, Op, MODE>(p, kcontig, s) : stream_tiles<4, Op, MODE>(p, kcontig, s);
}

}  // namespace

int32_t planes(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, const float* amax, char* to, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div64(ceil_div64(k, 16), 4) * ceil_div64(rows, 32)));
  if (transposed && amax) hipLaunchKernelGGL((planes_kernel<false, Pair>), grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, amax, to);
  else if (transposed) hipLaunchKernelGGL((planes_kernel<false, Triple>), grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, amax, to);
  else if (amax) hipLaunchKernelGGL((planes_kernel<true, Pair>), grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, amax, to);
  else hipLaunchKernelGGL((planes_kernel<true, Triple>), grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, amax, to);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int64_t direct_rows(int64_t N, int64_t rows) { return rows_per_group(N, rows); }
int32_t direct_stats(const Direct& p, bool kcontig, hipStream_t s) { return stream<STATS>(p, kcontig, s); }
int32_t direct_dz(const Direct& p, bool kcontig, hipStream_t s) { return stream<DZ>(p, kcontig, s); }
int32_t direct_dx(const Direct& p, bool kcontig, hipStream_t s) { return stream<DX>(p, kcontig, s); }

int32_t direct_dw(const Outer& q, bool by_d, hipStream_t s) {
  Outer p = q;
  const int64_t vg = ceil_div64(p.cols, 128), groups = ceil_div64(p.D, p.x_amax ? 256 : 128);
  int64_t cuts = ceil_div64(4 * endia::ctx().cu_count, vg);  // work-groups along x's columns, when the classes alone do not fill the chip
  if (cuts > groups) cuts = groups;
  p.groups = (int)ceil_div64(groups, cuts);
  const dim3 grid((unsigned)vg, (unsigned)ceil_div64(groups, p.groups));
  if (p.x_amax) {
    if (by_d) hipLaunchKernelGGL((outer_kernel<true, Pair>), grid, dim3(TPB), 0, s, p);
    else hipLaunchKernelGGL((outer_kernel<false, Pair>), grid, dim3(TPB), 0, s, p);
  } else {
    if (by_d) hipLaunchKernelGGL((outer_kernel<true, Triple>), grid, dim3(TPB), 0, s, p);
    else hipLaunchKernelGGL((outer_kernel<false, Triple>), grid, dim3(TPB), 0, s, p);
  }
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace lce
