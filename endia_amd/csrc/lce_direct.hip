// The linear cross entropy for few rows (up to a few hundred): the weight is what there is to read, so it is read as it lies, in
// fp32 and in either storage order, straight into matrix operands; no copy of it in another form is made.
//
// An fp32 number is held as three bf16 (hi, mid, lo: 8 + 8 + 8 bits, with fp32's exponent, so nothing has to be scaled and no pass
// over the weight has to find a maximum first). A product is six bf16 products,
//   x y = hi hi + hi mid + mid hi + hi lo + mid mid + lo hi   (the rest is below 2^-24 of it),
// accumulated in fp32. The small operand (x, or the cotangents) is turned into such triples once, in operand order ("planes").
//
// A work-group of 4 waves takes 128 rows of the streamed operand (32 per wave) against up to 128 columns; the waves share the
// columns' planes through LDS, and the next chunk of both travels while this one is multiplied.
// Bound: HBM up to about 96 columns (per 2 KiB of weight and wave 6 x 32 cycles of the matrix pipe per 32 columns and about 200 of
// the vector ALU, against some 900 cycles that its share of the memory takes), the matrix pipe beyond.
#include "linear_cross_entropy.h"

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
constexpr int kStepBytes = 3 * 1024;  // planes of 32 columns x 16 of k

struct Triple {
  bf16x8 p[3];
};

__device__ __forceinline__ Triple triple(const float (&x)[8]) {
  Triple t;
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
  return t;
}

__device__ __forceinline__ floatx16 mfma(bf16x8 a, bf16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ floatx16 mfma_triples(const Triple& a, const Triple& b, floatx16 c) {
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

// Elements k0 + k_of(half, e) of row r of an operand that lies contiguous along k (x[r * ld + k]) or along r (x[k * ld + r]). Loads
// go out unconditionally, clamped to the operand; what lies behind its end becomes zero.
template <bool KCONTIG, bool VEC>
__device__ __forceinline__ void load_step(const float* __restrict__ x, int64_t ld, int64_t r, int64_t rows, int64_t k0, int64_t k, int half, float (&v)[8]) {
  r = min(r, rows - 1);
  if (KCONTIG && VEC) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = k0 + 8 * j + 4 * half;
      const float4 f = *reinterpret_cast<const float4*>(x + r * ld + min(at, k - 4));
      v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t at = min(k0 + k_of(half, e), k - 1);
      v[e] = KCONTIG ? x[r * ld + at] : x[at * ld + r];
    }
  }
  if (k0 + 16 > k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k0 + k_of(half, e) < k ? v[e] : 0.f;
  }
}

// Planes of an operand [rows, k]: per 32 rows and step of 16: hi, mid, lo, each 64 lanes x 16 bytes. One wave per step.
template <bool KCONTIG>
__global__ __launch_bounds__(TPB) void planes_kernel(const float* __restrict__ x, int64_t ld, int64_t rows, int64_t k, const float* __restrict__ left_out,
                                                     char* __restrict__ planes) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int64_t steps = (k + 15) / 16, step = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), block = blockIdx.y, r = block * 32 + (lane & 31);
  if (step >= steps) return;
  float v[8];
  load_step<KCONTIG, false>(x, ld, r, rows, step * 16, k, half, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t i = KCONTIG ? r : step * 16 + k_of(half, e);  // index along x's first axis
    const bool skip = r >= rows || (left_out && i < (KCONTIG ? rows : k) && left_out[i] < 0.f);
    v[e] = skip ? 0.f : v[e];
  }
  const Triple t = triple(v);
  char* to = planes + (block * steps + step) * kStepBytes + lane * 16;
#pragma unroll
  for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(to + j * 1024) = t.p[j];
}

enum { STATS, DZ, DX };

template <int NB, bool KCONTIG, bool VEC, int MODE>
__global__ __launch_bounds__(TPB, 2) void stream_kernel(Direct p) {
  constexpr int CS = NB == 4 ? 2 : 4;                // steps per chunk
  constexpr int STAGE = CS * NB * kStepBytes;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * 128 + wave * 32;
  const int n0 = blockIdx.y * NB * 32, part = blockIdx.z;
  const int steps = (int)((p.k + 15) / 16), chunks = (steps + CS - 1) / CS, per = (chunks + p.parts - 1) / p.parts;
  const int c0 = min(part * per, chunks), c1 = min(c0 + per, chunks);
  const int blocks = (int)((p.N + 31) / 32), first_block = n0 / 32;

  // planes of chunk c: NB blocks of columns, CS steps each (clamped: a step or block behind the end is read again and not used)
  auto request = [&](int c, char* to) {
    constexpr int LINES = CS * NB * 3;  // of 1 KiB
#pragma unroll
    for (int i = 0; i < (LINES + 3) / 4; ++i) {
      const int line = i * 4 + wave;
      if (LINES % 4 == 0 || line < LINES) {
        const int b = line / (CS * 3), s = line / 3 % CS, j = line % 3;
        const int64_t from = ((int64_t)min(first_block + b, blocks - 1) * steps + min(c * CS + s, steps - 1)) * kStepBytes + j * 1024;
        pairs::load_to_lds(p.planes + from + lane * 16, to + line * 1024);
      }
    }
  };
  float next[CS][8], now[CS][8];
  auto fetch = [&](int c) {
#pragma unroll
    for (int s = 0; s < CS; ++s) load_step<KCONTIG, VEC>(p.a, p.lda, r0 + col, p.rows, (int64_t)(c * CS + s) * 16, p.k, half, next[s]);
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
      const Triple a = triple(now[s]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        Triple x;
#pragma unroll
        for (int j = 0; j < 3; ++j) x.p[j] = *reinterpret_cast<const bf16x8*>(stage + ((b * CS + s) * 3 + j) * 1024 + lane * 16);
        acc[b] = mfma_triples(a, x, acc[b]);
      }
    }
    pairs::wait_loads();
    __syncthreads();
  }

  const int left = (int)min(p.rows - r0, (int64_t)32);  // rows of this wave (can be none)
  if (MODE == STATS) {
    float* red = reinterpret_cast<float*>(smem);  // [4 waves][NB * 32][2]
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int n = n0 + b * 32 + col;
      float m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int i = k_of(half, v & 7) + 16 * (v >> 3);
        acc[b][v] = i < left ? acc[b][v] : -INFINITY;
        m = fmaxf(m, acc[b][v]);
      }
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float top = m * kLog2e;
      const float t = n < p.N ? p.target[n] : -1.f, local = t - (float)(p.v0 + r0);
      const int hot = local >= 0.f && local < 32.f ? (int)local : -1;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float z = acc[b][v];
        if (hot == k_of(half, v & 7) + 16 * (v >> 3) && hot < left) p.zt[n] = z;
        sum += z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -top));
      }
      sum += __shfl_xor(sum, 32, 64);
      if (half == 0) {
        red[(wave * NB * 32 + b * 32 + col) * 2] = m;
        red[(wave * NB * 32 + b * 32 + col) * 2 + 1] = sum;
      }
    }
    __syncthreads();
    if (tid < NB * 32 && n0 + tid < p.N) {
      float m = -INFINITY, sum = 0.f;
      for (int w = 0; w < 4; ++w) m = fmaxf(m, red[(w * NB * 32 + tid) * 2]);
      for (int w = 0; w < 4; ++w) {
        const float mw = red[(w * NB * 32 + tid) * 2], lw = red[(w * NB * 32 + tid) * 2 + 1];
        sum += lw == 0.f ? 0.f : lw * __builtin_amdgcn_exp2f((mw - m) * kLog2e);
      }
      float* to = p.stats + ((int64_t)blockIdx.x * p.N + n0 + tid) * 2;
      to[0] = m;
      to[1] = sum;
    }
  } else if (MODE == DZ) {
    // cotangents: fp32 [N, rows] for the weight's gradient, and as planes (columns: rows of x, k: classes) for x's
    const int64_t zsteps = (p.rows + 15) / 16;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int n = n0 + b * 32 + col;
      const float t = n < p.N ? p.target[n] : -1.f, e = p.lse[min((int64_t)n, p.N - 1)] * kLog2e - (float)kUp, local = t - (float)(p.v0 + r0);
      const int hot = local >= 0.f && local < 32.f ? (int)local : -1;
      float d[2][8];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int i = k_of(half, v & 7) + 16 * (v >> 3);
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[b][v], kLog2e, -e)) - (i == hot ? (float)(1ll << kUp) : 0.f);
        d[v >> 3][v & 7] = i < left && !(t < 0.f) ? y : 0.f;
      }
      if (p.dz && n < p.N) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int i = k_of(half, v & 7) + 16 * (v >> 3);
          if (i < left) p.dz[(int64_t)n * p.dz_ld + r0 + i] = d[v >> 3][v & 7];
        }
      }
      if (p.dz_planes && first_block + b < blocks)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (16 * s < left) {
            const Triple y = triple(d[s]);
            char* to = p.dz_planes + ((int64_t)(first_block + b) * zsteps + r0 / 16 + s) * kStepBytes + lane * 16;
#pragma unroll
            for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8*>(to + j * 1024) = y.p[j];
          }
    }
  } else {
    const float c = p.count[0] > 0.f ? __builtin_ldexpf(p.g[0] / p.count[0], -kUp) : 0.f;
    float* out = p.out + part * p.N * p.rows;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int n = n0 + b * 32 + col;
      if (n >= p.N) continue;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int i = k_of(half, v & 7) + 16 * (v >> 3);
        float* to = out + n * p.rows + r0 + i;
        if (i < left) *to = p.accumulate ? *to + acc[b][v] * c : acc[b][v] * c;
      }
    }
  }
}

// dW[d, v] = c sum_n x[n, d] dz[n, v]: a wave takes 32 classes against 4 x 32 of x's columns at a time, whose planes the four waves
// share through LDS. Bound: HBM (the gradient is written once) up to about 128 rows.
template <bool BY_D>
__global__ __launch_bounds__(TPB, 2) void outer_kernel(Outer p) {
  constexpr int DB = 4, CS = 2, STAGE = DB * CS * kStepBytes;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int64_t v0 = (int64_t)blockIdx.x * 128 + wave * 32, v = v0 + col;
  const int steps = (int)((p.N + 15) / 16), chunks = (steps + CS - 1) / CS, blocks = (int)((p.D + 31) / 32);
  const int groups = (blocks + DB - 1) / DB, g0 = blockIdx.y * p.groups, g1 = min(g0 + p.groups, groups);
  const float c = p.count[0] > 0.f ? __builtin_ldexpf(p.g[0] / p.count[0], -kUp) : 0.f;
  const int turns = (g1 - g0) * chunks;
  auto request = [&](int turn, char* to) {
    const int g = g0 + turn / chunks, ch = turn % chunks;
#pragma unroll
    for (int i = 0; i < DB * CS * 3 / 4; ++i) {
      const int line = i * 4 + wave, b = line / (CS * 3), s = line / 3 % CS, j = line % 3;
      const int64_t from = ((int64_t)min(g * DB + b, blocks - 1) * steps + min(ch * CS + s, steps - 1)) * kStepBytes + j * 1024;
      pairs::load_to_lds(p.planes + from + lane * 16, to + line * 1024);
    }
  };
  float next[CS][8], now[CS][8];
  auto fetch = [&](int turn) {
    const int ch = turn % chunks;
#pragma unroll
    for (int s = 0; s < CS; ++s) load_step<false, false>(p.dz, p.dz_ld, v, p.cols, (int64_t)(ch * CS + s) * 16, p.N, half, next[s]);
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
      const Triple z = triple(now[s]);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        Triple x;
#pragma unroll
        for (int j = 0; j < 3; ++j) x.p[j] = *reinterpret_cast<const bf16x8*>(stage + ((b * CS + s) * 3 + j) * 1024 + lane * 16);
        acc[b] = BY_D ? mfma_triples(x, z, acc[b]) : mfma_triples(z, x, acc[b]);
      }
    }
    if (turn % chunks == chunks - 1) {
      const int d0 = (g0 + turn / chunks) * DB * 32;
      // the axis that lies contiguous in the output is the one along the lanes
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = k_of(half, i & 7) + 16 * (i >> 3);
          if (BY_D) {
            const int d = d0 + b * 32 + k;
            if (v < p.cols && d < p.D) p.out[(int64_t)d * p.ld + v] = acc[b][i] * c;
          } else {
            const int d = d0 + b * 32 + col;
            if (d < p.D && v0 + k < p.cols) p.out[(v0 + k) * p.ld + d] = acc[b][i] * c;
          }
        }
#pragma unroll
      for (int b = 0; b < DB; ++b) acc[b] = floatx16{};
    }
    pairs::wait_loads();
    __syncthreads();
  }
}

template <int NB, int MODE>
int32_t stream(const Direct& p, bool kcontig, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64(p.rows, 128), (unsigned)ceil_div64(p.N, NB * 32), (unsigned)p.parts);
  if (!kcontig) hipLaunchKernelGGL((stream_kernel<NB, false, false, MODE>), grid, dim3(TPB), 0, s, p);
  else if (vec) hipLaunchKernelGGL((stream_kernel<NB, true, true, MODE>), grid, dim3(TPB), 0, s, p);
  else hipLaunchKernelGGL((stream_kernel<NB, true, false, MODE>), grid, dim3(TPB), 0, s, p);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

template <int MODE>
int32_t stream(const Direct& p, bool kcontig, hipStream_t s) {
  const bool vec = kcontig && p.lda % 4 == 0 && p.k % 4 == 0 && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0;
  return p.N <= 32 ? stream<1, MODE>(p, kcontig, vec, s) : p.N <= 64 ? stream<2, MODE>(p, kcontig, vec, s) : stream<4, MODE>(p, kcontig, vec, s);
}

}  // namespace

int32_t planes(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, char* to, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64(ceil_div64(k, 16), 4), (unsigned)ceil_div64(rows, 32));
  if (transposed) hipLaunchKernelGGL(planes_kernel<false>, grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, to);
  else hipLaunchKernelGGL(planes_kernel<true>, grid, dim3(TPB), 0, s, x, ld, rows, k, left_out, to);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t direct_stats(const Direct& p, bool kcontig, hipStream_t s) { return stream<STATS>(p, kcontig, s); }
int32_t direct_dz(const Direct& p, bool kcontig, hipStream_t s) { return stream<DZ>(p, kcontig, s); }
int32_t direct_dx(const Direct& p, bool kcontig, hipStream_t s) { return stream<DX>(p, kcontig, s); }

int32_t direct_dw(const Outer& q, bool by_d, hipStream_t s) {
  Outer p = q;
  const int64_t vg = ceil_div64(p.cols, 128), groups = ceil_div64(p.D, 128);
  int64_t cuts = ceil_div64(4 * endia::ctx().cu_count, vg);  // work-groups along x's columns, when the classes alone do not fill the chip
  if (cuts > groups) cuts = groups;
  p.groups = (int)ceil_div64(groups, cuts);
  const dim3 grid((unsigned)vg, (unsigned)ceil_div64(groups, p.groups));
  if (by_d) hipLaunchKernelGGL(outer_kernel<true>, grid, dim3(TPB), 0, s, p);
  else hipLaunchKernelGGL(outer_kernel<false>, grid, dim3(TPB), 0, s, p);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace lce
