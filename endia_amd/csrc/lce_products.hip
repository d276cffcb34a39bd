// The products of the linear cross entropy over many rows: logits with their statistics, logits with their cotangents, and the
// two gradients. All are C[a, b] = sum_k A[a, k] B[b, k] over panels of fp16 pairs (linear_cross_entropy.h).
//
// A work-group of 8 waves owns 256 x 256 of C, a wave 128 (a) x 64 (b) in blocks of v_mfma_f32_32x32x16_f16, three products per
// block and 16 of k. A block of 32 k is one 32 KiB image of each operand; the next one travels from memory straight into the other
// half of the LDS (128 KiB, one work-group per CU, two waves per SIMD) while this one is multiplied: per block and SIMD 96 matrix
// instructions of 32 cycles against 48 LDS reads of 16 bytes a lane. The accumulator holds one b (a row of x, or a class) per lane
// and four consecutive a per register quad, so that what is needed per row of x (maximum, sum, cotangent) stays within a lane but
// for one exchange.
// Bound: the matrix pipe. Measured at 8192 rows, width 4096, as fp32 products: statistics of 16384 classes 2.53 to 2.58 ms = 426 to 434
// TFLOP/s (1.28 to 1.3 PFLOP/s of fp16 ones; a large library product reaches 1.17 on this card), cotangents of 4096 classes 722 to 732 us =
// 376 to 381, a gradient of them 677 to 688 us = 400 to 406. Tiles of 128 x 128 reach about three quarters of that rate, two to a CU.
#include "linear_cross_entropy.h"
#include "mfma_tile.h"

namespace lce {

namespace {

using namespace pairs;
constexpr float kLog2e = 1.4426950408889634f;

// T x T of C: 256 (8 waves, 2 x 4, of 128 x 64) or 128 (4 waves, 2 x 2, of 64 x 64, two work-groups per CU)
template <int T>
struct Tile {
  static constexpr int TPB = T == 256 ? 512 : 256, WB = T == 256 ? 4 : 2, FA = T == 256 ? 4 : 2, FB = 2;  // FA x FB blocks of 32 x 32 per wave
  static constexpr int STAGE = 2 * T * 128, PER_PANEL = kPanel / T;
  typedef floatx16 Acc[FA][FB];
  int lane, wave, col, half, wa, wb;  // the wave's place along a and b
  __device__ __forceinline__ Tile() {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    col = lane & 31;
    half = lane >> 5;
    wa = wave / WB;
    wb = wave % WB;
  }
  __device__ __forceinline__ int a_of(int fa, int v) const { return wa * FA * 32 + fa * 32 + 8 * (v >> 2) + 4 * half + (v & 3); }
  __device__ __forceinline__ int b_of(int fb) const { return wb * FB * 32 + fb * 32 + col; }
  // block 0 of k of tile t (a panel of 256 rows holds PER_PANEL tiles)
  __device__ __forceinline__ static const char* panel(const char* x, int t, int64_t kblocks) {
    return x + (t / PER_PANEL) * kblocks * kBlockBytes + t % PER_PANEL * T * 128;
  }
};
typedef Tile<256> Tile256;
constexpr int FA = Tile256::FA, FB = Tile256::FB, TPB = Tile256::TPB;  // dz_kernel's

template <int T>
__device__ __forceinline__ void request(const char* a, const char* b, char* stage, const Tile<T>& t) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int at = (p * (Tile<T>::TPB / 64) + t.wave) * 1024;
    load_to_lds(a + at + t.lane * 16, stage + at);
    load_to_lds(b + at + t.lane * 16, stage + Tile<T>::STAGE / 2 + at);
  }
}

__device__ __forceinline__ void read_line(const char* lines, int line, int s, int h, half8& hi, half8& lo) {
  const char* at = lines + line * 128;
  hi = *reinterpret_cast<const half8*>(at + (((2 * s + h) ^ (line & 7)) << 4));
  lo = *reinterpret_cast<const half8*>(at + (((4 + 2 * s + h) ^ (line & 7)) << 4));
}

template <int T>
__device__ __forceinline__ void multiply(const char* stage, const Tile<T>& t, typename Tile<T>::Acc& acc) {
  constexpr int FA = Tile<T>::FA, FB = Tile<T>::FB;
  const char *sa = stage + t.wa * FA * 32 * 128, *sb = stage + Tile<T>::STAGE / 2 + t.wb * FB * 32 * 128;
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    half8 ah[FA], al[FA], bh[FB], bl[FB];
#pragma unroll
    for (int f = 0; f < FB; ++f) read_line(sb, f * 32 + t.col, st, t.half, bh[f], bl[f]);
#pragma unroll
    for (int f = 0; f < FA; ++f) read_line(sa, f * 32 + t.col, st, t.half, ah[f], al[f]);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
    }
  }
}

template <int T>
__device__ __forceinline__ void clear(typename Tile<T>::Acc& acc) {
#pragma unroll
  for (int i = 0; i < Tile<T>::FA; ++i)
#pragma unroll
    for (int j = 0; j < Tile<T>::FB; ++j) acc[i][j] = floatx16{};
}

// z in place of the accumulator: the scales of both operands come off (classes behind the piece's end become -inf). The factors
// wait in LDS (2 T floats at `lds`).
template <int T>
__device__ __forceinline__ void to_logits(const Logits& p, const Tile<T>& t, int64_t a0, int64_t b0, float* lds, typename Tile<T>::Acc& acc) {
  constexpr int FA = Tile<T>::FA, FB = Tile<T>::FB;
  {
    const int i = threadIdx.x & (T - 1);
    const float amax = threadIdx.x < T ? p.w_amax[min(a0 + i, p.cols - 1)] : p.x_amax[min(b0 + i, p.N - 1)];
    lds[threadIdx.x] = __builtin_ldexpf(1.f, -shift_of(amax));
  }
  __syncthreads();
  float cb[FB];
#pragma unroll
  for (int j = 0; j < FB; ++j) cb[j] = lds[T + t.b_of(j)];
  const int left = (int)min(p.cols - a0, (int64_t)T);
#pragma unroll
  for (int i = 0; i < FA; ++i) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const float ca = lds[t.a_of(i, v)];
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j][v] = acc[i][j][v] * ca * cb[j];
    }
    if (left < T) {
#pragma unroll
      for (int v = 0; v < 16; ++v)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j][v] = t.a_of(i, v) < left ? acc[i][j][v] : -INFINITY;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int T>
__device__ __forceinline__ void logits_tile(const Logits& p, const Tile<T>& t, int ta, int tb, char* smem, typename Tile<T>::Acc& acc) {
  constexpr int STAGE = Tile<T>::STAGE;
  const int kblocks = (int)((p.D + kBlock - 1) / kBlock);
  const char *a = t.panel(p.w, ta, kblocks), *b = t.panel(p.x, tb, kblocks);
  clear<T>(acc);
  request(a, b, smem, t);
  wait_loads();
  __syncthreads();
  for (int kb = 0; kb < kblocks; ++kb) {
    if (kb + 1 < kblocks) request(a + (kb + 1) * kBlockBytes, b + (kb + 1) * kBlockBytes, smem + ((kb + 1) & 1) * STAGE, t);
    multiply(smem + (kb & 1) * STAGE, t, acc);
    wait_loads();
    __syncthreads();
  }
}

template <int T>
__global__ __launch_bounds__(Tile<T>::TPB, 2) void stats_kernel(Logits p) {
  constexpr int FA = Tile<T>::FA, FB = Tile<T>::FB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile<T> t;
  int ta, tb;
  const int tiles_a = (int)((p.cols + T - 1) / T), tiles_b = (int)((p.N + T - 1) / T);
  mfma::tile_of_block(blockIdx.x, gridDim.x, tiles_a, tiles_b, ta, tb);
  typename Tile<T>::Acc acc;
  logits_tile(p, t, ta, tb, smem, acc);
  const int64_t a0 = (int64_t)ta * T, b0 = (int64_t)tb * T;
  to_logits(p, t, a0, b0, reinterpret_cast<float*>(smem) + 4 * T, acc);
  float* red = reinterpret_cast<float*>(smem);  // [2 (wa)][T rows of x][2]
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const int64_t n = b0 + t.b_of(j);
    const float target = n < p.N ? p.target[n] : -1.f;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) m = fmaxf(m, acc[i][j][v]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float top = m * kLog2e;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float z = acc[i][j][v];
        sum += m == -INFINITY && !(z != z) ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -top));
      }
    sum += __shfl_xor(sum, 32, 64);
    const float local = target - (float)(p.v0 + a0);
    if (local >= 0.f && local < (float)T) {
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if ((int)local == t.a_of(i, v)) p.zt[n] = acc[i][j][v];
    }
    if (t.half == 0) {
      red[(t.wa * T + t.b_of(j)) * 2] = m;
      red[(t.wa * T + t.b_of(j)) * 2 + 1] = sum;
    }
  }
  __syncthreads();
  const int64_t n = b0 + threadIdx.x;
  if (threadIdx.x < T && n < p.N) {
    const float m0 = red[threadIdx.x * 2], l0 = red[threadIdx.x * 2 + 1], m1 = red[(T + threadIdx.x) * 2], l1 = red[(T + threadIdx.x) * 2 + 1];
    const float m = fmaxf(m0, m1);
    const float w0 = m0 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m0 - m) * kLog2e), w1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m1 - m) * kLog2e);
    float* to = p.stats + ((int64_t)ta * p.N + n) * 2;
    to[0] = m;
    to[1] = (m0 == -INFINITY && l0 == 0.f ? 0.f : w0 * l0) + (m1 == -INFINITY && l1 == 0.f ? 0.f : w1 * l1);
    if (l0 != l0 || l1 != l1) to[1] = NAN;
  }
}

// The largest shift of a tile's cotangents. gradient_kernel moves its sums from one tile's shift to the next one's, which is upwards
// where a tile of small cotangents, or of zeros (256 rows that are left out), follows one of large ones. |dz| <= 1 has a shift of at
// least 13, and the factors of a product are below 2^14. Along the classes a row's |dz| add up to 2 at most: sums below 2^28 that
// move up by 100 - 13 stay below 2^115. Along the rows there may be N < 2^b of size 1: sums below 2^(28 + b), so shifts up to
// 111 - b keep them below 2^126. (Up to 2047 rows that is no limit; a class of cotangents all below 2^(b - 98) lies lower in fp16's range.)
__device__ __forceinline__ int most_shift_of_class(int64_t N) { return min(kMaxShift, 79 + __clz((int)N)); }

// dz = exp(z - lse) - [class = target] (zeros for rows that are left out and behind the ends), stored twice as pairs: rows of x
// along k for the weight's gradient, classes along k for x's gradient. The scale of a row is one power of two per tile, from the
// tile's own largest, so that rows that are nearly right and classes that are hardly likely keep their precision.
__global__ __launch_bounds__(TPB, 2) void dz_kernel(Logits p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile256 t;
  int ta, tb;
  const int tiles_a = (int)((p.cols + kPanel - 1) / kPanel), tiles_b = (int)((p.N + kPanel - 1) / kPanel);
  mfma::tile_of_block(blockIdx.x, gridDim.x, tiles_a, tiles_b, ta, tb);
  floatx16 acc[FA][FB];
  logits_tile(p, t, ta, tb, smem, acc);
  const int64_t a0 = (int64_t)ta * kPanel, b0 = (int64_t)tb * kPanel;
  to_logits(p, t, a0, b0, reinterpret_cast<float*>(smem) + 2 * kPanel, acc);
  unsigned* row_max = reinterpret_cast<unsigned*>(smem);  // 256 rows of x, then 256 classes (magnitudes as bits)
  unsigned* class_max = row_max + kPanel;
  row_max[threadIdx.x] = 0;  // (512 threads: both)
  __syncthreads();
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const int64_t n = b0 + t.b_of(j);
    const float target = n < p.N ? p.target[n] : -1.f;
    const bool kept = !(target < 0.f);
    const float e = p.lse[min(n, p.N - 1)] * kLog2e, local = target - (float)(p.v0 + a0);
    const int hot = local >= 0.f && local < (float)kPanel ? (int)local : -1;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        float d = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][v], kLog2e, -e)) - (hot == t.a_of(i, v) ? 1.f : 0.f);
        d = kept ? d : 0.f;  // (classes behind the end have z = -inf)
        acc[i][j][v] = d;
        amax = fmaxf(amax, finite_abs(d));
      }
    atomicMax(&row_max[t.b_of(j)], __float_as_uint(amax));
  }
  // the largest of each class over the wave's 64 rows: halves are exchanged until a lane holds one class of sixteen
#pragma unroll
  for (int i = 0; i < FA; ++i) {
    float x[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = fmaxf(finite_abs(acc[i][0][v]), finite_abs(acc[i][1][v]));
#pragma unroll
    for (int w = 8; w; w >>= 1) {  // lanes 2w apart share 2w values
      const bool upper = t.col & (2 * w);
#pragma unroll
      for (int v = 0; v < w; ++v) {
        const float give = upper ? x[v] : x[v + w], keep = upper ? x[v + w] : x[v];
        x[v] = fmaxf(keep, __shfl_xor(give, 2 * w, 64));
      }
    }
    x[0] = fmaxf(x[0], __shfl_xor(x[0], 1, 64));
    const int v = (t.col & 16 ? 8 : 0) | (t.col & 8 ? 4 : 0) | (t.col & 4 ? 2 : 0) | (t.col & 2 ? 1 : 0);
    if (!(t.col & 1)) atomicMax(&class_max[t.a_of(i, v)], __float_as_uint(x[0]));
  }
  __syncthreads();
  int sb[FB];
#pragma unroll
  for (int j = 0; j < FB; ++j) sb[j] = shift_of(__uint_as_float(row_max[t.b_of(j)]));
  int own_shift = shift_of(__uint_as_float(row_max[threadIdx.x]));  // of a row, or of class threadIdx.x - 256
  if (threadIdx.x >= kPanel) own_shift = min(own_shift, most_shift_of_class(p.N));
  if (threadIdx.x < kPanel) p.p_shift[(int64_t)ta * tiles_b * kPanel + b0 + threadIdx.x] = own_shift;
  else p.pt_shift[(int64_t)tb * tiles_a * kPanel + a0 + threadIdx.x - kPanel] = own_shift;
  __syncthreads();
  // Four images of 64 KiB each, two at a time in LDS (128 KiB): first the rows' lines (k: classes), in halves of 128 rows ...
  const int64_t kb_p = (p.cols + kPanel - 1) / kPanel * 8, kb_t = (p.N + kPanel - 1) / kPanel * 8;  // blocks of k in p and pt
  if (p.p)
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if ((t.wb >> 1) == half) {
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int i = 0; i < FA; ++i) {
          const int row = t.b_of(j);
          char* line = smem + ((t.wa * 4 + i) * 128 + (row & 127)) * 128;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            half2v h0, l0, h1, l1;
            split2(scaled(acc[i][j][4 * q], sb[j]), scaled(acc[i][j][4 * q + 1], sb[j]), h0, l0);
            split2(scaled(acc[i][j][4 * q + 2], sb[j]), scaled(acc[i][j][4 * q + 3], sb[j]), h1, l1);
            half2v* at = reinterpret_cast<half2v*>(line + ((q ^ (row & 7)) << 4) + 8 * t.half);
            at[0] = h0;
            at[1] = h1;
            at = reinterpret_cast<half2v*>(line + (((4 + q) ^ (row & 7)) << 4) + 8 * t.half);
            at[0] = l0;
            at[1] = l1;
          }
        }
    }
    __syncthreads();
    char* to = p.p + ((int64_t)tb * kb_p + (int64_t)ta * 8) * kBlockBytes + half * 128 * 128;
    for (int i = threadIdx.x; i < 8 * 128 * 8; i += TPB)  // 8 blocks of k x 128 lines x 8 pieces
      *reinterpret_cast<float4*>(to + (int64_t)(i >> 10) * kBlockBytes + (i & 1023) * 16) = *reinterpret_cast<const float4*>(smem + i * 16);
    __syncthreads();
  }
  // ... then the classes' lines (k: rows), in halves of 128 rows = 4 blocks of k. Neighbouring lanes hold neighbouring rows of x:
  // they trade registers so that each stores two rows of one class. First everything is brought to its class's scale.
  if (!p.pt) return;
  int* class_shift = reinterpret_cast<int*>(smem);
  if (threadIdx.x >= kPanel) class_shift[threadIdx.x - kPanel] = own_shift;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FA; ++i) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int sa = class_shift[t.a_of(i, v)];
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j][v] = scaled(acc[i][j][v], sa);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if ((t.wb >> 1) == half) {
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int v = 0; v < 16; v += 2) {
            const bool odd = t.col & 1;
            const float a = acc[i][j][v], b = acc[i][j][v + 1];
            const float other = __shfl_xor(odd ? a : b, 1, 64);
            half2v hi, lo;
            split2(odd ? other : a, odd ? b : other, hi, lo);
            const int cls = t.a_of(i, v) + (odd ? 1 : 0), kk = t.col & ~1;  // two rows kk, kk + 1 of the block of 32
            char* line = smem + (((t.wb & 1) * 2 + j) * kPanel + cls) * 128;
            *reinterpret_cast<half2v*>(line + (((kk >> 3) ^ (cls & 7)) << 4) + 2 * (kk & 7)) = hi;
            *reinterpret_cast<half2v*>(line + (((4 + (kk >> 3)) ^ (cls & 7)) << 4) + 2 * (kk & 7)) = lo;
          }
    }
    __syncthreads();
    char* to = p.pt + ((int64_t)ta * kb_t + (int64_t)tb * 8 + half * 4) * kBlockBytes;
    for (int i = threadIdx.x; i < 4 * kPanel * 8; i += TPB)
      *reinterpret_cast<float4*>(to + (int64_t)i * 16) = *reinterpret_cast<const float4*>(smem + i * 16);
    __syncthreads();
  }
}

template <int T>
__global__ __launch_bounds__(Tile<T>::TPB, 2) void gradient_kernel(Gradient p) {
  constexpr int FA = Tile<T>::FA, FB = Tile<T>::FB, STAGE = Tile<T>::STAGE;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Tile<T> t;
  const int tiles_a = (int)((p.rows_a + T - 1) / T), tiles_b = (int)((p.rows_b + T - 1) / T), tiles = tiles_a * tiles_b;
  const int part = blockIdx.x / tiles;
  int ta, tb;
  mfma::tile_of_block(blockIdx.x % tiles, tiles, tiles_a, tiles_b, ta, tb);
  const int kblocks = (int)((p.k + kBlock - 1) / kBlock), panels = (kblocks + 7) / 8;
  const int64_t b_blocks = (int64_t)panels * 8;  // b was written in whole panels of k
  const int per = (panels + p.parts - 1) / p.parts, k0 = min(part * per * 8, kblocks), k1 = min(k0 + per * 8, kblocks);
  const char *a = t.panel(p.a, ta, kblocks), *b = t.panel(p.b, tb, b_blocks);
  const int64_t a0 = (int64_t)ta * T, b0 = (int64_t)tb * T;
  typename Tile<T>::Acc acc;
  clear<T>(acc);
  int shift[FB];
  const int* shifts = p.b_shift + b0;
#pragma unroll
  for (int j = 0; j < FB; ++j) shift[j] = k0 < k1 ? shifts[(int64_t)(k0 / 8) * p.b_shift_ld + t.b_of(j)] : 0;
  if (k0 < k1) request(a + k0 * kBlockBytes, b + k0 * kBlockBytes, smem, t);
  wait_loads();
  __syncthreads();
  for (int kb = k0; kb < k1; ++kb) {
    if ((kb & 7) == 0 && kb != k0) {  // the next 256 of k have scales of their own: the sums so far move to them (see most_shift_of_class)
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        const int now = shifts[(int64_t)(kb / 8) * p.b_shift_ld + t.b_of(j)];
        const float f = __builtin_ldexpf(1.f, now - shift[j]);
        shift[j] = now;
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[i][j][v] *= f;
      }
    }
    if (kb + 1 < k1) request(a + (kb + 1) * kBlockBytes, b + (kb + 1) * kBlockBytes, smem + ((kb + 1 - k0) & 1) * STAGE, t);
    multiply(smem + ((kb - k0) & 1) * STAGE, t, acc);
    wait_loads();
    __syncthreads();
  }
  const Mean c = mean_of(p.g, p.count);
  float* out = p.out + part * p.part_stride;
  const bool vec = p.vec;
#pragma unroll
  for (int j = 0; j < FB; ++j) {
    const int64_t bi = b0 + t.b_of(j);
    if (bi >= p.rows_b) continue;
    const bool skip = p.left_out && p.left_out[bi] < 0.f;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t ai = a0 + t.a_of(i, 4 * q);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __builtin_ldexpf((skip ? 0.f : acc[i][j][4 * q + e]) * c.m, c.e - shift[j] - shift_of(p.a_amax[min(ai + e, p.rows_a - 1)]));
        if (vec) {
          if (ai < p.rows_a) {
            float4* to = reinterpret_cast<float4*>(out + bi * p.ld + ai);
            float4 o = make_float4(y[0], y[1], y[2], y[3]);
            if (p.accumulate) {
              const float4 was = *to;
              o = make_float4(o.x + was.x, o.y + was.y, o.z + was.z, o.w + was.w);
            }
            *to = o;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (ai + e < p.rows_a) {
              float* to = out + (p.by_a ? (ai + e) * p.ld + bi : bi * p.ld + ai + e);
              *to = p.accumulate ? *to + y[e] : y[e];
            }
        }
      }
  }
}

template <int T, typename Kernel, typename Params>
int32_t launch(Kernel* kernel, const Params& p, int64_t groups, hipStream_t s) {
  constexpr int lds = 2 * Tile<T>::STAGE;
  ENDIA_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(Tile<T>::TPB), lds, s, p);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

// 256 x 256 tiles run at the higher rate, 128 x 128 ones (two to a CU, about three quarters of the rate) waste less of the last
// round and of ragged edges: whichever takes fewer rounds of the chip, in units of a quarter tile.
int64_t tiles_of(int64_t a, int64_t b, int T) { return ceil_div64(a, T) * ceil_div64(b, T); }

}  // namespace

int product_tile(int64_t a, int64_t b) {
  const int64_t cus = endia::ctx().cu_count;
  const int64_t big = ceil_div64(tiles_of(a, b, 256), cus) * 4 * 3, small = ceil_div64(tiles_of(a, b, 128), 2 * cus) * 2 * 4;
  return small < big ? 128 : 256;
}

int32_t logits_stats(const Logits& p, hipStream_t s) {
  return product_tile(p.cols, p.N) == 256 ? launch<256>(stats_kernel<256>, p, tiles_of(p.cols, p.N, 256), s)
                                          : launch<128>(stats_kernel<128>, p, tiles_of(p.cols, p.N, 128), s);
}
int32_t logits_dz(const Logits& p, hipStream_t s) { return launch<256>(dz_kernel, p, tiles_of(p.cols, p.N, 256), s); }
int32_t gradient(const Gradient& q, hipStream_t s) {
  Gradient p = q;
  p.vec = !p.by_a && p.ld % 4 == 0 && p.rows_a % 4 == 0 && p.part_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  return product_tile(p.rows_a, p.rows_b) == 256 ? launch<256>(gradient_kernel<256>, p, tiles_of(p.rows_a, p.rows_b, 256) * p.parts, s)
                                                 : launch<128>(gradient_kernel<128>, p, tiles_of(p.rows_a, p.rows_b, 128) * p.parts, s);
}

}  // namespace lce
