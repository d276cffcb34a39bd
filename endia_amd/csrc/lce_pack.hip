// Operands of the linear cross entropy as panels of fp16 pairs (linear_cross_entropy.h), scaled by one power of two per row.
// Bound: HBM; 4 bytes read (8 where the scale takes a walk of its own and the source is larger than the last-level cache) and 4
// written per element. Measured: 32768 classes x 2048 stored by class (0.27 GB read, as much written) about 120 us =
// 4.4 TB/s; stored by width, transposed through LDS, 2.9 TB/s (74 us on average over the 41 blocks of a step over 131072 x 4096).
#include "linear_cross_entropy.h"

namespace lce {

namespace {

using namespace pairs;
constexpr int TPB = 256;
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void store_chunk(char* line, int row, int chunk, const float (&v)[8], int shift) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = scaled(v[e], shift);
  half8 hi, lo;
  split8(y, hi, lo);
  *reinterpret_cast<half8*>(line + ((chunk ^ (row & 7)) << 4)) = hi;
  *reinterpret_cast<half8*>(line + (((4 + chunk) ^ (row & 7)) << 4)) = lo;
}

// Source rows contiguous along k: one wave per row, the row twice (the second time from cache).
__global__ __launch_bounds__(TPB) void pack_rows_kernel(const float* __restrict__ x, int64_t ld, int64_t rows, int64_t k, const float* __restrict__ left_out,
                                                        char* __restrict__ panels, float* __restrict__ amax_out, int known) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const bool skip = left_out && left_out[row] < 0.f;
  const float* r = x + row * ld;
  float amax = 0.f;
  auto load8 = [&](int64_t k0, float (&v)[8]) {
    if (k0 + 8 <= k) {  // (global memory gives 16 bytes from any multiple of 4)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4u f = *reinterpret_cast<const float4u*>(r + k0 + 4 * j);
        v[4 * j] = f[0]; v[4 * j + 1] = f[1]; v[4 * j + 2] = f[2]; v[4 * j + 3] = f[3];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k0 + e < k ? r[k0 + e] : 0.f;
    }
  };
  if (!skip && !known)
    for (int64_t k0 = lane * 8; k0 < k; k0 += 512) {
      float v[8];
      load8(k0, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[e]));
    }
#pragma unroll
  for (int o = 32; o; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
  if (known) amax = amax_out[row];
  else if (lane == 0) amax_out[row] = amax;
  if (!panels) return;
  const int shift = shift_of(amax);
  const int64_t kblocks = (k + kBlock - 1) / kBlock;
  for (int64_t k0 = lane * 8; k0 < kblocks * kBlock; k0 += 512) {
    float v[8] = {};
    if (!skip) load8(k0, v);
    store_chunk(line_at(panels, row, k0 / kBlock, kblocks), (int)(row & 7), (int)(k0 % kBlock / 8), v, shift);
  }
}

// Source [k][row]: the largest of each column first (a maximum does not depend on the order, so atomics will do) ...
__global__ __launch_bounds__(TPB) void zero_kernel(float* __restrict__ x, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (i < n) x[i] = 0.f;
}

__global__ __launch_bounds__(TPB) void col_amax_kernel(const float* __restrict__ x, int64_t ld, int64_t rows, int64_t k, int64_t per,
                                                       const float* __restrict__ left_out, float* __restrict__ amax) {
  const int64_t r = (int64_t)blockIdx.x * TPB + threadIdx.x, k0 = (int64_t)blockIdx.y * per, k1 = k0 + per < k ? k0 + per : k;
  if (r >= rows) return;
  float m = 0.f;
#pragma unroll 8
  for (int64_t i = k0; i < k1; ++i) {
    const float v = finite_abs(x[i * ld + r]);
    m = fmaxf(m, left_out && left_out[i] < 0.f ? 0.f : v);
  }
  atomicMax(reinterpret_cast<unsigned*>(amax) + r, __float_as_uint(m));
}

// ... then blocks of 32 k x 128 rows through LDS.
__global__ __launch_bounds__(TPB) void pack_cols_kernel(const float* __restrict__ x, int64_t ld, int64_t rows, int64_t k, const float* __restrict__ left_out,
                                                        char* __restrict__ panels, const float* __restrict__ amax) {
  __shared__ float t[kBlock][129];
  const int tid = threadIdx.x;
  const int64_t row_groups = (rows + 127) / 128, r0 = blockIdx.x % row_groups * 128, kb = blockIdx.x / row_groups, kblocks = (k + kBlock - 1) / kBlock;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int kk = i * 2 + (tid >> 7), rr = tid & 127;
    const int64_t kg = kb * kBlock + kk, r = r0 + rr;
    const bool in = kg < k && r < rows && !(left_out && left_out[kg] < 0.f);
    t[kk][rr] = in ? x[kg * ld + r] : 0.f;
  }
  __syncthreads();
  const int rr = tid & 127;
  const int64_t row = r0 + rr;
  if (row >= rows) return;
  const int shift = shift_of(amax[row]);
  char* line = line_at(panels, row, kb, kblocks);
#pragma unroll
  for (int c = tid >> 7; c < 4; c += 2) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[c * 8 + e][rr];
    store_chunk(line, (int)(row & 7), c, v, shift);
  }
}

}  // namespace

int32_t row_amax(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, float* amax, hipStream_t s) {
  if (!transposed) return pack(x, ld, false, rows, k, left_out, nullptr, amax, false, s);
  hipLaunchKernelGGL(zero_kernel, dim3((unsigned)ceil_div64(rows, TPB)), dim3(TPB), 0, s, amax, rows);
  const int64_t groups = ceil_div64(rows, TPB);
  int64_t cuts = ceil_div64(4096, groups);
  if (cuts > ceil_div64(k, 16)) cuts = ceil_div64(k, 16);
  if (cuts > 65535) cuts = 65535;
  const int64_t per = ceil_div64(k, cuts);
  hipLaunchKernelGGL(col_amax_kernel, dim3((unsigned)groups, (unsigned)ceil_div64(k, per)), dim3(TPB), 0, s, x, ld, rows, k, per, left_out, amax);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t pack(const float* x, int64_t ld, bool transposed, int64_t rows, int64_t k, const float* left_out, char* panels, float* amax, bool known,
             hipStream_t s) {
  if (!transposed) {
    hipLaunchKernelGGL(pack_rows_kernel, dim3((unsigned)ceil_div64(rows, 4)), dim3(TPB), 0, s, x, ld, rows, k, left_out, panels, amax, known ? 1 : 0);
    ENDIA_LAUNCH_CHECK();
    return ENDIA_HIP_OK;
  }
  int32_t rc = known ? ENDIA_HIP_OK : row_amax(x, ld, true, rows, k, left_out, amax, s);
  if (rc) return rc;
  hipLaunchKernelGGL(pack_cols_kernel, dim3((unsigned)(ceil_div64(rows, 128) * ceil_div64(k, kBlock))), dim3(TPB), 0, s, x, ld, rows, k, left_out,
                     panels, amax);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace lce
