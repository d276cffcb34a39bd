// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient, in pieces of the vocabulary: the
// logits z = x W [N, V] are never kept. The loss stands beside mse (endia/functional/loss_ops/mse_op.mojo:17-20).
//
//   lse_i = log sum_j exp z_ij        loss = (1 / n) sum over kept rows of (lse_i - z_{i, t_i}),  n = kept rows
//   dz_ij = (g / n) (exp(z_ij - lse_i) - [j = t_i]),   dx = dz W^T,   dW = x^T dz
//
// A row with a negative target is left out: it adds nothing to the loss or to a gradient, whatever x holds there.
// The forward pass walks the vocabulary once and keeps, per row, the running maximum and the running sum of exp(z - max);
// the backward pass forms each piece of z again, turns it into dz and multiplies it from both sides.
#include "common.h"

using namespace endia;

namespace {

constexpr int TPB = 256;

struct Scratch {  // a pooled buffer for the time of one call (work on the one stream is ordered, so it can go back at once)
  void* p = nullptr;
  int32_t get(int64_t bytes) { return endia_hip_malloc(bytes, &p); }
  ~Scratch() {
    if (p) endia_hip_free(p);
  }
  float* f() const { return static_cast<float*>(p); }
};

__device__ __forceinline__ float block_reduce(float v, float* red, bool maximum) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = maximum ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < TPB / 64; ++w) v = maximum ? fmaxf(v, red[w]) : v + red[w];
  return v;
}

__device__ __forceinline__ bool left_out(float t) { return t < 0.f; }

// One group per row: the piece's columns [v0, v0 + cols) of the logits meet the row's running maximum m, sum l and the
// logit of its target.
__global__ __launch_bounds__(TPB) void row_stats_kernel(const float* __restrict__ z, int64_t cols, int64_t v0, const float* __restrict__ target,
                                                        float* __restrict__ m, float* __restrict__ l, float* __restrict__ zt, int first) {
  __shared__ float red[TPB / 64];
  const int64_t row = blockIdx.x;
  const float* zr = z + row * cols;
  float top = -INFINITY;
  for (int64_t c = threadIdx.x; c < cols; c += TPB) top = fmaxf(top, zr[c]);
  top = block_reduce(top, red, true);
  const float before = first ? -INFINITY : m[row];
  const float now = fmaxf(before, top);
  float sum = 0.f;
  for (int64_t c = threadIdx.x; c < cols; c += TPB) sum += expf(zr[c] - now);
  sum = block_reduce(sum, red, false);
  if (threadIdx.x == 0) {
    l[row] = (first ? 0.f : l[row] * expf(before - now)) + sum;
    m[row] = now;
    const float t = target[row];
    if (t >= (float)v0 && t < (float)(v0 + cols)) zt[row] = zr[(int64_t)t - v0];
  }
}

// lse per row and the mean loss. A target that is no class (NaN, or V and above) makes the loss NaN.
__global__ __launch_bounds__(TPB) void loss_kernel(int64_t N, int64_t V, const float* __restrict__ target, const float* __restrict__ m,
                                                   const float* __restrict__ l, const float* __restrict__ zt, float* __restrict__ lse,
                                                   float* __restrict__ loss) {
  __shared__ double red[TPB];
  __shared__ int cnt[TPB];
  double sum = 0.0;
  int kept = 0;
  for (int64_t i = threadIdx.x; i < N; i += TPB) {
    const float t = target[i];
    float e = m[i] + logf(l[i]);
    if (!left_out(t)) {
      if (!(t < (float)V)) e = NAN;
      else sum += (double)e - (double)zt[i];
      if (!(t < (float)V)) sum += (double)NAN;
      ++kept;
    }
    lse[i] = e;
  }
  red[threadIdx.x] = sum;
  cnt[threadIdx.x] = kept;
  __syncthreads();
  for (int s = TPB / 2; s; s >>= 1) {
    if (threadIdx.x < s) {
      red[threadIdx.x] += red[threadIdx.x + s];
      cnt[threadIdx.x] += cnt[threadIdx.x + s];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    lse[N] = (float)cnt[0];
    *loss = cnt[0] ? (float)(red[0] / cnt[0]) : 0.f;
  }
}

// logits -> cotangents, in place
__global__ __launch_bounds__(TPB) void dz_kernel(float* __restrict__ z, int64_t cols, int64_t v0, int64_t N, const float* __restrict__ target,
                                                 const float* __restrict__ lse, const float* __restrict__ g) {
  const int64_t row = blockIdx.x;
  float* zr = z + row * cols;
  const float t = target[row];
  const float kept = lse[N];
  if (left_out(t)) {
    for (int64_t c = threadIdx.x; c < cols; c += TPB) zr[c] = 0.f;
    return;
  }
  const float scale = g[0] / kept, e = lse[row];
  const int64_t at = t < (float)(v0 + cols) && t >= (float)v0 ? (int64_t)t - v0 : -1;
  for (int64_t c = threadIdx.x; c < cols; c += TPB) zr[c] = (expf(zr[c] - e) - (c == at ? 1.f : 0.f)) * scale;
}

// x with zeros in the rows that are left out, contiguous
__global__ __launch_bounds__(TPB) void kept_rows_kernel(const float* __restrict__ x, int64_t ldx, int64_t D, const float* __restrict__ target,
                                                        float* __restrict__ out) {
  const int64_t row = blockIdx.x;
  const bool skip = left_out(target[row]);
  for (int64_t d = threadIdx.x; d < D; d += TPB) out[row * D + d] = skip ? 0.f : x[row * ldx + d];
}

int64_t piece_columns(int64_t N, int64_t V) {
  int64_t cols = (64ll << 20) / N / 256 * 256;  // 256 MiB of logits at most
  if (cols < 256) cols = 256;
  return cols < V ? cols : V;
}

int32_t check(const char* who, int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw,
              const float* target, const float* lse) {
  ENDIA_CHECK_ARG(N > 0 && D > 0 && V > 0, "%s: sizes must be positive (N = %lld, D = %lld, V = %lld)", who, (long long)N, (long long)D,
                  (long long)V);
  ENDIA_CHECK_ARG(N < (1ll << 24) && V <= (1ll << 24) && D < (1ll << 24),
                  "%s: more than 2^24 rows, columns or classes (class numbers and the row count are held in fp32)", who);
  ENDIA_CHECK_ARG(x && W && target && lse, "%s: null pointer", who);
  ENDIA_CHECK_ARG(transW == 0 || transW == 1, "%s: transW must be 0 or 1", who);
  ENDIA_CHECK_ARG(ldx >= D && ldw >= (transW ? D : V), "%s: leading dimension too small", who);
  return ENDIA_HIP_OK;
}

int32_t logits_piece(int64_t N, int64_t D, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, int64_t v0, int64_t cols,
                     float* z) {
  return endia_hip_sgemm(0, transW, N, cols, D, x, ldx, W + (transW ? v0 * ldw : v0), ldw, z, cols, 1, 0, 0, 0, ENDIA_EPI_NONE,
                         ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr);
}

}  // namespace

extern "C" {

int32_t endia_hip_linear_cross_entropy_fwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W,
                                           int64_t ldw, const float* target, float* loss, float* lse) {
  int32_t rc = check("endia_hip_linear_cross_entropy_fwd", N, D, V, x, ldx, transW, W, ldw, target, lse);
  if (rc) return rc;
  ENDIA_CHECK_ARG(loss, "endia_hip_linear_cross_entropy_fwd: null pointer");
  ENDIA_REQUIRE_INIT();
  hipStream_t s = ctx().stream;
  const int64_t piece = piece_columns(N, V);
  Scratch z, stats;
  if ((rc = z.get(4 * N * piece)) || (rc = stats.get(12 * N))) return rc;
  float *m = stats.f(), *l = m + N, *zt = l + N;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    if ((rc = logits_piece(N, D, x, ldx, transW, W, ldw, v0, cols, z.f()))) return rc;
    hipLaunchKernelGGL(row_stats_kernel, dim3((unsigned)N), dim3(TPB), 0, s, z.f(), cols, v0, target, m, l, zt, v0 == 0 ? 1 : 0);
    ENDIA_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(TPB), 0, s, N, V, target, m, l, zt, lse, loss);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t endia_hip_linear_cross_entropy_bwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W,
                                           int64_t ldw, const float* target, const float* lse, const float* g, float* dx, float* dW) {
  int32_t rc = check("endia_hip_linear_cross_entropy_bwd", N, D, V, x, ldx, transW, W, ldw, target, lse);
  if (rc) return rc;
  ENDIA_CHECK_ARG(g, "endia_hip_linear_cross_entropy_bwd: null pointer");
  ENDIA_CHECK_ARG(dx || dW, "endia_hip_linear_cross_entropy_bwd: nothing to compute");
  ENDIA_REQUIRE_INIT();
  hipStream_t s = ctx().stream;
  const int64_t piece = piece_columns(N, V);
  Scratch z, xk;
  if ((rc = z.get(4 * N * piece))) return rc;
  if (dW) {
    if ((rc = xk.get(4 * N * D))) return rc;
    hipLaunchKernelGGL(kept_rows_kernel, dim3((unsigned)N), dim3(TPB), 0, s, x, ldx, D, target, xk.f());
    ENDIA_LAUNCH_CHECK();
  }
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    if ((rc = logits_piece(N, D, x, ldx, transW, W, ldw, v0, cols, z.f()))) return rc;
    hipLaunchKernelGGL(dz_kernel, dim3((unsigned)N), dim3(TPB), 0, s, z.f(), cols, v0, N, target, lse, g);
    ENDIA_LAUNCH_CHECK();
    if (dx && (rc = endia_hip_sgemm(0, !transW, N, D, cols, z.f(), cols, W + (transW ? v0 * ldw : v0), ldw, dx, D, 1, 0, 0, 0,
                                    v0 ? ENDIA_EPI_NONE | ENDIA_GEMM_ACCUMULATE : ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
      return rc;
    if (dW) {
      if (transW)
        rc = endia_hip_sgemm(1, 0, cols, D, N, z.f(), cols, xk.f(), D, dW + v0 * D, D, 1, 0, 0, 0, ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr,
                             nullptr, nullptr);
      else
        rc = endia_hip_sgemm(1, 0, D, cols, N, xk.f(), D, z.f(), cols, dW + v0, V, 1, 0, 0, 0, ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr,
                             nullptr, nullptr);
      if (rc) return rc;
    }
  }
  return ENDIA_HIP_OK;
}

}  // extern "C"
