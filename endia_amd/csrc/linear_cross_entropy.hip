// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient, in pieces of the vocabulary: the
// logits z = x W [N, V] are never kept. The loss stands beside mse (endia/functional/loss_ops/mse_op.mojo:17-20).
//
//   lse_i = log sum_j exp z_ij        loss = (1 / n) sum over kept rows of (lse_i - z_{i, t_i}),  n = kept rows
//   dz_ij = (g / n) (exp(z_ij - lse_i) - [j = t_i]),   dx = dz W^T,   dW = x^T dz
//
// A row with a negative target is left out: it adds nothing to the loss or to a gradient, whatever x holds there.
// The forward pass walks the vocabulary once and keeps, per row, the running maximum and the running sum of exp(z - max);
// the backward pass forms each piece of z again, turns it into dz and multiplies it from both sides.
// Many rows: products of fp16 pairs (lce_products.hip), the statistics and the cotangents in the products' epilogues.
// Fewer rows: endia_hip_sgemm on pieces of fp32 logits.
#include "linear_cross_entropy.h"

using namespace endia;

namespace {

constexpr int TPB = 256;

struct Scratch {  // a pooled buffer for the time of one call (work on the one stream is ordered, so it can go back at once)
  void* p = nullptr;
  int64_t used = 0;
  int32_t get(int64_t bytes) { return endia_hip_malloc(bytes, &p); }
  int64_t want(int64_t bytes) {  // offset of a piece
    const int64_t at = used;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
  char* at(int64_t offset) const { return static_cast<char*>(p) + offset; }
  float* f(int64_t offset) const { return reinterpret_cast<float*>(at(offset)); }
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

// ---- many rows ------------------------------------------------------------------------------------------------
constexpr int64_t kManyRows = 512;

// the statistics of a piece's tiles join the running ones of each row
__global__ __launch_bounds__(TPB) void join_stats_kernel(const float* __restrict__ stats, int64_t tiles, int64_t N, float* __restrict__ m, float* __restrict__ l,
                                                         int first) {
  const int64_t n = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (n >= N) return;
  float top = first ? -INFINITY : m[n], sum = first ? 0.f : l[n];
  for (int64_t t = 0; t < tiles; ++t) {
    const float2 s = *reinterpret_cast<const float2*>(stats + (t * N + n) * 2);
    const float now = fmaxf(top, s.x);
    sum = sum * (top == now ? 1.f : expf(top - now)) + s.y * (s.x == now ? 1.f : expf(s.x - now));
    top = now;
  }
  m[n] = top;
  l[n] = sum;
}

__global__ __launch_bounds__(TPB) void add_parts_kernel(const float* __restrict__ part, int64_t n, int parts, float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (i >= n) return;
  float sum = part[i];
  for (int s = 1; s < parts; ++s) sum += part[s * n + i];
  out[i] = sum;
}

// classes per piece: panels of the weight's piece of at most 256 MiB, and (backward) at most 2^25 cotangents, 256 MiB as
// two sets of pairs; a multiple of 256
int64_t panel_columns(int64_t N, int64_t D, int64_t V, bool backward) {
  int64_t cols = (64ll << 20) / D;
  if (backward && cols > (32ll << 20) / N) cols = (32ll << 20) / N;
  cols = cols / lce::kPanel * lce::kPanel;
  if (cols < lce::kPanel) cols = lce::kPanel;
  return cols < V ? cols : V;
}

int32_t many_rows_fwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, const float* target,
                      float* loss, float* lse, hipStream_t s) {
  const int64_t piece = panel_columns(N, D, V, false), tiles = ceil_div64(piece, lce::kPanel);
  Scratch w;
  const int64_t xp = w.want(lce::panel_bytes(N, D)), wp = w.want(lce::panel_bytes(piece, D)), xa = w.want(4 * N), wa = w.want(4 * piece),
                st = w.want(8 * tiles * N), run = w.want(12 * N);
  int32_t rc = w.get(w.used);
  if (rc || (rc = lce::pack(x, ldx, false, N, D, target, w.at(xp), w.f(xa), s))) return rc;
  float *m = w.f(run), *l = m + N, *zt = l + N;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    if ((rc = lce::pack(W + (transW ? v0 * ldw : v0), ldw, !transW, cols, D, nullptr, w.at(wp), w.f(wa), s))) return rc;
    lce::Logits a = {};
    a.w = w.at(wp); a.x = w.at(xp); a.w_amax = w.f(wa); a.x_amax = w.f(xa); a.target = target;
    a.N = N; a.cols = cols; a.v0 = v0; a.D = D;
    a.stats = w.f(st); a.zt = zt;
    if ((rc = lce::logits_stats(a, s))) return rc;
    hipLaunchKernelGGL(join_stats_kernel, dim3((unsigned)ceil_div64(N, TPB)), dim3(TPB), 0, s, w.f(st), ceil_div64(cols, lce::kPanel), N, m, l,
                       v0 == 0 ? 1 : 0);
  }
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(TPB), 0, s, N, V, target, m, l, zt, lse, loss);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t many_rows_bwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, const float* target,
                      const float* lse, const float* g, float* dx, float* dW, hipStream_t s) {
  const int64_t piece = panel_columns(N, D, V, true), rows = ceil_div64(N, lce::kPanel) * lce::kPanel, ptiles = ceil_div64(piece, lce::kPanel);
  const int64_t dx_tiles = rows / lce::kPanel * ceil_div64(D, lce::kPanel);
  int parts = (int)ceil_div64(ctx().cu_count, dx_tiles);  // x's gradient has few tiles and a long k: cut k until the chip is full
  if (parts > ptiles) parts = (int)ptiles;
  if (parts > 16) parts = 16;
  Scratch w;
  const int64_t xp = w.want(lce::panel_bytes(N, D)), wp = w.want(lce::panel_bytes(piece, D)), xa = w.want(4 * N), wa = w.want(4 * piece),
                xt = w.want(dW ? lce::panel_bytes(D, N) : 0), xta = w.want(4 * D), wt = w.want(dx ? lce::panel_bytes(D, piece) : 0), wta = w.want(4 * D),
                p = w.want(dx ? rows * ptiles * lce::kPanel * 4 : 0), pt = w.want(dW ? rows * ptiles * lce::kPanel * 4 : 0),
                ps = w.want(4 * ptiles * rows), pts = w.want(4 * rows / lce::kPanel * ptiles * lce::kPanel),
                dxp = w.want(dx && parts > 1 ? 4 * parts * N * D : 0);
  int32_t rc = w.get(w.used);
  if (rc || (rc = lce::pack(x, ldx, false, N, D, target, w.at(xp), w.f(xa), s))) return rc;
  if (dW && (rc = lce::pack(x, ldx, true, D, N, target, w.at(xt), w.f(xta), s))) return rc;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    const float* Wv = W + (transW ? v0 * ldw : v0);
    if ((rc = lce::pack(Wv, ldw, !transW, cols, D, nullptr, w.at(wp), w.f(wa), s))) return rc;
    lce::Logits a = {};
    a.w = w.at(wp); a.x = w.at(xp); a.w_amax = w.f(wa); a.x_amax = w.f(xa); a.target = target;
    a.N = N; a.cols = cols; a.v0 = v0; a.D = D;
    a.lse = lse;
    a.p = dx ? w.at(p) : nullptr;
    a.pt = dW ? w.at(pt) : nullptr;
    a.p_shift = reinterpret_cast<int*>(w.at(ps));
    a.pt_shift = reinterpret_cast<int*>(w.at(pts));
    if ((rc = lce::logits_dz(a, s))) return rc;
    lce::Gradient q = {};
    q.g = g;
    q.count = lse + N;
    if (dx) {
      if ((rc = lce::pack(Wv, ldw, transW, D, cols, nullptr, w.at(wt), w.f(wta), s))) return rc;
      q.a = w.at(wt); q.b = a.p; q.a_amax = w.f(wta); q.b_shift = a.p_shift; q.b_shift_ld = rows;
      q.rows_a = D; q.rows_b = N; q.k = cols;
      q.out = parts > 1 ? w.f(dxp) : dx;
      q.ld = D; q.by_a = 0; q.accumulate = v0 ? 1 : 0; q.parts = parts; q.part_stride = N * D;
      if ((rc = lce::gradient(q, s))) return rc;
    }
    if (dW) {
      q.a = w.at(xt); q.b = a.pt; q.a_amax = w.f(xta); q.b_shift = a.pt_shift; q.b_shift_ld = ceil_div64(cols, lce::kPanel) * lce::kPanel;
      q.rows_a = D; q.rows_b = cols; q.k = N;
      q.out = transW ? dW + v0 * D : dW + v0;
      q.ld = transW ? D : V;
      q.by_a = !transW; q.accumulate = 0; q.parts = 1; q.part_stride = 0;
      if ((rc = lce::gradient(q, s))) return rc;
    }
  }
  if (dx && parts > 1) {
    hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)ceil_div64(N * D, TPB)), dim3(TPB), 0, s, w.f(dxp), N * D, parts, dx);
    ENDIA_LAUNCH_CHECK();
  }
  return ENDIA_HIP_OK;
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
  if (N >= kManyRows) return many_rows_fwd(N, D, V, x, ldx, transW, W, ldw, target, loss, lse, s);
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
  if (N >= kManyRows) return many_rows_bwd(N, D, V, x, ldx, transW, W, ldw, target, lse, g, dx, dW, s);
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
