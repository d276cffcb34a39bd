// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient, in pieces of the vocabulary: the
// logits z = x W [N, V] are never kept. The loss stands beside mse (endia/functional/loss_ops/mse_op.mojo:17-20).
//
//   lse_i = log sum_j exp z_ij        loss = (1 / n) sum over kept rows of (lse_i - z_{i, t_i}),  n = kept rows
//   dz_ij = (g / n) (exp(z_ij - lse_i) - [j = t_i]),   dx = dz W^T,   dW = x^T dz
//
// A row with a negative target is left out: it adds nothing to the loss or to a gradient, whatever x holds there.
// The forward pass walks the vocabulary once and keeps, per row, the running maximum and the running sum of exp(z - max);
// the backward pass forms each piece of z again, turns it into dz and multiplies it from both sides.
// Many rows: products of fp16 pairs (lce_pack.hip, lce_products.hip), the statistics and the cotangents in the products'
// epilogues. Fewer rows: the weight streamed as it lies (lce_direct.hip).
#include "linear_cross_entropy.h"

using namespace endia;

namespace {

constexpr int TPB = 256;

__device__ __forceinline__ bool left_out(float t) { return t < 0.f; }

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
    if ((int)threadIdx.x < s) {
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

// the statistics of a piece's tiles join the running ones of each row; one wave per row
__global__ __launch_bounds__(TPB) void join_stats_kernel(const float* __restrict__ stats, int64_t tiles, int64_t N, float* __restrict__ m, float* __restrict__ l,
                                                         int first) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  float top = first ? -INFINITY : m[n];
  const float before = top;
  for (int64_t t = lane; t < tiles; t += 64) top = fmaxf(top, stats[(t * N + n) * 2]);
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  float sum = 0.f;
  for (int64_t t = lane; t < tiles; t += 64) {
    const float2 s = *reinterpret_cast<const float2*>(stats + (t * N + n) * 2);
    sum += s.x == top ? s.y : s.y * expf(s.x - top);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) {
    if (!first) sum += l[n] * (before == top ? 1.f : expf(before - top));
    m[n] = top;
    l[n] = sum;
  }
}

// out[r * ld + c] = the sum of the parts' [rows, cols]: a work-group takes 64 elements and the parts in four interleaved runs, which
// meet in order
__global__ __launch_bounds__(TPB) void add_parts_kernel(const float* __restrict__ part, int64_t rows, int64_t cols, int parts, float* __restrict__ out, int64_t ld) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane, n = rows * cols;
  float sum = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int s = run; s < parts; s += 4) sum += part[s * n + i];
  }
  red[run][lane] = sum;
  __syncthreads();
  if (run == 0 && i < n) out[i / cols * ld + i % cols] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

int32_t join_stats(const float* stats, int64_t tiles, int64_t N, float* m, float* l, bool first, hipStream_t s) {
  hipLaunchKernelGGL(join_stats_kernel, dim3((unsigned)ceil_div64(N, 4)), dim3(TPB), 0, s, stats, tiles, N, m, l, first ? 1 : 0);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t add_parts(const float* part, int64_t rows, int64_t cols, int parts, float* out, int64_t ld, hipStream_t s) {
  hipLaunchKernelGGL(add_parts_kernel, dim3((unsigned)ceil_div64(rows * cols, 64)), dim3(TPB), 0, s, part, rows, cols, parts, out, ld);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

// Work-groups for a product whose tiles alone do not fill the chip: its long axis of `steps` is cut into that many parts.
int cut(int64_t tiles, int64_t want, int64_t steps, int64_t most) {
  int64_t p = ceil_div64(want, tiles);
  p = p < steps ? p : steps;
  p = p < most ? p : most;
  return (int)(p < 1 ? 1 : p);
}

// ---- few rows -------------------------------------------------------------------------------------------------
// From here on the weight is brought into panels. Both sides, a step with the weight by class and by width: 417 rows, 79335 classes x
// 1668 2.66 and 2.85 ms streamed, 3.22 and 3.61 in panels; 512 rows, 65536 x 2048 2.49 and 2.67, 2.68 and 2.93; 1000 rows, 30000 x 4096 4.33
// and 4.65, 3.81 and 4.05.
constexpr int64_t kManyRows = 512;

int32_t few_rows_fwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, const float* target,
                     float* loss, float* lse, hipStream_t s) {
  const int64_t tiles = ceil_div64(V, lce::direct_rows(N, V));
  const bool scaled = N > lce::kTripleRows;
  float* wa = lse + N + 1;
  Scratch w;
  const int64_t xp = w.want(lce::plane_bytes(N, D)), st = w.want(8 * tiles * N), run = w.want(12 * N), xa = w.want(4 * N);
  int32_t rc = w.get();
  if (rc) return rc;
  if (scaled && ((rc = lce::row_amax(W, ldw, !transW, V, D, nullptr, wa, s)) || (rc = lce::row_amax(x, ldx, false, N, D, target, w.at<float>(xa), s)))) return rc;
  if ((rc = lce::planes(x, ldx, false, N, D, target, scaled ? w.at<float>(xa) : nullptr, w.at<char>(xp), s))) return rc;
  float *m = w.at<float>(run), *l = m + N, *zt = l + N;
  lce::Direct a = {};
  a.a = W; a.lda = ldw; a.rows = V; a.k = D;
  a.planes = w.at<char>(xp); a.N = N; a.parts = 1; a.target = target;
  a.a_amax = wa; a.x_amax = w.at<float>(xa);
  a.stats = w.at<float>(st); a.zt = zt;
  if ((rc = lce::direct_stats(a, transW, s)) || (rc = join_stats(w.at<float>(st), tiles, N, m, l, true, s))) return rc;
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(TPB), 0, s, N, V, target, m, l, zt, lse, loss);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t few_rows_bwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, const float* target,
                     const float* lse, const float* g, float* dx, float* dW, hipStream_t s) {
  int64_t piece = (24ll << 20) / N / 128 * 128;  // cotangents of a piece: 4 + 6 bytes each, 240 MiB
  if (piece > V) piece = V;
  const int64_t groups = ceil_div64(D, 128) * ceil_div64(N, N <= 32 ? 32 : N <= 64 ? 64 : 128);
  const bool scaled = N > lce::kTripleRows;
  const int parts = cut(groups, 2 * ctx().cu_count, ceil_div64(piece, 256), 256);
  Scratch w;
  const int64_t xp = w.want(lce::plane_bytes(N, D)), xt = w.want(dW ? lce::plane_bytes(D, N) : 0), dz = w.want(dW ? 4 * N * piece : 0),
                zp = w.want(dx ? lce::plane_bytes(N, piece) : 0), dxp = w.want(dx && parts > 1 ? 4 * parts * N * D : 0), xa = w.want(4 * N),
                xta = w.want(4 * D);
  int32_t rc = w.get();
  if (rc) return rc;
  if (scaled && ((rc = lce::row_amax(x, ldx, false, N, D, target, w.at<float>(xa), s)) ||
                 (dW && (rc = lce::row_amax(x, ldx, true, D, N, target, w.at<float>(xta), s)))))
    return rc;
  if ((rc = lce::planes(x, ldx, false, N, D, target, scaled ? w.at<float>(xa) : nullptr, w.at<char>(xp), s))) return rc;
  if (dW && (rc = lce::planes(x, ldx, true, D, N, target, scaled ? w.at<float>(xta) : nullptr, w.at<char>(xt), s))) return rc;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    lce::Direct a = {};
    a.a = W + (transW ? v0 * ldw : v0); a.lda = ldw; a.rows = cols; a.k = D;
    a.planes = w.at<char>(xp); a.N = N; a.v0 = v0; a.parts = 1; a.target = target; a.lse = lse;
    a.a_amax = lse + N + 1 + v0; a.x_amax = w.at<float>(xa);
    a.dz = dW ? w.at<float>(dz) : nullptr;
    a.dz_ld = cols;
    a.dz_planes = dx ? w.at<char>(zp) : nullptr;
    a.g = g; a.count = lse + N;
    if ((rc = lce::direct_dz(a, transW, s))) return rc;
    if (dx) {
      a.rows = D; a.k = cols;
      a.planes = w.at<char>(zp);
      a.parts = parts;
      a.out = parts > 1 ? w.at<float>(dxp) : dx;
      a.accumulate = v0 ? 1 : 0;
      if ((rc = lce::direct_dx(a, !transW, s))) return rc;
    }
    if (dW) {
      lce::Outer o = {};
      o.planes = w.at<char>(xt); o.x_amax = scaled ? w.at<float>(xta) : nullptr; o.dz = w.at<float>(dz); o.dz_ld = cols; o.N = N; o.D = D; o.cols = cols;
      o.out = transW ? dW + v0 * D : dW + v0;
      o.ld = transW ? D : V;
      o.g = g; o.count = lse + N;
      if ((rc = lce::direct_dw(o, !transW, s))) return rc;
    }
  }
  return dx && parts > 1 ? add_parts(w.at<float>(dxp), N, D, parts, dx, D, s) : ENDIA_HIP_OK;
}

// ---- many rows ------------------------------------------------------------------------------------------------
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
  const int64_t piece = panel_columns(N, D, V, false), tiles = ceil_div64(piece, 128);
  Scratch w;
  const int64_t xp = w.want(lce::panel_bytes(N, D)), wp = w.want(lce::panel_bytes(piece, D)), xa = w.want(4 * N),
                st = w.want(8 * tiles * N), run = w.want(12 * N);
  int32_t rc = w.get();
  if (rc || (rc = lce::pack(x, ldx, false, N, D, target, w.at<char>(xp), w.at<float>(xa), false, s))) return rc;
  float *m = w.at<float>(run), *l = m + N, *zt = l + N;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    if ((rc = lce::pack(W + (transW ? v0 * ldw : v0), ldw, !transW, cols, D, nullptr, w.at<char>(wp), lse + N + 1 + v0, false, s))) return rc;
    lce::Logits a = {};
    a.w = w.at<char>(wp); a.x = w.at<char>(xp); a.w_amax = lse + N + 1 + v0; a.x_amax = w.at<float>(xa); a.target = target;
    a.N = N; a.cols = cols; a.v0 = v0; a.D = D;
    a.stats = w.at<float>(st); a.zt = zt;
    if ((rc = lce::logits_stats(a, s))) return rc;
    if ((rc = join_stats(w.at<float>(st), ceil_div64(cols, lce::product_tile(cols, N)), N, m, l, v0 == 0, s))) return rc;
  }
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(TPB), 0, s, N, V, target, m, l, zt, lse, loss);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t many_rows_bwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W, int64_t ldw, const float* target,
                      const float* lse, const float* g, float* dx, float* dW, hipStream_t s) {
  const int64_t piece = panel_columns(N, D, V, true), rows = ceil_div64(N, lce::kPanel) * lce::kPanel, ptiles = ceil_div64(piece, lce::kPanel);
  // a gradient of few tiles and a long k: k is cut until the chip is full
  auto parts_of = [&](int64_t a, int64_t b, int64_t panels) {
    const int64_t T = lce::product_tile(a, b);
    return cut(ceil_div64(a, T) * ceil_div64(b, T), T == 256 ? ctx().cu_count : 2 * ctx().cu_count, panels, 16);
  };
  const int parts = parts_of(D, N, ptiles), w_parts = parts_of(D, piece, rows / lce::kPanel);
  Scratch w;
  const int64_t xp = w.want(lce::panel_bytes(N, D)), wp = w.want(lce::panel_bytes(piece, D)), xa = w.want(4 * N),
                xt = w.want(dW ? lce::panel_bytes(D, N) : 0), xta = w.want(4 * D), wt = w.want(dx ? lce::panel_bytes(D, piece) : 0), wta = w.want(4 * D),
                p = w.want(dx ? rows * ptiles * lce::kPanel * 4 : 0), pt = w.want(dW ? rows * ptiles * lce::kPanel * 4 : 0),
                ps = w.want(4 * ptiles * rows), pts = w.want(4 * rows / lce::kPanel * ptiles * lce::kPanel),
                dxp = w.want(dx && parts > 1 ? 4 * parts * N * D : 0), dwp = w.want(dW && w_parts > 1 ? 4 * w_parts * piece * D : 0);
  int32_t rc = w.get();
  if (rc || (rc = lce::pack(x, ldx, false, N, D, target, w.at<char>(xp), w.at<float>(xa), false, s))) return rc;
  if (dW && (rc = lce::pack(x, ldx, true, D, N, target, w.at<char>(xt), w.at<float>(xta), false, s))) return rc;
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t cols = V - v0 < piece ? V - v0 : piece;
    const float* Wv = W + (transW ? v0 * ldw : v0);
    if ((rc = lce::pack(Wv, ldw, !transW, cols, D, nullptr, w.at<char>(wp), const_cast<float*>(lse) + N + 1 + v0, true, s))) return rc;
    lce::Logits a = {};
    a.w = w.at<char>(wp); a.x = w.at<char>(xp); a.w_amax = lse + N + 1 + v0; a.x_amax = w.at<float>(xa); a.target = target;
    a.N = N; a.cols = cols; a.v0 = v0; a.D = D;
    a.lse = lse;
    a.p = dx ? w.at<char>(p) : nullptr;
    a.pt = dW ? w.at<char>(pt) : nullptr;
    a.p_shift = w.at<int>(ps);
    a.pt_shift = w.at<int>(pts);
    if ((rc = lce::logits_dz(a, s))) return rc;
    lce::Gradient q = {};
    q.g = g;
    q.count = lse + N;
    if (dx) {
      if ((rc = lce::pack(Wv, ldw, transW, D, cols, nullptr, w.at<char>(wt), w.at<float>(wta), false, s))) return rc;
      q.a = w.at<char>(wt); q.b = a.p; q.a_amax = w.at<float>(wta); q.b_shift = a.p_shift; q.b_shift_ld = rows;
      q.rows_a = D; q.rows_b = N; q.k = cols;
      q.out = parts > 1 ? w.at<float>(dxp) : dx;
      q.ld = D; q.by_a = 0; q.accumulate = v0 ? 1 : 0; q.parts = parts; q.part_stride = N * D;
      q.left_out = target;
      if ((rc = lce::gradient(q, s))) return rc;
      q.left_out = nullptr;
    }
    if (dW) {
      q.a = w.at<char>(xt); q.b = a.pt; q.a_amax = w.at<float>(xta); q.b_shift = a.pt_shift; q.b_shift_ld = ceil_div64(cols, lce::kPanel) * lce::kPanel;
      q.rows_a = D; q.rows_b = cols; q.k = N;
      q.out = transW ? dW + v0 * D : dW + v0;
      q.ld = transW ? D : V;
      q.by_a = !transW; q.accumulate = 0; q.parts = w_parts; q.part_stride = cols * D;
      float* out = q.out;
      const int64_t ld = q.ld;
      if (w_parts > 1) {
        q.out = w.at<float>(dwp);
        q.ld = transW ? D : cols;
      }
      if ((rc = lce::gradient(q, s))) return rc;
      if (w_parts > 1 && (rc = add_parts(q.out, transW ? cols : D, transW ? D : cols, w_parts, out, ld, s))) return rc;
    }
  }
  return dx && parts > 1 ? add_parts(w.at<float>(dxp), N, D, parts, dx, D, s) : ENDIA_HIP_OK;
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
  return N >= kManyRows ? many_rows_fwd(N, D, V, x, ldx, transW, W, ldw, target, loss, lse, s)
                        : few_rows_fwd(N, D, V, x, ldx, transW, W, ldw, target, loss, lse, s);
}

int32_t endia_hip_linear_cross_entropy_bwd(int64_t N, int64_t D, int64_t V, const float* x, int64_t ldx, int32_t transW, const float* W,
                                           int64_t ldw, const float* target, const float* lse, const float* g, float* dx, float* dW) {
  int32_t rc = check("endia_hip_linear_cross_entropy_bwd", N, D, V, x, ldx, transW, W, ldw, target, lse);
  if (rc) return rc;
  ENDIA_CHECK_ARG(g, "endia_hip_linear_cross_entropy_bwd: null pointer");
  ENDIA_CHECK_ARG(dx || dW, "endia_hip_linear_cross_entropy_bwd: nothing to compute");
  ENDIA_REQUIRE_INIT();
  hipStream_t s = ctx().stream;
  return N >= kManyRows ? many_rows_bwd(N, D, V, x, ldx, transW, W, ldw, target, lse, g, dx, dW, s)
                        : few_rows_bwd(N, D, V, x, ldx, transW, W, ldw, target, lse, g, dx, dW, s);
}

}  // extern "C"
