// Attention of queries over keys of another length, with an optional learned position bias by buckets, and its gradient.
// Stands beside matmul and linear (endia/functional/binary_ops/matmul_op.mojo): the products of a sequence model's layer.
//
//   s_ij = scale q_i . k_j + table[bucket(j - (i + query_offset))]     masked: j >= key_lengths[b], causal j > i + query_offset
//   p = softmax over the keys that are left (a row with none: zeros)   o = p v
//   dv = p^T do,  dp = do v^T,  ds = p (dp - sum_j p dp),  dq = scale ds k,  dk = scale ds^T q,  dtable = sums of ds by bucket
//
// First form: one batch entry at a time with the score matrix in memory, products by endia_hip_sgemm.
#include "common.h"

#include <math.h>

using namespace endia;

namespace {

constexpr int TPB = 256;
constexpr int kMaxSide = 128;  // buckets of one side

struct Scratch {
  void* p = nullptr;
  int32_t get(int64_t bytes) { return endia_hip_malloc(bytes, &p); }
  ~Scratch() {
    if (p) endia_hip_free(p);
  }
  float* f() const { return static_cast<float*>(p); }
};

// bucket of n steps: n itself below `exact`, then the largest i with start[i] <= n
struct Buckets {
  int side, exact, both;
  int start[kMaxSide];
};

__device__ __forceinline__ int bucket_of(const Buckets& t, int64_t rel) {
  int base = 0;
  int64_t n = -rel;
  if (t.both) {
    if (rel > 0) {
      base = t.side;
      n = rel;
    }
  } else if (n < 0) {
    n = 0;
  }
  if (n < t.exact) return base + (int)n;
  int i = t.exact;
  while (i + 1 < t.side && t.start[i + 1] <= n) ++i;
  return base + i;
}

int32_t make_buckets(const endia_hip_attention_desc* d, Buckets* t) {
  t->both = d->both_sides;
  t->side = d->both_sides ? d->buckets / 2 : d->buckets;
  t->exact = t->side / 2;
  const int steps = t->side - t->exact;
  for (int i = 0; i < kMaxSide; ++i) t->start[i] = i < t->exact ? i : 0x7fffffff;
  int i = t->exact;
  for (int n = t->exact; n <= d->max_distance && i < t->side; ++n) {
    // 1e-9: a whole number of steps lands on its own bucket (the next nearest quotient is further off than that)
    const int far = t->exact + (int)floor(log((double)n / t->exact) / log((double)d->max_distance / t->exact) * steps + 1e-9);
    while (i < t->side && i <= far) t->start[i++] = n;
  }
  return ENDIA_HIP_OK;
}

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

__device__ __forceinline__ int64_t key_count(const float* lengths, int64_t b, int64_t K) {
  if (!lengths) return K;
  const float n = lengths[b];
  return n > 0.f ? (n < (float)K ? (int64_t)n : K) : 0;
}

// k or v of one batch entry as [Hk, K, D], zeros behind the entry's length
__global__ __launch_bounds__(TPB) void clean_kernel(const float* __restrict__ x, int64_t sp, int64_t sh, const float* __restrict__ lengths, int64_t b,
                                                    int64_t K, int64_t D, float* __restrict__ out) {
  const int64_t j = blockIdx.x, h = blockIdx.y, n = key_count(lengths, b, K);
  for (int64_t d = threadIdx.x; d < D; d += TPB) out[(h * K + j) * D + d] = j < n ? x[j * sp + h * sh + d] : 0.f;
}

__global__ __launch_bounds__(TPB) void softmax_kernel(float* __restrict__ s, int64_t Q, int64_t K, int64_t b, int64_t H, const float* __restrict__ lengths,
                                                      float scale, int causal, int64_t off, const float* __restrict__ table, Buckets bk,
                                                      float* __restrict__ lse) {
  __shared__ float red[TPB / 64];
  const int64_t i = blockIdx.x, h = blockIdx.y;
  int64_t n = key_count(lengths, b, K);
  if (causal && i + off + 1 < n) n = i + off + 1 > 0 ? i + off + 1 : 0;
  float* row = s + (h * Q + i) * K;
  float top = -INFINITY;
  for (int64_t j = threadIdx.x; j < n; j += TPB) {
    float t = row[j] * scale;
    if (table) t += table[bucket_of(bk, j - (i + off)) * H + h];
    row[j] = t;
    top = fmaxf(top, t);
  }
  top = block_reduce(top, red, true);
  float sum = 0.f;
  for (int64_t j = threadIdx.x; j < n; j += TPB) sum += expf(row[j] - top);
  sum = block_reduce(sum, red, false);
  const float e = top + logf(sum);
  for (int64_t j = threadIdx.x; j < K; j += TPB) row[j] = j < n ? expf(row[j] - e) : 0.f;
  if (threadIdx.x == 0 && lse) lse[(b * H + h) * Q + i] = n ? e : -INFINITY;
}

__global__ __launch_bounds__(TPB) void ds_kernel(const float* __restrict__ p, float* __restrict__ dp, int64_t K) {
  __shared__ float red[TPB / 64];
  const int64_t r = blockIdx.x * K;
  float sum = 0.f;
  for (int64_t j = threadIdx.x; j < K; j += TPB) sum += p[r + j] * dp[r + j];
  sum = block_reduce(sum, red, false);
  for (int64_t j = threadIdx.x; j < K; j += TPB) dp[r + j] = p[r + j] * (dp[r + j] - sum);
}

// dtable[bucket, h] (+)= the sum of ds over the pairs of that bucket; one group per (bucket, h)
__global__ __launch_bounds__(TPB) void table_grad_kernel(const float* __restrict__ ds, int64_t Q, int64_t K, int64_t H, int64_t off, Buckets bk,
                                                         float* __restrict__ dtable, int first) {
  __shared__ double red[TPB];
  const int b = blockIdx.x;
  const int64_t h = blockIdx.y;
  double sum = 0.0;
  for (int64_t j = threadIdx.x; j < Q * K; j += TPB)
    if (bucket_of(bk, j % K - (j / K + off)) == b) sum += (double)ds[h * Q * K + j];
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int s = TPB / 2; s; s >>= 1) {
    if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) dtable[b * H + h] = (first ? 0.f : dtable[b * H + h]) + (float)red[0];
}

__global__ __launch_bounds__(TPB) void scale_kernel(float* __restrict__ x, int64_t n, float c) {
  const int64_t i = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (i < n) x[i] *= c;
}

int32_t check(const char* who, const endia_hip_attention_desc* d, const float* q, const float* k, const float* v, const float* table) {
  ENDIA_CHECK_ARG(d && q && k && v, "%s: null pointer", who);
  ENDIA_CHECK_ARG(d->B > 0 && d->Q > 0 && d->K > 0 && d->H > 0 && d->Hk > 0 && d->D > 0, "%s: sizes must be positive", who);
  ENDIA_CHECK_ARG(d->H % d->Hk == 0, "%s: %lld query heads cannot share %lld key heads evenly", who, (long long)d->H, (long long)d->Hk);
  ENDIA_CHECK_ARG(d->Q < (1ll << 24) && d->K <= (1ll << 24), "%s: more than 2^24 positions (lengths are held in fp32)", who);
  ENDIA_CHECK_ARG(d->query_offset > -(1ll << 30) && d->query_offset < (1ll << 30), "%s: query_offset out of range", who);
  ENDIA_CHECK_ARG(isfinite(d->scale), "%s: scale must be finite", who);
  if (d->D > ENDIA_ATTENTION_MAX_DIM || d->B * d->H > 65535)
    return fail(ENDIA_HIP_ERR_UNSUPPORTED, "%s: head dimension %lld above %d, or more than 65535 heads over the batch", who, (long long)d->D,
                ENDIA_ATTENTION_MAX_DIM);
  if (table) {
    const int side = d->both_sides ? d->buckets / 2 : d->buckets;
    ENDIA_CHECK_ARG(side >= 2 && (!d->both_sides || d->buckets % 2 == 0) && d->max_distance > side / 2,
                    "%s: %d buckets and max_distance %d do not make a bucket table", who, d->buckets, d->max_distance);
    if (side > kMaxSide || d->max_distance > ENDIA_ATTENTION_MAX_DISTANCE)
      return fail(ENDIA_HIP_ERR_UNSUPPORTED, "%s: at most %d buckets a side and max_distance at most %d", who, kMaxSide,
                  ENDIA_ATTENTION_MAX_DISTANCE);
  }
  return ENDIA_HIP_OK;
}

}  // namespace

extern "C" {

int32_t endia_hip_attention_fwd(const endia_hip_attention_desc* d, const float* q, const float* k, const float* v, const float* key_lengths,
                                const float* table, float* o, float* lse) {
  int32_t rc = check("endia_hip_attention_fwd", d, q, k, v, table);
  if (rc) return rc;
  ENDIA_CHECK_ARG(o, "endia_hip_attention_fwd: null pointer");
  ENDIA_REQUIRE_INIT();
  hipStream_t st = ctx().stream;
  const int64_t B = d->B, Q = d->Q, K = d->K, H = d->H, Hk = d->Hk, D = d->D, G = H / Hk;
  Buckets bk = {};
  if (table) make_buckets(d, &bk);
  Scratch s, kc, vc;
  if ((rc = s.get(4 * H * Q * K)) || (rc = kc.get(4 * Hk * K * D)) || (rc = vc.get(4 * Hk * K * D))) return rc;
  for (int64_t b = 0; b < B; ++b) {
    hipLaunchKernelGGL(clean_kernel, dim3((unsigned)K, (unsigned)Hk), dim3(TPB), 0, st, k + b * d->k_strides[0], d->k_strides[1], d->k_strides[2],
                       key_lengths, b, K, D, kc.f());
    hipLaunchKernelGGL(clean_kernel, dim3((unsigned)K, (unsigned)Hk), dim3(TPB), 0, st, v + b * d->v_strides[0], d->v_strides[1], d->v_strides[2],
                       key_lengths, b, K, D, vc.f());
    for (int64_t c = 0; c < Hk; ++c)
      if ((rc = endia_hip_sgemm(0, 1, Q, K, D, q + b * d->q_strides[0] + c * G * d->q_strides[2], d->q_strides[1], kc.f() + c * K * D, D,
                                s.f() + c * G * Q * K, K, G, d->q_strides[2], 0, Q * K, ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr,
                                nullptr)))
        return rc;
    hipLaunchKernelGGL(softmax_kernel, dim3((unsigned)Q, (unsigned)H), dim3(TPB), 0, st, s.f(), Q, K, b, H, key_lengths, d->scale, d->causal,
                       d->query_offset, table, bk, lse);
    for (int64_t h = 0; h < H; ++h)
      if ((rc = endia_hip_sgemm(0, 0, Q, D, K, s.f() + h * Q * K, K, vc.f() + h / G * K * D, D, o + b * Q * H * D + h * D, H * D, 1, 0, 0, 0,
                                ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
        return rc;
  }
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t endia_hip_attention_bwd(const endia_hip_attention_desc* d, const float* q, const float* k, const float* v, const float* key_lengths,
                                const float* table, const float* o, const float* lse, const float* go, float* dq, float* dk, float* dv,
                                float* dtable) {
  int32_t rc = check("endia_hip_attention_bwd", d, q, k, v, table);
  if (rc) return rc;
  ENDIA_CHECK_ARG(o && lse && go, "endia_hip_attention_bwd: null pointer");
  ENDIA_CHECK_ARG(dq || dk || dv || dtable, "endia_hip_attention_bwd: nothing to compute");
  ENDIA_CHECK_ARG(!dtable || table, "endia_hip_attention_bwd: dtable without a table");
  ENDIA_REQUIRE_INIT();
  hipStream_t st = ctx().stream;
  const int64_t B = d->B, Q = d->Q, K = d->K, H = d->H, Hk = d->Hk, D = d->D, G = H / Hk;
  Buckets bk = {};
  if (table) make_buckets(d, &bk);
  Scratch s, ds, kc, vc;
  if ((rc = s.get(4 * H * Q * K)) || (rc = ds.get(4 * H * Q * K)) || (rc = kc.get(4 * Hk * K * D)) || (rc = vc.get(4 * Hk * K * D))) return rc;
  for (int64_t b = 0; b < B; ++b) {
    hipLaunchKernelGGL(clean_kernel, dim3((unsigned)K, (unsigned)Hk), dim3(TPB), 0, st, k + b * d->k_strides[0], d->k_strides[1], d->k_strides[2],
                       key_lengths, b, K, D, kc.f());
    hipLaunchKernelGGL(clean_kernel, dim3((unsigned)K, (unsigned)Hk), dim3(TPB), 0, st, v + b * d->v_strides[0], d->v_strides[1], d->v_strides[2],
                       key_lengths, b, K, D, vc.f());
    const float* qb = q + b * d->q_strides[0];
    const float* gb = go + b * Q * H * D;
    for (int64_t c = 0; c < Hk; ++c) {
      if ((rc = endia_hip_sgemm(0, 1, Q, K, D, qb + c * G * d->q_strides[2], d->q_strides[1], kc.f() + c * K * D, D, s.f() + c * G * Q * K, K, G,
                                d->q_strides[2], 0, Q * K, ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)) ||
          (rc = endia_hip_sgemm(0, 1, Q, K, D, gb + c * G * D, H * D, vc.f() + c * K * D, D, ds.f() + c * G * Q * K, K, G, D, 0, Q * K,
                                ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
        return rc;
    }
    hipLaunchKernelGGL(softmax_kernel, dim3((unsigned)Q, (unsigned)H), dim3(TPB), 0, st, s.f(), Q, K, b, H, key_lengths, d->scale, d->causal,
                       d->query_offset, table, bk, nullptr);
    hipLaunchKernelGGL(ds_kernel, dim3((unsigned)(H * Q)), dim3(TPB), 0, st, s.f(), ds.f(), K);
    if (dtable)
      hipLaunchKernelGGL(table_grad_kernel, dim3((unsigned)d->buckets, (unsigned)H), dim3(TPB), 0, st, ds.f(), Q, K, H, d->query_offset, bk, dtable,
                         b == 0 ? 1 : 0);
    for (int64_t h = 0; h < H; ++h) {
      const int64_t c = h / G, at = h * Q * K;
      const int32_t more = h % G ? ENDIA_EPI_NONE | ENDIA_GEMM_ACCUMULATE : ENDIA_EPI_NONE;
      if (dv && (rc = endia_hip_sgemm(1, 0, K, D, Q, s.f() + at, K, gb + h * D, H * D, dv + b * K * Hk * D + c * D, Hk * D, 1, 0, 0, 0, more,
                                      ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
        return rc;
      if (dk && (rc = endia_hip_sgemm(1, 0, K, D, Q, ds.f() + at, K, qb + h * d->q_strides[2], d->q_strides[1], dk + b * K * Hk * D + c * D, Hk * D,
                                      1, 0, 0, 0, more, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
        return rc;
      if (dq && (rc = endia_hip_sgemm(0, 0, Q, D, K, ds.f() + at, K, kc.f() + c * K * D, D, dq + b * Q * H * D + h * D, H * D, 1, 0, 0, 0,
                                      ENDIA_EPI_NONE, ENDIA_OP_IDENTITY, nullptr, nullptr, nullptr)))
        return rc;
    }
  }
  if (dq) hipLaunchKernelGGL(scale_kernel, dim3((unsigned)ceil_div64(B * Q * H * D, TPB)), dim3(TPB), 0, st, dq, B * Q * H * D, d->scale);
  if (dk) hipLaunchKernelGGL(scale_kernel, dim3((unsigned)ceil_div64(B * K * Hk * D, TPB)), dim3(TPB), 0, st, dk, B * K * Hk * D, d->scale);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // extern "C"
