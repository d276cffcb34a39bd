// Attention for few queries per key head: the serving form, one or a few new tokens over a long cache. Bound: HBM, k and v are
// read once.
//
// A work-group of four waves takes R rows (query i of query head g, numbered g Q + i, of the G heads that share a key head) and
// one part of the keys; a key's row is read by LPK lanes, 16 bytes each, so a wave has 64 / LPK keys in hand at a time, UNROLL of
// them in flight per lane group. Scores are sums over a lane group; every lane group keeps its own running maximum, sum and
// output (a wave reads neither LDS nor other lanes' state per key), and the groups and waves meet once at the end. With few
// sequences the keys are cut into parts, and combine_kernel joins the parts' results. Measured: 64 sequences of 2000 to 4000 keys, 16
// heads of 64: 290 us = 5.4 TB/s; one sequence of 77 keys and 12 heads: 6 us, a launch.
// Used up to 16 rows per key head; from there on the tiles of the matrix cores take over (they would fill half of their 32 columns).
#include "attention.h"

namespace attention {

namespace {

constexpr int TPB = 256;

// A group's maximum may still be -inf (no key seen): nothing to carry over then.
__device__ __forceinline__ float carry(float m, float now) { return m == -INFINITY ? 0.f : exp2_fast(m - now); }

template <int LPK, int R, bool VEC>
__global__ __launch_bounds__(TPB) void rows_kernel(Args a) {
  constexpr int KPW = 64 / LPK, UNROLL = R <= 2 ? 4 : 2, DP = LPK * 4;
  constexpr int GROUPS = 4 * KPW;  // lane groups of the work-group
  __shared__ float lds_m[R][GROUPS], lds_l[R][GROUPS];
  __shared__ __attribute__((aligned(16))) float lds_o[R][GROUPS][DP];
  extern __shared__ float bias_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = lane / LPK, dl = lane % LPK;
  const int64_t b = blockIdx.z / (uint32_t)a.Hk, kh = blockIdx.z % (uint32_t)a.Hk;
  const int64_t rows = a.G * a.Q, r0 = (int64_t)blockIdx.x * R;
  const int D = (int)a.D;

  float4 q[R];
  int64_t place[R];   // position of the row's query
  int limit[R];       // keys the row may see
  const int n = key_count(a, b);
  int most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = r0 + r;
    const bool in = row < rows;
    const uint32_t g = in ? (uint32_t)row / (uint32_t)a.Q : 0, i = in ? (uint32_t)row % (uint32_t)a.Q : 0;
    q[r] = load4<VEC>(a.q + b * a.qs[0] + i * a.qs[1] + (kh * a.G + g) * a.qs[2], 4 * dl, D, in);
    const float c = a.scale * kLog2e;
    q[r].x *= c; q[r].y *= c; q[r].z *= c; q[r].w *= c;
    place[r] = i + a.off;
    int64_t see = n;
    if (a.causal && place[r] + 1 < see) see = place[r] + 1;
    limit[r] = in && see > 0 ? (int)see : 0;
    most = max(most, limit[r]);
  }
  const bool bias = a.table != nullptr;
  const int near = a.bk.near, span = 2 * near + 1;
  if (bias) {  // the heads of the work-group's rows, one table after the other (all rows of one head: one)
    const int64_t g0 = r0 / a.Q, g1 = min(r0 + R - 1, rows - 1) / a.Q;
    for (int64_t g = g0; g <= g1; ++g) load_bias(a, (int)(kh * a.G + g), bias_lds + (g - g0) * span, tid, TPB);
    __syncthreads();
  }
  float m[R], l[R];
  float4 o[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // this part's keys: whole steps of GROUPS * UNROLL
  constexpr int STEP = GROUPS * UNROLL;
  const int steps = (most + STEP - 1) / STEP, per = (steps + a.splits - 1) / a.splits;
  const int first = blockIdx.y * per * STEP, last = min(most, first + per * STEP);
  const float* kb = a.k + b * a.ks[0] + kh * a.ks[2];
  const float* vb = a.v + b * a.vs[0] + kh * a.vs[2];
  for (int j0 = first + wave * KPW + sub; j0 < last; j0 += STEP) {
    float4 kf[UNROLL], vf[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int j = min(j0 + u * GROUPS, last - 1);
      kf[u] = load4<VEC>(kb + (int64_t)j * a.ks[1], 4 * dl, D, true);
      vf[u] = load4<VEC>(vb + (int64_t)j * a.vs[1], 4 * dl, D, true);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float t[UNROLL], top = m[r];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        float d = (q[r].x * kf[u].x + q[r].y * kf[u].y) + (q[r].z * kf[u].z + q[r].w * kf[u].w);
#pragma unroll
        for (int w = LPK / 2; w; w >>= 1) d += __shfl_xor(d, w, 64);
        const int j = j0 + u * GROUPS;
        if (bias) {
          const int64_t g = (r0 + r) / a.Q - r0 / a.Q;
          const int64_t rel = (int64_t)j - place[r];
          const int at = rel < -near ? 0 : (rel > near ? 2 * near : (int)rel + near);
          d += (r0 + r < rows) ? bias_lds[g * span + at] : 0.f;
        }
        t[u] = j < limit[r] && j < last ? d : -INFINITY;
        top = fmaxf(top, t[u]);
      }
      const float keep = carry(m[r], top);
      m[r] = top;
      l[r] *= keep;
      o[r].x *= keep; o[r].y *= keep; o[r].z *= keep; o[r].w *= keep;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (t[u] == -INFINITY) continue;  // a key that is left out adds nothing, whatever its row holds (a NaN score does: fmaxf drops it from top)
        const float p = exp2_fast(t[u] - top);
        l[r] += p;
        o[r].x += p * vf[u].x; o[r].y += p * vf[u].y; o[r].z += p * vf[u].z; o[r].w += p * vf[u].w;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int g = wave * KPW + sub;
    if (dl == 0) {
      lds_m[r][g] = m[r];
      lds_l[r][g] = l[r];
    }
    *reinterpret_cast<float4*>(&lds_o[r][g][4 * dl]) = o[r];
  }
  __syncthreads();
  // thread t: element t % DP of row t / DP (+ more rows)
  for (int at = tid; at < R * DP; at += TPB) {
    const int r = at / DP, d = at % DP;
    const int64_t row = r0 + r;
    if (row >= rows) continue;
    float top = -INFINITY;
    for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, lds_m[r][g]);
    float sum = 0.f, out = 0.f;
    for (int g = 0; g < GROUPS; ++g) {  // (all maxima -inf: no key, and zeros are joined, or nothing but NaN scores, and NaN are)
      const float w = carry(lds_m[r][g], top);
      sum += w * lds_l[r][g];
      out += w * lds_o[r][g][d];
    }
    const int64_t h = kh * a.G + row / a.Q, i = row % a.Q;
    if (a.splits == 1) {
      if (d < D) a.o[((b * a.Q + i) * a.H + h) * D + d] = sum != 0.f ? out / sum : 0.f;
      if (d == 0 && a.lse) a.lse[(b * a.H + h) * a.Q + i] = sum != 0.f ? (top + log2_fast(sum)) * kLn2 : -INFINITY;
    } else {
      const int64_t part = ((b * a.H + h) * a.Q + i) * a.splits + blockIdx.y;
      if (d < D) a.part[part * D + d] = out;
      if (d == 0) {
        a.part_ml[2 * part] = top;
        a.part_ml[2 * part + 1] = sum;
      }
    }
  }
}

// One wave per row: joins the parts' outputs, each relative to its part's maximum. The lanes first share the parts' weights out
// among them. A part whose maximum is -inf has weight 0 and holds zeros (no key) or NaN (nothing but NaN scores), which 0 leaves NaN.
__global__ __launch_bounds__(TPB) void combine_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b H + h) Q + i
  if (row >= a.B * a.H * a.Q) return;
  const uint32_t bh = (uint32_t)(row / a.Q), i = (uint32_t)(row % a.Q), h = bh % (uint32_t)a.H, b = bh / (uint32_t)a.H;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * a.splits;
  float top = -INFINITY, sum = 0.f;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, ml[s].x);
  top = wave_max(top);
  float o0 = 0.f, o1 = 0.f;
  const float* part = a.part + row * a.splits * a.D;
  for (int s0 = 0; s0 < a.splits; s0 += 64) {
    float w = 0.f;
    if (s0 + lane < a.splits) {
      const float2 f = ml[s0 + lane];
      w = carry(f.x, top);
      sum += w * f.y;
    }
    const int n = min(64, a.splits - s0);
    for (int s = 0; s < n; ++s) {
      const float ws = __shfl(w, s, 64);
      const float* from = part + (s0 + s) * a.D;
      if (lane < a.D) o0 += ws * from[lane];
      if (lane + 64 < a.D) o1 += ws * from[lane + 64];
    }
  }
#pragma unroll
  for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w, 64);
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  float* out = a.o + (((int64_t)b * a.Q + i) * a.H + h) * a.D;
  if (lane < a.D) out[lane] = o0 * inv;
  if (lane + 64 < a.D) out[lane + 64] = o1 * inv;
  if (lane == 0 && a.lse) a.lse[row] = sum != 0.f ? (top + log2_fast(sum)) * kLn2 : -INFINITY;
}

template <int LPK, int R>
int32_t launch(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div64(a.G * a.Q, R), (unsigned)a.splits, (unsigned)(a.B * a.Hk));
  size_t lds = 0;
  if (a.table) {  // heads that R consecutive rows can touch
    const int64_t heads = a.Q >= R ? 2 : ceil_div64(R, a.Q) + 1;
    lds = (size_t)((heads < a.G ? heads : a.G) * (2 * a.bk.near + 1)) * 4;
  }
  if (a.vec) hipLaunchKernelGGL((rows_kernel<LPK, R, true>), grid, dim3(TPB), lds, s, a);
  else hipLaunchKernelGGL((rows_kernel<LPK, R, false>), grid, dim3(TPB), lds, s, a);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

template <int LPK>
int32_t launch(const Args& a, int R, hipStream_t s) {
  return R == 1 ? launch<LPK, 1>(a, s) : R == 2 ? launch<LPK, 2>(a, s) : launch<LPK, 4>(a, s);
}

}  // namespace

int32_t launch_rows(const Args& a, int R, hipStream_t s) {
  int32_t rc = a.D <= 32 ? launch<8>(a, R, s) : a.D <= 64 ? launch<16>(a, R, s) : launch<32>(a, R, s);
  return rc || a.splits == 1 ? rc : launch_combine(a, s);
}

int32_t launch_combine(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL(combine_kernel, dim3((unsigned)ceil_div64(a.B * a.H * a.Q, 4)), dim3(TPB), 0, s, a);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace attention
