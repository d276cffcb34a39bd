// Gradients of attention on the matrix cores, operands as pairs of fp16 (fp16_pairs.h). The scores are formed again from q and k
// and the forward pass's lse: p = exp2(s - lse), ds = p (dp - delta) with delta = sum_j p dp = do . o (tiles_kernel).
//
// dq_kernel: as in the forward pass a wave owns 32 queries and walks over the keys: S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.
// dkv_kernel: a wave owns 32 keys and walks over the queries of all heads that share them: S = Q K^T, dP = dO V^T,
// dV^T += dO^T P, dK^T += Q^T dS. In both the lane holds 16 scores of one of its own rows, which are the next product's
// operand as they lie. Two kernels with 3 and 4 products rather than one with 5: nothing is added across work-groups, so the
// sums have one order (no atomics), and a group that is cut into parts writes each part's sum for reduce_parts_kernel.
// p and ds are scaled per key (or query) by a running power of two, lowered with the accumulator when a block exceeds it.
// Bound: the matrix pipe at DP = 128, the vector ALU at DP = 64 and below; with a table the 16 LDS additions of a tile near the
// diagonal (half of dq's time at 512 keys). Measured, as fp32 products: 4096 queries x 16384 keys, 16 heads of 128: dq 2.62 ms = 315
// TFLOP/s, dkv 3.76 ms = 293; 8 x 448 x 1500, 16 heads of 64: dq 122 us = 212, dkv 182 us = 189; 5001 causal with buckets: dq 813 to
// 822 us = 187 to 189, dkv 1.02 ms = 201.
#include "attention.h"

namespace attention {

namespace {

using namespace pairs;
constexpr int TPB = 256;
constexpr float kMost = 32768.f;  // a scaled p or ds stays below this

// Brings the running shift F of the lane's accumulator column (2^F times the sums; both halves of the wave agree on it) and the
// factor of the block at hand together: the block's values x times 2^(F - shift) have to stay below kMost. Returns that factor.
// A column of its own for every key (or query): one that is hardly attended to keeps its precision beside the others. Only
// blocks far below the column's largest so far may vanish, which is what they add beside it.
template <int N>
__device__ __forceinline__ float fit(const float (&x)[16], int shift, int& F, floatx16 (&acc)[N]) {
  float amax = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) amax = fmaxf(amax, __builtin_fabsf(x[v]));
  const int up = F - shift;
  if (__any(amax > 0.f && (up > kMaxShift || amax * pow2i(up) >= kMost))) {
    const float most = finite_abs(fmaxf(amax, __shfl_xor(amax, 32, 64)));
    const int e = max((int)(__float_as_uint(most) >> 23) - 127, -88);
    const int to = 12 - e + shift;  // (two bits of room, so that a slowly growing ds does not come here each time)
    if (most > 0.f && to < F) {
      const float down = pow2i(to - F);
#pragma unroll
      for (int d = 0; d < N; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[d][v] *= down;
      F = to;
    }
  }
  return pow2i(min(F - shift, kMaxShift));
}

__device__ __forceinline__ void as_operand(const float (&x)[16], float c, half8 (&hi)[2], half8 (&lo)[2]) {
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[8 * st + e] * c;
    split8(y, hi[st], lo[st]);
  }
}

// acc (columns: the lane's row of D values) -> out[d], times c
template <int DP>
__device__ __forceinline__ void store_row(float* out, const floatx16 (&acc)[DP / 32], float c, int D, int half, int vec) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = d * 32 + 8 * j + 4 * half;
      if (vec) {
        if (at < D)
          *reinterpret_cast<float4*>(out + at) = make_float4(acc[d][4 * j] * c, acc[d][4 * j + 1] * c, acc[d][4 * j + 2] * c, acc[d][4 * j + 3] * c);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at + e < D) out[at + e] = acc[d][4 * j + e] * c;
      }
    }
}

__device__ __forceinline__ float far_part(float ds, float p, float p_all, float row_sum) {
  return p_all > 0.f ? (ds - p * (row_sum / p_all)) / p_all : ds;
}

template <int DP, bool BIAS>
__global__ __launch_bounds__(TPB, DP <= 64 ? 2 : 1) void dq_kernel(Args a, const TileInfo* __restrict__ k_info, const TileInfo* __restrict__ v_info,
                                                                   const float* __restrict__ meta) {
  constexpr int STAGE = DP * 384;  // row images of k and v, column image of k
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int near = a.bk.near, span = 2 * near + 1;
  float* bias_lds = reinterpret_cast<float*>(smem + a.stages * STAGE);
  float* bins = bias_lds + span;  // one set per wave: sums of ds by position difference
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int64_t qgroups = (a.Q + 127) / 128;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const uint32_t split = id % (uint32_t)a.splits;
  id /= (uint32_t)a.splits;
  const uint32_t hb = id / (uint32_t)qgroups;
  const int64_t qt = a.causal ? qgroups - 1 - id % (uint32_t)qgroups : id % (uint32_t)qgroups, h = hb % (uint32_t)a.H, b = hb / (uint32_t)a.H, kh = (uint32_t)h / (uint32_t)a.G;
  const int D = (int)a.D;
  const int64_t q0 = qt * 128 + wave * 32, i = q0 + col;
  const bool in = i < a.Q;
  const bool sum_table = BIAS && a.part_table;

  half8 qh[DP / 16], ql[DP / 16], gh[DP / 16], gl[DP / 16];
  const int64_t iv = min(i, a.Q - 1);
  const int qshift = load_fragments<DP>(a.q + b * a.qs[0] + iv * a.qs[1] + h * a.qs[2], in, D, a.vec, half, qh, ql);
  const int gshift = load_fragments<DP>(a.go + ((b * a.Q + iv) * a.H + h) * D, in, D, a.vec, half, gh, gl);
  // The matrix instruction's sums are a little low on average (3e-8 of |do| |v| here, far below one rounding), which shows where
  // ds is added up over a million pairs: every other query's dp is formed with its sign turned, so that it cancels over the rows.
  const float turn = col & 1 ? -1.f : 1.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    gh[s] *= (_Float16)turn;
    gl[s] *= (_Float16)turn;
  }
  const float cq = a.scale * kLog2e * pow2i(-qshift), cg = turn * pow2i(-gshift);
  const int64_t qtiles = (a.Q + kTile - 1) / kTile;
  const int64_t mt = ((b * a.H + h) * qtiles + min(q0 / 32, qtiles - 1)) * 64;
  const float lse = in ? meta[mt + col] : INFINITY, delta = in ? meta[mt + 32 + col] : 0.f;
  if (BIAS) {
    load_bias(a, (int)h, bias_lds, tid, TPB);
    if (sum_table)
      for (int j = tid; j < 4 * span; j += TPB) bins[j] = 0.f;
  }
  float* my_bins = bins + wave * span;
  // The sum of a row's p is 1, that of its ds 0, and a bucket far away holds most of both: what lse and delta are off by (they come
  // from rounded results) would add up there over all keys. So the row's own sums are taken too, and the far buckets' are set right
  // by them: ds_far := (ds_far - p_far sum(ds) / sum(p)) / sum(p).
  float far_low = 0.f, far_high = 0.f, p_low = 0.f, p_high = 0.f, p_all = 0.f, row_sum = 0.f;

  const int n = key_count(a, b);
  const int64_t place = i + a.off;
  int64_t see = n;
  if (a.causal && place + 1 < see) see = place + 1 > 0 ? place + 1 : 0;
  const int limit = (int)see;
  int64_t most = n;
  if (a.causal) {
    const int64_t last = min(a.Q - 1, qt * 128 + 127) + a.off + 1;
    most = last < most ? (last > 0 ? last : 0) : most;
  }
  const int tiles = (int)((most + kTile - 1) / kTile), per = (tiles + a.splits - 1) / a.splits;
  const int t0 = (int)split * per, t1 = min(tiles, t0 + per);
  const int64_t wave_first = q0 + a.off;
  int64_t clear_keys = n;
  if (a.causal && wave_first + 1 < clear_keys) clear_keys = wave_first + 1 > 0 ? wave_first + 1 : 0;

  const int64_t ktiles = (a.K + kTile - 1) / kTile, tile_at = (b * a.Hk + kh) * ktiles;
  auto request = [&](int t, int stage) {
    const int64_t from = (tile_at + t) * (DP * 128) + lane * 16;
    char* to = smem + stage * STAGE;
#pragma unroll
    for (int p = 0; p < DP / 32; ++p) {
      const int at = (p * 4 + wave) * 1024;
      load_to_lds(a.k_rows + from + at, to + at);
      load_to_lds(a.v_rows + from + at, to + DP * 128 + at);
      load_to_lds(a.k_cols + from + at, to + DP * 256 + at);
    }
  };

  floatx16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dq[d] = floatx16{};
  int F = 2 * kMaxShift;
  const bool ahead = a.stages == 2;
  if (t0 < t1) request(t0, 0);
  wait_loads();
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int stage = ahead ? (t - t0) & 1 : 0;
    const int ks = k_info[tile_at + t].shift, vs = v_info[tile_at + t].shift;
    if (ahead && t + 1 < t1) request(t + 1, stage ^ 1);
    const char* kimg = smem + stage * STAGE;
    const char* vimg = kimg + DP * 128;
    const char* kcol = kimg + DP * 256;
    if (q0 < a.Q && (int64_t)t * kTile < clear_keys + 31) {
      floatx16 s = {}, dp = {};
#pragma unroll
      for (int kb = 0; kb < DP / 32; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 ah, al;
          read_line(kimg + kb * 4096, col, st, half, ah, al);
          s = mfma_pairs(ah, al, qh[2 * kb + st], ql[2 * kb + st], s);
          read_line(vimg + kb * 4096, col, st, half, ah, al);
          dp = mfma_pairs(ah, al, gh[2 * kb + st], gl[2 * kb + st], dp);
        }
      const float c = cq * pow2i(-ks), cd = cg * pow2i(-vs);
      const int key0 = t * kTile + 4 * half;
      const int rel = BIAS ? (int)max(min(key0 - place, (int64_t)1 << 20), -((int64_t)1 << 20)) : 0;
      const int64_t lo = (int64_t)t * kTile - (wave_first + 31), hi = (int64_t)t * kTile + 31 - wave_first;
      const bool far = BIAS && (lo >= near || hi <= -near);
      float x[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = s[v] * c;
      if (BIAS) {
        if (far) {
          const float f = bias_lds[hi <= -near ? 0 : 2 * near];
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] += f;
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] += bias_lds[near_index(rel + 8 * (v >> 2) + (v & 3), near)];
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = exp2_fast(x[v] - lse);
      // (a row without keys has lse = inf here, which leaves p = 0 but not ds = 0 if dp is not finite)
      const bool mask = (int64_t)(t + 1) * kTile > clear_keys || q0 + 31 >= a.Q;
      if (mask) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = in && key0 + 8 * (v >> 2) + (v & 3) < limit ? x[v] : 0.f;
      }
      if (sum_table) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) sum += x[v];
        p_all += sum;
        if (far) {
          if (hi <= -near) p_low += sum;
          else p_high += sum;
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] *= dp[v] * cd - delta;
      if (mask) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = in && key0 + 8 * (v >> 2) + (v & 3) < limit ? x[v] : 0.f;
      }
      if (sum_table) {
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) sum += x[v];
        row_sum += sum;
        if (far) {
          if (hi <= -near) far_low += sum;
          else far_high += sum;
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) atomicAdd(&my_bins[near_index(rel + 8 * (v >> 2) + (v & 3), near)], x[v]);
        }
      }
      const float up = fit<DP / 32>(x, ks, F, dq);
      half8 xh[2], xl[2];
      as_operand(x, up, xh, xl);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 ah, al;
          read_line(kcol, d * 32 + col, st, half, ah, al);
          dq[d] = mfma_pairs(ah, al, xh[st], xl[st], dq[d]);
        }
    }
    if (!ahead && t + 1 < t1) {  // one stage: everybody is done with it before the next tile comes
      __syncthreads();
      request(t + 1, 0);
    }
    wait_loads();
    __syncthreads();
  }
  if (in && a.dq) {
    const float c = pow2i(-F) * a.scale;
    const int64_t row = (b * a.Q + i) * a.H + h;
    float* out = a.splits == 1 ? a.dq + row * D : a.part + ((int64_t)split * a.B * a.Q * a.H + row) * D;
    store_row<DP>(out, dq, c, D, half, a.vec);
  }
  if (sum_table) {
    // (both halves of the wave hold parts of a row)
    float* sums[] = {&far_low, &far_high, &p_low, &p_high, &p_all, &row_sum};
#pragma unroll
    for (float* x : sums) *x += __shfl_xor(*x, 32, 64);
    if (a.splits == 1) {
      far_low = far_part(far_low, p_low, p_all, row_sum);
      far_high = far_part(far_high, p_high, p_all, row_sum);
    } else if (in && half == 0) {  // a row that is cut: table_grad_kernel adds its parts up first
      float4* to = reinterpret_cast<float4*>(a.part_rows + (((b * a.H + h) * a.Q + i) * a.splits + split) * 8);
      to[0] = make_float4(far_low, far_high, p_low, p_high);
      to[1] = make_float4(p_all, row_sum, 0.f, 0.f);
    }
    if (a.splits > 1 || half) far_low = far_high = 0.f;
    // the wave's far sums join its bins at the ends, then the waves' bins are added in order
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      far_low += __shfl_xor(far_low, o, 64);
      far_high += __shfl_xor(far_high, o, 64);
    }
    if (lane == 0) {
      my_bins[0] += far_low;
      my_bins[2 * near] += far_high;
    }
    __syncthreads();
    float* to = a.part_table + (((b * a.H + h) * qgroups + qt) * a.splits + split) * span;
    for (int j = tid; j < span; j += TPB) to[j] = (bins[j] + bins[span + j]) + (bins[2 * span + j] + bins[3 * span + j]);
  }
}

template <int DP, bool BIAS>
__global__ __launch_bounds__(TPB, DP <= 64 ? 2 : 1) void dkv_kernel(Args a, const TileInfo* __restrict__ q_info, const TileInfo* __restrict__ g_info,
                                                                    const float* __restrict__ meta) {
  constexpr int STAGE = DP * 512 + 256;  // row and column images of q and do; lse and delta
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* bias_lds = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = BIAS ? __builtin_amdgcn_readfirstlane(tid >> 6) : tid >> 6, col = lane & 31, half = lane >> 5;
  const int near = a.bk.near;  // (with a table the wave's number is made scalar, so that addresses take no vector registers: with the
                               // order of ds below 1.03 ms against 1.35 at 5001 causal queries and 16 heads of 128)
  const int64_t kgroups = (a.K + 127) / 128;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const uint32_t split = id % (uint32_t)a.splits;
  id /= (uint32_t)a.splits;
  const uint32_t hb = id / (uint32_t)kgroups;
  const int64_t kt = id % (uint32_t)kgroups, kh = hb % (uint32_t)a.Hk, b = hb / (uint32_t)a.Hk;
  const int D = (int)a.D;
  const int64_t k0 = kt * 128 + wave * 32, j = k0 + col;
  const int n = key_count(a, b);
  const bool in = j < n;

  half8 kfh[DP / 16], kfl[DP / 16], vfh[DP / 16], vfl[DP / 16];
  const int64_t jv = min(j, a.K - 1);
  const int kshift = load_fragments<DP>(a.k + b * a.ks[0] + jv * a.ks[1] + kh * a.ks[2], in, D, a.vec, half, kfh, kfl);
  const int vshift = load_fragments<DP>(a.v + b * a.vs[0] + jv * a.vs[1] + kh * a.vs[2], in, D, a.vec, half, vfh, vfl);
  const float ck = a.scale * kLog2e * pow2i(-kshift), cv = pow2i(-vshift);

  // the queries of one head that see the group's keys, tile by tile, head after head
  const int qtiles = (int)((a.Q + kTile - 1) / kTile);
  int64_t first_q = 0;
  if (a.causal) first_q = max((int64_t)0, kt * 128 - a.off);
  const int qt0 = kt * 128 < n ? (int)min((int64_t)qtiles, first_q / kTile) : qtiles;
  const int each = qtiles - qt0, all = each * (int)a.G, per = (all + a.splits - 1) / a.splits;
  const int u0 = (int)split * per, u1 = min(all, u0 + per);

  auto tile_of = [&](int u) { return (b * a.H + kh * a.G + u / each) * qtiles + qt0 + u % each; };
  auto request = [&](int u, int stage) {
    const int64_t t = tile_of(u), from = t * (DP * 128) + lane * 16;
    char* to = smem + stage * STAGE;
#pragma unroll
    for (int p = 0; p < DP / 32; ++p) {
      const int at = (p * 4 + wave) * 1024;
      load_to_lds(a.q_rows + from + at, to + at);
      load_to_lds(a.g_rows + from + at, to + DP * 128 + at);
      load_to_lds(a.q_cols + from + at, to + DP * 256 + at);
      load_to_lds(a.g_cols + from + at, to + DP * 384 + at);
    }
    if (wave == 0 && lane < 16) load_to_lds(reinterpret_cast<const char*>(meta + t * 64) + lane * 16, to + DP * 512);
  };

  floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = floatx16{};
  int FK = 2 * kMaxShift, FV = 2 * kMaxShift;
  int64_t bias_head = -1;
  unsigned bad = 0;
  if (u0 < u1) request(u0, 0);
  wait_loads();
  __syncthreads();
  for (int u = u0; u < u1; ++u) {
    const int stage = (u - u0) & 1;
    const int64_t t = tile_of(u);
    const int qs = q_info[t].shift, gs = g_info[t].shift;
    bad |= g_info[t].bad;
    if (u + 1 < u1) request(u + 1, stage ^ 1);
    if (BIAS && bias_head != u / each) {  // (uniform over the work-group; everybody is behind the barrier of the last turn)
      bias_head = u / each;
      load_bias(a, (int)(kh * a.G + bias_head), bias_lds, tid, TPB);
      __syncthreads();
    }
    const char* qimg = smem + stage * STAGE;
    const char* gimg = qimg + DP * 128;
    const char* qcol = qimg + DP * 256;
    const char* gcol = qimg + DP * 384;
    const float* row_lse = reinterpret_cast<const float*>(qimg + DP * 512);
    const int64_t q0 = (int64_t)(qt0 + u % each) * kTile, p0 = q0 + a.off;  // first query of the tile, its position
    if (k0 < n && (!a.causal || p0 + 31 >= k0)) {
      floatx16 s = {}, dp = {};
#pragma unroll
      for (int kb = 0; kb < DP / 32; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 ah, al;
          read_line(qimg + kb * 4096, col, st, half, ah, al);
          s = mfma_pairs(ah, al, kfh[2 * kb + st], kfl[2 * kb + st], s);
          read_line(gimg + kb * 4096, col, st, half, ah, al);
          dp = mfma_pairs(ah, al, vfh[2 * kb + st], vfl[2 * kb + st], dp);
        }
      const float c = ck * pow2i(-qs), cd = cv * pow2i(-gs);
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) p[v] = s[v] * c;
      if (BIAS) {
        const int64_t lo = k0 - (p0 + 31), hi = k0 + 31 - p0;
        if (lo >= near || hi <= -near) {
          const float f = bias_lds[hi <= -near ? 0 : 2 * near];
#pragma unroll
          for (int v = 0; v < 16; ++v) p[v] += f;
        } else {
          const int rel = (int)(j - p0) - 4 * half;
#pragma unroll
          for (int v = 0; v < 16; ++v) p[v] += bias_lds[near_index(rel - (8 * (v >> 2) + (v & 3)), near)];
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 e = *reinterpret_cast<const float4*>(row_lse + 8 * g + 4 * half);
        p[4 * g] = exp2_fast(p[4 * g] - e.x);
        p[4 * g + 1] = exp2_fast(p[4 * g + 1] - e.y);
        p[4 * g + 2] = exp2_fast(p[4 * g + 2] - e.z);
        p[4 * g + 3] = exp2_fast(p[4 * g + 3] - e.w);
      }
      const bool mask = k0 + 31 >= n || q0 + 31 >= a.Q || (a.causal && p0 < k0 + 31);
      // the first and the last of the tile's queries that see the lane's key, counted from the lane's first one
      const int from = a.causal ? (int)max(min(j - p0, (int64_t)32), (int64_t)0) - 4 * half : -4, to = in ? (int)min(a.Q - q0, (int64_t)32) - 4 * half : -4;
      if (mask) {
#pragma unroll
        for (int v = 0; v < 16; ++v) p[v] = 8 * (v >> 2) + (v & 3) >= from && 8 * (v >> 2) + (v & 3) < to ? p[v] : 0.f;
      }
      // ds, before dv's products (more for the vector ALU to do beside them: 3.7 ms against 4.0 at 4096 x 16384) or, where the table
      // leaves no registers for both p and ds, behind them
      float x[16];
      auto form_ds = [&]() {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 dl = *reinterpret_cast<const float4*>(row_lse + 32 + 8 * g + 4 * half);
          x[4 * g] = p[4 * g] * (dp[4 * g] * cd - dl.x);
          x[4 * g + 1] = p[4 * g + 1] * (dp[4 * g + 1] * cd - dl.y);
          x[4 * g + 2] = p[4 * g + 2] * (dp[4 * g + 2] * cd - dl.z);
          x[4 * g + 3] = p[4 * g + 3] * (dp[4 * g + 3] * cd - dl.w);
        }
        if (mask) {  // (p = 0 leaves 0 only where dp is finite)
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] = 8 * (v >> 2) + (v & 3) >= from && 8 * (v >> 2) + (v & 3) < to ? x[v] : 0.f;
        }
      };
      if (!BIAS) form_ds();
      half8 xh[2], xl[2];
      as_operand(p, fit<DP / 32>(p, gs, FV, dv), xh, xl);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 ah, al;
          read_line(gcol, d * 32 + col, st, half, ah, al);
          dv[d] = mfma_pairs(ah, al, xh[st], xl[st], dv[d]);
        }
      if (BIAS) form_ds();
      as_operand(x, fit<DP / 32>(x, qs, FK, dk), xh, xl);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 ah, al;
          read_line(qcol, d * 32 + col, st, half, ah, al);
          dk[d] = mfma_pairs(ah, al, xh[st], xl[st], dk[d]);
        }
    }
    wait_loads();
    __syncthreads();
  }
  if (j >= a.K) return;
  const int64_t row = (b * a.K + j) * a.Hk + kh, part = (int64_t)split * 2 * a.B * a.K * a.Hk;
  float* dk_out = a.splits > 1 ? a.part + (part + row) * D : a.dk ? a.dk + row * D : nullptr;
  float* dv_out = a.splits > 1 ? a.part + (part + a.B * a.K * a.Hk + row) * D : a.dv ? a.dv + row * D : nullptr;
  if (dk_out) store_row<DP>(dk_out, dk, pow2i(-FK) * a.scale, D, half, a.vec);
  if (!dv_out) return;
  store_row<DP>(dv_out, dv, pow2i(-FV), D, half, a.vec);
  if (bad && in)
    for (int u = u0; u < u1; ++u)
      for (unsigned left = g_info[tile_of(u)].bad; left; left &= left - 1) {
        const int64_t i = (int64_t)(qt0 + u % each) * kTile + __builtin_ctz(left);
        if (!a.causal || j <= i + a.off) put_bad(a.go + ((b * a.Q + i) * a.H + kh * a.G + u / each) * D, D, half, dv_out);
      }
}

// out[i] = sum over the parts of part[s][i], in order
__global__ __launch_bounds__(TPB) void reduce_parts_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, int64_t stride, int splits) {
  const int64_t i = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
  for (int s = 0; s < splits; ++s) sum += part[s * stride + i];
  out[i] = sum;
}

// Sums by position difference of one head over its work-groups, in double and in order: a group of 256 threads takes 64
// differences and the work-groups in four interleaved runs, which meet in order.
__global__ __launch_bounds__(TPB) void table_diff_kernel(Args a, int64_t per_head, double* __restrict__ diff) {
  __shared__ double red[4][64];
  const int span = 2 * a.bk.near + 1, lane = threadIdx.x & 63, run = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
  const int64_t h = blockIdx.y;
  double sum = 0.0;
  if (d < span)
    for (int64_t b = 0; b < a.B; ++b) {
      const float* from = a.part_table + (b * a.H + h) * per_head * span + d;
#pragma unroll 4
      for (int64_t g = run; g < per_head; g += 4) sum += (double)from[g * span];
    }
  red[run][lane] = sum;
  __syncthreads();
  if (run == 0 && d < span) diff[h * span + d] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// dtable[bucket, h] from the sums by difference, and from the rows' far sums where rows were cut in parts.
__global__ __launch_bounds__(TPB) void table_grad_kernel(Args a, const double* __restrict__ diff, float* __restrict__ dtable) {
  __shared__ double red[2][TPB];
  const int span = 2 * a.bk.near + 1, tid = threadIdx.x, buckets = a.bk.both ? 2 * a.bk.side : a.bk.side;
  const int64_t h = blockIdx.x;
  double low = 0.0, high = 0.0;
  if (a.splits > 1)
    for (int64_t r = tid; r < a.B * a.Q; r += TPB) {
      const float* from = a.part_rows + ((r / a.Q * a.H + h) * a.Q + r % a.Q) * a.splits * 8;
      float sum[6] = {};
      for (int s = 0; s < a.splits; ++s) {
        const float4 f = *reinterpret_cast<const float4*>(from + s * 8), g = *reinterpret_cast<const float4*>(from + s * 8 + 4);
        sum[0] += f.x; sum[1] += f.y; sum[2] += f.z; sum[3] += f.w; sum[4] += g.x; sum[5] += g.y;
      }
      low += (double)far_part(sum[0], sum[2], sum[4], sum[5]);
      high += (double)far_part(sum[1], sum[3], sum[4], sum[5]);
    }
  red[0][tid] = low;
  red[1][tid] = high;
  __syncthreads();
  for (int s = TPB / 2; s; s >>= 1) {
    if (tid < s) {
      red[0][tid] += red[0][tid + s];
      red[1][tid] += red[1][tid + s];
    }
    __syncthreads();
  }
  // A bucket's differences lie side by side: a wave adds up one bucket after another.
  const int lane = tid & 63, near = a.bk.near;
  for (int bucket = __builtin_amdgcn_readfirstlane(tid >> 6); bucket < buckets; bucket += TPB / 64) {
    const bool later = bucket >= a.bk.side;  // two sides: keys behind the query
    const int i = later ? bucket - a.bk.side : bucket;
    const int n0 = a.bk.start[i], n1 = i + 1 < a.bk.side ? a.bk.start[i + 1] - 1 : near;
    const int first = later ? near + max(n0, 1) : near - n1, last = later ? near + n1 : (!a.bk.both && i == 0 ? 2 * near : near - n0);
    double sum = 0.0;
    for (int d = first + lane; d <= last; d += 64) sum += diff[h * span + d];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (bucket == bucket_of(a.bk, -a.bk.near)) sum += red[0][0];
    if (bucket == bucket_of(a.bk, a.bk.near)) sum += red[1][0];
    if (lane == 0) dtable[bucket * a.H + h] = (float)sum;
  }
}

template <typename Kernel>
int32_t allow_lds(Kernel* kernel, size_t lds) {
  if (lds > 65536) ENDIA_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  return ENDIA_HIP_OK;
}

template <int DP, bool BIAS>
int32_t dq_launch(Args a, hipStream_t s) {
  // Five tables of position differences (the bias, and a set of sums per wave) stand beside the stages: with the widest tables
  // there is room for one stage only.
  const size_t tables = BIAS ? 5 * (2 * a.bk.near + 1) * 4 : 0;
  a.stages = 2 * DP * 384 + tables <= 160 * 1024 ? 2 : 1;
  const size_t lds = a.stages * DP * 384 + tables;
  int32_t rc = allow_lds(dq_kernel<DP, BIAS>, lds);
  if (rc) return rc;
  const int64_t groups = ceil_div64(a.Q, 128) * a.H * a.B * a.splits;
  hipLaunchKernelGGL((dq_kernel<DP, BIAS>), dim3((unsigned)groups), dim3(TPB), lds, s, a, a.k_info, a.v_info, a.meta);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

template <int DP, bool BIAS>
int32_t dkv_launch(const Args& a, hipStream_t s) {
  const size_t lds = 2 * (DP * 512 + 256) + (BIAS ? (2 * a.bk.near + 1) * 4 : 0);
  int32_t rc = allow_lds(dkv_kernel<DP, BIAS>, lds);
  if (rc) return rc;
  const int64_t groups = ceil_div64(a.K, 128) * a.Hk * a.B * a.splits;
  hipLaunchKernelGGL((dkv_kernel<DP, BIAS>), dim3((unsigned)groups), dim3(TPB), lds, s, a, a.q_info, a.g_info, a.meta);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

template <int DP>
int32_t dq_launch(const Args& a, hipStream_t s) {
  return a.table ? dq_launch<DP, true>(a, s) : dq_launch<DP, false>(a, s);
}
template <int DP>
int32_t dkv_launch(const Args& a, hipStream_t s) {
  return a.table ? dkv_launch<DP, true>(a, s) : dkv_launch<DP, false>(a, s);
}

int32_t reduce_parts(const float* part, float* out, int64_t n, int64_t stride, int splits, hipStream_t s) {
  hipLaunchKernelGGL(reduce_parts_kernel, dim3((unsigned)ceil_div64(n, TPB)), dim3(TPB), 0, s, part, out, n, stride, splits);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace

int64_t table_groups(const Args& a) { return a.B * a.H * ceil_div64(a.Q, 128) * a.splits; }

int32_t launch_dq(const Args& a, int DP, hipStream_t s) {
  int32_t rc = DP == 32 ? dq_launch<32>(a, s) : DP == 64 ? dq_launch<64>(a, s) : DP == 96 ? dq_launch<96>(a, s) : dq_launch<128>(a, s);
  if (rc || a.splits == 1 || !a.dq) return rc;
  const int64_t n = a.B * a.Q * a.H * a.D;
  return reduce_parts(a.part, a.dq, n, n, a.splits, s);
}

int32_t launch_dkv(const Args& a, int DP, hipStream_t s) {
  int32_t rc = DP == 32 ? dkv_launch<32>(a, s) : DP == 64 ? dkv_launch<64>(a, s) : DP == 96 ? dkv_launch<96>(a, s) : dkv_launch<128>(a, s);
  if (rc || a.splits == 1) return rc;
  const int64_t n = a.B * a.K * a.Hk * a.D;
  if (a.dk && (rc = reduce_parts(a.part, a.dk, n, 2 * n, a.splits, s))) return rc;
  return a.dv ? reduce_parts(a.part + n, a.dv, n, 2 * n, a.splits, s) : ENDIA_HIP_OK;
}

int32_t launch_table_grad(const Args& a, double* diff, float* dtable, hipStream_t s) {
  const int span = 2 * a.bk.near + 1;
  hipLaunchKernelGGL(table_diff_kernel, dim3((unsigned)ceil_div64(span, 64), (unsigned)a.H), dim3(TPB), 0, s, a, table_groups(a) / (a.B * a.H), diff);
  hipLaunchKernelGGL(table_grad_kernel, dim3((unsigned)a.H), dim3(TPB), 0, s, a, diff, dtable);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

}  // namespace attention
