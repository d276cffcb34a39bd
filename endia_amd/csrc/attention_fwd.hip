// Attention over tiles of keys on the matrix cores, operands as pairs of fp16 (fp16_pairs.h).
//
// A wave owns 32 queries of one head, a work-group 4 x 32. Per tile of 32 keys it forms S^T = K Q^T (the tile's row image from
// LDS times the wave's queries, which stay in registers), so that a lane holds 16 scores of ONE query: maximum and sum need a
// single exchange between the two halves of the wave, and the probabilities, split into pairs where they are, already are the
// right operand of O^T = V^T P^T (the column image holds the positions in accumulator order). Scores live in base 2; the running
// maximum may lag behind by up to 4 (kSlack) before the sums are brought to the new one, and since a tile of v carries a shift of
// its own, the output accumulator has a running shift as it has a running maximum. The next tile's images travel from memory
// straight into the other half of the LDS meanwhile.
// Bound: the matrix pipe and the vector ALU about evenly (per 32 x 32 block 6 DP / 16 matrix instructions of 32 cycles and about
// 20 vector instructions for each of 16 scores a lane). Measured, as fp32 products: 4096 queries x 16384 keys, 16 heads of 128: 1.46 ms =
// 376 TFLOP/s; 8 x 448 x 1500, 16 heads of 64: 93 us = 185; 5001 causal, 16 heads of 128, with buckets: 394 to 404 us = 253 to 260.
#include "attention.h"

namespace attention {

namespace {

using namespace pairs;
constexpr int TPB = 256;
constexpr float kSlack = 4.f;  // p <= 2^kSlack
constexpr int kPTop = 11;      // probabilities are scaled by up to 2^kPTop: 2^(kPTop + kSlack) fits fp16

template <int DP, bool BIAS>
__global__ __launch_bounds__(TPB, 2) void forward_kernel(Args a, const TileInfo* __restrict__ k_info, const TileInfo* __restrict__ v_info) {
  constexpr int STAGE = DP * 256;  // row image of k, column image of v
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* bias_lds = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int64_t qtiles = (a.Q + 127) / 128;
  uint32_t id = xcd_contiguous(blockIdx.x, gridDim.x);
  const uint32_t split = id % (uint32_t)a.splits;
  id /= (uint32_t)a.splits;
  const uint32_t hb = id / (uint32_t)qtiles;
  // (causal: the last queries see the most keys and go first)
  const int64_t qt = a.causal ? qtiles - 1 - id % (uint32_t)qtiles : id % (uint32_t)qtiles, h = hb % (uint32_t)a.H, b = hb / (uint32_t)a.H, kh = (uint32_t)h / (uint32_t)a.G;
  const int D = (int)a.D;
  const int64_t i = qt * 128 + wave * 32 + col;
  const bool in = i < a.Q;

  half8 qh[DP / 16], ql[DP / 16];
  const float* qrow = a.q + b * a.qs[0] + min(i, a.Q - 1) * a.qs[1] + h * a.qs[2];
  const int qshift = load_fragments<DP>(qrow, in, D, a.vec, half, qh, ql);
  const float cq = a.scale * kLog2e * pow2i(-qshift);
  if (BIAS) load_bias(a, (int)h, bias_lds, tid, TPB);

  const int n = key_count(a, b);
  const int64_t place = i + a.off;
  int64_t see = n;
  if (a.causal && place + 1 < see) see = place + 1 > 0 ? place + 1 : 0;
  const int limit = (int)see;  // keys this lane's query may see
  // tiles of the work-group (its last query sees the most keys), of this part, and those that no lane of the wave masks
  int64_t most = n;
  if (a.causal) {
    const int64_t last = min(a.Q - 1, qt * 128 + 127) + a.off + 1;
    most = last < most ? (last > 0 ? last : 0) : most;
  }
  const int tiles = (int)((most + kTile - 1) / kTile), per = (tiles + a.splits - 1) / a.splits;
  const int t0 = (int)split * per, t1 = min(tiles, t0 + per);
  const int64_t wave_first = qt * 128 + wave * 32 + a.off;  // position of the wave's first query
  int64_t clear_keys = n;
  if (a.causal && wave_first + 1 < clear_keys) clear_keys = wave_first + 1 > 0 ? wave_first + 1 : 0;

  const int64_t ktiles = (a.K + kTile - 1) / kTile, tile_at = (b * a.Hk + kh) * ktiles;
  auto request = [&](int t, int stage) {
    const char* kr = a.k_rows + (tile_at + t) * (DP * 128) + lane * 16;
    const char* vc = a.v_cols + (tile_at + t) * (DP * 128) + lane * 16;
    char* to = smem + stage * STAGE;
#pragma unroll
    for (int p = 0; p < DP / 32; ++p) {
      const int at = (p * 4 + wave) * 1024;
      load_to_lds(kr + at, to + at);
      load_to_lds(vc + at, to + DP * 128 + at);
    }
  };

  floatx16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) o[d] = floatx16{};
  float m = -INFINITY, l = 0.f;
  unsigned bad = 0;
  int F = 2 * kMaxShift;  // the output accumulator holds 2^F times the sums of p v
  if (t0 < t1) request(t0, 0);
  wait_loads();
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int stage = (t - t0) & 1;
    if (t + 1 < t1) request(t + 1, stage ^ 1);
    const char* kimg = smem + stage * STAGE;
    const char* vimg = kimg + DP * 128;
    if (qt * 128 + wave * 32 < a.Q) {
      floatx16 s = {};
#pragma unroll
      for (int kb = 0; kb < DP / 32; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 kh8, kl8;
          read_line(kimg + kb * 4096, col, st, half, kh8, kl8);
          s = mfma_pairs(kh8, kl8, qh[2 * kb + st], ql[2 * kb + st], s);
        }
      const float c = cq * pow2i(-k_info[tile_at + t].shift);
      const int key0 = t * kTile + 4 * half;
      float x[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = s[v] * c;
      if (BIAS) {
        const int64_t lo = (int64_t)t * kTile - (wave_first + 31), hi = (int64_t)t * kTile + 31 - wave_first;
        if (lo >= a.bk.near || hi <= -a.bk.near) {  // every pair of the block is in a last bucket
          const float far = bias_lds[hi <= -a.bk.near ? 0 : 2 * a.bk.near];
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] += far;
        } else {
          const int rel = (int)(key0 - place);  // (within the block's reach of +-near: far from 32-bit limits)
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] += bias_lds[near_index(rel + 8 * (v >> 2) + (v & 3), a.bk.near)];
        }
      }
      if ((int64_t)(t + 1) * kTile > clear_keys) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = key0 + 8 * (v >> 2) + (v & 3) < limit ? x[v] : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int v = 1; v < 16; ++v) top = fmaxf(top, x[v]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m + kSlack || (m == -INFINITY && top > m))) {
        const float now = fmaxf(m, top);
        const float keep = m == -INFINITY ? 0.f : exp2_fast(m - now);
        m = now;
        l *= keep;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= keep;
      }
      const int vs = v_info[tile_at + t].shift;
      bad |= v_info[tile_at + t].bad;
      if (kPTop + vs < F) {
        if (F < 2 * kMaxShift) {
          const float down = pow2i(kPTop + vs - F);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d][v] *= down;
        }
        F = kPTop + vs;
      }
      // A tile whose v is 2^70 below the largest so far would leave no bits of p: below 2^-60 it is added as if it were larger. (What is
      // below 2^-36 of the largest v so far is lost beside it: nothing to the rows that attend to that one too.)
      const int up = max(F - vs, -60);
      const float base = m == -INFINITY ? -INFINITY : m - (float)up;  // -inf: no key yet, exp2(-inf - -inf) is caught below
      float sum = 0.f;
      half8 ph[2], pl[2];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        x[v] = x[v] == -INFINITY ? 0.f : exp2_fast(x[v] - base);
        sum += x[v];
      }
      l += sum * pow2i(-up);
      {
        float y[8];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[8 * st + e];
          split8(y, ph[st], pl[st]);
        }
      }
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          half8 vh8, vl8;
          read_line(vimg, d * 32 + col, st, half, vh8, vl8);
          o[d] = mfma_pairs(vh8, vl8, ph[st], pl[st], o[d]);
        }
    }
    wait_loads();
    __syncthreads();
  }

  if (!in) return;
  l += __shfl_xor(l, 32, 64);
  const float down = pow2i(-F);
  const int64_t part = ((b * a.H + h) * a.Q + i) * a.splits + split;
  float* out = a.splits == 1 ? a.o + ((b * a.Q + i) * a.H + h) * D : a.part + part * D;
  if (a.splits == 1) {
    const float inv = l != 0.f ? down / l : 0.f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = d * 32 + 8 * j + 4 * half;
        if (a.vec) {
          if (at < D)
            *reinterpret_cast<float4*>(out + at) = make_float4(o[d][4 * j] * inv, o[d][4 * j + 1] * inv, o[d][4 * j + 2] * inv, o[d][4 * j + 3] * inv);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at + e < D) out[at + e] = o[d][4 * j + e] * inv;
        }
      }
    if (half == 0 && a.lse) a.lse[(b * a.H + h) * a.Q + i] = l != 0.f ? (m + log2_fast(l)) * kLn2 : -INFINITY;
  } else {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int at = d * 32 + 8 * (v >> 2) + 4 * half + (v & 3);
        if (at < D) out[at] = o[d][v] * down;
      }
    if (half == 0) {
      a.part_ml[2 * part] = m;
      a.part_ml[2 * part + 1] = l;
    }
  }
  if (bad)
    for (int t = t0; t < t1; ++t)
      for (unsigned left = v_info[tile_at + t].bad; left; left &= left - 1) {
        const int j = t * kTile + __builtin_ctz(left);
        if (j < limit) put_bad(a.v + b * a.vs[0] + j * a.vs[1] + kh * a.vs[2], D, half, out);
      }
}

template <int DP, bool BIAS>
int32_t launch(const Args& a, hipStream_t s) {
  const int64_t groups = ceil_div64(a.Q, 128) * a.H * a.B * a.splits;
  const size_t lds = 2 * DP * 256 + (BIAS ? (2 * a.bk.near + 1) * 4 : 0);
  if (lds > 65536)
    ENDIA_HIP_CALL(hipFuncSetAttribute(reinterpret_cast<const void*>(forward_kernel<DP, BIAS>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL((forward_kernel<DP, BIAS>), dim3((unsigned)groups), dim3(TPB), lds, s, a, a.k_info, a.v_info);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

template <int DP>
int32_t launch(const Args& a, hipStream_t s) {
  return a.table ? launch<DP, true>(a, s) : launch<DP, false>(a, s);
}

}  // namespace

int32_t launch_forward(const Args& a, int DP, hipStream_t s) {
  int32_t rc = DP == 32 ? launch<32>(a, s) : DP == 64 ? launch<64>(a, s) : DP == 96 ? launch<96>(a, s) : launch<128>(a, s);
  return rc || a.splits == 1 ? rc : launch_combine(a, s);
}

}  // namespace attention
