// The operands of the attention products that every work-group reads again, split into pairs of fp16 once per call and laid
// out as the LDS images that the matrix-core kernels load.
//
// A tile is 32 positions of one head. Its row image holds, per 32 elements of the head dimension, 32 lines (one per position)
// of 128 bytes: 32 hi, 32 lo; its column image one line per element of the head dimension: the 32 positions' hi, then lo,
// with the positions in the order in which an accumulator of the 32 x 32 product holds its rows (see the order below), so
// that a product of probabilities can take them from the accumulator registers as they are. One shift per tile. Infinities and NaN
// stay what they are in the row image, whose products are masked by selection, and are zeros in the column image (see put_bad).
// Bound: HBM. Reads 4 and writes 4 or 8 bytes per element; keys that no query sees and queries that see no key become zeros. Measured: 36 us on
// average for the three launches of a step over 8 x 448 queries and 8 x 1500 keys of 16 heads of 64 (0.49 GB in all: 4.5 TB/s).
#include "attention.h"

namespace attention {

namespace {

constexpr int TPB = 256;

struct Source {
  const float* x;
  int64_t sb, sp, sh, L, H;
  int64_t first;    // positions before it become zeros: queries that see no key
  int use_lengths;  // so do those behind the sequence's keys
  char *rows, *cols;
  TileInfo* info;
  const float *o, *lse;  // with meta: the forward pass's output and lse beside go = x
  float* meta;
};

template <int DP, bool VEC>
__global__ __launch_bounds__(TPB) void tiles_kernel(Args a, Source s0, Source s1) {
  constexpr int PER_ROW = DP / 8, ITEMS = (32 * PER_ROW + TPB - 1) / TPB;
  __shared__ __attribute__((aligned(16))) char cols[DP * 128];
  __shared__ float red[TPB / 64];
  __shared__ unsigned bad_positions[TPB / 64];
  __shared__ float dsum[32][PER_ROW];
  const bool second = blockIdx.y >= s0.H;
  const Source& src = second ? s1 : s0;
  const int64_t h = blockIdx.y - (second ? s0.H : 0), b = blockIdx.z, tile = blockIdx.x;
  const int64_t tiles = (src.L + kTile - 1) / kTile;
  if (tile >= tiles) return;
  const int64_t at = (b * src.H + h) * tiles + tile;
  const int n = src.use_lengths ? key_count(a, b) : (int)src.L;
  const int D = (int)a.D, tid = threadIdx.x;
  float x[ITEMS][8];
  float amax = 0.f;
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int item = tid + i * TPB, row = item / PER_ROW, ch = item % PER_ROW;
    const int64_t p = tile * kTile + row;
    const bool in = item < 32 * PER_ROW && p >= src.first && p < n;
    const float* base = src.x + b * src.sb + min(p, src.L - 1) * src.sp + h * src.sh;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int d = ch * 8 + 4 * j;
      const float4 f = load4<VEC>(base, d, D, in);
      x[i][4 * j] = f.x;
      x[i][4 * j + 1] = f.y;
      x[i][4 * j + 2] = f.z;
      x[i][4 * j + 3] = f.w;
      if (src.meta) {
        const float4 o = load4<VEC>(src.o + ((b * src.L + min(p, src.L - 1)) * src.H + h) * D, d, D, in);
        dot += (f.x * o.x + f.y * o.y) + (f.z * o.z + f.w * o.w);
      }
    }
    if (src.meta && item < 32 * PER_ROW) dsum[row][ch] = dot;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      amax = fmaxf(amax, pairs::finite_abs(x[i][e]));
      bad |= __builtin_fabsf(x[i][e]) < INFINITY ? 0u : 1u << (row & 31);
    }
  }
  amax = wave_max(amax);
  if (__any(bad != 0)) {
#pragma unroll
    for (int o = 32; o; o >>= 1) bad |= (unsigned)__shfl_xor((int)bad, o, 64);
  }
  if ((tid & 63) == 0) {
    red[tid >> 6] = amax;
    bad_positions[tid >> 6] = bad;
  }
  __syncthreads();
  const int shift = pairs::shift_of(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  bad = bad_positions[0] | bad_positions[1] | bad_positions[2] | bad_positions[3];
  if (tid == 0) src.info[at] = {shift, bad};
  if (src.meta && tid < 32) {
    const int64_t p = tile * kTile + tid;
    float delta = 0.f;
    for (int c = 0; c < PER_ROW; ++c) delta += dsum[tid][c];
    // a row without keys, or behind the last query: exp2(s - inf) = 0 for every score
    const float e = p < src.L ? src.lse[(b * src.H + h) * src.L + p] : -INFINITY;
    src.meta[at * 64 + tid] = e == -INFINITY ? INFINITY : e * kLog2e;
    src.meta[at * 64 + 32 + tid] = delta;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int item = tid + i * TPB, row = item / PER_ROW, ch = item % PER_ROW;
    if (item >= 32 * PER_ROW) break;
    pairs::half8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = pairs::scaled(x[i][e], shift);
    pairs::split8(x[i], hi, lo);
    if (src.rows) {
      char* line = src.rows + at * (DP * 128) + ((ch >> 2) * 32 + row) * 128;
      *reinterpret_cast<pairs::half8*>(line + (((ch & 3) ^ (row & 7)) << 4)) = hi;
      *reinterpret_cast<pairs::half8*>(line + (((4 + (ch & 3)) ^ (row & 7)) << 4)) = lo;
    }
    if (src.cols) {
      if (bad) {  // (uniform: of the whole tile)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = __builtin_fabsf(x[i][e]) < INFINITY ? x[i][e] : 0.f;
        pairs::split8(x[i], hi, lo);
      }
      // accumulator order: slot 8 h + e of a group of 16 holds position 8 (e / 4) + 4 h + e % 4
      const int w = row & 15, piece = 2 * (row >> 4) + ((w >> 2) & 1), e = ((w >> 3) << 2) | (w & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int line = ch * 8 + j;
        *reinterpret_cast<_Float16*>(cols + line * 128 + ((piece ^ (line & 7)) << 4) + 2 * e) = hi[j];
        *reinterpret_cast<_Float16*>(cols + line * 128 + (((4 + piece) ^ (line & 7)) << 4) + 2 * e) = lo[j];
      }
    }
  }
  if (src.cols) {
    __syncthreads();
    for (int i = tid; i < DP * 8; i += TPB)
      *reinterpret_cast<float4*>(src.cols + at * (DP * 128) + i * 16) = *reinterpret_cast<const float4*>(cols + i * 16);
  }
}

template <int DP>
int32_t launch(const Args& a, const Source& s0, const Source& s1, hipStream_t s) {
  const int64_t L = s0.L > s1.L ? s0.L : s1.L;
  const dim3 grid((unsigned)ceil_div64(L, kTile), (unsigned)(s0.H + s1.H), (unsigned)a.B);
  if (a.vec) hipLaunchKernelGGL((tiles_kernel<DP, true>), grid, dim3(TPB), 0, s, a, s0, s1);
  else hipLaunchKernelGGL((tiles_kernel<DP, false>), grid, dim3(TPB), 0, s, a, s0, s1);
  ENDIA_LAUNCH_CHECK();
  return ENDIA_HIP_OK;
}

int32_t launch(const Args& a, int DP, const Source& s0, const Source& s1, hipStream_t s) {
  switch (DP) {
    case 32: return launch<32>(a, s0, s1, s);
    case 64: return launch<64>(a, s0, s1, s);
    case 96: return launch<96>(a, s0, s1, s);
    default: return launch<128>(a, s0, s1, s);
  }
}

}  // namespace

int32_t launch_tiles(const Args& a, int DP, bool backward, hipStream_t s) {
  const Source k = {a.k, a.ks[0], a.ks[1], a.ks[2], a.K, a.Hk, 0, 1, a.k_rows, a.k_cols, a.k_info, nullptr, nullptr, nullptr};
  const Source v = {a.v, a.vs[0], a.vs[1], a.vs[2], a.K, a.Hk, 0, 1, a.v_rows, a.v_cols, a.v_info, nullptr, nullptr, nullptr};
  int32_t rc = launch(a, DP, k, v, s);
  if (rc || !backward) return rc;
  const int64_t first = a.causal && a.off < 0 ? -a.off : 0;
  const Source q = {a.q, a.qs[0], a.qs[1], a.qs[2], a.Q, a.H, first, 0, a.q_rows, a.q_cols, a.q_info, nullptr, nullptr, nullptr};
  const Source g = {a.go, a.Q * a.H * a.D, a.H * a.D, a.D, a.Q, a.H, first, 0, a.g_rows, a.g_cols, a.g_info, a.out, a.lse, a.meta};
  return launch(a, DP, q, g, s);
}

}  // namespace attention
