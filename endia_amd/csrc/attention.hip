// Attention of queries over keys of another length, with an optional learned position bias by buckets, and its gradient: the
// entry points, their checks, and the choice of kernels. Stands beside matmul and linear
// (endia/functional/binary_ops/matmul_op.mojo): the reference would spell it in matmul, exp, sum and div nodes.
//
//   s_ij = scale q_i . k_j + table[bucket(j - (i + query_offset))]     masked: j >= key_lengths[b], causal j > i + query_offset
//   p = softmax over the keys that are left (a row with none: zeros)   o = p v
//   dv = p^T do,  dp = do v^T,  ds = p (dp - do . o),  dq = scale ds k,  dk = scale ds^T q,  dtable = sums of ds by bucket
#include "attention.h"

#include <math.h>

using namespace endia;
using namespace attention;

namespace {

void make_buckets(const endia_hip_attention_desc* d, Buckets* t) {
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
  t->near = t->start[t->side - 1];  // (max_distance itself is in the last bucket, so all starts are set)
}

int32_t check(const char* who, const endia_hip_attention_desc* d, const float* q, const float* k, const float* v, const float* table) {
  ENDIA_CHECK_ARG(d && q && k && v, "%s: null pointer", who);
  ENDIA_CHECK_ARG(d->B > 0 && d->Q > 0 && d->K > 0 && d->H > 0 && d->Hk > 0 && d->D > 0, "%s: sizes must be positive", who);
  ENDIA_CHECK_ARG(d->H % d->Hk == 0, "%s: %lld query heads cannot share %lld key heads evenly", who, (long long)d->H, (long long)d->Hk);
  ENDIA_CHECK_ARG(d->Q < (1ll << 24) && d->K <= (1ll << 24), "%s: more than 2^24 positions (lengths are held in fp32)", who);
  ENDIA_CHECK_ARG(d->query_offset > -(1ll << 30) && d->query_offset < (1ll << 30), "%s: query_offset out of range", who);
  ENDIA_CHECK_ARG(isfinite(d->scale), "%s: scale must be finite", who);
  if (d->D > ENDIA_ATTENTION_MAX_DIM || d->B > 65535 || d->H > 32767 || d->B * d->H > 65535 || d->B * d->H * ceil_div64(d->Q, 32) >= (1ll << 31) ||
      d->B * d->Hk * ceil_div64(d->K, 32) >= (1ll << 31))
    return fail(ENDIA_HIP_ERR_UNSUPPORTED, "%s: head dimension %lld above %d, more than 65535 heads over the batch, or too many rows", who,
                (long long)d->D, ENDIA_ATTENTION_MAX_DIM);
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

bool on16(const float* p, const int64_t* strides) {
  bool ok = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  for (int i = 0; strides && i < 3; ++i) ok = ok && strides[i] % 4 == 0;
  return ok;
}

Args make_args(const endia_hip_attention_desc* d, const float* q, const float* k, const float* v, const float* lengths, const float* table) {
  Args a = {};
  a.B = d->B; a.Q = d->Q; a.K = d->K; a.H = d->H; a.Hk = d->Hk; a.D = d->D; a.G = d->H / d->Hk;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d->q_strides[i];
    a.ks[i] = d->k_strides[i];
    a.vs[i] = d->v_strides[i];
  }
  a.off = d->query_offset;
  a.scale = d->scale;
  a.causal = d->causal ? 1 : 0;
  a.seen = d->K;
  if (a.causal && d->Q + d->query_offset < a.seen) a.seen = d->Q + d->query_offset > 0 ? d->Q + d->query_offset : 0;
  a.q = q; a.k = k; a.v = v; a.lengths = lengths; a.table = table;
  a.vec = d->D % 4 == 0 && on16(q, d->q_strides) && on16(k, d->k_strides) && on16(v, d->v_strides);
  a.splits = 1;
  if (table) make_buckets(d, &a.bk);
  return a;
}

int padded_dim(int64_t D) { return (int)((D + 31) / 32 * 32); }

// Into how many parts a walk of `steps` is cut so that `groups` work-groups become about `want`; a part has at least `least` steps.
int parts(int64_t groups, int64_t want, int64_t steps, int64_t least) {
  int64_t p = (want + groups - 1) / groups;
  if (p > steps / least) p = steps / least;
  return (int)(p < 1 ? 1 : p > 256 ? 256 : p);
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
  Args a = make_args(d, q, k, v, key_lengths, table);
  a.vec = a.vec && on16(o, nullptr);
  a.o = o;
  a.lse = lse;
  const int64_t rows = a.G * a.Q, cus = ctx().cu_count;
  Scratch w;
  // Up to 16 rows per key head they are streamed past the keys, up to 4 at a time (8 at a time, with half the waves
  // in flight: 332 us against 256 for 8 rows of 64 sequences); from there on the tiles of the matrix cores are
  // faster (16 heads of 64, 64 sequences of 1000 to 2000 keys: 16 rows 466 us against 579, 24 rows 676 against 582).
  if (rows <= 16) {
    int R = rows == 1 ? 1 : rows == 2 ? 2 : 4;
    while (table && R > 1 && R * (2 * a.bk.near + 1) * 4 > 32 * 1024) R /= 2;  // a bias table per head of the rows
    const int64_t step = (a.D <= 32 ? 32 : a.D <= 64 ? 16 : 8) * (R <= 2 ? 4 : 2);
    a.splits = parts(ceil_div64(rows, R) * a.B * a.Hk, 4 * cus, ceil_div64(a.K, step), 2);
    if (a.splits > 1) {
      const int64_t n = a.B * a.H * a.Q * a.splits, part = w.want(4 * n * a.D), ml = w.want(8 * n);
      if ((rc = w.get())) return rc;
      a.part = w.at<float>(part);
      a.part_ml = w.at<float>(ml);
    }
    return launch_rows(a, R, st);
  }
  const int DP = padded_dim(a.D);
  const int64_t tiles = ceil_div64(a.K, kTile), images = a.B * a.Hk * tiles * DP * 128;
  a.splits = parts(ceil_div64(a.Q, 128) * a.H * a.B, cus, tiles, 4);
  const int64_t n = a.splits > 1 ? a.B * a.H * a.Q * a.splits : 0;
  const int64_t kr = w.want(images), vc = w.want(images), ks = w.want(sizeof(TileInfo) * a.B * a.Hk * tiles), vs = w.want(sizeof(TileInfo) * a.B * a.Hk * tiles),
                part = w.want(4 * n * a.D), ml = w.want(8 * n);
  if ((rc = w.get())) return rc;
  a.k_rows = w.at<char>(kr);
  a.v_cols = w.at<char>(vc);
  a.k_info = w.at<TileInfo>(ks);
  a.v_info = w.at<TileInfo>(vs);
  a.part = w.at<float>(part);
  a.part_ml = w.at<float>(ml);
  if ((rc = launch_tiles(a, DP, false, st))) return rc;
  return launch_forward(a, DP, st);
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
  Args a = make_args(d, q, k, v, key_lengths, table);
  a.vec = a.vec && on16(o, nullptr) && on16(go, nullptr) && on16(dq, nullptr) && on16(dk, nullptr) && on16(dv, nullptr);
  a.out = o;
  a.lse = const_cast<float*>(lse);
  a.go = go;
  a.dq = dq; a.dk = dk; a.dv = dv;
  const int DP = padded_dim(a.D);
  const int64_t cus = ctx().cu_count, kt = ceil_div64(a.K, kTile), qt = ceil_div64(a.Q, kTile);
  const int64_t kn = a.B * a.Hk * kt, qn = a.B * a.H * qt, image = DP * 128;
  const bool queries = dq || dtable, keys = dk || dv;
  Args aq = a, ak = a;
  aq.splits = parts(ceil_div64(a.Q, 128) * a.H * a.B, cus, kt, 4);
  ak.splits = parts(ceil_div64(a.K, 128) * a.Hk * a.B, cus, a.G * qt, 4);
  Scratch w;
  const int64_t kr = w.want(kn * image), kc = w.want(kn * image), vr = w.want(kn * image), qr = w.want(qn * image), qc = w.want(qn * image),
                gr = w.want(qn * image), gc = w.want(qn * image), ki = w.want(sizeof(TileInfo) * kn), vi = w.want(sizeof(TileInfo) * kn),
                qi = w.want(sizeof(TileInfo) * qn), gi = w.want(sizeof(TileInfo) * qn), meta = w.want(256 * qn);
  const int64_t part_q = aq.splits > 1 ? 4 * aq.splits * a.B * a.Q * a.H * a.D : 0, part_k = ak.splits > 1 ? 8 * ak.splits * a.B * a.K * a.Hk * a.D : 0;
  const int64_t part = w.want(part_q > part_k ? part_q : part_k);  // (one after the other on the stream)
  const int64_t span = 2 * a.bk.near + 1, table_part = w.want(dtable ? table_groups(aq) * span * 4 : 0), diff = w.want(dtable ? 8 * a.H * span : 0),
                table_rows = w.want(dtable && aq.splits > 1 ? 32 * a.B * a.H * a.Q * aq.splits : 0);
  if ((rc = w.get())) return rc;
  for (Args* x : {&a, &aq, &ak}) {
    x->k_rows = w.at<char>(kr); x->k_cols = w.at<char>(kc); x->v_rows = w.at<char>(vr); x->q_rows = w.at<char>(qr);
    x->q_cols = w.at<char>(qc); x->g_rows = w.at<char>(gr); x->g_cols = w.at<char>(gc);
    x->k_info = w.at<TileInfo>(ki); x->v_info = w.at<TileInfo>(vi); x->q_info = w.at<TileInfo>(qi); x->g_info = w.at<TileInfo>(gi);
    x->meta = w.at<float>(meta);
    x->part = w.at<float>(part);
    x->part_table = dtable ? w.at<float>(table_part) : nullptr;
    x->part_rows = w.at<float>(table_rows);
  }
  if ((rc = launch_tiles(a, DP, true, st))) return rc;
  if (queries && (rc = launch_dq(aq, DP, st))) return rc;
  if (dtable && (rc = launch_table_grad(aq, w.at<double>(diff), dtable, st))) return rc;
  if (keys && (rc = launch_dkv(ak, DP, st))) return rc;
  return ENDIA_HIP_OK;
}

}  // extern "C"
