// fc_grouped.hip -- bz_grouped_fc: every group's layer on its rows in one launch.
#include "fc_groups.h"

namespace {

using namespace bz::groups;

template <int DT>
int run(const Layer& l, bool gated, hipStream_t st) {
  const Call call = {"bz_grouped_fc", st};
  return gated ? run_layer<DT, true, false>(l, call) : run_layer<DT, false, false>(l, call);
}

}  // namespace

extern "C" int bz_grouped_fc(const bz_grouped_fc_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_grouped_fc: null descriptor");
  const bz_grouped_fc_desc& d = *desc;
  const bool gated = d.act == BZ_ACT_SWIGLU;
  BZ_REQUIRE(d.in_dtype == BZ_F32 || d.in_dtype == BZ_F16 || d.in_dtype == BZ_BF16, "bz_grouped_fc: in_dtype %d", d.in_dtype);
  BZ_REQUIRE(d.out_dtype == d.in_dtype || d.out_dtype == BZ_F32, "bz_grouped_fc: out_dtype %d of in_dtype %d", d.out_dtype, d.in_dtype);
  BZ_REQUIRE(d.m >= 0 && d.n >= 1 && d.k >= 1, "bz_grouped_fc: m %d, n %d, k %d", d.m, d.n, d.k);
  BZ_REQUIRE(!gated || d.n < 1 << 30, "bz_grouped_fc: n %d", d.n);
  BZ_REQUIRE(d.groups >= 1 && d.groups <= BZ_GROUP_MAX_GROUPS, "bz_grouped_fc: groups %d (1..%d)", d.groups, BZ_GROUP_MAX_GROUPS);
  BZ_REQUIRE(d.lda >= d.k && d.ldw >= d.k && d.ldy >= d.n, "bz_grouped_fc: pitches %lld, %lld and %lld for k %d, n %d", (long long)d.lda,
             (long long)d.ldw, (long long)d.ldy, d.k, d.n);
  const int64_t w_rows = gated ? 2 * (int64_t)d.n : d.n;
  BZ_REQUIRE(d.groups == 1 || d.w_stride >= (w_rows - 1) * d.ldw + d.k, "bz_grouped_fc: w_stride %lld", (long long)d.w_stride);
  BZ_REQUIRE(d.rows == nullptr || d.rows_per >= 1, "bz_grouped_fc: rows_per %d", d.rows_per);
  BZ_REQUIRE(d.a_count >= 0 && (d.rows != nullptr || d.a_count >= d.m), "bz_grouped_fc: %lld rows of a, m %d", (long long)d.a_count, d.m);
  if (!gated) {
    const int rc = bz::layer_act("bz_grouped_fc", d.act, d.act_size, d.act_p0, d.act_p1, d.act_p2, d.n);
    if (rc != BZ_OK) return rc;
  }
  if (d.m == 0) return BZ_OK;
  BZ_REQUIRE((d.a || d.a_count == 0) && d.w && d.y && d.offsets, "bz_grouped_fc: null pointer");
  Layer l = {};
  l.a = (const char*)d.a;
  l.w = (const char*)d.w;
  l.y = d.y;
  l.rows = d.rows;
  l.offsets = d.offsets;
  l.a_count = d.a_count;
  l.lda = d.lda;
  l.ldw = d.ldw;
  l.w_stride = d.w_stride;
  l.ldy = d.ldy;
  l.m = d.m;
  l.n = d.n;
  l.k = d.k;
  l.groups = d.groups;
  l.rows_per = d.rows ? d.rows_per : 1;
  l.ep.bias = d.bias;
  l.ep.p0 = d.act_p0;
  l.ep.p1 = d.act_p1;
  l.ep.p2 = d.act_p2;
  l.ep.bias_rows = d.bias ? 1 : 0;
  l.ep.act = gated ? BZ_ACT_NONE : d.act;
  l.ep.act_size = d.act_size;
  l.ep.dice_nosqrt = d.dice_nosqrt;
  l.ep.alpha = l.ep.beta = 1.f;
  l.ep.act_alpha = d.act_alpha;
  l.p_stride = d.act == BZ_ACT_PRELU ? d.act_size : d.n;
  const hipStream_t st = bz::as_stream(stream);
  l.out_f32 = d.out_dtype == BZ_F32;
  if (d.in_dtype == BZ_F32) return run<BZ_F32>(l, gated, st);
  if (d.in_dtype == BZ_F16) return run<BZ_F16>(l, gated, st);
  return run<BZ_BF16>(l, gated, st);
}
