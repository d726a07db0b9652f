// fc_adapters.hip -- bz_fc_adapters: a shared layer and beside it each row's own low-rank product.  Two launches: the low-rank factors of
// all rows, then the layer, which adds their products with the adapters' second factors to its tiles.
#include "fc_groups.h"

namespace {

using namespace bz::groups;

// Low-rank factors: low[r] = scale[g] * (a[r] * down[g]^T), g = ids[r].  A workgroup owns 32 rows and 32 of the rank, its waves share K
// (Split); the distinct adapters of the rows are taken one after the other, or by several workgroups where rows are few (adapters whose
// first row is a workgroup's, every gridDim.z-th row), and each row keeps its own one's.  An adapter of few rows (kDots) is left to plain vector instructions.
// 2-byte layers keep a factor as two bf16s, together 16 bits of its mantissa (an infinite one as itself and 0), fp32 layers as it is; zeros
// between rank and low_rank.  Rows without an adapter are not written, and nobody reads them into a result.
// Bound by the rows' way in, and by blocks whose rows have two adapters, which take two turns: 8192 bf16 rows of 4096, rank 32, 67 MB in
// 29 us (37 with blocks dealt over the XCDs).  Few rows by the chain ids, rows, sums: 32 rows of 2048 with an adapter each 4.9 us.
struct Low {
  const char* a;
  const char* down;
  const int32_t* ids;
  const float* scale;
  char* low;
  int64_t lda, ld_down, down_stride;
  int m, k, adapters, rank, low_rank;
};

template <int DT>
__device__ __forceinline__ void put_low(const Low& l, int row, int r, float v) {
  char* out = l.low + (int64_t)row * l.low_rank * 4;
  if constexpr (DT == BZ_F32) {
    ((float*)out)[r] = v;
  } else {
    // (above the largest bf16 by less than half a step that one, not infinity)
    const float most = 0x1.fep127f, in_reach = fabsf(v) < __builtin_huge_valf() ? fminf(fmaxf(v, -most), most) : v;
    const __hip_bfloat16 hi = __float2bfloat16(in_reach);
    const float rest = v - __bfloat162float(hi);
    ((__hip_bfloat16*)out)[r] = hi;
    ((__hip_bfloat16*)out)[l.low_rank + r] = __float2bfloat16(fabsf(rest) < __builtin_huge_valf() ? rest : 0.f);
  }
}

constexpr int kLowWaves = 8, kDots = 4;

// Factors of the rows of `match` (ROWS of them, or fewer) and `ranks` rows of `down` from r0 on: a wave takes two of those at a time, its
// lanes 16 bytes side by side of each and of the rows, so that all of them are on their way together.
template <int DT, int ROWS>
__device__ __forceinline__ void dots(const Low& l, int m0, uint32_t match, const char* down, float scale, int r0, int ranks) {
  constexpr int ES = In<DT>::kSize, CH = In<DT>::kChunk, AT_ONCE = 2;
  using bz::rows::Chunk;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const char* x[ROWS];
  int row[ROWS];
  uint32_t left = match;
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    row[t] = m0 + __builtin_ctz(left != 0 ? left : match);  // (one of them again where there are fewer)
    left &= left - 1;
    x[t] = l.a + (int64_t)row[t] * l.lda * ES;
  }
  for (int r = wave * AT_ONCE; r < ranks; r += kLowWaves * AT_ONCE) {
    const char* d[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) d[i] = down + (int64_t)min(r0 + r + i, l.rank - 1) * l.ld_down * ES;
    float sum[AT_ONCE][ROWS] = {};
    auto add = [&](const Chunk<DT> (&u)[AT_ONCE], const Chunk<DT> (&v)[ROWS]) {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int t = 0; t < ROWS; ++t)
#pragma unroll
          for (int e = 0; e < CH; ++e) sum[i][t] = fmaf(u[i].at(e), v[t].at(e), sum[i][t]);
    };
    const int whole = l.k / (64 * CH);  // steps that all lanes take: no lane's loads wait for another's end
#pragma unroll 4
    for (int step = 0; step < whole; ++step) {
      const int64_t at = ((int64_t)step * 64 + lane) * 16;
      Chunk<DT> u[AT_ONCE], v[ROWS];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) __builtin_memcpy(&u[i].raw, d[i] + at, 16);
#pragma unroll
      for (int t = 0; t < ROWS; ++t) __builtin_memcpy(&v[t].raw, x[t] + at, 16);
      add(u, v);
    }
    const int k = (whole * 64 + lane) * CH;
    if (k < l.k) {
      Chunk<DT> u[AT_ONCE], v[ROWS];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) u[i].raw = row_chunk<DT>(d[i], k, l.k);
#pragma unroll
      for (int t = 0; t < ROWS; ++t) v[t].raw = row_chunk<DT>(x[t], k, l.k);
      add(u, v);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int t = 0; t < ROWS; ++t) {
        const float v = bz::rows::reduce<64>(sum[i][t], [](float a, float b) { return a + b; });
        if (lane == 0 && r + i < ranks) put_low<DT>(l, row[t], r0 + r + i, r0 + r + i < l.rank ? scale * v : 0.f);
      }
  }
}

template <int DT, bool ALIGNED, int COLS>
__global__ __launch_bounds__(kLowWaves * 64) void bz_adapters_low_kernel(Low l) {
  using Parts = Split<DT, kLowWaves, ALIGNED, COLS>;
  constexpr int ES = In<DT>::kSize, NT = kLowWaves * 64;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, frow = tid & 31;
  // blocks side by side on one XCD, whose L2 their adapters' `down` then comes from
  const int each = gridDim.x / 8, more = gridDim.x % 8, xcd = blockIdx.x % 8;
  const int m0 = (xcd * each + min(xcd, more) + (int)blockIdx.x / 8) * 32, r0 = blockIdx.y * COLS, ranks = min(COLS, l.low_rank - r0);
  int id = m0 + frow < l.m ? l.ids[m0 + frow] : -1;
  id = (uint32_t)id < (uint32_t)l.adapters ? id : -1;
  uint32_t todo = (uint32_t)__ballot(id >= 0 && frow % (int)gridDim.z == (int)blockIdx.z);
  while (todo != 0) {
    const int first = __builtin_ctz(todo);
    const int g = __builtin_amdgcn_readlane(id, first);
    const uint32_t match = (uint32_t)__ballot(id == g);
    todo &= ~match;
    if (__builtin_ctz(match) != first) continue;  // (another workgroup's)
    const char* down = l.down + (int64_t)g * l.down_stride * ES;
    const float s = l.scale != nullptr ? l.scale[g] : 1.f;
    if (__popc(match) <= kDots) {
      const int rows = __popc(match);
      if (rows == 1)
        dots<DT, 1>(l, m0, match, down, s, r0, ranks);
      else if (rows == 2)
        dots<DT, 2>(l, m0, match, down, s, r0, ranks);
      else
        dots<DT, kDots>(l, m0, match, down, s, r0, ranks);
      continue;
    }
    Parts split(smem);
#pragma unroll
    for (int q = 0; q < 4; ++q) split.row[q] = l.a + (int64_t)min(m0 + split.row_of(q), l.m - 1) * l.lda * ES;
#pragma unroll
    for (int q = 4; q < Parts::NQ; ++q) {
      const int r = r0 + split.row_of(q) - 32;
      split.row[q] = r < l.rank ? down + (int64_t)r * l.ld_down * ES : nullptr;
    }
    typename Parts::Sums acc;
    split.start(l.k);
    split.run(l.k, acc, (match & 0xffffu) != 0, match >> 16 != 0);
    __syncthreads();
    split.put_sums(smem, acc, 1.f);
    __syncthreads();
    for (int q = tid; q < 32 * COLS; q += NT) {
      const int row = q / COLS, r = q % COLS;
      // (behind the rank zeros, also of a row of infinities, whose sums with zeros are no numbers; nor are an infinite scale's products with the
      // sums of waves that have no part of K, so that it comes last)
      if ((match >> row & 1) && r < ranks) put_low<DT>(l, m0 + row, r0 + r, r0 + r < l.rank ? s * Parts::sum(smem, row, r) : 0.f);
    }
    __syncthreads();
  }
}

template <int DT>
int run_low(const bz_fc_adapters_desc& d, int low_rank, hipStream_t st) {
  constexpr int ES = In<DT>::kSize;
  const bool aligned = (uintptr_t)d.a % 16 == 0 && (uintptr_t)d.down % 16 == 0 && d.lda * ES % 16 == 0 && d.ld_down * ES % 16 == 0 &&
                       d.down_stride * ES % 16 == 0 && (int64_t)d.k * ES % 16 == 0;
  auto launch = [&](auto aligned_c, auto cols_c) {
    constexpr bool ALIGNED = decltype(aligned_c)::value;
    constexpr int COLS = decltype(cols_c)::value, LDS = Split<DT, kLowWaves, ALIGNED, COLS>::LDS;
    auto* kernel = bz_adapters_low_kernel<DT, ALIGNED, COLS>;
    static Lds lds;
    const int rc = lds.allow((const void*)kernel, LDS);
    if (rc != BZ_OK) return rc;
    constexpr int64_t kPart = 1 << 26;  // rows of a launch, which has fewer than 2^32 threads
    for (int64_t r0 = 0; r0 < d.m; r0 += kPart) {
      const int m = (int)std::min<int64_t>(kPart, d.m - r0), blocks = (m + 31) / 32, parts = (low_rank + COLS - 1) / COLS;
      const Low l = {(const char*)d.a + r0 * d.lda * ES, (const char*)d.down, d.ids + r0, d.scale, (char*)d.scratch + r0 * low_rank * 4, d.lda, d.ld_down,
                     d.down_stride, m, d.k, d.adapters, d.rank, low_rank};
      const int turns = std::max(1, std::min(32, 512 / std::min(512, blocks * parts)));
      hipLaunchKernelGGL(kernel, dim3(blocks, parts, turns), dim3(kLowWaves * 64), LDS, st, l);
      BZ_LAUNCH_OK("bz_adapters_low_kernel");
    }
    return (int)BZ_OK;
  };
  auto by_rank = [&](auto aligned_c) {
    return low_rank <= 16 ? launch(aligned_c, std::integral_constant<int, 16>()) : launch(aligned_c, std::integral_constant<int, 32>());
  };
  return aligned ? by_rank(std::true_type()) : by_rank(std::false_type());
}

template <int DT>
int run(const Layer& l, const Call& call) {
  return l.adapters > 0 ? run_layer<DT, false, true>(l, call) : run_layer<DT, false, false>(l, call);
}
int run(int dtype, const Layer& l, const Call& call) {
  return dtype == BZ_F32 ? run<BZ_F32>(l, call) : dtype == BZ_F16 ? run<BZ_F16>(l, call) : run<BZ_BF16>(l, call);
}

int low_rank_of(int rank) { return (rank + 15) / 16 * 16; }

}  // namespace

extern "C" {

int64_t bz_fc_adapters_scratch_bytes(int64_t m, int rank) {
  return m > 0 && rank > 0 ? m * low_rank_of(rank) * 4 : 0;
}

int bz_fc_adapters(const bz_fc_adapters_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_fc_adapters: null descriptor");
  const bz_fc_adapters_desc& d = *desc;
  BZ_REQUIRE(d.in_dtype == BZ_F32 || d.in_dtype == BZ_F16 || d.in_dtype == BZ_BF16, "bz_fc_adapters: in_dtype %d", d.in_dtype);
  BZ_REQUIRE(d.out_dtype == d.in_dtype || d.out_dtype == BZ_F32, "bz_fc_adapters: out_dtype %d of in_dtype %d", d.out_dtype, d.in_dtype);
  BZ_REQUIRE(d.m >= 0 && d.n >= 1 && d.k >= 1, "bz_fc_adapters: m %d, n %d, k %d", d.m, d.n, d.k);
  BZ_REQUIRE(d.adapters >= 0, "bz_fc_adapters: adapters %d", d.adapters);
  BZ_REQUIRE(d.lda >= d.k && d.ldw >= d.k && d.ldy >= d.n, "bz_fc_adapters: pitches %lld, %lld and %lld for k %d, n %d", (long long)d.lda,
             (long long)d.ldw, (long long)d.ldy, d.k, d.n);
  const int rc = bz::layer_act("bz_fc_adapters", d.act, d.act_size, d.act_p0, d.act_p1, d.act_p2, d.n);
  if (rc != BZ_OK) return rc;
  if (d.adapters > 0) {
    BZ_REQUIRE(d.rank >= 1 && d.rank <= BZ_ADAPTER_MAX_RANK, "bz_fc_adapters: rank %d (1..%d)", d.rank, BZ_ADAPTER_MAX_RANK);
    BZ_REQUIRE(d.ld_down >= d.k && d.ld_up >= d.rank, "bz_fc_adapters: pitches %lld and %lld for k %d, rank %d", (long long)d.ld_down,
               (long long)d.ld_up, d.k, d.rank);
    BZ_REQUIRE(d.adapters == 1 || (d.down_stride >= (d.rank - 1) * d.ld_down + d.k && d.up_stride >= (d.n - 1) * d.ld_up + d.rank),
               "bz_fc_adapters: strides %lld and %lld", (long long)d.down_stride, (long long)d.up_stride);
  }
  if (d.m == 0) return BZ_OK;
  BZ_REQUIRE(d.a && d.w && d.y, "bz_fc_adapters: null pointer");
  if (d.adapters > 0) {
    BZ_REQUIRE(d.down && d.up && d.ids, "bz_fc_adapters: null pointer");
    const int64_t need = bz_fc_adapters_scratch_bytes(d.m, d.rank);
    BZ_REQUIRE(d.scratch != nullptr && (uintptr_t)d.scratch % 16 == 0 && d.scratch_bytes >= need,
               "bz_fc_adapters: scratch of %lld bytes, %lld on a 16-byte boundary needed", (long long)(d.scratch ? d.scratch_bytes : 0), (long long)need);
  }
  Layer l = {};
  l.a = (const char*)d.a;
  l.w = (const char*)d.w;
  l.y = d.y;
  l.a_count = d.m;
  l.lda = d.lda;
  l.ldw = d.ldw;
  l.ldy = d.ldy;
  l.m = d.m;
  l.n = d.n;
  l.k = d.k;
  l.groups = 1;
  l.rows_per = 1;
  l.ep.bias = d.bias;
  l.ep.p0 = d.act_p0;
  l.ep.p1 = d.act_p1;
  l.ep.p2 = d.act_p2;
  l.ep.bias_rows = d.bias ? 1 : 0;
  l.ep.act = d.act;
  l.ep.act_size = d.act_size;
  l.ep.dice_nosqrt = d.dice_nosqrt;
  l.ep.alpha = d.alpha;
  l.ep.beta = d.beta;
  l.ep.act_alpha = d.act_alpha;
  l.adapters = d.adapters;
  l.out_f32 = d.out_dtype == BZ_F32;
  const hipStream_t st = bz::as_stream(stream);
  if (d.adapters > 0) {
    l.rank = d.rank;
    l.low_rank = low_rank_of(d.rank);
    l.ids = d.ids;
    l.low = (const char*)d.scratch;
    l.up = (const char*)d.up;
    l.ld_up = d.ld_up;
    l.up_stride = d.up_stride;
    // what can be refused is refused before the factors are launched (no kernel has more than a thread an output, 32 by 16 of them whole)
    if (((int64_t)d.m + 31) * ((int64_t)d.n + 15) >= (int64_t)1 << 31) {
      const int rc = run(d.in_dtype, l, {"bz_fc_adapters", st, true});
      if (rc != BZ_OK) return rc;
    }
    const int done = d.in_dtype == BZ_F32 ? run_low<BZ_F32>(d, l.low_rank, st)
                     : d.in_dtype == BZ_F16 ? run_low<BZ_F16>(d, l.low_rank, st) : run_low<BZ_BF16>(d, l.low_rank, st);
    if (done != BZ_OK) return done;
  }
  return run(d.in_dtype, l, {"bz_fc_adapters", st});
}

}  // extern "C"
