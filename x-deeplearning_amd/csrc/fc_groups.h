// fc_groups.h -- layers whose rows go through different weights (fc_grouped.hip, fc_adapters.hip): three kernels and the choice between them
// (run_layer).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <atomic>

#include "bz_common.h"
#include "fc_common.h"
#include "rows_common.h"

namespace bz {
namespace groups {

using bz::fc::floatx16;
using bz::fc::floatx4;
using bz::fc::In;
using bz::rows::Elem;

static __device__ uint4 kZeros = {0u, 0u, 0u, 0u};  // never written: what is read for a chunk behind K, or of a row of zeros

// 16 bytes of a row from element k on, or where K ends in them or before them, the row's last 16 bytes: row_moved(.., k, K) makes of them
// what begins at k, with zeros at and behind K.  Nothing outside the row's K elements (16 bytes at least) is read, and no branch keeps many from
// being on their way together.  The row may begin at any element; null: zeros.
template <int DT>
__device__ __forceinline__ uint4 row_raw(const char* row, int k, int K) {
  uint4 v;
  __builtin_memcpy(&v, row != nullptr ? row + (int64_t)min(k, K - In<DT>::kChunk) * In<DT>::kSize : (const char*)&kZeros, 16);
  return v;
}
template <int DT>
__device__ __forceinline__ uint4 row_moved(uint4 v, int k, int K) {
  const int b = min(max(k - (K - In<DT>::kChunk), 0) * In<DT>::kSize, 16);
  if (In<DT>::kSize == 2) {
    const uint32_t s = (b & 2) * 8;
    v = make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, s), __builtin_amdgcn_alignbit(v.z, v.y, s), __builtin_amdgcn_alignbit(v.w, v.z, s), v.w >> s);
  }
  v = b & 4 ? make_uint4(v.y, v.z, v.w, 0u) : v;
  v = b & 8 ? make_uint4(v.z, v.w, 0u, 0u) : v;
  return b & 16 ? make_uint4(0u, 0u, 0u, 0u) : v;
}
// both in one, and rows of less than 16 bytes
template <int DT>
__device__ __forceinline__ uint4 row_chunk(const char* row, int k, int K) {
  if (K >= In<DT>::kChunk) return row_moved<DT>(row_raw<DT>(row, k, K), k, K);
  return row != nullptr && k < K ? bz::rows::Chunk<DT>::load(row + (int64_t)k * In<DT>::kSize, K - k).raw : make_uint4(0u, 0u, 0u, 0u);
}

// What every kernel of these layers needs of its call.  A group's (an adapter layer: the only) weight is w + g * w_stride.
struct Layer {
  const char* a;
  const char* w;
  void* y;
  const int32_t* rows;     // where row r's input is: a[rows[r] / rows_per]; null: a[r]
  const int32_t* offsets;  // [groups + 1]; null: one group of m rows
  int64_t a_count, lda, ldw, w_stride, ldy;
  int m, n, k, groups, rows_per;
  int out_f32;             // y is fp32, whatever the operands
  bz::fc::Epilogue ep;     // p0.. of group 0
  int p_stride;            // parameters (p0) a group
  // adapters (null: none): a row's number, its low-rank factor (two bf16s, or an fp32), the second factors
  const int32_t* ids;
  const char* low;
  const char* up;
  int64_t ld_up, up_stride;
  int adapters, rank, low_rank;  // low_rank: rank rounded up to 16
};

// The rows [begin, end) of a group, wherever its offsets point
__device__ __forceinline__ void group_range(const int32_t* offsets, int g, int m, int& begin, int& end) {
  begin = min(max(offsets[g], 0), m);
  end = min(max(offsets[g + 1], begin), m);
}

// Tiles of BM rows, a group's after another's: the group and first row of tile `tile`; false: there are fewer.  Every lane of the wave
// looks at one group's offsets, 64 groups at a time.
template <int BM>
__device__ __forceinline__ bool find_tile(const Layer& l, int tile, int& group, int& m0, int& m1) {
  if (l.offsets == nullptr) {
    group = 0;
    m0 = tile * BM;
    m1 = l.m;
    return m0 < l.m;
  }
  const int lane = threadIdx.x & 63;
  int left = tile;
  for (int g0 = 0; g0 < l.groups; g0 += 64) {
    const int g = g0 + lane;
    int begin = 0, end = 0;
    if (g < l.groups) group_range(l.offsets, g, l.m, begin, end);
    const int tiles = (end - begin + BM - 1) / BM;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(upto, o);
      upto += lane >= o ? u : 0;
    }
    const uint64_t here = __ballot(upto > left);
    if (here != 0) {
      const int src = __ffsll((long long)here) - 1;
      group = __builtin_amdgcn_readlane(g, src);
      m0 = __builtin_amdgcn_readlane(begin + (left - (upto - tiles)) * BM, src);
      m1 = __builtin_amdgcn_readlane(end, src);
      return true;
    }
    left -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}
// how many tiles of bm rows there can be
__host__ __device__ inline int64_t most_tiles(int64_t m, int groups, int bm) { return m / bm + (groups < m ? groups : m); }
// The number of tiles of BM rows that all groups have together.  Offsets that run backwards count rows again and again: no more tiles than a
// launch is made for (64 times as many fit 32 bits: it has a workgroup of 256 threads for each).
template <int BM>
__device__ __forceinline__ int count_tiles(const Layer& l) {
  if (l.offsets == nullptr) return (l.m + BM - 1) / BM;
  const int lane = threadIdx.x & 63, most = (int)most_tiles(l.m, l.groups, BM);
  int tiles = 0;
  for (int g = lane; g < l.groups; g += 64) {
    int begin, end;
    group_range(l.offsets, g, l.m, begin, end);
    tiles += (end - begin + BM - 1) / BM;
  }
  return __builtin_amdgcn_readfirstlane(min(bz::rows::reduce<64>(min(tiles, most), [](int a, int b) { return a + b; }), most));
}
// Who asks for a layer, and where; check_only: whether it can be launched, and no more
struct Call {
  const char* who;
  hipStream_t stream;
  bool check_only = false;
};
// (a launch has fewer than 2^32 threads)
constexpr const char* kTooManyTiles = "%s: %lld tiles of %d rows and %d columns are too many for a launch";


// address of row r's input, null for a row of zeros
__device__ __forceinline__ const char* input_row(const Layer& l, int r, int es) {
  int64_t at = r;
  if (l.rows != nullptr) {
    const int from = l.rows[r];
    at = from < 0 ? -1 : from / l.rows_per;  // (a division alone makes row 0 of -1)
  }
  return at >= 0 && at < l.a_count ? l.a + at * l.lda * es : nullptr;
}

// y[at] = v, rounded to the output's type
template <int DT>
__device__ __forceinline__ void put_out(const Layer& l, int64_t at, float v) {
  if (DT == BZ_F32 || l.out_f32)
    ((float*)l.y)[at] = v;
  else
    bz::fc::store_out<typename Elem<DT>::type>((typename Elem<DT>::type*)l.y + at, v);
}

__device__ __forceinline__ float silu(float v) { return v / (1.f + expf(-v)); }

// Eight bf16s: whether any is infinite or no number, and the same with zeros in the place of those
__device__ __forceinline__ bool any_unbounded(const uint4& v) {
  auto carry = [](uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; };  // an exponent of ones reaches the sign's place
  return ((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u) != 0;
}
__device__ __forceinline__ uint4 bounded(const uint4& v) {
  auto keep = [](uint32_t w) {
    const uint32_t top = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    return w & ~(top | (top - (top >> 15)));
  };
  return make_uint4(keep(v.x), keep(v.y), keep(v.z), keep(v.w));
}

// One step of K = 32 bytes of a low-rank product, added to d: what of a row's factor and of a row of `up` the lane brings.
// An operand in two pieces has its infinity, or what is no number, in the first alone: times that, the second pieces of the other
// operand, of any sign or 0, would make NaNs of infinities, and are left out.
template <int DT>
struct LowStep {
  uint4 hi, lo, u;
  // plain: no chunk of a row of `up` reaches behind its end
  __device__ __forceinline__ void load(const Layer& l, const char* low, const char* up, int k, int half, bool plain) {
    constexpr int CH = In<DT>::kChunk;
    if constexpr (DT == BZ_F32) {
      hi = *(const uint4*)(low + (k + half * 4) * 4);
    } else {
      hi = *(const uint4*)(low + (k + half * 8) * 2);
      lo = *(const uint4*)(low + (l.low_rank + k + half * 8) * 2);
    }
    if (plain)
      __builtin_memcpy(&u, up + (int64_t)(k + half * CH) * In<DT>::kSize, 16);
    else
      u = row_chunk<DT>(up, k + half * CH, l.rank);
  }
  __device__ __forceinline__ void multiply(floatx16& d) const {
    if constexpr (DT == BZ_F32) {
      In<BZ_F32>::mma(hi, u, d);
    } else if constexpr (DT == BZ_BF16) {
      uint4 u_some = u;
      if (__builtin_expect(any_unbounded(u), 0)) u_some = bounded(u);
      In<BZ_BF16>::mma(lo, u_some, d);
      In<BZ_BF16>::mma(hi, u, d);
    } else {
      // (an fp16 `up` is split the same way as the factor, so that a factor beyond fp16 does no harm)
      typedef _Float16 h8 __attribute__((ext_vector_type(8)));
      const h8 f = __builtin_bit_cast(h8, u);
      uint32_t uh[4], ul[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = (float)f[2 * i], x1 = (float)f[2 * i + 1];
        uh[i] = bz::fc::nearest_bf16x2(x0, x1);
        ul[i] = bz::fc::nearest_bf16x2(x0 - __uint_as_float(uh[i] << 16), x1 - __uint_as_float(uh[i] & 0xffff0000u));
      }
      const uint4 u_hi = make_uint4(uh[0], uh[1], uh[2], uh[3]);
      uint4 u_lo = make_uint4(ul[0], ul[1], ul[2], ul[3]), u_some = u_hi, hi_some = hi;
      if (__builtin_expect(any_unbounded(u_hi), 0)) {
        u_some = bounded(u_hi);
        u_lo = bounded(u_lo);  // (an infinity less itself)
      }
      if (__builtin_expect(any_unbounded(hi), 0)) hi_some = bounded(hi);
      In<BZ_BF16>::mma(lo, u_lo, d);  // (up to 2^-16 of the product, as much as a factor's own rounding)
      In<BZ_BF16>::mma(lo, u_some, d);
      In<BZ_BF16>::mma(hi_some, u_lo, d);
      In<BZ_BF16>::mma(hi, u_hi, d);
    }
  }
};

// Adds the low-rank products of 32 rows (row0..) to their TN blocks of 32 columns (col0.., col_step apart), each row with its own
// adapter's: add(block, i, product, take) for the i-th sum of the lane, `take` telling whether its row has it.  The distinct adapters of
// the 32 rows are taken AT_ONCE at a time: a product of all rows' factors with each adapter's, of which the rows that have the adapter take
// theirs and no other row is touched.  Lane l brings row row0 + l % 32's adapter in `id` (-1: none).
// The adapter of row r is taken where no row before has it, and r is the `share`-th of every `shares` (waves that add the same block up share
// the rows). AT_ONCE of them at a time.
// UNROLL: blocks at once (add's block is a constant where that is TN).
template <int DT, int TN, int UNROLL, int AT_ONCE, typename Add>
__device__ __forceinline__ void add_adapters(const Layer& l, int id, int row0, int m1, int col0, int col_step, const Add& add, int share = 0,
                                             int shares = 1) {
  constexpr int STEP = 2 * In<DT>::kChunk;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (no address below is computed, and kept, in front of a loop that this is in)
  const int frow = lane & 31, half = lane >> 5;
  const char* low = l.low + (int64_t)min(row0 + frow, m1 - 1) * l.low_rank * 4;
  const bool plain = l.rank % STEP == 0;
  uint32_t todo = (uint32_t)__ballot(id >= 0 && frow % shares == share);
  while (todo != 0) {
    int g[AT_ONCE];
    uint32_t match[AT_ONCE];
    int n = 0;
#pragma unroll
    for (int b = 0; b < AT_ONCE; ++b) {
      g[b] = 0;
      match[b] = 0;
      while (todo != 0 && match[b] == 0) {
        const int r = __builtin_ctz(todo);
        const int one = __builtin_amdgcn_readlane(id, r);
        const uint32_t same = (uint32_t)__ballot(id == one);
        todo &= ~same;
        if (shares == 1 || __builtin_ctz(same) == r) {
          g[b] = one;
          match[b] = same;
          n = b + 1;
        }
      }
    }
    if (n == 0) break;
#pragma unroll UNROLL
    for (int j = 0; j < TN; ++j) {
      const int c = min(col0 + j * col_step + frow, l.n - 1);
      floatx16 d[AT_ONCE];
      const char* up[AT_ONCE];
#pragma unroll
      for (int b = 0; b < AT_ONCE; ++b) {
        up[b] = l.up + ((int64_t)g[b] * l.up_stride + (int64_t)c * l.ld_up) * In<DT>::kSize;
#pragma unroll
        for (int i = 0; i < 16; ++i) d[b][i] = 0.f;
      }
      for (int k = 0; k < l.rank; k += STEP) {
        LowStep<DT> s[AT_ONCE];
#pragma unroll
        for (int b = 0; b < AT_ONCE; ++b)
          if (b < n) s[b].load(l, low, up[b], k, half, plain);
#pragma unroll
        for (int b = 0; b < AT_ONCE; ++b)
          if (b < n) s[b].multiply(d[b]);
      }
#pragma unroll
      for (int b = 0; b < AT_ONCE; ++b)
        if (b < n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) add(j, i, d[b][i], (match[b] >> (8 * (i >> 2) + 4 * half + (i & 3)) & 1) != 0);
        }
    }
  }
}

// The layers' activation.  Sigmoid is 1 / (1 + e^-v), which has a value for any v; the shared layers' e^v / (1 + e^v) is NaN from v = 88.73 on.
// A leaky ReLU of slope 0 is ReLU: 0 below 0, where the product with -infinity is NaN.  fp32 layers have an exact Dice, whose error does not
// grow as fast with the distance from the mean (v_exp_f32's argument, rounded after a product with log2(e), is 2^-24 of itself off: 60
// deviations from the mean 60 steps of the result).  p2 is what dice_column makes of a column's variance.
template <int DT, int ACT>
__device__ __forceinline__ float activated(float v, const bz::fc::Epilogue& ep, float p0, float p1, float p2) {
  if constexpr (DT == BZ_F32 && ACT == BZ_ACT_DICE) {
    const float p = 1.f / (1.f + expf((p1 - v) / p2));
    return fmaf(1.f - p, p0, p) * v;
  }
  if constexpr (ACT == BZ_ACT_SIGMOID) return 1.f / (1.f + expf(-v));
  if constexpr (ACT == BZ_ACT_LEAKY_RELU) return v >= 0.f ? v : v < 0.f && ep.act_alpha == 0.f ? 0.f : ep.act_alpha * v;
  return bz::fc::apply_act_t<ACT>(v, ep, p0, p1, p2);
}

template <int DT>
__device__ __forceinline__ float dice_column(const bz::fc::Epilogue& ep, float var) {
  return DT == BZ_F32 ? bz::fc::dice_den(ep, var) : bz::fc::dice_inv_den(ep, var);
}

// The parameters of column c of group g
template <int DT, int ACT>
struct Column {
  float bias = 0.f, p0 = 0.f, p1 = 0.f, p2 = 0.f;
  __device__ __forceinline__ Column(const Layer& l, int g, int c, int bias_cols) {
    const bz::fc::Epilogue& ep = l.ep;
    if (ep.bias != nullptr) bias = ep.beta * ep.bias[(int64_t)g * bias_cols + c];
    const int64_t p = (int64_t)g * l.p_stride;
    if constexpr (ACT == BZ_ACT_PRELU) p0 = ep.p0[p + (ep.act_size == 1 ? 0 : c)];
    if constexpr (ACT == BZ_ACT_DICE) {
      p0 = ep.p0[p + c];
      p1 = ep.p1[p + c];
      p2 = dice_column<DT>(ep, ep.p2[p + c]);
    }
  }
  __device__ __forceinline__ float of(const Layer& l, float v) const {
    return activated<DT, ACT>(fmaf(l.ep.alpha, v, bias), l.ep, p0, p1, p2);
  }
};

// ---------------------------------------------------------------------------------------------
// tile kernel
// ---------------------------------------------------------------------------------------------
// A workgroup of four waves owns BM rows of one group and BN columns (with GATED: BN / 2 columns, each with its gate's); a wave BM / 2 x
// BN / 2 of them in 32x32 blocks.  K goes by in steps of 128 bytes a row, from global memory through registers into one of two LDS
// buffers, the next step's loads in flight while this one is multiplied.  Chunk c of row r lies at position c ^ (r & 7).
// It takes what the wide kernel cannot: rows that begin anywhere, operands beyond 4 GB, an `a` without rows.  Bound by the loads at odd addresses, two requests
// where one would do: 2000 rows of 1023 -> 1023 bf16 23.1 us, 182 TFLOP/s (1024 -> 1024 by this kernel 20.0, by
// the wide one 13.0).
template <int DT, int BM, int BN, bool GATED, bool ADAPTERS>
__global__ __launch_bounds__(256) void bz_groups_tile_kernel(Layer l, int tiles_n) {
  using T = In<DT>;
  constexpr int ES = T::kSize, CH = T::kChunk, BK = 8 * CH, TM = BM / 64, TN = BN / 64, NA = BM * 8 / 256, NW = BN * 8 / 256;
  static_assert(!GATED || TN == 2, "a wave has both of a column's");
  __shared__ __attribute__((aligned(16))) char lds[2][(BM + BN) * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int tile_n = blockIdx.x % tiles_n;
  int group, m0, m1;
  if (!find_tile<BM>(l, blockIdx.x / tiles_n, group, m0, m1)) return;
  const int n0 = tile_n * (GATED ? BN / 2 : BN);
  const char* w = l.w + (int64_t)group * l.w_stride * ES;

  const char* pa[NA];
  const char* pw[NW];
  const int c = tid & 7;
#pragma unroll
  for (int i = 0; i < NA; ++i) pa[i] = input_row(l, min(m0 + (tid >> 3) + i * 32, m1 - 1), ES);
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int r = (tid >> 3) + i * 32;  // GATED: blocks of 32 columns and 32 gates in turn
    const int col = GATED ? min(n0 + r / 64 * 32 + r % 32, l.n - 1) + (r / 32 % 2 ? l.n : 0) : min(n0 + r, l.n - 1);
    pw[i] = w + (int64_t)col * l.ldw * ES;
  }
  uint4 ra[NA], rw[NW];
  auto load = [&](int k) {
    if (l.k >= CH) {
#pragma unroll
      for (int i = 0; i < NA; ++i) ra[i] = row_raw<DT>(pa[i], k + c * CH, l.k);
#pragma unroll
      for (int i = 0; i < NW; ++i) rw[i] = row_raw<DT>(pw[i], k + c * CH, l.k);
    } else {
#pragma unroll
      for (int i = 0; i < NA; ++i) ra[i] = row_chunk<DT>(pa[i], k + c * CH, l.k);
#pragma unroll
      for (int i = 0; i < NW; ++i) rw[i] = row_chunk<DT>(pw[i], k + c * CH, l.k);
    }
  };
  auto put = [&](int buf, int k) {
    const int r0 = tid >> 3;
    if (l.k >= CH && k + BK > l.k) {
#pragma unroll
      for (int i = 0; i < NA; ++i) ra[i] = row_moved<DT>(ra[i], k + c * CH, l.k);
#pragma unroll
      for (int i = 0; i < NW; ++i) rw[i] = row_moved<DT>(rw[i], k + c * CH, l.k);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) *(uint4*)&lds[buf][(r0 + i * 32) * 128 + ((c ^ (r0 & 7)) << 4)] = ra[i];
#pragma unroll
    for (int i = 0; i < NW; ++i) *(uint4*)&lds[buf][(BM + r0 + i * 32) * 128 + ((c ^ (r0 & 7)) << 4)] = rw[i];
  };
  floatx16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const int frow = lane & 31, half = lane >> 5;
  load(0);
  put(0, 0);
  __syncthreads();
  for (int k = 0, buf = 0; k < l.k; k += BK, buf ^= 1) {
    const bool more = k + BK < l.k;
    if (more) load(k + BK);
    const char* base = &lds[buf][0];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = ((2 * s + half) ^ (frow & 7)) << 4;
      uint4 fa[TM], fw[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = *(const uint4*)(base + (wm * (BM / 2) + i * 32 + frow) * 128 + at);
#pragma unroll
      for (int j = 0; j < TN; ++j) fw[j] = *(const uint4*)(base + (BM + wn * (BN / 2) + j * 32 + frow) * 128 + at);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) T::mma(fa[i], fw[j], acc[i][j]);
    }
    if (more) put(buf ^ 1, k + BK);
    __syncthreads();
  }
  const int col0 = n0 + wn * (GATED ? BN / 4 : BN / 2);
  if constexpr (ADAPTERS) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row0 = m0 + wm * (BM / 2) + i * 32;
      int id = row0 + frow < m1 ? l.ids[row0 + frow] : -1;
      id = (uint32_t)id < (uint32_t)l.adapters ? id : -1;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] *= l.ep.alpha;
      if (row0 < m1)
        add_adapters<DT, TN, TN, 1>(l, id, row0, m1, col0, 32, [&](int j, int r, float d, bool take) { acc[i][j][r] += take ? d : 0.f; });
    }
  }
  // lane: column frow of each block, rows 8 * (r / 4) + 4 * half + r % 4
  auto finish = [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    constexpr int COLS = GATED ? 1 : TN;
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      const int col = col0 + j * 32 + frow, cc = min(col, l.n - 1);
      const Column<DT, ACT> p(l, group, cc, GATED ? 2 * l.n : l.n);
      const float gate_bias = p.bias, up_bias = GATED && l.ep.bias != nullptr ? l.ep.bias[(int64_t)group * 2 * l.n + l.n + cc] : 0.f;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = m0 + wm * (BM / 2) + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
          float v;
          if constexpr (GATED)
            v = silu(acc[i][0][r] + gate_bias) * (acc[i][TN - 1][r] + up_bias);
          else if constexpr (ADAPTERS)
            v = activated<DT, ACT>(acc[i][j][r] + p.bias, l.ep, p.p0, p.p1, p.p2);
          else
            v = p.of(l, acc[i][j][r]);
          if (row < m1 && col < l.n) put_out<DT>(l, (int64_t)row * l.ldy + col, v);
        }
    }
  };
  if constexpr (GATED)
    finish(std::integral_constant<int, BZ_ACT_NONE>());
  else
    bz::fc::with_act(l.ep.act, finish);
}

template <int DT, int BM, int BN, bool GATED, bool ADAPTERS>
int launch_tile(const Layer& l, const Call& call) {
  const int bn = GATED ? BN / 2 : BN;
  const int64_t tiles_n = (l.n + bn - 1) / bn, tiles = most_tiles(l.m, l.offsets ? l.groups : 1, BM) * tiles_n;
  BZ_REQUIRE(tiles * 256 < (int64_t)1 << 32, kTooManyTiles, call.who, (long long)tiles, l.m, l.n);
  if (call.check_only) return BZ_OK;
  hipLaunchKernelGGL((bz_groups_tile_kernel<DT, BM, BN, GATED, ADAPTERS>), dim3((uint32_t)tiles), dim3(256), 0, call.stream, l, (int)tiles_n);
  BZ_LAUNCH_OK("bz_groups_tile_kernel");
  return BZ_OK;
}

// ---------------------------------------------------------------------------------------------
// split kernel: few rows
// ---------------------------------------------------------------------------------------------
// 16 bytes per lane from global memory to LDS at lds_addr + 16 * lane (lds_addr is the same in all lanes).  A scalar write of M0 needs
// a wait state before a load to LDS reads it.
typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ void lds_load(const char* g, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds_addr) : "memory", "m0");
}

// Products of 32 rows with 32 rows (COLS: or with 16) over K by waves that share K, 128 bytes of every row at a time (stage t is wave t % NW's), each wave
// for itself: a stage's rows go from global memory straight to one of two places in the wave's own LDS, eight lanes a row, are read from there
// as fragments, and the stage after next is asked for where they were.  Nobody waits for another wave until the sums meet.
// Bound by the weights' way from HBM: 64 rows x 4 of 16 gated experts, 2048 -> 1024 bf16, 134 MB in 33.8 us, 4.0 TB/s of a copy's 4.9; 29.6
// with the weights in the 256 MB cache.  Five waves (80 KB of LDS, more on its way) took 33.5 there and 20.1 for 19.7 at K 1024, eight 37.7.
// ALIGNED: rows begin on 16 bytes and K is whole chunks; else they come through registers, from any element.
// Row r of a stage is at 128 * r, its chunk c at position c ^ ((r >> 1) & 7): sixteen lanes that read one chunk of sixteen rows are on all banks.
// COLS 16: in 16x16 blocks, of which a half of the rows that nobody has is left out.
template <int DT, int NW, bool ALIGNED, int COLS = 32>
struct Split {
  static constexpr int ES = In<DT>::kSize, CH = In<DT>::kChunk, BK = 8 * CH, NQ = (32 + COLS) / 8, SLOT = NQ * 1024, PITCH = 33;
  static constexpr int LDS = NW * 2 * SLOT;
  static_assert(LDS >= NW * 32 * PITCH * 4, "the partial sums fit where the operands were");
  using Sums = typename std::conditional<COLS == 32, floatx16, floatx4[2]>::type;
  const char* row[NQ];  // load q brings rows q * 8 + lane / 8, the first 32 of one operand, the last of the other; null: zeros
  char* lds;           // the wave's two places
  int lane, wave;
  __device__ __forceinline__ Split(char* lds_of_all) : lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {
    lds = lds_of_all + wave * (2 * SLOT);
  }
  // (of the lane, in load q)
  __device__ __forceinline__ int row_of(int q) const { return q * 8 + (lane >> 3); }
  __device__ __forceinline__ int chunk_of(int q) const { return (lane & 7) ^ ((q & 1) * 4 + (lane >> 4)); }

  // the wave's stages of K
  __device__ __forceinline__ int count(int K) const {
    const int stages = (K + BK - 1) / BK;
    return wave < stages ? (stages - 1 - wave) / NW + 1 : 0;
  }
  __device__ __forceinline__ void issue(int K, int i) {
    const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char*)lds) + (i & 1) * SLOT;
    const int k0 = (wave + i * NW) * BK;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int k = k0 + chunk_of(q) * CH;
      lds_load(row[q] != nullptr && k < K ? row[q] + (int64_t)k * ES : (const char*)&kZeros, to + q * 1024);
    }
  }
  // asks for what run begins with (to be called before it): what stands between takes its time while that is on its way
  __device__ __forceinline__ void start(int K) {
    if constexpr (ALIGNED) {
      const int n = count(K);
      if (n > 0) issue(K, 0);
      if (n > 1) issue(K, 1);
    }
  }

  // upper, lower: whether anybody has rows 0 to 15, 16 to 31
  __device__ __forceinline__ void run(int K, Sums& acc, bool upper, bool lower) {
    constexpr int L = COLS == 32 ? 32 : 16;  // rows of a block
    const int n = count(K), frow = lane % L, part = lane / L, swizzle = (frow >> 1) & 7;
    if constexpr (COLS == 32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    } else {
      acc[0] = acc[1] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    uint4 r[NQ];
    auto load = [&](int i) {
      const int k0 = (wave + i * NW) * BK;
      if (K >= CH) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) r[q] = row_raw<DT>(row[q], k0 + chunk_of(q) * CH, K);
      } else {
#pragma unroll
        for (int q = 0; q < NQ; ++q) r[q] = row_chunk<DT>(row[q], k0 + chunk_of(q) * CH, K);
      }
    };
    auto put = [&](int i) {
      const int k0 = (wave + i * NW) * BK;
      if (K >= CH && k0 + BK > K) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) r[q] = row_moved<DT>(r[q], k0 + chunk_of(q) * CH, K);
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q) *(uint4*)(lds + (i & 1) * SLOT + q * 1024 + lane * 16) = r[q];
    };
    if constexpr (!ALIGNED) {
      if (n > 0) {
        load(0);
        put(0);
        if (n > 1) load(1);
      }
    }
    for (int i = 0; i < n; ++i) {
      if constexpr (ALIGNED) {
        if (i + 1 < n)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NQ) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      } else {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      const char* s = lds + (i & 1) * SLOT + frow * 128;
      // fa: chunks of the first 16 or 32 rows and, in 16x16 blocks, of the next 16
      uint4 fa[4], fw[COLS == 32 ? 4 : 2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = (((COLS == 32 ? 2 * c : 4 * (c & 1)) + part) ^ swizzle) << 4;
        fa[c] = *(const uint4*)(s + (COLS == 32 ? 0 : (c >> 1) * 16 * 128) + at);
        if (COLS == 32 || c < 2) fw[COLS == 32 ? c : c & 1] = *(const uint4*)(s + 32 * 128 + at);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (ALIGNED) {
        if (i + 2 < n) issue(K, i + 2);
      } else if (i + 1 < n) {
        put(i + 1);
        if (i + 2 < n) load(i + 2);
      }
      if constexpr (COLS == 32) {
#pragma unroll
        for (int c = 0; c < 4; ++c) In<DT>::mma(fa[c], fw[c], acc);
      } else {
        if (upper) {
          In<DT>::mma16(fa[0], fw[0], acc[0]);
          In<DT>::mma16(fa[1], fw[1], acc[0]);
        }
        if (lower) {
          In<DT>::mma16(fa[2], fw[0], acc[1]);
          In<DT>::mma16(fa[3], fw[1], acc[1]);
        }
      }
    }
  }

  // the wave's sums, to where sum() finds them (behind a barrier: that is where the operands were)
  __device__ __forceinline__ void put_sums(char* lds_of_all, const Sums& acc, float alpha) const {
    float* to = (float*)lds_of_all + wave * (32 * PITCH);
    if constexpr (COLS == 32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) to[(8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * PITCH + (lane & 31)] = alpha * acc[i];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(16 * h + 4 * (lane >> 4) + i) * PITCH + (lane & 15)] = alpha * acc[h][i];
    }
  }
  static __device__ __forceinline__ float sum(const char* lds_of_all, int row, int col) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += ((const float*)lds_of_all)[w * (32 * PITCH) + row * PITCH + col];
    return v;
  }
};

// A workgroup owns 32 rows of one group and COLS columns (GATED: 16, each with its gate), its NW waves share K.
template <int DT, int NW, bool ALIGNED, bool GATED, bool ADAPTERS, int COLS>
__global__ __launch_bounds__(NW * 64) void bz_groups_split_kernel(Layer l, int tiles_n) {
  using Parts = Split<DT, NW, ALIGNED, COLS>;
  static_assert(!GATED || COLS == 32);
  constexpr int ES = In<DT>::kSize;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int group, m0, m1;
  if (!find_tile<32>(l, blockIdx.x / tiles_n, group, m0, m1)) return;
  const int n0 = (int)(blockIdx.x % tiles_n) * (GATED ? 16 : COLS);
  const char* w = l.w + (int64_t)group * l.w_stride * ES;
  Parts split(smem);
#pragma unroll
  for (int q = 0; q < 4; ++q) split.row[q] = input_row(l, min(m0 + split.row_of(q), m1 - 1), ES);
#pragma unroll
  for (int q = 4; q < Parts::NQ; ++q) {
    const int r = split.row_of(q) - 32;  // GATED: 16 gates, then their columns
    const int col = GATED ? min(n0 + r % 16, l.n - 1) + r / 16 * l.n : min(n0 + r, l.n - 1);
    split.row[q] = w + (int64_t)col * l.ldw * ES;
  }
  split.start(l.k);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, frow = lane & 31, half = lane >> 5;
  // the parameters of the column that this thread finishes, on their way meanwhile
  constexpr int OUT = GATED ? 16 : COLS;
  const int c = tid % OUT, col = n0 + c;
  float bias = 0.f, p0 = 0.f, p1 = 0.f, p2 = 0.f;
  {
    const bz::fc::Epilogue& ep = l.ep;
    const int cc = min(col, l.n - 1);
    const int64_t at = (int64_t)group * l.p_stride + (ep.act == BZ_ACT_PRELU && ep.act_size == 1 ? 0 : cc);
    if (ep.bias != nullptr) bias = ep.bias[(int64_t)group * (GATED ? 2 * l.n : l.n) + cc];
    if (GATED && ep.bias != nullptr) p0 = ep.bias[(int64_t)group * 2 * l.n + l.n + cc];  // (the other factor's)
    if (!GATED && (ep.act == BZ_ACT_PRELU || ep.act == BZ_ACT_DICE)) p0 = ep.p0[at];
    if (!GATED && ep.act == BZ_ACT_DICE) {
      p1 = ep.p1[at];
      p2 = ep.p2[at];
    }
  }
  floatx16 low;
#pragma unroll
  for (int i = 0; i < 16; ++i) low[i] = 0.f;
  if constexpr (ADAPTERS) {
    int id = m0 + frow < m1 ? l.ids[m0 + frow] : -1;
    id = (uint32_t)id < (uint32_t)l.adapters ? id : -1;
    add_adapters<DT, 1, 1, 4>(l, id, m0, m1, n0, 0, [&](int, int r, float d, bool take) { low[r] += take ? d : 0.f; }, wave, NW);
  }
  typename Parts::Sums acc;
  split.run(l.k, acc, true, m1 - m0 > 16);
  __syncthreads();
  split.put_sums(smem, acc, ADAPTERS ? l.ep.alpha : 1.f);
  if constexpr (ADAPTERS) {
    __builtin_amdgcn_wave_barrier();
    float* own = (float*)smem + wave * (32 * Parts::PITCH);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (frow < COLS) own[(8 * (i >> 2) + 4 * half + (i & 3)) * Parts::PITCH + frow] += low[i];
  }
  __syncthreads();
  auto sum = [&](int row, int col) { return Parts::sum(smem, row, col); };
  auto finish = [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    if (col >= l.n) return;
    const float q2 = ACT == BZ_ACT_DICE ? dice_column<DT>(l.ep, p2) : 0.f, b = l.ep.beta * bias;
    for (int r = tid / OUT; r < 32 && m0 + r < m1; r += NW * 64 / OUT) {
      float v;
      if constexpr (GATED)
        v = silu(sum(r, c) + bias) * (sum(r, c + 16) + p0);
      else
        v = activated<DT, ACT>(ADAPTERS ? sum(r, c) + b : fmaf(l.ep.alpha, sum(r, c), b), l.ep, p0, p1, q2);
      put_out<DT>(l, (int64_t)(m0 + r) * l.ldy + col, v);
    }
  };
  if constexpr (GATED)
    finish(std::integral_constant<int, BZ_ACT_NONE>());
  else
    bz::fc::with_act(l.ep.act, finish);
}

// Lets a kernel have more than the 64 KB of dynamic LDS that it may have without asking, once per device (one of these per kernel).
struct Lds {
  std::atomic<uint64_t> done{0};
  int allow(const void* kernel, int bytes) {
    int dev = 0;
    BZ_HIP_OK(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
      BZ_HIP_OK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
      done.fetch_or(bit, std::memory_order_relaxed);
    }
    return BZ_OK;
  }
};

template <int DT, int NW, bool ALIGNED, bool GATED, bool ADAPTERS, int COLS = 32>
int launch_split(const Layer& l, const Call& call) {
  const int bn = GATED ? 16 : COLS;
  const int64_t tiles_n = (l.n + bn - 1) / bn, tiles = most_tiles(l.m, l.offsets ? l.groups : 1, 32) * tiles_n;
  BZ_REQUIRE(tiles * (NW * 64) < (int64_t)1 << 32, kTooManyTiles, call.who, (long long)tiles, l.m, l.n);
  if (call.check_only) return BZ_OK;
  constexpr int LDS = Split<DT, NW, ALIGNED, COLS>::LDS;
  auto* kernel = bz_groups_split_kernel<DT, NW, ALIGNED, GATED, ADAPTERS, COLS>;
  if constexpr (LDS > 64 << 10) {
    static Lds lds;
    const int rc = lds.allow((const void*)kernel, LDS);
    if (rc != BZ_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((uint32_t)tiles), dim3(NW * 64), LDS, call.stream, l, (int)tiles_n);
  BZ_LAUNCH_OK("bz_groups_split_kernel");
  return BZ_OK;
}

// ---------------------------------------------------------------------------------------------
// wide kernel: many rows
// ---------------------------------------------------------------------------------------------
// A workgroup of four waves owns 64 * TM x 64 * TN outputs, a wave 32 * TM x 32 * TN of them in 32x32 blocks; its rows begin on 16 bytes and
// lie within 4 GB of where their operand (a group's weight) begins.
//  - K goes by in stages of 128 bytes a row (a line: the L2 answers a request of half a line in the time of a whole one), from global
//    memory straight to one of S places in LDS; an address is a scalar base that moves on and a lane's 32-bit offset that does not, so a load costs no
//    vector instruction.
//  - A stage is four steps of K = 32 bytes; a step multiplies one set of fragments while the next one is read.  In front of the last the
//    waves meet: the next stage has landed, and nobody reads this one any more, so that the S-th after it goes there.
//  - Reads and loads stand between the matrix instructions, which take longer than they do, and nothing moves from there.
//  - Row r of a stage lies at 128 * r, its chunk c at position c ^ ((r >> 1) & 7): sixteen lanes that read one chunk of sixteen rows are
//    on all banks.
//  - The eight XCDs take turns at consecutive workgroups: XCD x walks its own part of the tiles, eight tiles of rows beside each other and
//    then the next columns, so that the 32 workgroups that it runs at a time share few rows of either operand in its L2.
// Bound by the matrix cores, at the clocks that their power leaves: the main loop of 256x256 tiles takes the same time without loads and
// without reads of LDS.  One group of 8192 rows, K and N 4096, bf16: 242 us, 1140 TFLOP/s (a large library product: 1220 to 1290); 32 gated
// experts, 8192 rows x 4, 2048 -> 1024: 339 us, 811 TFLOP/s; what is missing are tiles that groups do not fill, the last round of
// workgroups and the starts and ends of tiles, which nothing covers.
constexpr int kWideBand = 8;
// which tile of tiles_m x tiles_n (their product and 8 more below 2^31) workgroup `block` has; false: none
__host__ __device__ inline bool wide_tile(int tiles_m, int tiles_n, uint32_t block, int& tile_m, int& tile_n) {
  const int each = (tiles_m * tiles_n + 7) / 8;
  int t = (int)(block >> 3);
  if (t >= each) return false;
  t += (int)(block & 7) * each;
  if (t >= tiles_m * tiles_n) return false;
  const int band = t / (kWideBand * tiles_n), in_band = t - band * (kWideBand * tiles_n), left = tiles_m - band * kWideBand;
  const int high = left < kWideBand ? left : kWideBand;
  tile_n = in_band / high;
  tile_m = band * kWideBand + in_band % high;
  return true;
}
// The loads are free to move among reads of LDS: only the waits and barriers keep them apart.
__device__ __forceinline__ void lds_load_free(const char* g, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds_addr) : "m0");
}
__device__ __forceinline__ void lds_load_free(const char* base, uint32_t off, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_addr) : "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The lane's number, from nothing that would have to be kept in a register meanwhile
__device__ __forceinline__ int lane_number() {
  int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(lane));  // (nor is an address that is computed from it, in front of a loop that this is in)
  return lane;
}

// Low-rank products of a strip of 32 rows with TN blocks of 32 columns, K of the rank at a time: what the lane brings of the rows'
// factors, and of one adapter's rows of `up`, which are kept from strip to strip.  All of it is asked for at once.
template <int DT>
struct StripLow {
  static constexpr int STEPS = 2, STEP = 2 * In<DT>::kChunk;
  uint4 hi[STEPS], lo[STEPS];
  __device__ __forceinline__ void load(const Layer& l, int row, int m1, int k) {
    const int lane = lane_number();
    const char* low = l.low + (int64_t)min(row + (lane & 31), m1 - 1) * l.low_rank * 4;
    const int half = lane >> 5;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int at = min(k + s * STEP, l.low_rank - STEP) + half * (STEP / 2);  // (steps behind the rank are not multiplied)
      if constexpr (DT == BZ_F32) {
        hi[s] = *(const uint4*)(low + at * 4);
      } else {
        hi[s] = *(const uint4*)(low + at * 2);
        lo[s] = *(const uint4*)(low + (l.low_rank + at) * 2);
      }
    }
  }
};
template <int DT, int TN>
struct StripUp {
  static constexpr int STEPS = StripLow<DT>::STEPS, STEP = StripLow<DT>::STEP, K = STEPS * STEP;
  uint4 u[TN][STEPS];
  int group = -1, k = 0;
  __device__ __forceinline__ void load(const Layer& l, int g, int col0, int from) {
    const int lane = lane_number();
    group = g;
    k = from;
    const bool plain = l.rank % STEP == 0 && l.ld_up % In<DT>::kChunk == 0;  // no chunk of a row reaches behind its end
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const char* up = l.up + ((int64_t)g * l.up_stride + (int64_t)min(col0 + j * 32 + (lane & 31), l.n - 1) * l.ld_up) * In<DT>::kSize;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int at = from + s * STEP + (lane >> 5) * (STEP / 2);
        if (plain)
          __builtin_memcpy(&u[j][s], up + (int64_t)min(at, l.rank - STEP / 2) * In<DT>::kSize, 16);
        else
          u[j][s] = row_chunk<DT>(up, at, l.rank);
      }
    }
  }
  __device__ __forceinline__ void multiply(const StripLow<DT>& low, int j, int left, floatx16& d) const {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (s * STEP < left) LowStep<DT>{low.hi[s], low.lo[s], u[j][s]}.multiply(d);
  }
};

template <int DT, int TM, int TN, int S, bool GATED, bool ADAPTERS>
__global__ __launch_bounds__(256, TM * TN > 8 || (DT == BZ_F32 && TM * TN > 2) ? 1 : 2) void bz_groups_wide_kernel(Layer l, int tiles_n) {
  using T = In<DT>;
  constexpr int ES = T::kSize, CH = T::kChunk, BK = 8 * CH, BM = 64 * TM, BN = 64 * TN, ROWS = BM + BN, STAGE = ROWS * 128;
  constexpr int LOADS = ROWS / 32;  // of 8 rows each, a wave's share of a stage
  constexpr int FRAGS = TM + TN, BLOCKS = TM * TN;
  static_assert(!GATED || TN % 2 == 0, "a wave has both of a column's");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
  const int tiles_m = count_tiles<BM>(l);
  int tile_m, tile_n, group, m0, m1;
  if (!wide_tile(tiles_m, tiles_n, blockIdx.x, tile_m, tile_n) || !find_tile<BM>(l, tile_m, group, m0, m1)) return;
  const int n0 = tile_n * (GATED ? BN / 2 : BN);
  const char* a = l.a;
  const char* w = l.w + (int64_t)group * l.w_stride * ES;

  // this lane's part of its wave's loads: row q * 32 + wave * 8 + lane / 8 of the stage, the chunk that belongs at position lane % 8
  const int lrow = wave * 8 + (lane >> 3), chunk = (lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7);
  auto a_off = [&](int r) {
    const char* row = input_row(l, min(m0 + r, m1 - 1), ES);
    return row != nullptr ? (uint32_t)(row - l.a) : 0u;  // (a row of zeros: the first one, whose sums are passed over)
  };
  auto w_off = [&](int r) {  // GATED: 32 columns and their 32 gates in turn
    const int col = GATED ? min(n0 + r / 64 * 32 + r % 32, l.n - 1) + (r / 32 % 2 ? l.n : 0) : min(n0 + r, l.n - 1);
    return (uint32_t)((int64_t)col * l.ldw * ES);
  };
  uint32_t off[LOADS];
#pragma unroll
  for (int q = 0; q < LOADS; ++q) {
    off[q] = (q < 2 * TM ? a_off(q * 32 + lrow) : w_off((q - 2 * TM) * 32 + lrow)) + chunk * 16;
  }
  const int stages = (l.k + BK - 1) / BK, whole_stages = l.k / BK;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)smem + wave * 1024;
  // what the end needs of the tile's columns and rows, fetched now and behind the places: bias (GATED: of columns and gates in turn) and
  // activation's parameters, a row's adapter (or whether it is a row of zeros)
  float* params = (float*)(smem + S * STAGE);
  int* of_row = (int*)(params + 4 * BN);
  if (tid < BN) {
    const int col = GATED ? min(n0 + tid / 64 * 32 + tid % 32, l.n - 1) + (tid / 32 % 2 ? l.n : 0) : min(n0 + tid, l.n - 1);
    const bz::fc::Epilogue& ep = l.ep;
    const int64_t at = (int64_t)group * l.p_stride + (ep.act == BZ_ACT_PRELU && ep.act_size == 1 ? 0 : col);
    const bool dice = !GATED && ep.act == BZ_ACT_DICE;
    params[tid] = ep.bias != nullptr ? ep.beta * ep.bias[(int64_t)group * (GATED ? 2 * l.n : l.n) + col] : 0.f;
    params[BN + tid] = !GATED && (ep.act == BZ_ACT_PRELU || dice) ? ep.p0[at] : 0.f;
    params[2 * BN + tid] = dice ? ep.p1[at] : 0.f;
    params[3 * BN + tid] = dice ? dice_column<DT>(ep, ep.p2[at]) : 0.f;
  }
  if (tid < BM) {
    const int row = min(m0 + tid, m1 - 1);
    if constexpr (ADAPTERS)
      of_row[tid] = (uint32_t)l.ids[row] < (uint32_t)l.adapters && m0 + tid < m1 ? l.ids[row] : -1;
    else
      of_row[tid] = input_row(l, row, ES) != nullptr;
  }
  // load q of stage i into place p; WHOLE: of a stage that does not reach behind K (what does, and stages behind the last, bring zeros there)
  auto issue = [&](int i, int p, int q, auto whole_c) {
    uint64_t at = (uint64_t)((q < 2 * TM ? a : w) + (int64_t)i * 128);
    if constexpr (DT == BZ_F32)  // (there the compiler would add it up in vector registers)
      at = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
    const char* base = (const char*)at;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + p * STAGE + q * 4096);
    if constexpr (decltype(whole_c)::value)
      lds_load_free(base, off[q], to);
    else
      lds_load_free(i * BK + chunk * CH < l.k ? base + off[q] : (const char*)&kZeros, to);
  };
  constexpr std::true_type kWhole;
  constexpr std::false_type kPart;

  floatx16 acc[TM][TN];
  const int frow = lane & 31, half = lane >> 5;
  int p, next;  // the places of this stage and the next
  auto turn = [&]() {
    p = next;
    next = next + 1 == S ? 0 : next + 1;
  };
  auto begin = [&]() {
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < whole_stages) {
#pragma unroll
        for (int q = 0; q < LOADS; ++q) issue(i, i, q, kWhole);
      } else {
#pragma unroll
        for (int q = 0; q < LOADS; ++q) issue(i, i, q, kPart);
      }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    p = 0;
    next = 1 % S;
    wait_loads<(S - 1) * LOADS>();
    asm volatile("s_barrier" ::: "memory");
  };
  // The two halves of the waves have every other 32 rows, so that both have less to multiply where the group ends in the tile: `live` blocks
  // (8192 rows x 4 through 32 gated experts 348 -> 339 us).
  auto block_row = [&](int f) { return (2 * f + wm) * 32; };
  const int live = min(TM, max(0, m1 - m0 - wm * 32 + 63) / 64);
  // chunk c of the lane's row of block f: the rows' blocks, then the columns'
  auto fragment = [&](int place, int f, int c) {
    const int row = f < TM ? block_row(f) : BM + wn * 32 * TN + (f - TM) * 32;
    return *(const uint4*)(smem + place * STAGE + (row + frow) * 128 + ((c ^ ((frow >> 1) & 7)) << 4));
  };
  // (every read of this stage has returned, and the next one has landed)
  auto meet = [&]() {
    wait_loads<(S - 2) * LOADS>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto multiply = [&]() {
    begin();
    uint4 fa[2][TM], fw[2][TN];
    auto read = [&](int set, int place, int step, int f) {
      if (f < TM)
        fa[set][f] = fragment(place, f, 2 * step + half);
      else
        fw[set][f - TM] = fragment(place, f, 2 * step + half);
    };
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) read(0, 0, 0, f);
    auto stage = [&](int i, auto whole_c, auto all_c) {
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        if (step == 3) meet();
        // one block of rows with all columns' blocks, and what stands between its products
        auto row_of_blocks = [&](int x, bool products) {
#pragma unroll
          for (int b = x * TN; b < (x + 1) * TN; ++b) {
            if (products) T::mma(fa[step & 1][x], fw[step & 1][b % TN], acc[x][b % TN]);
#pragma unroll
            for (int f = b * FRAGS / BLOCKS; f < (b + 1) * FRAGS / BLOCKS; ++f) {
              if (step < 3)
                read((step + 1) & 1, p, step + 1, f);
              else
                read(0, next, 0, f);
            }
            if (step == 3) {
#pragma unroll
              for (int q = b * LOADS / BLOCKS; q < (b + 1) * LOADS / BLOCKS; ++q) issue(i + S, p, q, whole_c);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        };
#pragma unroll
        for (int x = 0; x < TM; ++x) {
          if (decltype(all_c)::value || x < live)
            row_of_blocks(x, true);
          else
            row_of_blocks(x, false);
        }
      }
      turn();
    };
    int i = 0;
    if (TM == 1 || live == TM) {
      for (; i + S < whole_stages; ++i) stage(i, kWhole, std::true_type());
      for (; i < stages; ++i) stage(i, kPart, std::true_type());
    } else {
      for (; i < stages; ++i) stage(i, kPart, std::false_type());
    }
    // (loads of zeros are still on their way to LDS, which is used again)
    wait_loads<0>();
    __syncthreads();
  };
  // fp32 on the bf16 matrix cores: every operand as three bf16s (bz::fc::Bf16x3), six of whose nine products are multiplied, in 192 clocks for
  // 32x32x16 where the fp32 instructions take 512.  An operand is converted once for all four waves, on its way to LDS: it comes through
  // registers, two stages ahead, and a stage's pieces lie in one of two places as three matrices of 64 bytes a row, chunk c of row r at
  // position c ^ ((r >> 2) & 3).  Bound by the conversions and the instructions that feed the matrix cores: 8192 rows, 2048 -> 2048 475 us, 145
  // TFLOP/s (730 with fp32 instructions, in the tile kernel); 2048 x 2 rows of 896 -> 512 through 8 experts 41.2 (44.7 with each wave converting
  // the fragments that it read, and without what finds doubtful sums).
  // A sum that is not finite, or small enough that what a split drops of its operands may count in it, is doubtful (bz::fc::doubtful): the
  // tile is multiplied again with fp32 instructions then, and such sums are taken from there (the others stay, so that no row's result
  // depends on what is in another).  For that the largest operand of each row is kept on the way, a twelfth of the
  // conversion's instructions: one group of 8192 rows, 2048 -> 2048, 459 -> 475 us, 2048 x 2 rows of 896 -> 512 40.4 -> 41.2.
  uint32_t again[TM][TN];  // the doubtful ones of a block's sums
  auto multiply_split = [&]() {
    using bz::fc::Bf16x3;
    constexpr int ITEMS = ROWS / 64, PLANE = ROWS * 64;  // eight floats an item
    static_assert(DT != BZ_F32 || 2 * 3 * PLANE <= S * STAGE, "two places");
    const int irow = tid >> 2, ichunk = tid & 3;
    uint32_t item_off[ITEMS];
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) item_off[q] = (q < TM ? a_off(q * 64 + irow) : w_off((q - TM) * 64 + irow)) + ichunk * 32;
    struct Raw {
      uint4 x[ITEMS][2];
    } raw[2];
    auto load = [&](Raw& to, int i) {
      const int64_t at = (int64_t)i * 128;
      if (i < whole_stages) {
#pragma unroll
        for (int q = 0; q < ITEMS; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) to.x[q][c] = *(const uint4*)((q < TM ? a : w) + at + item_off[q] + c * 16);
      } else {
#pragma unroll
        for (int q = 0; q < ITEMS; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            to.x[q][c] = make_uint4(0, 0, 0, 0);
            if (i * BK + ichunk * 8 + c * 4 < l.k) to.x[q][c] = *(const uint4*)((q < TM ? a : w) + at + item_off[q] + c * 16);
          }
      }
    };
    float most[ITEMS];  // the largest |operand| that the thread has seen of the item's row
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) most[q] = 0.f;
    auto put = [&](const Raw& from, int place, int q) {
      const Bf16x3 v = bz::fc::split_floats(from.x[q][0], from.x[q][1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        bz::fc::largest(most[q], __uint_as_float(from.x[q][c].x), __uint_as_float(from.x[q][c].y));
        bz::fc::largest(most[q], __uint_as_float(from.x[q][c].z), __uint_as_float(from.x[q][c].w));
      }
      const int row = q * 64 + irow;
      char* to = smem + place * (3 * PLANE) + row * 64 + ((ichunk ^ ((row >> 2) & 3)) << 4);
      *(uint4*)to = v.hi;
      *(uint4*)(to + PLANE) = v.mid;
      *(uint4*)(to + 2 * PLANE) = v.lo;
    };
    struct Pieces {
      Bf16x3 v[FRAGS];
    } first, second;
    auto read = [&](Pieces& to, int place, int step) {
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int row = (f < TM ? block_row(f) : BM + wn * 32 * TN + (f - TM) * 32) + frow;
        const char* from = smem + place * (3 * PLANE) + row * 64 + (((2 * step + half) ^ ((frow >> 2) & 3)) << 4);
        to.v[f].hi = *(const uint4*)from;
        to.v[f].mid = *(const uint4*)(from + PLANE);
        to.v[f].lo = *(const uint4*)(from + 2 * PLANE);
      }
    };
    auto products = [&](const Pieces& p) {
      auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) f(p.v[i], p.v[TM + j], acc[i][j]);
      };
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.lo, y.hi, c); });
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.hi, y.lo, c); });
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.mid, y.mid, c); });
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.mid, y.hi, c); });
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.hi, y.mid, c); });
      each([](const Bf16x3& x, const Bf16x3& y, floatx16& c) { In<BZ_BF16>::mma(x.hi, y.hi, c); });
    };
    // a step's products, and between them the conversion of items from..to
    auto step = [&](const Pieces& p, const Raw& r, int place, auto from_c, auto to_c) {
      constexpr int FROM = decltype(from_c)::value, TO = decltype(to_c)::value, MFMAS = 6 * BLOCKS, EACH = ((TO - FROM) * 54 + MFMAS - 1) / MFMAS;
      __builtin_amdgcn_sched_barrier(0);
      products(p);
#pragma unroll
      for (int q = FROM; q < TO; ++q) put(r, place, q);
#pragma unroll
      for (int m = 0; m < MFMAS; ++m) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, EACH, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    load(raw[0], 0);
    load(raw[1], 1);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) put(raw[0], 0, q);
    load(raw[0], 2);
    constexpr std::integral_constant<int, 0> kNone;
    constexpr std::integral_constant<int, ITEMS / 2> kSome;
    constexpr std::integral_constant<int, ITEMS> kAll;
    // stage i lies in place i % 2; raw i + 1 % 2 holds the next one, the other the one after
    auto stage = [&](int i, auto odd_c) {
      constexpr int ODD = decltype(odd_c)::value;
      __syncthreads();
      read(first, ODD, 0);
      read(second, ODD, 1);
      step(first, raw[1 - ODD], 1 - ODD, kNone, kSome);
      step(second, raw[1 - ODD], 1 - ODD, kSome, kAll);
      load(raw[1 - ODD], i + 3);
    };
    int i = 0;
    for (; i + 1 < stages; i += 2) {
      stage(i, std::integral_constant<int, 0>());
      stage(i + 1, std::integral_constant<int, 1>());
    }
    if (i < stages) stage(i, std::integral_constant<int, 0>());
    // |v| from what is doubtful for kOrdinary up to infinity, as bits without the sign's: one look at the tile
    const uint32_t least = __float_as_uint((float)l.k * (bz::fc::kSplitDrops * bz::fc::kOrdinary)) << 1;
    uint32_t worst = 0;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) worst = max(worst, (__float_as_uint(acc[i][j][r]) << 1) - least);
    bool look = worst >= 0xff000000u - least;
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) look |= most[q] > bz::fc::kOrdinary;
    if (__syncthreads_or(look) == 0) return false;
    // the rows' largest operands, where the stages were: four threads have seen parts of a row
    float* row_most = (float*)smem;
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
      most[q] = fmaxf(most[q], __shfl_xor(most[q], 1));
      most[q] = fmaxf(most[q], __shfl_xor(most[q], 2));
      if (ichunk == 0) row_most[q * 64 + irow] = most[q];
    }
    __syncthreads();
    bool off = false;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        again[i][j] = 0;
        const float max_w = row_most[BM + wn * 32 * TN + j * 32 + frow];
#pragma unroll
        for (int r = 0; r < 16; ++r)
          again[i][j] |= bz::fc::doubtful(acc[i][j][r], l.k, row_most[block_row(i) + 8 * (r >> 2) + 4 * half + (r & 3)], max_w) ? 1u << r : 0u;
        off |= again[i][j] != 0;
      }
    return __syncthreads_or(off) != 0;
  };
  if constexpr (DT == BZ_F32) {
    if (multiply_split()) {
      floatx16 split[TM][TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) split[i][j] = acc[i][j];
      multiply();
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = again[i][j] >> r & 1 ? acc[i][j][r] : split[i][j][r];
    }
  } else {
    multiply();
  }

  // 32 rows at a time: the adapters' products, then the sums through LDS of the wave's own, so that a lane has neighbouring columns of a
  // row: their bias and activation, and a store of 16 bytes.  A block's sums are in lane l: column l % 32, rows 8 * (r / 4) + 4 * (l / 32) + r % 4.
  const int late = lane_number(), col_of = late & 31, half_of = late >> 5;
  const int col0 = n0 + wn * (GATED ? 16 * TN : 32 * TN);
  constexpr int PITCH = 32 * TN + 4;
  static_assert(4 * 32 * PITCH * 4 <= S * STAGE, "the strips fit where the operands were");
  float* mine = (float*)smem + wave * (32 * PITCH);
  auto finish = [&](auto act_c, auto* out, int row) {
    constexpr int ACT = decltype(act_c)::value;
    using OutT = std::remove_pointer_t<decltype(out)>;
    constexpr int OCH = 16 / sizeof(OutT), COLS = GATED ? 16 * TN : 32 * TN, PER_ROW = COLS / OCH;
    static_assert(64 % PER_ROW == 0, "a lane's columns are the same in all rows");
    const int ln = lane_number();
    const int c = ln % PER_ROW * OCH, col = col0 + c, from = GATED ? c / 32 * 64 + c % 32 : c;
    if (col >= l.n) return;
    const float* p = params + wn * 32 * TN + from;
    float p0[OCH], p1[OCH], p2[OCH], bias[OCH];
#pragma unroll
    for (int x = 0; x < OCH; ++x) {
      bias[x] = p[x];
      p0[x] = p[GATED ? x + 32 : BN + x];  // (GATED: the other factor's bias)
      p1[x] = ACT == BZ_ACT_DICE ? p[2 * BN + x] : 0.f;
      p2[x] = ACT == BZ_ACT_DICE ? p[3 * BN + x] : 0.f;
    }
    const bool whole = (uintptr_t)out % 16 == 0 && l.ldy % OCH == 0 && col + OCH <= l.n;
    auto one = [&](int r, bool fast) {
      float y[OCH];
      const float* v = mine + r * PITCH + from;
      const bool there = ADAPTERS || of_row[row + r - m0] != 0;
#pragma unroll
      for (int x = 0; x < OCH; ++x) {
        const float sum = there ? v[x] : 0.f;
        if constexpr (GATED)
          y[x] = silu(sum + bias[x]) * ((there ? v[x + 32] : 0.f) + p0[x]);
        else
          y[x] = activated<DT, ACT>(ADAPTERS ? sum + bias[x] : fmaf(l.ep.alpha, sum, bias[x]), l.ep, p0[x], p1[x], p2[x]);
      }
      OutT* to = out + (int64_t)(row + r) * l.ldy + col;
      if (fast) {
        typename bz::rows::Native<OutT>::type u[OCH];
#pragma unroll
        for (int x = 0; x < OCH; ++x) u[x] = bz::rows::narrow<typename bz::rows::Native<OutT>::type>(y[x]);
        *(uint4*)to = *(const uint4*)u;
      } else {
#pragma unroll
        for (int x = 0; x < OCH; ++x)
          if (col + x < l.n) bz::fc::store_out<OutT>(to + x, y[x]);
      }
    };
    constexpr int TURNS = 32 * PER_ROW / 64;
    if (row + 32 <= m1 && __ballot(!whole) == 0) {
#pragma unroll
      for (int t = 0; t < TURNS; ++t) one(ln / PER_ROW + t * (64 / PER_ROW), true);
    } else {
#pragma unroll 1
      for (int t = 0; t < TURNS; ++t)
        if (row + ln / PER_ROW + t * (64 / PER_ROW) < m1) one(ln / PER_ROW + t * (64 / PER_ROW), false);
    }
  };
  auto at = [&](int j, int r) -> float& { return mine[(8 * (r >> 2) + 4 * half_of + (r & 3)) * PITCH + j * 32 + col_of]; };
  StripLow<DT> strip_low;
  StripUp<DT, TN> strip_up;
  // (one strip's code for all of them: four times over it did not fit the registers)
#pragma unroll 1
  for (int i = 0; i < TM; ++i) {
    const int row = m0 + block_row(i);
    if (row >= m1) break;
#pragma unroll
    for (int x = 0; x < TM; ++x)
      if (x == i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) at(j, r) = ADAPTERS ? l.ep.alpha * acc[x][j][r] : acc[x][j][r];
      }
    if constexpr (ADAPTERS) {
      if (row < m1) {
        strip_low.load(l, row, m1, 0);
        uint32_t todo = (uint32_t)__ballot(of_row[row - m0 + col_of] >= 0);
        const int id = of_row[row - m0 + col_of];
        while (todo != 0) {
          const int g = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
          const uint32_t match = (uint32_t)__ballot(id == g);
          todo &= ~match;
          for (int k = 0; k < l.rank; k += strip_up.K) {
            if (k > 0) strip_low.load(l, row, m1, k);
            if (strip_up.group != g || strip_up.k != k) strip_up.load(l, g, col0, k);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              floatx16 d;
#pragma unroll
              for (int r = 0; r < 16; ++r) d[r] = 0.f;
              strip_up.multiply(strip_low, j, l.rank - k, d);
              float sum[16];
#pragma unroll
              for (int r = 0; r < 16; ++r) sum[r] = at(j, r);
#pragma unroll
              for (int r = 0; r < 16; ++r) at(j, r) = sum[r] + (match >> (8 * (r >> 2) + 4 * half_of + (r & 3)) & 1 ? d[r] : 0.f);
            }
          }
          if (todo != 0 && l.rank > strip_up.K) strip_low.load(l, row, m1, 0);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto typed = [&](auto act_c) {
      if (DT == BZ_F32 || l.out_f32)
        finish(act_c, (float*)l.y, row);
      else
        finish(act_c, (typename Elem<DT>::type*)l.y, row);
    };
    if constexpr (GATED)
      typed(std::integral_constant<int, BZ_ACT_NONE>());
    else
      bz::fc::with_act(l.ep.act, typed);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

template <int DT, int TM, int TN, int S, bool GATED, bool ADAPTERS>
int launch_wide(const Layer& l, const Call& call) {
  const int bm = 64 * TM, bn = GATED ? 32 * TN : 64 * TN;
  const int64_t tiles_n = (l.n + bn - 1) / bn, tiles = most_tiles(l.m, l.offsets ? l.groups : 1, bm) * tiles_n;
  BZ_REQUIRE((tiles + 7) * 256 < (int64_t)1 << 32, kTooManyTiles, call.who, (long long)tiles, l.m, l.n);
  if (call.check_only) return BZ_OK;
  constexpr int LDS = S * 64 * (TM + TN) * 128 + (4 * 64 * TN + 64 * TM) * 4;
  auto* kernel = bz_groups_wide_kernel<DT, TM, TN, S, GATED, ADAPTERS>;
  if constexpr (LDS > 64 << 10) {
    static Lds lds;
    const int rc = lds.allow((const void*)kernel, LDS);
    if (rc != BZ_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((uint32_t)((tiles + 7) / 8 * 8)), dim3(256), LDS, call.stream, l, (int)tiles_n);
  BZ_LAUNCH_OK("bz_groups_wide_kernel");
  return BZ_OK;
}

// whether the rows of both operands begin on 16 bytes and K is whole chunks
inline bool rows_aligned(const Layer& l, int es) {
  return (uintptr_t)l.a % 16 == 0 && (uintptr_t)l.w % 16 == 0 && l.lda * es % 16 == 0 && l.ldw * es % 16 == 0 && l.w_stride * es % 16 == 0 &&
         (int64_t)l.k * es % 16 == 0;
}

// How many tiles of `rows` rows m rows of so many groups make, about: half a tile of each group stays empty
inline int64_t about_tiles(int64_t m, int64_t groups, int64_t rows) {
  return groups == 1 ? (m + rows - 1) / rows : m / rows + std::min(groups, m) / 2 + 1;
}

// What `tiles` workgroups of a wide kernel take, in hundredths of the time of one of 256x256 that has a CU for itself: AT_ONCE of them share
// one of the 256 CUs, and `part[i]` is what i + 1 of them take that run side by side.
template <int AT_ONCE>
inline int64_t wide_cost(int64_t tiles, const int (&part)[AT_ONCE]) {
  const int64_t round = 256 * AT_ONCE, rest = tiles % round;
  return tiles / round * part[AT_ONCE - 1] + (rest > 0 ? part[(rest - 1) / 256] : 0);
}

// Which kernel.
// Few rows, or few tiles: 32 rows by 32 columns, the waves sharing K (us by it and by the best other one: bf16, K and N 1024, 8 groups of 32
// rows 8.6 and 10.3, of 64 rows 12.1 and 10.6; one layer with adapters, 300 rows 17.4 and 19.9, 512 rows 17.3 and 16.4; fp32 512 rows 29.4
// and 34.1).  Eight waves rather than four where the CUs are not full (bf16 64 rows, 1024x1024, with adapters: 13.2 and 14.2), four where
// they are (8 groups of 32 rows: 8.6 and 10.7), but eight with adapters, whose rows the waves share (128 rows, 4096x4096: 30.7 and 34.6).
// Where tiles of 16 columns still leave a CU each, those: half the matrix instructions, a quarter of them for at most 16 rows, which is what
// fp32 takes (2 rows x 3 through 16 experts, 2508 -> 216 10.7 and 19.3, 68 rows through 6, 1616 -> 128 8.6 and 14.4; fp16 6.9 and 7.7, 100 rows
// through 4, 512 -> 512 5.5 and 5.8); beyond, rows are read twice for nothing (fp32 200 rows of 512 -> 512 9.5 and 8.2).
// Longer, aligned: the wide kernel, and 2-byte layers with the tile that fills the rounds of workgroups best.  Larger tiles take less time
// a product, but a round that is begun costs a whole one (us by 256x256, 128x128, 64x128 and 64x64: bf16, one layer of 8192 rows, K 1024,
// N 2048 44.2, 48.5, -, -; 8192 rows x 2 of 8 groups, 1024x1024 76.8, 60.3, -, -; 2048 rows x 2 38.6, 22.7, 26.6, 24.6; 1536 rows x 2 37.7,
// 19.7, 18.2, 23.0; 256 rows x 2 32.2, 15.2, 12.7, 10.6; 512 rows x 8 of 64 groups, K 768, N 2048 68.3, 55.5, 47.7, 52.1).  fp32 layers keep to 64
// rows and columns, which is what few tiles want (us by 64x64, 64x128 and 128x64: 2048 rows x 2 of 8 groups, 896 -> 512 46.5, 51.7, 53.0; 4096 x 2
// of 16, 512 -> 512 48.5, 52.2, 53.8; 1000 x 4 of 32, 256 -> 1024 31.0, 33.2, 35.3; 3000 x 2 of 4, 1024 -> 256 38.1, 37.7, 39.4), though long batches
// would take less with 64x128 (8192 rows of one group, 2048 -> 2048 490, 444, 445; 8192 x 2 of 8, 1024 -> 1024 261, 243, 250).
// What is not aligned: the tile kernel, which needs no alignment (where not the few rows' one: 1023x1023, 500 rows 11.6 by that and 16.7 by
// tiles, fp32 700 rows 54.7 and 49.6, with adapters fp16 300 rows 24.7 and 24.2).
template <int DT, bool GATED, bool ADAPTERS>
int run_layer(const Layer& l, const Call& call) {
  const int groups = l.offsets ? l.groups : 1;
  const bool aligned = rows_aligned(l, In<DT>::kSize);
  const int64_t limit = (int64_t)1 << 32, es = In<DT>::kSize;
  // (the wide kernel reads some row where a row of zeros is asked for, so there has to be one)
  const bool near = l.a_count > 0 && l.a_count * l.lda * es <= limit && (int64_t)l.n * (GATED ? 2 : 1) * l.ldw * es <= limit;
  auto tiles = [&](int rows, int cols) { return about_tiles(l.m, groups, rows) * ((l.n + cols - 1) / cols); };
  constexpr int G = GATED ? 2 : 1;
  const int64_t small = tiles(32, 32 / G);
  if (l.m <= 48 * (int64_t)groups || small <= (!aligned ? (ADAPTERS ? 256 : 512) : DT == BZ_F32 ? 768 : 512)) {
    if constexpr (!GATED)
      if (small <= 128)
        return aligned ? launch_split<DT, 8, true, false, ADAPTERS, 16>(l, call) : launch_split<DT, 8, false, false, ADAPTERS, 16>(l, call);
    if (!aligned) return launch_split<DT, 4, false, GATED, ADAPTERS>(l, call);
    if constexpr (!ADAPTERS)
      if (small > 256) return launch_split<DT, 4, true, GATED, ADAPTERS>(l, call);
    return launch_split<DT, 8, true, GATED, ADAPTERS>(l, call);
  }
  if (aligned && near) {
    if constexpr (DT != BZ_F32) {
      const int64_t c44 = wide_cost<1>(tiles(256, 256 / G), {100}), c22 = wide_cost<2>(tiles(128, 128 / G), {33, 56});
      const int64_t c12 = wide_cost<2>(tiles(64, 128 / G), {26, 33});
      const int64_t c11 = wide_cost<3>(tiles(64, 64), {19, 25, 31});
      const int64_t large = std::min(std::min(c44, c22), c12), least = GATED ? large : std::min(large, c11);
      if (c44 == least) return launch_wide<DT, 4, 4, 2, GATED, ADAPTERS>(l, call);
      if (c12 == least) return launch_wide<DT, 1, 2, 3, GATED, ADAPTERS>(l, call);
      if (c22 == least) return launch_wide<DT, 2, 2, 2, GATED, ADAPTERS>(l, call);
    }
    return launch_wide<DT, 1, GATED ? 2 : 1, 3, GATED, ADAPTERS>(l, call);
  }
  return launch_tile<DT, 64, GATED ? 128 : 64, GATED, ADAPTERS>(l, call);
}

}  // namespace groups

// checks that the layers' activation and its parameters make sense, and what goes into their epilogue
inline int layer_act(const char* who, int act, int act_size, const float* p0, const float* p1, const float* p2, int n) {
  BZ_REQUIRE(act == BZ_ACT_NONE || act == BZ_ACT_PRELU || act == BZ_ACT_DICE || act == BZ_ACT_LEAKY_RELU || act == BZ_ACT_SIGMOID,
             "%s: activation %d", who, act);
  if (act == BZ_ACT_PRELU) BZ_REQUIRE(p0 && (act_size == 1 || act_size == n), "%s: PRelu with %d slopes for %d columns", who, p0 ? act_size : 0, n);
  if (act == BZ_ACT_DICE) {
    BZ_REQUIRE(p0 && p1 && p2, "%s: Dice without its parameters", who);
    BZ_REQUIRE(act_size == 0 || act_size == n, "%s: Dice with %d parameters for %d columns", who, act_size, n);
  }
  return BZ_OK;
}

}  // namespace bz
