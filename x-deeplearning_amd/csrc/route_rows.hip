// route_rows.hip -- the moves of a mixture of experts: the gate's choice (bz_route_topk), entries and rows in their experts' order
// (bz_group_rows), results back at their rows (bz_merge_rows) and the gradient of that (bz_merge_rows_grad).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "bz_common.h"
#include "rows_common.h"

namespace {

using namespace bz::rows;

// ---------------------------------------------------------------------------------------------
// the gate's choice
// ---------------------------------------------------------------------------------------------
// L lanes own a row, V neighbouring logits each.  The k largest are found one after the other: the largest of a lane's, of the
// lanes' (lane rotations inside 16 lanes, no LDS), then the lowest index that has it, and its owner drops it.  Nothing but
// comparisons decides, so the choice is exact whatever the type.  Lane j keeps the j-th.
// A 2-byte logit and its index make one 32-bit word that orders both: the value's bits, turned so that they order as the value does, above
// 65535 - index (0: none), and one search finds the two (16384 x 128 bf16, 8 of them: 6.0 us with a search for each, 5.2 this way).
// That is 1.0 TB/s; what bounds it are the instructions of k searches in a row, and one launch where rows are few (one row of 8: 1.5 us).
template <int DT, int L, int V>
__global__ __launch_bounds__(256) void bz_route_kernel(const char* __restrict__ logits, int64_t ld, int64_t rows, int n, int k,
                                                       int32_t* __restrict__ ids, float* __restrict__ weights, int score,
                                                       int renormalize, float scale) {
  constexpr int ES = Elem<DT>::kSize;
  const float kNone = -__builtin_huge_valf();
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const bool there = row < rows;
  const char* p = logits + ((there ? row : rows - 1) * ld + lane * V) * ES;
  float v[V];
  if (lane * V + V <= n) {
    char raw[V * ES];
    __builtin_memcpy(raw, p, V * ES);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = Elem<DT>::get(raw + i * ES);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = lane * V + i < n ? Elem<DT>::get(p + i * ES) : kNone;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = v[i] != v[i] ? kNone : v[i];
  float first = kNone, total = 0.f, mine = kNone;
  int my_id = -1;
  // the largest is known: what the others' weights are measured by
  auto begin = [&](float m) {
    first = m;
    if (score == BZ_ROUTE_SOFTMAX && !renormalize) {
#pragma unroll
      for (int i = 0; i < V; ++i) total += v[i] == kNone ? 0.f : exp_from(v[i], first);
      total = reduce<L>(total, [](float a, float b) { return a + b; });
    }
  };
  if constexpr (ES == 2) {
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t bits = DT == BZ_BF16 ? __float_as_uint(v[i]) >> 16 : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[i]);
      const uint32_t order = bits == 0x8000u || bits == 0 ? 0x8000u : bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u;
      key[i] = v[i] == kNone ? 0u : order << 16 | (0xffffu - (lane * V + i));
    }
    for (int j = 0; j < k; ++j) {
      uint32_t m = key[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = max(m, key[i]);
      m = reduce<L>(m, [](uint32_t a, uint32_t b) { return max(a, b); });
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = key[i] == m ? 0u : key[i];
      const uint32_t order = m >> 16, bits = order & 0x8000u ? order & 0x7fffu : ~order & 0xffffu;
      const float value = m == 0 ? kNone : DT == BZ_BF16 ? __uint_as_float(bits << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
      if (j == 0) begin(value);
      if (lane == j && m != 0) {
        my_id = 0xffff - (int)(m & 0xffffu);
        mine = value;
      }
    }
  } else {
    for (int j = 0; j < k; ++j) {
      float m = v[0];
#pragma unroll
      for (int i = 1; i < V; ++i) m = fmaxf(m, v[i]);
      const float lane_m = m;
      m = reduce<L>(m, [](float a, float b) { return fmaxf(a, b); });
      if (j == 0) begin(m);
      int at = 0x7fffffff;
      if (lane_m == m) {
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = v[i] == m ? lane * V + i : at;
      }
      at = reduce<L>(at, [](int a, int b) { return min(a, b); });
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at == lane * V + i) v[i] = kNone;
      if (lane == j && m != kNone) {
        my_id = at;
        mine = m;
      }
    }
  }
  float w = 0.f;
  if (my_id >= 0) w = score == BZ_ROUTE_SOFTMAX ? exp_from(mine, first) : 1.f / (1.f + expf(-mine));
  if (renormalize) total = reduce<L>(w, [](float a, float b) { return a + b; });
  if (renormalize || score == BZ_ROUTE_SOFTMAX) w = total > 0.f ? w / total : 0.f;
  if (there && lane < k) {
    ids[row * k + lane] = my_id;
    weights[row * k + lane] = w * scale;
  }
}

// A launch has fewer than 2^32 threads: more rows, of `threads` each, go by in parts.  f(first row, rows of the part)
constexpr int64_t kPartThreads = (int64_t)1 << 31;
template <typename F>
int in_parts(int64_t rows, int64_t threads, const F& f) {
  const int64_t part = std::max<int64_t>(1, kPartThreads / threads);
  for (int64_t r = 0; r < rows; r += part) {
    const int rc = f(r, std::min(part, rows - r));
    if (rc != BZ_OK) return rc;
  }
  return BZ_OK;
}

template <int DT, int L, int V>
int launch_route(const bz_route_desc& d, hipStream_t st) {
  return in_parts(d.rows, L, [&](int64_t r0, int64_t rows) {
    hipLaunchKernelGGL((bz_route_kernel<DT, L, V>), dim3((uint32_t)((rows * L + 255) / 256)), dim3(256), 0, st,
                       (const char*)d.logits + r0 * d.ld * Elem<DT>::kSize, d.ld, rows, d.n, d.k, d.ids + r0 * d.k, d.weights + r0 * d.k, d.score,
                       d.renormalize, d.scale);
    BZ_LAUNCH_OK("bz_route_kernel");
    return (int)BZ_OK;
  });
}

template <int DT>
int route(const bz_route_desc& d, hipStream_t st) {
  if (d.n <= 16) return launch_route<DT, 16, 1>(d, st);
  if (d.n <= 64) return launch_route<DT, 16, 4>(d, st);
  if (d.n <= 128) return launch_route<DT, 16, 8>(d, st);
  if (d.n <= 256) return launch_route<DT, 64, 4>(d, st);
  return launch_route<DT, 64, 16>(d, st);
}

// ---------------------------------------------------------------------------------------------
// entries in their groups' order
// ---------------------------------------------------------------------------------------------
// A counting sort that keeps the order within a group.  A workgroup owns a run of entries; an entry's position is
//   entries of lower groups + entries of its group in earlier runs + those in its own run before it.
// The first two come from counts, the last from the wave's ballots: the lanes whose group has the same bits are an entry's peers.
// Integer sums only, so the result does not depend on the order in which anything runs.
// Counting and placing are chains of trips to memory, not bytes: 131072 entries of 128 groups (1.6 MB) take 5.0 and 7.1 us.
constexpr int kGroupThreads = 256, kGroupWaves = 4;
constexpr int kGroupRun = 1024;      // entries of a workgroup where counts come from a launch in front
constexpr int kGroupMaxRuns = 256;   // (each reads the counts of all)

// the lanes that hold the same group as this one; `bits` of the number tell groups apart
__device__ __forceinline__ uint64_t peers(int g, int bits) {
  uint64_t same = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const uint64_t has = __ballot((g >> b) & 1);
    same &= (g >> b) & 1 ? has : ~has;
  }
  return same;
}

// group of entry i, `groups` where it has none or is not below end; any entry is read in its place then, so that loads need no branch
// and many are on their way together (end > 0)
__device__ __forceinline__ int group_at(const int32_t* ids, int64_t i, int64_t end, int groups) {
  const uint32_t g = (uint32_t)ids[min(i, end - 1)];
  return i < end && g < (uint32_t)groups ? (int)g : groups;
}

// f(group, entry) for the entries begin + lane, begin + lane + step, ..: below end; kAhead entries are on their way at a time (one trip
// to memory each took 0.6 us).  early: the groups of the first of them, if they are there already.
constexpr int kAhead = 8;
template <typename F>
__device__ __forceinline__ void each_group(const int32_t* ids, int64_t begin, int64_t end, int lane, int64_t step, int groups, const F& f,
                                           const int* early = nullptr) {
  for (int64_t i0 = begin; i0 < end; i0 += kAhead * step) {  // (end > 0 in here)
    int g[kAhead];
    if (early != nullptr && i0 == begin) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) g[a] = early[a];
    } else {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) g[a] = group_at(ids, i0 + a * step + lane, end, groups);
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (i0 + a * step < end) f(g[a], i0 + a * step + lane);
  }
}

// What a run holds of every group: rows of whole 16 bytes, the last of which need not hold anything
__host__ __device__ __forceinline__ int counts_pitch(int groups) { return (groups + 3) / 4 * 4; }

__global__ __launch_bounds__(kGroupThreads) void bz_group_count_kernel(const int32_t* __restrict__ ids, int64_t n, int64_t run, int groups,
                                                                       int32_t* __restrict__ counts) {
  __shared__ int sum[BZ_GROUP_MAX_GROUPS];
  for (int g = threadIdx.x; g < groups; g += kGroupThreads) sum[g] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t begin = blockIdx.x * run, end = min(begin + run, n);
  each_group(ids, begin + wave * 64, end, lane, kGroupThreads, groups, [&](int g, int64_t) {
    if (g < groups) atomicAdd(&sum[g], 1);
  });
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kGroupThreads) counts[(int64_t)blockIdx.x * counts_pitch(groups) + g] = sum[g];
}

// The positions of a workgroup's run.  counts: what bz_group_count_kernel found in every run; NULL: the workgroup counts all entries
// itself (few of them: one launch instead of two).
__global__ __launch_bounds__(kGroupThreads) void bz_group_place_kernel(const int32_t* __restrict__ ids, int64_t n, int64_t run, int groups,
                                                                       int bits, const int32_t* __restrict__ counts,
                                                                       int32_t* __restrict__ offsets, int32_t* __restrict__ order,
                                                                       int32_t* __restrict__ position) {
  __shared__ int before[BZ_GROUP_MAX_GROUPS];  // entries of the group in earlier runs
  __shared__ int total[BZ_GROUP_MAX_GROUPS];
  __shared__ int in_wave[kGroupWaves][BZ_GROUP_MAX_GROUPS];  // entries of the group in the wave's stretch; later where the next one goes
  __shared__ int sums[kGroupWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t begin = blockIdx.x * run, end = min(begin + run, n);
  // a wave's share of the run is one stretch, so that earlier waves hold earlier entries
  const int64_t share = ((run + kGroupWaves - 1) / kGroupWaves + 63) / 64 * 64;
  const int64_t wbegin = min(begin + wave * share, end), wend = min(wbegin + share, end);
  int early[kAhead];  // the share's first entries, on their way beside the counts
#pragma unroll
  for (int a = 0; a < kAhead; ++a) early[a] = n > 0 ? group_at(ids, wbegin + a * 64 + lane, wend, groups) : groups;
  for (int g = tid; g < groups; g += kGroupThreads) {
    before[g] = total[g] = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) in_wave[w][g] = 0;
  }
  __syncthreads();
  if (counts != nullptr) {
    // four groups a thread, the runs shared by as many threads as there are for those
    const int quads = counts_pitch(groups) / 4, slices = kGroupThreads / quads, slice = tid / quads, g0 = tid % quads * 4, runs = gridDim.x;
    int b[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
    for (int r0 = slice < slices ? slice : runs; r0 < runs; r0 += 16 * slices) {
      int c[16][4];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        __builtin_memcpy(c[i], counts + (int64_t)min(r0 + i * slices, runs - 1) * counts_pitch(groups) + g0, 16);
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + i * slices;
          t[e] += r < runs ? c[i][e] : 0;
          b[e] += r < (int)blockIdx.x ? c[i][e] : 0;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (slice < slices && g0 + e < groups) {
        atomicAdd(&total[g0 + e], t[e]);
        atomicAdd(&before[g0 + e], b[e]);
      }
  }
  each_group(ids, wbegin, wend, lane, 64, groups, [&](int g, int64_t) {
    if (g < groups) atomicAdd(&in_wave[wave][g], 1);
  }, early);
  if (counts == nullptr) {
    each_group(ids, wave * 64, n, lane, kGroupThreads, groups, [&](int g, int64_t i) {
      if (g < groups) atomicAdd(&total[g], 1);
      if (g < groups && i < begin) atomicAdd(&before[g], 1);
    });
  }
  __syncthreads();
  // exclusive sums of the totals, a stretch of groups a thread
  const int stretch = (groups + kGroupThreads - 1) / kGroupThreads;
  int mine = 0;
  for (int i = 0; i < stretch; ++i) mine += tid * stretch + i < groups ? total[tid * stretch + i] : 0;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(upto, o);
    upto += lane >= o ? u : 0;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int base = upto - mine;
  for (int w = 0; w < wave; ++w) base += sums[w];
  for (int i = 0; i < stretch; ++i) {
    const int g = tid * stretch + i;
    if (g >= groups) break;
    if (blockIdx.x == 0) {
      offsets[g] = base;
      if (g == groups - 1) offsets[groups] = base + total[g];
    }
    int at = base + before[g];
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      const int c = in_wave[w][g];
      in_wave[w][g] = at;
      at += c;
    }
    base += total[g];
  }
  __syncthreads();
  each_group(ids, wbegin, wend, lane, 64, groups, [&](int g, int64_t i) {
    const uint64_t same = peers(g, bits);
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int at = g < groups ? in_wave[wave][g] + rank : -1;
    __builtin_amdgcn_wave_barrier();
    if (g < groups) {
      if (rank == 0) in_wave[wave][g] += __popcll(same);
      order[at] = (int32_t)i;
    }
    if (position != nullptr && i < wend) position[i] = at;
    __builtin_amdgcn_wave_barrier();
  }, early);
}

// Few entries (kFewEntries), rows and all, in one launch: every workgroup counts all entries and places a run of at most 64, whose rows it moves.  The
// rows' first chunks are on their way while it counts.  DT: the rows' type.
// 2048 x 2 rows of 896 fp16, 11 MB: 7.0 us, 1.6 TB/s (11.7 with loads under branches).  What bounds it is its chain: ids, counts, sums,
// the run's positions, stores.
constexpr int kFewRun = 64, kFewChunks = 4, kFewAhead = 16, kFewShift = 3;
template <int DT>
__global__ __launch_bounds__(kGroupThreads) void bz_group_few_kernel(const int32_t* __restrict__ ids, int n, int run, int groups, int bits,
                                                                     int32_t* __restrict__ offsets, int32_t* __restrict__ order,
                                                                     int32_t* __restrict__ position, const char* __restrict__ x,
                                                                     char* __restrict__ xs, int64_t ld_x, int64_t ld_xs, int dim, int per) {
  constexpr int ES = Elem<DT>::kSize, CH = 16 / ES;
  __shared__ uint32_t count[BZ_GROUP_MAX_GROUPS];  // entries of the group, and 65536 times those in front of the run; later where its first one goes
  __shared__ int sums[kGroupWaves];
  __shared__ int to[kFewRun];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int begin = blockIdx.x * run, end = min(begin + run, n);
  const uint32_t chunks = (uint32_t)(dim - 1) / CH + 1, items = (uint32_t)(end - begin) / (uint32_t)per * chunks;
  const int64_t row0 = (uint32_t)begin / (uint32_t)per;
  auto load = [&](uint32_t q) {
    const uint32_t row = q / chunks;
    const int c = chunk_start((int)(q - row * chunks), CH, dim);
    return Chunk<DT>::load(x + ((row0 + row) * ld_x + c) * ES, dim - c);
  };
  Chunk<DT> early[kFewChunks];
#pragma unroll
  for (int i = 0; i < kFewChunks; ++i)
    if (tid + i * kGroupThreads < items) early[i] = load(tid + i * kGroupThreads);
  const int own = group_at(ids, begin + lane, end, groups);
  // Eight counters a group where groups are few for so many entries: lanes that add to one wait for each other (8000 x 2 entries of 2 groups
  // 13.7 us and 23.6 with one, of 8 13.8 and 14.8, of 16 13.8 and 13.3; 2048 x 2 of 8 8.4 and 8.1).
  const int shift = groups <= 64 && n > 1024 * groups ? kFewShift : 0, copies = 1 << shift;
  for (int g = tid; g < groups << shift; g += kGroupThreads) count[g] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += kFewAhead * kGroupThreads) {
    int g[kFewAhead];
#pragma unroll
    for (int a = 0; a < kFewAhead; ++a) g[a] = group_at(ids, i0 + a * kGroupThreads + tid, n, groups);
#pragma unroll
    for (int a = 0; a < kFewAhead; ++a)
      if (g[a] < groups) atomicAdd(&count[(g[a] << shift) + (lane & (copies - 1))], i0 + a * kGroupThreads + tid < begin ? 65537u : 1u);
  }
  __syncthreads();
  if (shift > 0) {
    uint32_t sum = 0;
#pragma unroll
    for (int c = 0; c < 1 << kFewShift; ++c) sum += count[(min(tid, groups - 1) << kFewShift) + c];
    __syncthreads();
    if (tid < groups) count[tid] = sum;
    __syncthreads();
  }
  // exclusive sums of the totals, a stretch of groups a thread
  const int stretch = (groups + kGroupThreads - 1) / kGroupThreads;
  int mine = 0;
  for (int i = 0; i < stretch; ++i) mine += tid * stretch + i < groups ? (int)(count[tid * stretch + i] & 0xffffu) : 0;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(upto, o);
    upto += lane >= o ? u : 0;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int base = upto - mine;
  for (int w = 0; w < wave; ++w) base += sums[w];
  for (int i = 0; i < stretch; ++i) {
    const int g = tid * stretch + i;
    if (g >= groups) break;
    const int total = (int)(count[g] & 0xffffu);
    if (blockIdx.x == 0) {
      offsets[g] = base;
      if (g == groups - 1) offsets[groups] = base + total;
    }
    count[g] = base + (count[g] >> 16);
    base += total;
  }
  __syncthreads();
  if (wave == 0) {
    const uint64_t same = peers(own, bits);
    const int at = own < groups ? (int)count[own] + __popcll(same & ((1ull << lane) - 1)) : -1;
    if (begin + lane < end) {
      to[lane] = at;
      position[begin + lane] = at;
      if (at >= 0) order[at] = begin + lane;
    }
  }
  __syncthreads();
  auto put = [&](uint32_t q, const Chunk<DT>& v) {
    const uint32_t row = q / chunks;
    const int c = chunk_start((int)(q - row * chunks), CH, dim);
    for (int j = 0; j < per; ++j) {
      const int at = to[row * per + j];
      if (at >= 0) v.store(xs + ((int64_t)at * ld_xs + c) * ES, dim - c);
    }
  };
#pragma unroll
  for (int i = 0; i < kFewChunks; ++i)
    if (tid + i * kGroupThreads < items) put(tid + i * kGroupThreads, early[i]);
  for (uint32_t q = tid + kFewChunks * kGroupThreads; q < items; q += kGroupThreads) put(q, load(q));
}

// Rows to where their entries went: 16 bytes a thread, read once and stored `per` times.  ONCE: more than the caches keep (beyond_caches).
// Bound by HBM: 16384 x 8 rows of 2048 bf16, 604 MB, in 102 us, 5.9 TB/s.
template <int DT, bool ONCE>
__global__ __launch_bounds__(256) void bz_spread_kernel(const char* __restrict__ x, const int32_t* __restrict__ position, char* __restrict__ xs,
                                                        int64_t items, int64_t ld_x, int64_t ld_xs, int chunks, int dim, int per) {
  constexpr int ES = Elem<DT>::kSize, CH = 16 / ES;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= items) return;
  const int64_t row = item / chunks;
  const int c = chunk_start((int)(item - row * chunks), CH, dim);
  const Chunk<DT> v = Chunk<DT>::load(x + (row * ld_x + c) * ES, dim - c);
  for (int j = 0; j < per; ++j) {
    const int at = position[row * per + j];
    if (at >= 0) v.template store<ONCE>(xs + ((int64_t)at * ld_xs + c) * ES, dim - c);
  }
}

// ---------------------------------------------------------------------------------------------
// results back at their rows
// ---------------------------------------------------------------------------------------------
// 16 bytes of a row a thread; the results' chunks are all asked for before any is used.  K: as many as there may be (2, 4, 8, 16).
// Bound by HBM: 8192 x 8 rows of 2048 bf16, 302 MB, in 53 us, 5.7 TB/s (61 with loads that the caches keep); few rows by three trips to memory
// (300 x 4 rows of 445 fp32 2.9 us).
template <int DT, typename OutT, int K>
__global__ __launch_bounds__(256) void bz_merge_kernel(const char* __restrict__ xs, const int32_t* __restrict__ position,
                                                       const float* __restrict__ weights, OutT* __restrict__ y, int64_t items, int64_t n,
                                                       int64_t ld_xs, int64_t ld_y, int chunks, int dim, int k) {
  constexpr int ES = Elem<DT>::kSize, CH = 16 / ES;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= items) return;
  const int64_t row = item / chunks;
  const int c = chunk_start((int)(item - row * chunks), CH, dim), count = min(CH, dim - c);
  int at[K];
  float w[K], sum[CH];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    at[j] = j < k ? position[row * k + j] : -1;
    at[j] = (uint64_t)(int64_t)at[j] < (uint64_t)n ? at[j] : -1;
    w[j] = j < k && weights != nullptr ? weights[row * k + j] : 1.f;
  }
  Chunk<DT> v[K];
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (at[j] >= 0) v[j] = Chunk<DT>::template load<true>(xs + ((int64_t)at[j] * ld_xs + c) * ES, dim - c);
#pragma unroll
  for (int i = 0; i < CH; ++i) sum[i] = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < CH; ++i) sum[i] = at[j] >= 0 ? fmaf(w[j], v[j].at(i), sum[i]) : sum[i];
  store_floats<OutT, CH>(y + row * ld_y + c, sum, count);
}

// One wave a row: dy's chunk is read once, multiplied with each weight and stored, and multiplied with each result.  The results' chunks
// are all asked for before any is used.  K: as many results as there may be (2, 4, 8, 16).  ONCE: more is written than the caches keep.
// Bound by HBM: 8192 x 8 rows of 2048 bf16, 570 MB read and written, in 130 us, 4.4 TB/s of a copy's 4.9.
template <int DT, int K, bool ONCE>
__global__ __launch_bounds__(256) void bz_merge_grad_kernel(const char* __restrict__ dy, const char* __restrict__ xs,
                                                            const int32_t* __restrict__ position, const float* __restrict__ weights,
                                                            char* __restrict__ dxs, float* __restrict__ dweights, int64_t rows, int64_t n,
                                                            int64_t ld_dy, int64_t ld_xs, int64_t ld_dxs, int k, int dim) {
  constexpr int ES = Elem<DT>::kSize, CH = 16 / ES;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  const int chunks = (dim - 1) / CH + 1;
  int at[K];
  float w[K], dot[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int p = j < k ? position[row * k + j] : -1;
    at[j] = __builtin_amdgcn_readfirstlane((uint64_t)(int64_t)p < (uint64_t)n ? p : -1);
    w[j] = j < k && weights != nullptr ? weights[row * k + j] : 1.f;
    dot[j] = 0.f;
  }
  for (int q = lane; q < chunks; q += 64) {
    const int c = chunk_start(q, CH, dim), again = q * CH - c;  // the last chunk begins earlier: its first `again` are another's
    const Chunk<DT> g = Chunk<DT>::load(dy + (row * ld_dy + c) * ES, dim - c);
    if (dweights != nullptr) {
      Chunk<DT> v[K];
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (at[j] >= 0) v[j] = Chunk<DT>::template load<true>(xs + ((int64_t)at[j] * ld_xs + c) * ES, dim - c);
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (at[j] >= 0) {
#pragma unroll
          for (int i = 0; i < CH; ++i) dot[j] = i >= again ? fmaf(g.at(i), v[j].at(i), dot[j]) : dot[j];
        }
    }
    if (dxs != nullptr) {
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (at[j] >= 0) {
          float out[CH];
#pragma unroll
          for (int i = 0; i < CH; ++i) out[i] = w[j] * g.at(i);
          store_floats<typename Elem<DT>::type, CH, ONCE>((typename Elem<DT>::type*)(dxs + ((int64_t)at[j] * ld_dxs + c) * ES), out,
                                                          min(CH, dim - c));
        }
    }
  }
  if (dweights == nullptr) return;
  float mine = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const float s = reduce<64>(dot[j], [](float a, float b) { return a + b; });
    mine = lane == j ? s : mine;
  }
  if (lane < k) dweights[row * k + lane] = mine;
}

bool float_type(int dt) { return dt == BZ_F32 || dt == BZ_F16 || dt == BZ_BF16; }

template <typename F>
int by_type(int dt, const F& f) {
  if (dt == BZ_F32) return f(std::integral_constant<int, BZ_F32>());
  if (dt == BZ_F16) return f(std::integral_constant<int, BZ_F16>());
  return f(std::integral_constant<int, BZ_BF16>());
}

// Whether rows that are written are more than the 256 MB cache keeps for whoever reads them next.  Written past the caches they take a tenth
// less (16384 x 8 rows of 2048 bf16 moved in 115 us, 128 with ordinary stores; the gradient of 8192 x 8 such rows 134 and 144), but what
// reads fewer of them soon takes longer (8192 x 2 rows of 1024 bf16 moved, through two layers and merged: 194 us and 189).
bool beyond_caches(int64_t bytes) { return bytes > (int64_t)128 << 20; }

// entries of a workgroup's run, and the runs
int64_t run_length(int64_t n) {
  const int64_t run = std::max<int64_t>(kGroupRun, (n + kGroupMaxRuns - 1) / kGroupMaxRuns);
  return (run + 255) / 256 * 256;
}
// Up to here every workgroup counts all entries itself.
constexpr int64_t kGroupAlone = 8192;
// Up to here with their rows in the same launch (us there and in three: 8192 x 2 rows of 512 bf16 13.3 and 15.5, 4096 x 4 12.5 and 16.0, 16384 x 1
// 16.8 and 15.1, 8192 x 4 19.0 and 18.4).
constexpr int64_t kFewEntries = 16384, kFewRows = 8192;

}  // namespace

extern "C" {

int bz_route_topk(const bz_route_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_route_topk: null descriptor");
  const bz_route_desc& d = *desc;
  BZ_REQUIRE(float_type(d.dtype), "bz_route_topk: dtype %d", d.dtype);
  BZ_REQUIRE(d.n >= 1 && d.n <= BZ_ROUTE_MAX_N, "bz_route_topk: n %d (1..%d)", d.n, BZ_ROUTE_MAX_N);
  BZ_REQUIRE(d.k >= 1 && d.k <= BZ_ROUTE_MAX_K && d.k <= d.n, "bz_route_topk: k %d of %d (1..%d)", d.k, d.n, BZ_ROUTE_MAX_K);
  BZ_REQUIRE(d.score == BZ_ROUTE_SOFTMAX || d.score == BZ_ROUTE_SIGMOID, "bz_route_topk: score %d", d.score);
  BZ_REQUIRE(d.rows >= 0 && d.rows < (int64_t)1 << 31, "bz_route_topk: rows %lld", (long long)d.rows);
  BZ_REQUIRE(d.ld >= d.n, "bz_route_topk: ld %lld, n %d", (long long)d.ld, d.n);
  if (d.rows == 0) return BZ_OK;
  BZ_REQUIRE(d.logits && d.ids && d.weights, "bz_route_topk: null pointer");
  return by_type(d.dtype, [&](auto dt) { return route<decltype(dt)::value>(d, bz::as_stream(stream)); });
}

int64_t bz_group_scratch_bytes(int64_t n, int groups) {
  if (n <= kGroupAlone || groups < 1) return 0;
  const int64_t run = run_length(n);
  return (n + run - 1) / run * counts_pitch(std::min(groups, BZ_GROUP_MAX_GROUPS)) * (int64_t)sizeof(int32_t);
}

int bz_group_rows(const bz_group_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_group_rows: null descriptor");
  const bz_group_desc& d = *desc;
  BZ_REQUIRE(d.n >= 0 && d.n < (int64_t)1 << 31, "bz_group_rows: n %lld", (long long)d.n);
  BZ_REQUIRE(d.groups >= 1 && d.groups <= BZ_GROUP_MAX_GROUPS, "bz_group_rows: groups %d (1..%d)", d.groups, BZ_GROUP_MAX_GROUPS);
  BZ_REQUIRE(d.offsets != nullptr, "bz_group_rows: null pointer");
  BZ_REQUIRE(d.n == 0 || (d.ids && d.order), "bz_group_rows: null pointer");
  const int64_t need = bz_group_scratch_bytes(d.n, d.groups);
  BZ_REQUIRE(need == 0 || (d.scratch != nullptr && d.scratch_bytes >= need), "bz_group_rows: scratch of %lld bytes, %lld needed",
             (long long)(d.scratch ? d.scratch_bytes : 0), (long long)need);
  if (d.x != nullptr) {
    BZ_REQUIRE(float_type(d.dtype), "bz_group_rows: dtype %d", d.dtype);
    BZ_REQUIRE(d.per >= 1 && d.n % d.per == 0, "bz_group_rows: %lld entries, %d a row", (long long)d.n, d.per);
    BZ_REQUIRE(d.dim >= 1 && d.ld_x >= d.dim && d.ld_xs >= d.dim, "bz_group_rows: rows of %d at pitches %lld and %lld", d.dim,
               (long long)d.ld_x, (long long)d.ld_xs);
    BZ_REQUIRE(d.n == 0 || (d.xs && d.position), "bz_group_rows: null pointer");
  }
  const hipStream_t st = bz::as_stream(stream);
  int bits = 1;
  while (d.groups >> bits) ++bits;  // (the number `groups`, of entries in none, among them)
  int32_t* counts = need > 0 ? (int32_t*)d.scratch : nullptr;
  const int64_t few = (std::max<int64_t>(1, d.n / 512) + d.per - 1) / std::max(1, d.per) * d.per;  // about 512 workgroups, whole rows each
  if (d.x != nullptr && d.n > 0 && d.n <= kFewEntries && d.n / d.per <= kFewRows && few <= kFewRun && d.dim < 1 << 24)  // (its chunks of 32 bits)
    return by_type(d.dtype, [&](auto dt) {
      hipLaunchKernelGGL((bz_group_few_kernel<decltype(dt)::value>), dim3((uint32_t)((d.n + few - 1) / few)), dim3(kGroupThreads), 0, st, d.ids,
                         (int)d.n, (int)few, d.groups, bits, d.offsets, d.order, d.position, (const char*)d.x, (char*)d.xs, d.ld_x, d.ld_xs,
                         d.dim, d.per);
      BZ_LAUNCH_OK("bz_group_few_kernel");
      return (int)BZ_OK;
    });
  const int64_t run = counts != nullptr ? run_length(d.n) : 256;
  const uint32_t wg = (uint32_t)std::max<int64_t>(1, (d.n + run - 1) / run);
  if (counts != nullptr) {
    hipLaunchKernelGGL(bz_group_count_kernel, dim3(wg), dim3(kGroupThreads), 0, st, d.ids, d.n, run, d.groups, counts);
    BZ_LAUNCH_OK("bz_group_count_kernel");
  }
  hipLaunchKernelGGL(bz_group_place_kernel, dim3(wg), dim3(kGroupThreads), 0, st, d.ids, d.n, run, d.groups, bits, (const int32_t*)counts,
                     d.offsets, d.order, d.position);
  BZ_LAUNCH_OK("bz_group_place_kernel");
  if (d.x == nullptr || d.n == 0) return BZ_OK;
  return by_type(d.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const int chunks = (d.dim - 1) / (16 / Elem<DT>::kSize) + 1;
    constexpr int ES = Elem<DT>::kSize;
    auto* kernel = beyond_caches(d.n * d.dim * ES) ? bz_spread_kernel<DT, true> : bz_spread_kernel<DT, false>;
    return in_parts(d.n / d.per, chunks, [&](int64_t r0, int64_t rows) {
      const int64_t items = rows * chunks;
      hipLaunchKernelGGL(kernel, dim3((uint32_t)((items + 255) / 256)), dim3(256), 0, st, (const char*)d.x + r0 * d.ld_x * ES,
                         (const int32_t*)d.position + r0 * d.per, (char*)d.xs, items, d.ld_x, d.ld_xs, chunks, d.dim, d.per);
      BZ_LAUNCH_OK("bz_spread_kernel");
      return (int)BZ_OK;
    });
  });
}

int bz_merge_rows(const bz_merge_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_merge_rows: null descriptor");
  const bz_merge_desc& d = *desc;
  BZ_REQUIRE(float_type(d.dtype), "bz_merge_rows: dtype %d", d.dtype);
  BZ_REQUIRE(d.out_dtype == d.dtype || d.out_dtype == BZ_F32, "bz_merge_rows: out_dtype %d of dtype %d", d.out_dtype, d.dtype);
  BZ_REQUIRE(d.k >= 1 && d.k <= BZ_ROUTE_MAX_K, "bz_merge_rows: k %d (1..%d)", d.k, BZ_ROUTE_MAX_K);
  BZ_REQUIRE(d.rows >= 0 && d.rows < (int64_t)1 << 31 && d.n >= 0 && d.n < (int64_t)1 << 31, "bz_merge_rows: rows %lld, n %lld",
             (long long)d.rows, (long long)d.n);
  BZ_REQUIRE(d.dim >= 1 && d.ld_xs >= d.dim && d.ld_y >= d.dim, "bz_merge_rows: rows of %d at pitches %lld and %lld", d.dim,
             (long long)d.ld_xs, (long long)d.ld_y);
  if (d.rows == 0) return BZ_OK;
  BZ_REQUIRE((d.xs || d.n == 0) && d.position && d.y, "bz_merge_rows: null pointer");
  return by_type(d.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const int chunks = (d.dim - 1) / (16 / Elem<DT>::kSize) + 1;
    auto launch = [&](auto* y) {
      using OutT = std::remove_pointer_t<decltype(y)>;
      auto* kernel = d.k <= 2 ? bz_merge_kernel<DT, OutT, 2> : d.k <= 4 ? bz_merge_kernel<DT, OutT, 4> : d.k <= 8 ? bz_merge_kernel<DT, OutT, 8>
                                                                                                                  : bz_merge_kernel<DT, OutT, 16>;
      return in_parts(d.rows, chunks, [&](int64_t r0, int64_t rows) {
        const int64_t items = rows * chunks;
        hipLaunchKernelGGL(kernel, dim3((uint32_t)((items + 255) / 256)), dim3(256), 0, bz::as_stream(stream), (const char*)d.xs,
                           d.position + r0 * d.k, d.weights != nullptr ? d.weights + r0 * d.k : nullptr, y + r0 * d.ld_y, items, d.n, d.ld_xs, d.ld_y,
                           chunks, d.dim, d.k);
        BZ_LAUNCH_OK("bz_merge_kernel");
        return (int)BZ_OK;
      });
    };
    return d.out_dtype == DT ? launch((typename Elem<DT>::type*)d.y) : launch((float*)d.y);
  });
}

int bz_merge_rows_grad(const bz_merge_grad_desc* desc, bz_stream_t stream) {
  BZ_REQUIRE(desc != nullptr, "bz_merge_rows_grad: null descriptor");
  const bz_merge_grad_desc& d = *desc;
  BZ_REQUIRE(float_type(d.dtype), "bz_merge_rows_grad: dtype %d", d.dtype);
  BZ_REQUIRE(d.k >= 1 && d.k <= BZ_ROUTE_MAX_K, "bz_merge_rows_grad: k %d (1..%d)", d.k, BZ_ROUTE_MAX_K);
  BZ_REQUIRE(d.rows >= 0 && d.rows < (int64_t)1 << 31 && d.n >= 0 && d.n < (int64_t)1 << 31, "bz_merge_rows_grad: rows %lld, n %lld",
             (long long)d.rows, (long long)d.n);
  BZ_REQUIRE(d.dim >= 1 && d.ld_dy >= d.dim && (!d.dweights || d.ld_xs >= d.dim) && (!d.dxs || d.ld_dxs >= d.dim),
             "bz_merge_rows_grad: rows of %d at pitches %lld, %lld and %lld", d.dim, (long long)d.ld_dy, (long long)d.ld_xs, (long long)d.ld_dxs);
  if (d.rows == 0 || (!d.dxs && !d.dweights)) return BZ_OK;
  BZ_REQUIRE(d.dy && d.position && (d.xs || !d.dweights || d.n == 0), "bz_merge_rows_grad: null pointer");
  return by_type(d.dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto pick = [&](auto once) {
      constexpr bool ONCE = decltype(once)::value;
      return d.k <= 2   ? bz_merge_grad_kernel<DT, 2, ONCE>
             : d.k <= 4 ? bz_merge_grad_kernel<DT, 4, ONCE>
             : d.k <= 8 ? bz_merge_grad_kernel<DT, 8, ONCE>
                        : bz_merge_grad_kernel<DT, 16, ONCE>;
    };
    const int64_t bytes = d.dxs ? std::min<int64_t>(d.rows * d.k, d.n) * d.dim * Elem<DT>::kSize : 0;
    auto* kernel = beyond_caches(bytes) ? pick(std::true_type()) : pick(std::false_type());
    return in_parts(d.rows, 64, [&](int64_t r0, int64_t rows) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, bz::as_stream(stream),
                         (const char*)d.dy + r0 * d.ld_dy * Elem<DT>::kSize, (const char*)d.xs, d.position + r0 * d.k,
                         d.weights != nullptr ? d.weights + r0 * d.k : nullptr, (char*)d.dxs, d.dweights != nullptr ? d.dweights + r0 * d.k : nullptr,
                         rows, d.n, d.ld_dy, d.ld_xs, d.ld_dxs, d.k, d.dim);
      BZ_LAUNCH_OK("bz_merge_grad_kernel");
      return (int)BZ_OK;
    });
  });
}

}  // extern "C"
