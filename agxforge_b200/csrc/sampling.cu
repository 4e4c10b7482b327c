// sampling.cu — one token a row from logits, with temperature, top-k, top-p and min-p, at given uniform numbers.
//
// Weights are w = floor(2^40 exp((l - max) / T)) as 64-bit integers, so a row's sums are exact whatever their order and
// the token does not depend on how the row is split. Tokens are ranked by a 64-bit key, the logit's order in the high
// half and the index (lower first) in the low half; top-k and top-p each keep the keys from some key up, min-p compares
// exp((l - max) / T) itself, and the token is the first kept index whose cumulative weight exceeds floor(u * total).
//
// A cluster of CTAs takes a row: each CTA reads its range of the vocabulary once into shared memory (what does not fit
// is read again from global memory), and everything after that happens there and in its neighbours' shared memory.
//   1  the maximum (its first index is a greedy row's token) and the least finite logit
//   2  top-k: counts in 1,024 bins, equal steps of the logit down to weight zero or the least logit; the first CTA adds
//      the cluster's bins up and finds the one that holds rank k. Up to 2,048 elements in that bin and above are listed,
//      each CTA its own, and the first CTA collects them and finishes the row
//   3  top-p: the bins' exact weights (64 bits as two 32-bit shared-memory adds, the second with the first's carry, rarely
//      needed); the bin that holds the bar
//   4  where a bin holds a cut, only that bin is listed (and for top-p the weights above it are added up in the same pass).
//      The key the cut falls on: 1,024 finer bins, then a comparison of the few elements of one of them. A bin that is more
//      than a list (thousands of equal logits) is cut bit by bit
//   5  the kept weights' total and the token, in index order: the warp, then the element, that the target falls on
//
// 256 rows of 151,936 fp32 logits (155.6 MB, 23.8 us at the copy rate), eight CTAs a row, 37 rows at a time: 52 us greedy,
// 118 with the weights alone, 144 with top-k 50, 278 with top-p 0.95, 184 where rows mix all of these. The SMs bind it, not
// DRAM (fetching the next rows into L2 meanwhile gained nothing): of a top-p row's time (by clock, when the rows took 283) 5 us
// went to loading it and its maximum, 9.6 to the weights in bins (an exp and a shared-memory add each), 3.6 to the first CTA's
// sum of the cluster's bins, 6 to the list of the cut's bin and the weights above it, 2.7 to the cut and 2 to the draw, and
// the cluster's barriers between them leave warps waiting. One row with top-k 50: 12.9 us, steps and barriers; 64 rows of
// 92,544 with min-p: 22.3; 33 rows of 50,257 bf16, top-k 1,000: 27.4. Not kept: the listed keys sorted in place of finer bins
// (382 for the top-p rows, 43 for the 33), a pass of their own for the kept weights (310).
#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace agxc {
namespace {

namespace cg = cooperative_groups;

constexpr size_t align16(size_t v) { return (v + 15) / 16 * 16; }

struct SampleParams {
  const void* x;
  int64_t ld;
  int B, V, per, cached;  // per = elements of a CTA, cached = how many of them shared memory holds (a multiple of 16)
  const float* u;
  float T, top_p, min_p;
  int top_k;
  const float* T_a;
  const int32_t* k_a;
  const float* p_a;
  const float* m_a;
  int32_t* token;
  float* prob;
  unsigned* err;
};

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kFew = kThreads / 4, kBins = 1024, kList = 2048, kMaxCluster = 16;

constexpr int kCopies = 4;  // pieces that a CTA's range is copied in: the first is looked at while the last are on their way

template <int DT>
__device__ __forceinline__ float as_float(uint32_t bits) {
  if (DT == AGXC_F32) return __uint_as_float(bits);
  if (DT == AGXC_F16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  return __uint_as_float(bits << 16);
}

template <int DT>
struct Raw {
  using Type = uint32_t;
};
template <>
struct Raw<AGXC_F16> {
  using Type = uint16_t;
};
template <>
struct Raw<AGXC_BF16> {
  using Type = uint16_t;
};
template <int DT>
constexpr uint32_t kNaN = DT == AGXC_F32 ? 0x7FFFFFFFu : 0x7FFFu;
template <int DT>
constexpr uint32_t kMinusInf = DT == AGXC_F32 ? 0xFF800000u : DT == AGXC_F16 ? 0xFC00u : 0xFF80u;

// larger logits first, then lower indices: the larger key ranks first
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.f);  // the two zeros rank alike
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(o) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int key_index(uint64_t key) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key)); }

// floor(2^40 e) for 0 <= e <= 1
__device__ __forceinline__ uint64_t weight(float e) {
  const uint32_t b = __float_as_uint(e), m = (b & 0x7FFFFFu) | 0x800000u;
  const int up = static_cast<int>(b >> 23) - 110;
  return up >= 0 ? static_cast<uint64_t>(m) << up : static_cast<uint64_t>(m >> min(-up, 31));
}

// A sum of weights from their fp32 exps, 20 bits at a time: 8 + e rounded towards zero has floor(2^20 e) in its low bits,
// and 2^-17 plus what that leaves has the next 20. The constants' own bits are taken off by the count (at most 4,095).
struct WeightSum {
  uint32_t hi = 0, lo = 0, n = 0;
  __device__ void add(float e) {
    const float t = __fadd_rz(e, 8.f), u = __fadd_rz(__fsub_rn(e, __fsub_rn(t, 8.f)), 7.62939453125e-6f);
    hi += __float_as_uint(t);
    lo += __float_as_uint(u);
    ++n;
  }
  __device__ uint64_t get() const {
    return (static_cast<uint64_t>(hi - n * 0x41000000u) << 20) + (lo - n * 0x37000000u);
  }
};

struct Row {
  float best, inv_t, step;  // step = bins a unit of logit
  __device__ float e(float v) const { return expf(__fmul_rn(__fsub_rn(v, best), inv_t)); }
  __device__ float place(float v) const { return fminf(__fmul_rn(__fsub_rn(best, v), step), kBins - 1.f); }  // bin = its floor
};

struct Shared {
  float2 best;  // {largest, least}
  uint64_t sum[2];
  uint64_t copied[kCopies];
  int n_list, n_few, bin, first;
  uint64_t before, total, cut;
  uint64_t said[3];  // what the first CTA found
  uint64_t warp64[kWarps];
  uint64_t warp_kept[kWarps];
  alignas(16) uint32_t count[kBins];
  alignas(16) uint32_t lo[kBins];
  alignas(16) uint32_t hi[kBins];
  uint64_t few[kFew];
  uint64_t list[kList];
};

__device__ __forceinline__ int bin_of(float place) { return __float_as_int(__fadd_rz(place, 8388608.f)) - 0x4B000000; }

// one exact 64-bit sum among many in shared memory
__device__ __forceinline__ void add64(uint32_t* lo, uint32_t* hi, int at, uint64_t w) {
  const uint32_t l = static_cast<uint32_t>(w), old = atomicAdd(&lo[at], l);
  const uint32_t h = static_cast<uint32_t>(w >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(&hi[at], h);
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// The sum over a CTA, on every thread.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* sh) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += sh[w];
  return t;
}

// The sum over the threads below, and over all.
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* sh, uint64_t& total) {
  const int lane = threadIdx.x & 31;
  uint64_t up = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, up, m);
    if (lane >= m) up += o;
  }
  __syncthreads();
  if (lane == 31) sh[threadIdx.x >> 5] = up;
  __syncthreads();
  total = 0;
  uint64_t below = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == static_cast<int>(threadIdx.x >> 5)) below = total;
    total += sh[w];
  }
  return below + up - v;
}

// Sorts the list's first n keys (any n <= kList), the largest first.
__device__ void sort_list(uint64_t* list, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
  __syncthreads();
  for (int span = 2; span <= size; span <<= 1)
    for (int gap = span >> 1; gap >= 1; gap >>= 1) {
      for (int x = threadIdx.x; x < size / 2; x += kThreads) {
        const int i = (x & ~(gap - 1)) << 1 | (x & (gap - 1)), j = i | gap;
        const uint64_t a = list[i], b = list[j];
        if ((a < b) == ((i & span) == 0)) {
          list[i] = b;
          list[j] = a;
        }
      }
      __syncthreads();
    }
}

__device__ __forceinline__ uint64_t top_p_bar(float p, uint64_t total) {
  const double bar = ceil(__dmul_rn(static_cast<double>(p), __ll2double_rn(static_cast<long long>(total))));
  return bar > 1.0 ? static_cast<uint64_t>(bar) : 1;
}

__device__ __forceinline__ uint64_t target_of(float u, uint64_t total) {
  const double t = floor(__dmul_rn(static_cast<double>(u), __ll2double_rn(static_cast<long long>(total))));
  const uint64_t r = t > 0.0 ? static_cast<uint64_t>(t) : 0;
  return r < total ? r : total - 1;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  using T16 = typename Raw<DT>::Type;
  constexpr int kSize = sizeof(T16);
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  T16* cache = reinterpret_cast<T16*>(dyn + align16(sizeof(Shared)));
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / C;
  const int64_t base = static_cast<int64_t>(b) * p.ld;
  const int r0 = min(p.V, rank * p.per), n = min(p.V, r0 + p.per) - r0;
  // The range lies at `pad` in the CTA's space, so that its first 16-byte boundary is one there too; places before and
  // after it hold NaN, then -inf. Everything goes by fours of places; index = place + i0.
  const T16* src = static_cast<const T16*>(p.x) + base + r0;
  const int to16 = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / kSize;
  const int pad = (16 / kSize - to16) % (16 / kSize), i0 = r0 - pad, quads = (pad + n + 3) / 4;
  const int nc = min(n, p.cached - pad), head = min(nc, to16), bulk = (nc - head) / (16 / kSize) * (16 / kSize);

  // 1: the range into shared memory: bulk copies of its aligned middle, plain loads at its ends
  if (tid == 0) {
    for (int c = 0; c < kCopies; ++c) mbar_init(&sh.copied[c], 1);
    fence_mbar_init();
    sh.n_list = 0;
    sh.first = 0x7fffffff;
  }
  for (int x = tid; x < kBins; x += kThreads) sh.count[x] = sh.lo[x] = sh.hi[x] = 0;
  pdl_wait();  // what came before is done from here on
  pdl_launch_dependents();
  const int each = ((bulk + kCopies - 1) / kCopies + 15) / 16 * 16;  // of a copy
  if (tid == 0) {
    for (int c = 0; c < kCopies; ++c) {
      const int at = min(bulk, c * each), len = min(bulk, at + each) - at;
      mbar_arrive_expect_tx(&sh.copied[c], len * kSize);
      if (len) bulk_g2s(cache + pad + head + at, src + head + at, len * kSize, &sh.copied[c]);
    }
  }
  if (tid < 16) {
    if (tid < pad) cache[tid] = static_cast<T16>(kNaN<DT>);
    if (tid < head) cache[pad + tid] = src[tid];
    const int tail = head + bulk + tid;  // fewer than 16 bytes of the range, then fewer than four places
    if (tail < nc) cache[pad + tail] = src[tail];
    else if (nc == n && pad + tail < 4 * quads) cache[pad + tail] = static_cast<T16>(kNaN<DT>);
  }
  const float T_in = p.T_a ? p.T_a[b] : p.T, top_p = p.p_a ? p.p_a[b] : p.top_p, min_p = p.m_a ? p.m_a[b] : p.min_p;
  const bool no_T = !(T_in >= 0.f);  // below zero, where weights would pass 1 and leave the sums' range, or NaN
  // from the smallest normal number up, so that 1 / T is finite (only logits that are subnormal numbers themselves could
  // tell: any other below the maximum is further away than 28 T)
  const float T = T_in > 0.f ? fminf(fmaxf(T_in, FLT_MIN), FLT_MAX) : T_in;
  const int k_in = p.k_a ? p.k_a[b] : p.top_k;
  const bool use_k = k_in > 0 && k_in < p.V, use_p = top_p < 1.f;
  __syncthreads();

  bool has_inf = false;  // the row's maximum is +inf
  // four places' logits; NaN ranks as -inf, and beside +inf everything does
  auto get4 = [&](int q, float* f) {
    if (4 * q + 3 < p.cached) {
      if constexpr (kSize == 4) {
        const float4 v = *reinterpret_cast<const float4*>(cache + 4 * q);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(cache + 4 * q);
        f[0] = as_float<DT>(v.x & 0xffffu); f[1] = as_float<DT>(v.x >> 16);
        f[2] = as_float<DT>(v.y & 0xffffu); f[3] = as_float<DT>(v.y >> 16);
      }
    } else {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int x = 4 * q + y - pad;
        f[y] = x >= 0 && x < n ? as_float<DT>(src[x]) : -INFINITY;
        if (f[y] != f[y]) f[y] = -INFINITY;
        if (has_inf) f[y] = f[y] == INFINITY ? 0.f : -INFINITY;
      }
    }
  };
  auto put = [&](int x, float v) {  // a special value
    if (x < p.cached) cache[x] = DT == AGXC_F32 ? static_cast<T16>(__float_as_uint(v))
                                                : static_cast<T16>(v == 0.f ? 0u : kMinusInf<DT>);
  };
  float best = -INFINITY, least = INFINITY;
  bool came = true;
  for (int c = 0, q = tid; c < kCopies; ++c) {  // what each copy brings, as it lands
    came = came && mbar_wait_warp(&sh.copied[c], 0, p.err);
    const int end = c + 1 < kCopies ? min(quads, (pad + head + min(bulk, (c + 1) * each)) / 4) : quads;
    for (; q < end; q += kThreads) {
      float f[4];
      get4(q, f);
      best = fmaxf(fmaxf(best, fmaxf(f[0], f[1])), fmaxf(f[2], f[3]));
      least = fminf(fminf(least, fminf(f[0], f[1])), fminf(f[2], f[3]));
      if (f[0] != f[0] || f[1] != f[1] || f[2] != f[2] || f[3] != f[3]) {
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (f[y] != f[y]) {
            put(4 * q + y, -INFINITY);
            if (4 * q + y >= pad && 4 * q + y < pad + n) least = -INFINITY;
          }
      }
    }
  }
  best = warp_max(best);
  least = -warp_max(-least);
  if (lane == 0) reinterpret_cast<float2*>(sh.warp64)[warp] = make_float2(best, least);
  const bool lost = __syncthreads_or(!came);
  if (warp == 0) {
    const float2 o = lane < kWarps ? reinterpret_cast<float2*>(sh.warp64)[lane] : make_float2(-INFINITY, INFINITY);
    best = warp_max(o.x);
    least = -warp_max(-o.y);
    if (lane == 0) sh.best = make_float2(best, lost ? NAN : least);  // NaN: a copy did not land while it was waited for
  }
  cluster.sync();
  bool whole;
  {
    const float2 o = lane < C ? *cluster.map_shared_rank(&sh.best, lane) : make_float2(-INFINITY, INFINITY);
    whole = __all_sync(0xffffffffu, o.y == o.y);
    best = warp_max(o.x);
    least = -warp_max(-o.y);
  }
  if (!whole) {  // no token from part of a row; the error word says why
    for (int c = 0; c < kCopies; ++c) mbar_wait_warp(&sh.copied[c], 0, p.err);  // for the copies still on their way
    cluster.sync();
    if (rank == 0 && tid == 0) {
      p.token[b] = -1;
      if (p.prob) p.prob[b] = 0.f;
    }
    return;
  }
  if (best == -INFINITY || T == 0.f || no_T) {  // nothing finite or no temperature: none; greedy: the first maximum
    const bool none = best == -INFINITY || no_T || !(1.f >= min_p);
    if (no_T && rank == 0 && tid == 0) atomicOr(p.err, kErrBadOption);
    if (!none) {
      int first = 0x7fffffff;
      for (int q = tid; q < quads && first == 0x7fffffff; q += kThreads) {
        float f[4];
        get4(q, f);
#pragma unroll
        for (int y = 3; y >= 0; --y)
          if (f[y] == best) first = i0 + 4 * q + y;
      }
      if (first != 0x7fffffff) atomicMin(cluster.map_shared_rank(&sh.first, 0), first);
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      p.token[b] = none ? -1 : sh.first;
      if (p.prob) p.prob[b] = none ? 0.f : 1.f;
    }
    return;
  }
  if (best == INFINITY) {
    for (int q = tid; q < quads; q += kThreads) {
      float f[4];
      get4(q, f);
#pragma unroll
      for (int y = 0; y < 4; ++y) put(4 * q + y, f[y] == INFINITY ? 0.f : -INFINITY);
    }
    __syncthreads();
    has_inf = true;
    best = 0.f;
    least = least == INFINITY ? 0.f : -INFINITY;
  }
  Row r;
  r.best = best;
  r.inv_t = __fdiv_rn(1.f, T);
  const float zero_at = 28.f * T;  // 2^40 e^-28 < 1: weights are zero from here down
  const bool zero_last = best - least >= zero_at;
  const float range = zero_last ? zero_at : best - least;
  r.step = range > 1e-30f ? (kBins - 1) / range : 0.f;
  const float ends = zero_last ? kBins - 1.f : kBins;  // places from here on weigh nothing

  int round = 0;
  auto cluster_sum = [&](uint64_t v) {  // over the row, on every thread
    v = block_sum(v, sh.warp64);
    if (tid == 0) sh.sum[round] = v;
    cluster.sync();
    const uint64_t t = warp_sum64(lane < C ? *cluster.map_shared_rank(&sh.sum[round], lane) : 0);
    round ^= 1;
    return t;
  };
  // What the first CTA found, on every thread of the cluster. (It is past every reading of what it found before.)
  auto learn = [&](uint64_t* v) {
    cluster.sync();
    const uint64_t o = lane < 3 ? *cluster.map_shared_rank(&sh.said[lane], 0) : 0;
#pragma unroll
    for (int x = 0; x < 3; ++x) v[x] = __shfl_sync(0xffffffffu, o, x);
  };
  // The lists' length over the cluster, all of them in the first CTA's list where they fit, to that CTA.
  auto collect = [&]() {
    cluster.sync();
    int len = 0;
    if (rank == 0) {  // a warp for each CTA's list, behind this one's own
      if (lane == 0) sh.warp64[warp] = warp < C ? *cluster.map_shared_rank(&sh.n_list, warp) : 0;
      __syncthreads();
      int at = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) at = len;
        len += static_cast<int>(min(sh.warp64[w], static_cast<uint64_t>(kList + 1)));
      }
      if (warp > 0 && warp < C) {
        const uint64_t* other = cluster.map_shared_rank(sh.list, warp);
        const int m = static_cast<int>(sh.warp64[warp]);
        for (int x = lane; x < m && at + x < kList; x += 32) sh.list[at + x] = other[x];
      }
      __syncthreads();
    }
    return len;
  };
  // Lists the elements at places from `lo` to below `hi` whose keys reach `from`, and collects them.
  auto gather = [&](float lo, float hi, uint64_t from) {
    __syncthreads();
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    for (int q = tid; q < quads; q += kThreads) {
      float f[4];
      get4(q, f);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float at = r.place(f[y]);
        if (!(at >= lo && at < hi && f[y] > -INFINITY)) continue;
        const uint64_t key = rank_key(f[y], i0 + 4 * q + y);
        if (key < from) continue;
        const int x = atomicAdd(&sh.n_list, 1);
        if (x < kList) sh.list[x] = key;
      }
    }
    return collect();
  };
  // In the first CTA: the key among the list's first `len`, all at places from `lo` to below `hi`, from which up those
  // that reach `from` sum to `need`, by number or by weight.
  auto cut_list = [&](int len, float lo, float hi, uint64_t from, uint64_t need, bool by_weight) {
    const float scale = kBins / (hi - lo);
    auto sub = [&](uint64_t key) {
      return min(kBins - 1, max(0, __float2int_rz((r.place(key_logit(key)) - lo) * scale)));
    };
    auto value = [&](uint64_t key) -> uint64_t { return by_weight ? weight(r.e(key_logit(key))) : 1; };
    __syncthreads();
    sh.lo[tid] = sh.hi[tid] = sh.lo[tid + kThreads] = sh.hi[tid + kThreads] = 0;
    if (tid == 0) sh.n_few = 0;
    __syncthreads();
    for (int x = tid; x < len; x += kThreads)
      if (sh.list[x] >= from) add64(sh.lo, sh.hi, sub(sh.list[x]), value(sh.list[x]));
    __syncthreads();
    uint64_t a[2], unused;
#pragma unroll
    for (int y = 0; y < 2; ++y) a[y] = static_cast<uint64_t>(sh.hi[2 * tid + y]) << 32 | sh.lo[2 * tid + y];
    uint64_t at = block_before(a[0] + a[1], sh.warp64, unused);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      if (at < need && at + a[y] >= need) {
        sh.bin = 2 * tid + y;
        sh.before = at;
      }
      at += a[y];
    }
    __syncthreads();
    const int bin = sh.bin;
    at = sh.before;
    for (int x = tid; x < len; x += kThreads)
      if (sh.list[x] >= from && sub(sh.list[x]) == bin) {
        const int z = atomicAdd(&sh.n_few, 1);
        if (z < kFew) sh.few[z] = sh.list[x];
      }
    __syncthreads();
    const int m = sh.n_few;
    if (m <= kFew) {  // four threads an element
      const int x = tid >> 2;
      const uint64_t key = x < m ? sh.few[x] : 0;
      uint64_t ahead = 0;
      for (int y = tid & 3; y < m; y += 4)
        if (sh.few[y] > key) ahead += value(sh.few[y]);
      ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
      ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
      at += ahead;
      if (x < m && at < need && at + value(key) >= need) sh.cut = key;
    } else {  // many equal logits: sorted
      sort_list(sh.list, len);
      constexpr int kEach = kList / kThreads;
      uint64_t w[kEach], sum = 0;
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const int x = tid * kEach + y;
        w[y] = x < len && sh.list[x] >= from ? value(sh.list[x]) : 0;
        sum += w[y];
      }
      at = block_before(sum, sh.warp64, unused);
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        if (at < need && at + w[y] >= need) sh.cut = sh.list[tid * kEach + y];
        at += w[y];
      }
    }
    __syncthreads();
    return sh.cut;
  };
  auto tell = [&](int token, uint64_t w, uint64_t total) {
    p.token[b] = token;
    if (p.prob)
      p.prob[b] = total ? static_cast<float>(__ddiv_rn(__ll2double_rn(static_cast<long long>(w)),
                                                       __ll2double_rn(static_cast<long long>(total)))) : 0.f;
  };
  // The first CTA has every candidate in its list, at places below `hi`: cut, draw, done. Up to 128 candidates are ranked
  // by comparing each with all (four threads a candidate); for more, cuts as above and two histograms over the index.
  auto finish_list = [&](int len, float hi, int keep) {
    if (rank == 0 && len <= kThreads / 4) {
      const int x = tid >> 2;
      const uint64_t key = x < len ? sh.list[x] : 0;
      const float e = x < len ? r.e(key_logit(key)) : 0.f;
      if (x < len && (tid & 3) == 0) sh.list[kList / 2 + x] = weight(e);
      __syncthreads();
      int ahead = 0;
      uint64_t before = 0, total = 0;
      for (int y = tid & 3; y < len; y += 4) {
        const uint64_t o = sh.list[y];
        if (o > key) {
          ++ahead;
          before += sh.list[kList / 2 + y];
        }
      }
#pragma unroll
      for (int m = 1; m <= 2; m <<= 1) {
        ahead += __shfl_xor_sync(0xffffffffu, ahead, m);
        before += __shfl_xor_sync(0xffffffffu, before, m);
      }
      uint64_t w = x < len && ahead < keep ? weight(e) : 0;
      if (use_p) {
        total = block_sum((tid & 3) == 0 ? w : 0, sh.warp64);
        if (before >= top_p_bar(top_p, total)) w = 0;
      }
      if (!(e >= min_p)) w = 0;
      total = block_sum((tid & 3) == 0 ? w : 0, sh.warp64);  // and every thread is past the first weights
      if (x < len && (tid & 3) == 0) sh.list[kList / 2 + x] = w;
      __syncthreads();
      if (total == 0) {
        if (tid == 0) tell(-1, 0, 0);
      } else {
        const uint64_t target = target_of(p.u[b], total);
        before = 0;
        for (int y = tid & 3; y < len; y += 4)
          if (key_index(sh.list[y]) < key_index(key)) before += sh.list[kList / 2 + y];
#pragma unroll
        for (int m = 1; m <= 2; m <<= 1) before += __shfl_xor_sync(0xffffffffu, before, m);
        if ((tid & 3) == 0 && target >= before && target < before + w) tell(key_index(key), w, total);
      }
    } else if (rank == 0) {
      uint64_t from = len > keep ? cut_list(len, 0.f, hi, 0, keep, false) : 0;
      if (use_p) {
        uint64_t sum = 0;
        for (int x = tid; x < len; x += kThreads)
          if (sh.list[x] >= from) sum += weight(r.e(key_logit(sh.list[x])));
        sum = block_sum(sum, sh.warp64);
        from = cut_list(len, 0.f, hi, from, top_p_bar(top_p, sum), true);
      }
      constexpr int kEach = kList / kThreads;
      uint64_t w[kEach], sum = 0, total;
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const int x = tid + y * kThreads;
        const float e = x < len && sh.list[x] >= from ? r.e(key_logit(sh.list[x])) : 0.f;
        w[y] = e >= min_p ? weight(e) : 0;
        sum += w[y];
      }
      total = block_sum(sum, sh.warp64);
      if (total == 0) {
        if (tid == 0) tell(-1, 0, 0);
      } else {
        // the weights over the index in up to 1,024 steps, then over the indices of the step that the target falls in
        uint64_t left = target_of(p.u[b], total), w_at = 0;
        const int shift = max(0, 22 - __clz(p.V - 1));  // an index has at most 20 bits
        int at_index = 0;
        for (int level = 0; level < (shift ? 2 : 1); ++level) {
          sh.lo[tid] = sh.hi[tid] = sh.lo[tid + kThreads] = sh.hi[tid + kThreads] = 0;
          __syncthreads();
#pragma unroll
          for (int y = 0; y < kEach; ++y) {
            const int x = tid + y * kThreads, index = w[y] ? key_index(sh.list[x]) : 0;
            if (w[y] && level == 1 && (index >> shift) != at_index) w[y] = 0;
            if (w[y]) add64(sh.lo, sh.hi, level ? index & ((1 << shift) - 1) : index >> shift, w[y]);
          }
          __syncthreads();
          uint64_t a[2], unused;
#pragma unroll
          for (int y = 0; y < 2; ++y) a[y] = static_cast<uint64_t>(sh.hi[2 * tid + y]) << 32 | sh.lo[2 * tid + y];
          uint64_t at = block_before(a[0] + a[1], sh.warp64, unused);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if (left >= at && left < at + a[y]) {
              sh.bin = 2 * tid + y;
              sh.before = at;
              sh.total = a[y];
            }
            at += a[y];
          }
          __syncthreads();
          at_index = level ? at_index << shift | sh.bin : sh.bin;
          left -= sh.before;
          w_at = sh.total;
          __syncthreads();
        }
        if (tid == 0) tell(at_index, w_at, total);
      }
    }
    cluster.sync();
  };
  // the largest key from which up a bin's elements sum to `need`, bit by bit
  auto bisect = [&](auto sum_of, float lo, float hi, uint64_t from, uint64_t need) {
    uint64_t cut = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = cut | 1ull << bit, least_key = at > from ? at : from;
      uint64_t s = 0;
      for (int q = tid; q < quads; q += kThreads) {
        float f[4];
        get4(q, f);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float x = r.place(f[y]);
          if (x >= lo && x < hi && f[y] > -INFINITY && rank_key(f[y], i0 + 4 * q + y) >= least_key) s += sum_of(f[y]);
        }
      }
      if (cluster_sum(s) >= need) cut = at;
    }
    return cut > from ? cut : from;
  };

  uint64_t cut = 0;  // keys from `cut` up are kept
  // each warp has a contiguous part of the CTA's range where weights are added up
  const int part = (quads + kWarps - 1) / kWarps, q0 = min(quads, warp * part), q1 = min(quads, q0 + part);
  bool summed = false;  // the parts' kept weights are there
  if (use_k) {
    for (int q = tid; q < quads; q += kThreads) {
      float f[4];
      get4(q, f);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float x = r.place(f[y]);
        if (x < ends && f[y] > -INFINITY) atomicAdd(&sh.count[bin_of(x)], 1u);
      }
    }
    cluster.sync();
    if (rank == 0) {
      uint32_t c2[2] = {};
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < C) {
          const uint2 o = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.count, c) + 2 * tid);
          c2[0] += o.x;
          c2[1] += o.y;
        }
      uint64_t all;
      uint64_t below = block_before(static_cast<uint64_t>(c2[0]) + c2[1], sh.warp64, all);
      if (all < static_cast<uint64_t>(k_in) && tid == 0) sh.said[0] = kBins, sh.said[1] = 0, sh.said[2] = all;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (below < static_cast<uint64_t>(k_in) && below + c2[y] >= static_cast<uint64_t>(k_in)) {
          sh.said[0] = 2 * tid + y;
          sh.said[1] = below;
          sh.said[2] = below + c2[y];
        }
        below += c2[y];
      }
    }
    uint64_t v[3];
    learn(v);
    const bool some = v[0] < kBins;  // else fewer than k weigh anything
    const float lo = static_cast<float>(v[0]), hi = some ? lo + 1.f : ends;
    if (v[2] <= kList) {
      const int len = gather(0.f, hi, 0);
      finish_list(len, hi, k_in);
      return;
    }
    if (some) {
      const uint64_t left = k_in - v[1];
      if (v[2] - v[1] <= kList) {
        const int len = gather(lo, hi, 0);
        if (rank == 0) sh.said[0] = cut_list(len, lo, hi, 0, left, false);
        learn(v);
        cut = v[0];
      } else {
        cut = bisect([&](float) -> uint64_t { return 1; }, lo, hi, 0, left);
      }
    }
  }
  if (use_p) {
    if (use_k && rank == 0) {  // the finer bins were there
      __syncthreads();
      sh.lo[tid] = sh.hi[tid] = sh.lo[tid + kThreads] = sh.hi[tid + kThreads] = 0;
      __syncthreads();
    }
    for (int q = tid; q < quads; q += kThreads) {
      float f[4];
      get4(q, f);
      uint32_t hi[4], lo[4], old[4];
      int at[4];
      // the four's adds are on their way together
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float x = r.place(f[y]);
        const bool in = x < ends && f[y] > -INFINITY && (!cut || rank_key(f[y], i0 + 4 * q + y) >= cut);
        // the weight's two words: 2^15 + e rounded towards zero has floor(2^8 e) in its low bits, and what that leaves is exact
        const float e = in ? r.e(f[y]) : 0.f, t = __fadd_rz(e, 32768.f);
        hi[y] = __float_as_uint(t) - 0x47000000u;
        lo[y] = __float2uint_rz(__fmul_rn(__fsub_rn(e, __fsub_rn(t, 32768.f)), 1099511627776.f));
        at[y] = bin_of(x);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) old[y] = lo[y] ? atomicAdd(&sh.lo[at[y]], lo[y]) : 0;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t h = hi[y] + (old[y] + lo[y] < old[y] ? 1u : 0u);
        if (h) atomicAdd(&sh.hi[at[y]], h);
      }
    }
    cluster.sync();
    if (rank == 0) {
      uint64_t w2[2] = {};
#pragma unroll 8
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < C) {
          const uint2 l = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.lo, c) + 2 * tid);
          const uint2 h = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.hi, c) + 2 * tid);
          w2[0] += static_cast<uint64_t>(h.x) << 32 | l.x;
          w2[1] += static_cast<uint64_t>(h.y) << 32 | l.y;
        }
      uint64_t total;
      uint64_t below = block_before(w2[0] + w2[1], sh.warp64, total);
      const uint64_t bar = top_p_bar(top_p, total);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (below < bar && below + w2[y] >= bar) {  // exactly one bin
          sh.said[0] = 2 * tid + y;
          sh.said[1] = bar - below;
        }
        below += w2[y];
      }
    }
    uint64_t v[3];
    learn(v);
    const float lo = static_cast<float>(v[0]);
    const uint64_t need = v[1];
    // In one pass: the bin's elements are listed, and the weights of those above it, which are kept, added up.
    __syncthreads();
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    WeightSum above;
    for (int q = q0 + lane; q < q1; q += 32) {
      float f[4];
      get4(q, f);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float at = r.place(f[y]), e = r.e(f[y]);
        above.add(at < lo && e >= min_p ? e : 0.f);
        if (!(at >= lo && at < lo + 1.f && f[y] > -INFINITY)) continue;
        const uint64_t key = rank_key(f[y], i0 + 4 * q + y);
        if (key < cut) continue;
        const int x = atomicAdd(&sh.n_list, 1);
        if (x < kList) sh.list[x] = key;
      }
    }
    const uint64_t sum = warp_sum64(above.get());
    if (lane == 0) sh.warp_kept[warp] = sum;
    int len = collect();
    if (rank == 0) {
      const uint64_t key = len <= kList ? cut_list(len, lo, lo + 1.f, cut, need, true) : 0;
      if (tid == 0) sh.said[0] = key;
    }
    learn(v);
    summed = v[0] != 0;
    if (summed) {  // and the kept of the bin, each to its part
      cut = v[0];
      if (rank > 0) len = sh.n_list;
      for (int x = tid; x < len; x += kThreads) {
        const uint64_t key = sh.list[x];
        const int i = key_index(key);
        const float e = r.e(key_logit(key));
        if (key >= cut && i >= r0 && i < r0 + n && e >= min_p)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.warp_kept[((i - i0) >> 2) / part]),
                    static_cast<unsigned long long>(weight(e)));
      }
    } else {
      cut = bisect([&](float x) { return weight(r.e(x)); }, lo, lo + 1.f, cut, need);
    }
  }

  // 5: the parts' kept weights, and the part, the thread's fours and the element that the target falls on
  const float cut_v = cut ? key_logit(cut) : -INFINITY;  // kept: above the cut's logit, or equal and not after its index
  const int cut_i = cut ? key_index(cut) : 0x7fffffff;
  auto kept_e = [&](float v, int i) {
    const float e = r.e(v);
    return e >= min_p && (v > cut_v || (v == cut_v && i <= cut_i)) ? e : 0.f;
  };
  if (!summed) {
    WeightSum ws;
#pragma unroll 2
    for (int q = q0 + lane; q < q1; q += 32) {
      float f[4];
      get4(q, f);
#pragma unroll
      for (int y = 0; y < 4; ++y) ws.add(kept_e(f[y], i0 + 4 * q + y));
    }
    const uint64_t own = warp_sum64(ws.get());
    if (lane == 0) sh.warp_kept[warp] = own;
  }
  uint64_t sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += sh.warp_kept[w];
    sh.sum[round] = sum;
  }
  cluster.sync();
  sum = lane < C ? *cluster.map_shared_rank(&sh.sum[round], lane) : 0;
  const uint64_t total = warp_sum64(sum);                // of the row
  uint64_t ahead = warp_sum64(lane < rank ? sum : 0);    // of the CTAs before this one
  if (total == 0) {
    if (rank == 0 && tid == 0) tell(-1, 0, 0);
  } else {
    const uint64_t target = target_of(p.u[b], total);
    int found = -1;
    for (int w = 0; w < kWarps; ++w) {
      const uint64_t t = sh.warp_kept[w];
      if (found < 0 && target >= ahead && target < ahead + t) found = w;
      if (found < 0) ahead += t;
    }
    if (found >= 0) {  // this CTA, the part of warp `found`: every thread a few fours of it in order
      const int y0 = min(quads, found * part), y1 = min(quads, y0 + part), each = (part + kThreads - 1) / kThreads;
      const int z0 = min(y1, y0 + tid * each), z1 = min(y1, z0 + each);
      WeightSum mine;
      for (int q = z0; q < z1; ++q) {
        float f[4];
        get4(q, f);
#pragma unroll
        for (int y = 0; y < 4; ++y) mine.add(kept_e(f[y], i0 + 4 * q + y));
      }
      uint64_t unused;
      sum = mine.get();
      uint64_t at = ahead + block_before(sum, sh.warp64, unused);
      if (target >= at && target < at + sum) {
        for (int q = z0; q < z1; ++q) {
          float f[4];
          get4(q, f);
          for (int y = 0; y < 4; ++y) {
            const uint64_t w = weight(kept_e(f[y], i0 + 4 * q + y));
            if (target >= at && target < at + w) tell(i0 + 4 * q + y, w, total);
            at += w;
          }
        }
      }
    }
  }
  cluster.sync();  // the neighbours' shared memory stays until all have read it
}

// CTAs a row: doubled while the rows' CTAs are no more than the SMs, and so many that a CTA's range takes at most 96 KB. That
// limit was measured at one size, 64 rows of 92,544: 24.2 us with four CTAs a row, of 122,688 bytes each and so one an SM, 26.6
// with eight, two an SM; either way two waves.
template <int DT>
int sample_launch(const agxc_ctx* ctx, SampleParams p, cudaStream_t s) {
  static std::atomic<int> most[64] = {};  // the largest cluster that the device places
  int dev = 0;
  AGXC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return fail(AGXC_EINVAL, "sample: device index below 64");
  if (!most[dev]) {
    AGXC_CUDA(cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, ctx->max_smem_optin));
    AGXC_CUDA(cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t q = {};
    cudaLaunchAttribute qa[1];
    qa[0].id = cudaLaunchAttributeClusterDimension;
    qa[0].val.clusterDim.x = kMaxCluster;
    qa[0].val.clusterDim.y = qa[0].val.clusterDim.z = 1;
    q.gridDim = dim3(kMaxCluster);
    q.blockDim = dim3(kThreads);
    q.dynamicSmemBytes = ctx->max_smem_optin;
    q.attrs = qa;
    q.numAttrs = 1;
    int fit = 0;
    if (cudaOccupancyMaxActiveClusters(&fit, sample_kernel<DT>, &q) != cudaSuccess) {
      cudaGetLastError();
      fit = 0;
    }
    most[dev] = fit > 0 ? kMaxCluster : 8;
  }
  int c = 1;
  while (c < most[dev] && p.V > c * 2048 &&
         (static_cast<int64_t>(p.B) * c <= ctx->num_sms || p.V / c * static_cast<int64_t>(sizeof(typename Raw<DT>::Type)) > 96000))
    c *= 2;
  p.per = (p.V + c - 1) / c;
  const int size = static_cast<int>(sizeof(typename Raw<DT>::Type)), fixed = static_cast<int>(align16(sizeof(Shared)));
  const int room = (ctx->max_smem_optin - fixed) / size / 16 * 16, want = (p.per + 31) / 16 * 16;  // its ends' padding too
  p.cached = want < room ? want : room;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.B) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = fixed + size * static_cast<size_t>(p.cached);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  AGXC_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<DT>, p));
  return 0;
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" AGXC_API int agxc_sample_dev(agxc_ctx* ctx, const agxc_sample_args* a, void* stream) {
  if (!ctx || !a) return fail(AGXC_EINVAL, "sample: null argument");
  if (a->dtype < AGXC_F32 || a->dtype > AGXC_BF16) return fail(AGXC_EINVAL, "sample: logits fp32, fp16 or bf16");
  if (a->batch < 0 || a->batch > (1 << 26)) return fail(AGXC_EINVAL, "sample: batch 0 to 67,108,864");
  if (a->vocab < 1 || a->vocab > (1 << 20)) return fail(AGXC_EINVAL, "sample: vocab 1 to 1,048,576");
  if (a->logits_ld < a->vocab) return fail(AGXC_EINVAL, "sample: logits_ld < vocab");
  if (!a->temperature_dev && !(a->temperature >= 0.f)) return fail(AGXC_EINVAL, "sample: temperature >= 0");
  if (a->batch == 0) return 0;
  if (!a->logits_dev || !a->u_dev || !a->token_dev) return fail(AGXC_EINVAL, "sample: null buffer");
  const OnDevice on(ctx->device);
  if (on.rc()) return on.rc();
  SampleParams p;
  p.x = a->logits_dev; p.ld = a->logits_ld; p.B = a->batch; p.V = a->vocab; p.u = a->u_dev;
  p.T = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.T_a = a->temperature_dev; p.k_a = a->top_k_dev; p.p_a = a->top_p_dev; p.m_a = a->min_p_dev;
  p.token = a->token_dev; p.prob = a->prob_dev; p.err = ctx->err_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  if (a->dtype == AGXC_F32) return sample_launch<AGXC_F32>(ctx, p, s);
  if (a->dtype == AGXC_F16) return sample_launch<AGXC_F16>(ctx, p, s);
  return sample_launch<AGXC_BF16>(ctx, p, s);
}
