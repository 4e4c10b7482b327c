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
//   2  top-k: counts in 1,024 bins, equal steps of the logit down to weight zero or the least logit; the bin that holds
//      rank k. Up to 2,048 elements in that bin and above go to one CTA as a list; it sorts them and finishes the row
//   3  top-p: the same with the bins' exact weights (64 bits as two 32-bit shared-memory adds, the second with the
//      first's carry)
//   4  more than a list: only the bin of the cut is listed and sorted, to find the key it falls on; a bin that is more
//      than a list (thousands of equal logits) is cut bit by bit instead
//   5  the kept weights' total and the token, in index order: the warp, then the element, that the target falls on
#include <cooperative_groups.h>

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
  int B, V, per, cached;  // per = elements of a CTA, cached = how many of them shared memory holds
  const float* u;
  float T, top_p, min_p;
  int top_k;
  const float* T_a;
  const int32_t* k_a;
  const float* p_a;
  const float* m_a;
  int32_t* token;
  float* prob;
};

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 1024, kList = 2048, kMaxCluster = 16;

template <int DT>
__device__ __forceinline__ float as_logit(uint32_t bits) {  // NaN ranks as -inf, the two zeros alike
  float v;
  if (DT == AGXC_F32) v = __uint_as_float(bits);
  else if (DT == AGXC_F16) v = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  else v = __uint_as_float(bits << 16);
  return v != v ? -INFINITY : v + 0.f;
}

template <int DT>
__device__ __forceinline__ float logit(const void* x, int64_t i) {
  return DT == AGXC_F32 ? as_logit<DT>(static_cast<const uint32_t*>(x)[i])
                        : as_logit<DT>(static_cast<const unsigned short*>(x)[i]);
}

// larger logits first, then lower indices: the larger key ranks first
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  const uint32_t b = __float_as_uint(v);
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

struct Row {
  float best, inv_t, step;  // step = bins a unit of logit
  __device__ float down(float v) const { return v == best ? 0.f : __fsub_rn(v, best); }
  __device__ float e(float v) const { return v == -INFINITY ? 0.f : expf(__fmul_rn(down(v), inv_t)); }
  // -inf weighs nothing and is in none
  __device__ int bin(float v) const {
    return v == -INFINITY ? kBins : min(kBins - 1, __float2int_rz(-down(v) * step));
  }
};

struct Best {
  float v, least;
  int i;
};

struct Shared {
  Best best;
  uint64_t sum[2];
  int n_list, bin;
  uint64_t before, total, cut;
  uint64_t warp64[kWarps];
  uint64_t warp_kept[kWarps];
  Best warp_best[kWarps];
  alignas(16) uint32_t count[kBins];
  alignas(16) uint32_t lo[kBins];
  alignas(16) uint32_t hi[kBins];
  uint64_t list[kList];
};

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
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& sh = *reinterpret_cast<Shared*>(dyn);
  float* cache = reinterpret_cast<float*>(dyn + align16(sizeof(Shared)));
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x / C;
  const int64_t base = static_cast<int64_t>(b) * p.ld;
  const int i0 = min(p.V, rank * p.per), n = min(p.V, i0 + p.per) - i0, nc = min(n, p.cached);
  const float T = p.T_a ? p.T_a[b] : p.T, top_p = p.p_a ? p.p_a[b] : p.top_p, min_p = p.m_a ? p.m_a[b] : p.min_p;
  const int k_in = p.k_a ? p.k_a[b] : p.top_k;
  const bool use_k = k_in > 0 && k_in < p.V, use_p = top_p < 1.f;

  // 1: the range into shared memory, 16 bytes at a time from its first 16-byte boundary
  constexpr int kSize = DT == AGXC_F32 ? 4 : 2, kVec = 16 / kSize;
  const uint8_t* src = static_cast<const uint8_t*>(p.x) + (base + i0) * kSize;
  const int head = min(nc, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / kSize);
  cache += (4 - head % 4) % 4;
  Best mine = {-INFINITY, INFINITY, 0x7fffffff};
  auto see = [&](float v, int i) {
    if (v > mine.v || mine.i == 0x7fffffff) mine.v = v, mine.i = i;
    if (v > -INFINITY) mine.least = fminf(mine.least, v);
  };
  if (tid < head) {
    const float v = logit<DT>(p.x, base + i0 + tid);
    cache[tid] = v;
    see(v, i0 + tid);
  }
  const int vecs = (nc - head) / kVec;
#pragma unroll 4
  for (int x = tid; x < vecs; x += kThreads) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(src + head * kSize) + x);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float f[kVec];
#pragma unroll
    for (int y = 0; y < kVec; ++y)
      f[y] = kSize == 4 ? as_logit<DT>(u[y & 3]) : as_logit<DT>(u[y / 2] >> (16 * (y & 1)) & 0xffffu);
    const int at = head + x * kVec;
#pragma unroll
    for (int y = 0; y < kVec; y += 4) *reinterpret_cast<float4*>(cache + at + y) = make_float4(f[y], f[y + 1], f[y + 2], f[y + 3]);
#pragma unroll
    for (int y = 0; y < kVec; ++y) see(f[y], i0 + at + y);
  }
  for (int x = head + vecs * kVec + tid; x < n; x += kThreads) {
    const float v = logit<DT>(p.x, base + i0 + x);
    if (x < nc) cache[x] = v;
    see(v, i0 + x);
  }
  auto get = [&](int x) { return x < nc ? cache[x] : logit<DT>(p.x, base + i0 + x); };
  auto join = [](Best& a, float v, float least, int i) {
    if (v > a.v || (v == a.v && i < a.i)) a.v = v, a.i = i;
    a.least = fminf(a.least, least);
  };
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1)
    join(mine, __shfl_xor_sync(0xffffffffu, mine.v, m), __shfl_xor_sync(0xffffffffu, mine.least, m),
         __shfl_xor_sync(0xffffffffu, mine.i, m));
  if (lane == 0) sh.warp_best[warp] = mine;
  for (int x = tid; x < kBins; x += kThreads) sh.count[x] = sh.lo[x] = sh.hi[x] = 0;
  if (tid == 0) sh.n_list = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) join(mine, sh.warp_best[w].v, sh.warp_best[w].least, sh.warp_best[w].i);
    sh.best = mine;
  }
  cluster.sync();
  mine = {-INFINITY, INFINITY, 0x7fffffff};
  for (int c = 0; c < C; ++c) {
    const Best o = *cluster.map_shared_rank(&sh.best, c);
    join(mine, o.v, o.least, o.i);
  }
  if (mine.v == -INFINITY || T == 0.f) {
    if (rank == 0 && tid == 0) {
      const bool none = mine.v == -INFINITY || !(1.f >= min_p);
      p.token[b] = none ? -1 : mine.i;
      if (p.prob) p.prob[b] = none ? 0.f : 1.f;
    }
    cluster.sync();
    return;
  }
  Row r;
  r.best = mine.v;
  r.inv_t = __fdiv_rn(1.f, T);
  const float zero_at = 28.f * T;  // 2^40 e^-28 < 1: weights are zero from here down
  const bool zero_last = mine.v - mine.least >= zero_at;
  const float range = zero_last ? zero_at : mine.v - mine.least;
  r.step = range > 0.f ? (kBins - 1) / range : 0.f;
  const int ends = zero_last ? kBins - 1 : kBins;  // bins from here on weigh nothing

  int round = 0;
  auto cluster_sum = [&](uint64_t v) {  // over the row, on every thread
    v = block_sum(v, sh.warp64);
    if (tid == 0) sh.sum[round] = v;
    cluster.sync();
    uint64_t t = 0;
    for (int c = 0; c < C; ++c) t += *cluster.map_shared_rank(&sh.sum[round], c);
    round ^= 1;
    return t;
  };
  // elements that pass, as keys, into the first CTA's list (their number is known to fit)
  auto gather = [&](auto pass) {
    uint64_t* list = cluster.map_shared_rank(sh.list, 0);
    int* count = cluster.map_shared_rank(&sh.n_list, 0);
    for (int x0 = warp * 32; x0 < n; x0 += kThreads) {
      const int x = x0 + lane;
      const float v = x < n ? get(x) : -INFINITY;
      const bool in = x < n && pass(v, i0 + x);
      const unsigned some = __ballot_sync(0xffffffffu, in);
      if (!some) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(count, __popc(some));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(some & ((1u << lane) - 1));
      if (in && at < kList) list[at] = rank_key(v, i0 + x);
    }
    cluster.sync();
  };
  // the first CTA has every candidate in its list: cut, draw, done
  auto finish_list = [&](int len, int keep) {
    if (rank == 0) {
      sort_list(sh.list, len);
      len = min(len, keep);
      constexpr int kEach = kList / kThreads;
      uint64_t w[kEach], sum = 0, total, below;
      float e[kEach];
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const int x = tid * kEach + y;
        e[y] = x < len ? r.e(key_logit(sh.list[x])) : 0.f;
        w[y] = x < len ? weight(e[y]) : 0;
        sum += w[y];
      }
      below = block_before(sum, sh.warp64, total);
      const uint64_t bar = use_p ? top_p_bar(top_p, total) : ~0ull;
      sum = 0;
#pragma unroll
      for (int y = 0; y < kEach; ++y) {
        const uint64_t before = below;
        below += w[y];
        if (before >= bar || !(e[y] >= min_p)) w[y] = 0;
        sum += w[y];
      }
      total = block_sum(sum, sh.warp64);
      if (total == 0) {
        if (tid == 0) {
          p.token[b] = -1;
          if (p.prob) p.prob[b] = 0.f;
        }
      } else {
        const uint64_t target = target_of(p.u[b], total);
        // the largest index with at most `target` of the weight before it
        int at = 0;
        for (int bit = 31 - __clz(p.V); bit >= 0; --bit) {
          const int to = at | 1 << bit;
          sum = 0;
#pragma unroll
          for (int y = 0; y < kEach; ++y)
            if (w[y] && key_index(sh.list[tid * kEach + y]) < to) sum += w[y];
          if (block_sum(sum, sh.warp64) <= target) at = to;
        }
#pragma unroll
        for (int y = 0; y < kEach; ++y)
          if (w[y] && key_index(sh.list[tid * kEach + y]) == at) {
            p.token[b] = at;
            if (p.prob)
              p.prob[b] = static_cast<float>(__ddiv_rn(__ll2double_rn(static_cast<long long>(w[y])),
                                                       __ll2double_rn(static_cast<long long>(total))));
          }
      }
    }
    cluster.sync();
  };
  // the key at which `test` of the sum over keys from it up turns true, among the keys of one bin: bit by bit
  auto bisect = [&](auto sum_from, uint64_t need) {
    uint64_t cut = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = cut | 1ull << bit;
      uint64_t s = 0;
      for (int x = tid; x < n; x += kThreads) s += sum_from(get(x), i0 + x, at);
      if (cluster_sum(s) >= need) cut = at;
    }
    return cut;
  };

  uint64_t cut = 0;  // keys from `cut` up are kept
  if (use_k) {
    for (int x = tid; x < n; x += kThreads) {
      const int q = r.bin(get(x));
      if (q < ends) atomicAdd(&sh.count[q], 1u);
    }
    cluster.sync();
    uint32_t c2[2] = {};
    for (int c = 0; c < C; ++c) {
      const uint2 o = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.count, c) + 2 * tid);
      c2[0] += o.x; c2[1] += o.y;
    }
    uint64_t all;
    uint64_t below = block_before(static_cast<uint64_t>(c2[0]) + c2[1], sh.warp64, all);
    if (all <= static_cast<uint64_t>(k_in) && all <= kList && !use_p) {
      // every element that weighs anything is kept: nothing to cut
    } else {
      if (tid == 0) sh.bin = -1;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (below < static_cast<uint64_t>(k_in) && below + c2[y] >= static_cast<uint64_t>(k_in)) {
          sh.bin = 2 * tid + y;
          sh.before = below;
          sh.total = below + c2[y];
        }
        below += c2[y];
      }
      __syncthreads();
      const int bin = sh.bin;
      const uint64_t before = sh.before, through = bin < 0 ? all : sh.total;
      if (through <= kList) {
        gather([&](float v, int) { const int q = r.bin(v); return q < ends && (bin < 0 || q <= bin); });
        finish_list(static_cast<int>(through), k_in);
        return;
      }
      if (bin >= 0) {
        const int left = static_cast<int>(k_in - before);
        if (through - before <= kList) {
          gather([&](float v, int) { return r.bin(v) == bin; });
          if (rank == 0) {
            sort_list(sh.list, static_cast<int>(through - before));
            if (tid == 0) sh.cut = sh.list[left - 1], sh.n_list = 0;
          }
          cluster.sync();
          cut = *cluster.map_shared_rank(&sh.cut, 0);
        } else {
          cut = bisect([&](float v, int i, uint64_t at) -> uint64_t { return r.bin(v) == bin && rank_key(v, i) >= at; },
                       left);
        }
      }
    }
  }
  if (use_p) {
    if (use_k) {  // the counts were for top-k
      cluster.sync();
      for (int x = tid; x < kBins; x += kThreads) sh.count[x] = 0;
      __syncthreads();
    }
    for (int x = tid; x < n; x += kThreads) {
      const float v = get(x);
      const int q = r.bin(v);
      if (q >= ends || (cut && rank_key(v, i0 + x) < cut)) continue;
      const uint64_t w = weight(r.e(v));
      const uint32_t l = static_cast<uint32_t>(w), old = atomicAdd(&sh.lo[q], l);
      const uint32_t h = static_cast<uint32_t>(w >> 32) + (old + l < old ? 1u : 0u);
      if (h) atomicAdd(&sh.hi[q], h);
      atomicAdd(&sh.count[q], 1u);
    }
    cluster.sync();
    uint64_t w2[2] = {}, n2[2] = {};
    for (int c = 0; c < C; ++c) {
      const uint2 l = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.lo, c) + 2 * tid);
      const uint2 h = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.hi, c) + 2 * tid);
      const uint2 o = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(sh.count, c) + 2 * tid);
      w2[0] += static_cast<uint64_t>(h.x) << 32 | l.x;
      w2[1] += static_cast<uint64_t>(h.y) << 32 | l.y;
      n2[0] += o.x;
      n2[1] += o.y;
    }
    uint64_t total;
    uint64_t below = block_before(w2[0] + w2[1], sh.warp64, total);
    const uint64_t bar = top_p_bar(top_p, total);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      if (below < bar && below + w2[y] >= bar) {  // exactly one bin
        sh.bin = 2 * tid + y;
        sh.before = below;
        sh.total = n2[y];
      }
      below += w2[y];
    }
    __syncthreads();
    const int bin = sh.bin;
    const uint64_t before = sh.before, in_bin = sh.total;
    if (in_bin <= kList) {
      const uint64_t from = cut;
      gather([&](float v, int i) { return r.bin(v) == bin && rank_key(v, i) >= from; });
      if (rank == 0) {
        sort_list(sh.list, static_cast<int>(in_bin));
        constexpr int kEach = kList / kThreads;
        uint64_t w[kEach], sum = 0, unused;
#pragma unroll
        for (int y = 0; y < kEach; ++y) {
          const int x = tid * kEach + y;
          w[y] = x < static_cast<int>(in_bin) ? weight(r.e(key_logit(sh.list[x]))) : 0;
          sum += w[y];
        }
        uint64_t at = before + block_before(sum, sh.warp64, unused);
#pragma unroll
        for (int y = 0; y < kEach; ++y) {
          if (at < bar && at + w[y] >= bar) sh.cut = sh.list[tid * kEach + y];
          at += w[y];
        }
      }
      cluster.sync();
      cut = *cluster.map_shared_rank(&sh.cut, 0);
    } else {
      const uint64_t from = cut;
      cut = bisect(
          [&](float v, int i, uint64_t at) -> uint64_t {
            return r.bin(v) == bin && rank_key(v, i) >= (at > from ? at : from) ? weight(r.e(v)) : 0;
          },
          bar - before);
      cut = cut > from ? cut : from;
    }
  }

  // 5: each warp a contiguous part of the CTA's range
  auto kept = [&](int x) -> uint64_t {
    const float v = get(x), e = r.e(v);
    return e >= min_p && (!cut || rank_key(v, i0 + x) >= cut) ? weight(e) : 0;
  };
  const int part = (n + kWarps - 1) / kWarps, x0 = min(n, warp * part), x1 = min(n, x0 + part);
  uint64_t sum = 0;
  for (int x = x0 + lane; x < x1; x += 32) sum += kept(x);
  sum = warp_sum64(sum);
  if (lane == 0) sh.warp_kept[warp] = sum;
  cluster.sync();
  uint64_t total = 0, ahead = 0;  // of the row, and of the CTAs before this one
  for (int c = 0; c < C; ++c) {
    const uint64_t* o = cluster.map_shared_rank(sh.warp_kept, c);
    uint64_t t = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += o[w];
    if (c < rank) ahead += t;
    total += t;
  }
  if (total == 0) {
    if (rank == 0 && tid == 0) {
      p.token[b] = -1;
      if (p.prob) p.prob[b] = 0.f;
    }
  } else {
    const uint64_t target = target_of(p.u[b], total);
    int found = -1;
    for (int w = 0; w < kWarps; ++w) {
      const uint64_t t = sh.warp_kept[w];
      if (found < 0 && target >= ahead && target < ahead + t) found = w;
      if (found < 0) ahead += t;
    }
    if (found >= 0) {  // this CTA, the part of warp `found`: every thread a few elements of it in order
      const int y0 = min(n, found * part), y1 = min(n, y0 + part), each = (part + kThreads - 1) / kThreads;
      const int z0 = min(y1, y0 + tid * each), z1 = min(y1, z0 + each);
      sum = 0;
      for (int x = z0; x < z1; ++x) sum += kept(x);
      uint64_t unused;
      uint64_t at = ahead + block_before(sum, sh.warp64, unused);
      for (int x = z0; x < z1; ++x) {
        const uint64_t w = kept(x);
        if (target >= at && target < at + w) {
          p.token[b] = i0 + x;
          if (p.prob)
            p.prob[b] = static_cast<float>(__ddiv_rn(__ll2double_rn(static_cast<long long>(w)),
                                                     __ll2double_rn(static_cast<long long>(total))));
        }
        at += w;
      }
    }
  }
  cluster.sync();  // the neighbours' shared memory stays until all have read it
}

// CTAs a row: eight where the rows alone fill the GPU, up to sixteen where they do not.
template <int DT>
int sample_launch(const agxc_ctx* ctx, SampleParams p, cudaStream_t s) {
  static int most[64] = {};  // the largest cluster that the device places
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
  while (c < most[dev] && p.V > c * 2048 && (p.B * c < ctx->num_sms || p.V / c > 24000)) c *= 2;
  p.per = (p.V + c - 1) / c;
  const int fixed = static_cast<int>(align16(sizeof(Shared))) + 16;
  const int room = (ctx->max_smem_optin - fixed) / 4;
  p.cached = p.per < room ? p.per : room;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.B) * c);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = fixed + 4 * static_cast<size_t>(p.cached);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AGXC_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel<DT>, p));
  return 0;
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" AGXC_API int agxc_sample_dev(agxc_ctx* ctx, const agxc_sample_args* a, void* stream) {
  if (!ctx || !a) return fail(AGXC_EINVAL, "sample: null argument");
  if (a->dtype < AGXC_F32 || a->dtype > AGXC_BF16) return fail(AGXC_EINVAL, "sample: logits fp32, fp16 or bf16");
  if (a->batch < 0 || a->vocab < 1) return fail(AGXC_EINVAL, "sample: batch >= 0 and a vocabulary of at least one");
  if (a->logits_ld < a->vocab) return fail(AGXC_EINVAL, "sample: logits_ld < vocab");
  if (!a->temperature_dev && !(a->temperature >= 0.f)) return fail(AGXC_EINVAL, "sample: temperature >= 0");
  if (a->batch == 0) return 0;
  if (!a->logits_dev || !a->u_dev || !a->token_dev) return fail(AGXC_EINVAL, "sample: null buffer");
  SampleParams p;
  p.x = a->logits_dev; p.ld = a->logits_ld; p.B = a->batch; p.V = a->vocab; p.u = a->u_dev;
  p.T = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.T_a = a->temperature_dev; p.k_a = a->top_k_dev; p.p_a = a->top_p_dev; p.m_a = a->min_p_dev;
  p.token = a->token_dev; p.prob = a->prob_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  if (a->dtype == AGXC_F32) return sample_launch<AGXC_F32>(ctx, p, s);
  if (a->dtype == AGXC_F16) return sample_launch<AGXC_F16>(ctx, p, s);
  return sample_launch<AGXC_BF16>(ctx, p, s);
}
