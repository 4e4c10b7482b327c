// kv4_attention.cu — attention over the paged 4-bit KV cache (kv4.cuh): query row i of a sequence of length L with n
// rows sees keys 0 .. L - n + i, out = sum_t p_t v_t / sum_t p_t with p_t = 2^(q . k_t - m), one pass over the keys.
//
// Mathematics. With k = s code + b per group of 64 dims, q . k = sum_g s_g (q_g . code_g) + b_g sum(q_g), and
// sum_t p_t v_t = sum_t (p_t s_t) code_t + sum_t p_t b_t: the codes meet the tensor cores as they are (a 4-bit field
// masked out of a word IS an fp16 subnormal, code 2^-24 or code 2^-20, so one AND prepares two operands), and scales
// and biases are applied to the 16 x 8 scores, not to the 16 x head_dim values. A warp takes 32 keys at a time, as two
// tiles of 16:
//   scores   D[key][column] = codes (A, 16 keys x 16 dims) x q (B, 16 dims x 8 columns), a column = one (row, head)
//   values   O[dim][column] += (codes - 8) (A, 16 dims x 16 keys) x P (B, 16 keys x 8 columns); the score fragments
//            become P operands by one 8 x 8 transpose each (movmatrix)
// q is scaled by a power of two a column and the fields' 2^-24 is undone in fp32 (exact). P = p s / sref is rounded to
// fp16 (11 bits; the only rounding of the pass): sref is the running power of two above the group's scales and the
// reference m sits 8 below the running maximum, so P stays in fp16's normal range down to 2^-22 of the largest weight.
// The values' codes are taken about 8 (one subtraction of fp16 subnormals for two) and their bias as b + 8 s, so that P's
// rounding counts by a value's distance from its group's middle and the sums over thousands of keys stay small beside what
// the tensor core's accumulation drops (codes of one sign: 3.6e-4 off at 8,192 keys, 2-norm; about 8: 2.8e-4, of which the
// output's own fp16 rounding is 2.1e-4). m and sref move only when a score passes m + 12 or a scale passes 8 sref (one vote
// for 32 keys), which rescales the accumulators.
//
// Split. The 128-key blocks of every (sequence, KV head, block of columns) lie end to end; each CTA takes an equal
// share of that line, whatever the lengths are. A fifth warp copies the blocks, a bulk copy a tile (which is
// contiguous), into three stages of shared memory, and each of four warps computes on 32 keys of a block. A piece that
// is not a whole item leaves its maximum, sum and values in the workspace, and a second kernel joins the pieces in a
// fixed order (no atomics: equal calls give equal bits). A sum of weights is zero where no key was seen; one that is NaN,
// from a query or a seen key that is not finite, is carried along like any other. Few items are split over a cluster each
// instead, whose CTAs join their pieces in shared memory: one launch, and no second kernel to wait for.
//
// 64 sequences of 8,192 tokens, 32 heads over 8 KV heads of 128 dims (605 MB): 135 us, 4.48 TB/s (the copy rate would take
// 92.5). The SM's issue slots bind it, 59 of 100 taken at 12 warps an SM, with DRAM at 53: two ANDs, a subtraction and their
// share of an MMA for each pair of codes of K and V, about 300 instructions a 16-key tile and warp where 475 took 197 us.
// 128 ragged sequences of up to 1,792 tokens of 2 KV heads of 64 (18.6 MB): 18.6 us; one of 1,792 of 8: 6.7, both a launch, a
// chain of three dependent loads and a join. 16 rows of 8 sequences: 22 us, the 32 columns a KV head as two blocks, which
// dequantise each key twice. Not kept: compute warps that take the copy's turn (156 us), seven of them in two CTAs an
// SM (136), codes or-ed into 1,024 (148).
#include <cooperative_groups.h>

#include <atomic>

#include "kv4_attention.cuh"

namespace agxc {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;   // of the warps that compute; one more warp copies
constexpr int kBlock = 32 * kWarps;     // keys a block
constexpr float kNone = -1e30f;         // the maximum that stands for no key

__device__ __forceinline__ int blocks_of(int len) { return (len + kBlock - 1) / kBlock; }

// A CTA's place on the line of blocks: sequence b, item = kv_head * CB + column block, block t of its T, and how many
// blocks are left of the CTA's share.
struct Place {
  int b, item, t, T, len;
  long long rem;
  __device__ int end() const { return rem < T - t ? t + static_cast<int>(rem) : T; }
  __device__ void next(const Kv4AttnParams& p) {
    rem -= end() - t;
    t = 0;
    if (++item == p.c.kvh * p.CB) {
      item = 0;
      do {
        if (++b >= p.B) {
          rem = 0;
          return;
        }
        len = kv4_seq_len(p, b);
        T = blocks_of(len);
      } while (T == 0);
    }
  }
};

// Blocks a CTA: the line's length over the CTAs. Every warp computes it for itself.
__device__ __forceinline__ long long line_quota(const Kv4AttnParams& p, int lane) {
  long long sum = 0;
  for (int b = lane; b < p.B; b += 32) sum += blocks_of(kv4_seq_len(p, b));
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  sum *= p.c.kvh * p.CB;
  return quotient(sum + p.ctas - 1, p.ctas);
}

// The sequence that holds position `at` of the line, and where its items start.
__device__ __forceinline__ bool line_find(const Kv4AttnParams& p, int lane, long long at, int& seq, int& len,
                                          long long& start) {
  long long acc = 0;
  const int items = p.c.kvh * p.CB;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    const int l = b < p.B ? kv4_seq_len(p, b) : 0;
    const long long mine = static_cast<long long>(blocks_of(l)) * items;
    long long up = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, up, m);
      if (lane >= m) up += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, acc + up > at);
    if (past) {
      const int w = __ffs(past) - 1;
      seq = b0 + w;
      len = __shfl_sync(0xffffffffu, l, w);
      start = acc + __shfl_sync(0xffffffffu, up - mine, w);
      return true;
    }
    acc += __shfl_sync(0xffffffffu, up, 31);
  }
  return false;
}

// a barrier of the warps that compute
__device__ __forceinline__ void warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// code - 8 of the even (hi = 0) or 16 (code - 8) of the odd nibble in the low byte of each half of x, times 2^-24 (an
// exact difference of fp16 subnormals)
__device__ __forceinline__ uint32_t about8(uint32_t x, int hi) {
  const __half2 d = __hsub2(as_half2(x & (hi ? 0x00f000f0u : 0x000f000fu)), as_half2(hi ? 0x00800080u : 0x00080008u));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// D = A B + D and D = A B, m16n8k16 (not volatile: the compiler may order them among each other's operands)
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_zero(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(0.f));
}

// Shared memory of a CTA: stages of a block's tiles, the warps' results [warp][column][hd + 4], {max, sum} of each, the
// stages' barriers (filled, emptied) and which of their tiles were copied.
template <int HD, int NT>
struct Smem {
  static constexpr int kStages = 3;
  static constexpr int kStage = kBlock / 16 * Kv4Tile<HD>::kBytes;
  static constexpr int kCols = 8 * NT;
  static constexpr int kRow = HD + 4;
  static constexpr int kO = kStages * kStage;
  static constexpr int kMl = kO + kWarps * kCols * kRow * 4;
  static constexpr int kOwn = kMl + kWarps * kCols * 8;   // {max, sum} of the CTA, for its cluster
  static constexpr int kBar = kOwn + kCols * 8;
  static constexpr int kCame = kBar + 2 * kStages * 8;
  static constexpr int kBytes = kCame + kStages * 4;
};

// The results of `lanes` lanes (a power of two up to 16, lanes side by side) of one column's eight dims, {m, sum} and v
// each, as one: out on each of them.
__device__ __forceinline__ void join_lanes(int lanes, float m, float sum, float* v) {
  float mx = m;
#pragma unroll
  for (int x = 8; x >= 1; x >>= 1)
    if (x < lanes) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  const float f = ex2(m - mx);
  sum *= f;
#pragma unroll
  for (int x = 8; x >= 1; x >>= 1)
    if (x < lanes) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  const float inv = sum != 0.f ? f / sum : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= inv;
#pragma unroll
  for (int x = 8; x >= 1; x >>= 1)
    if (x < lanes) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], x);
    }
}

template <int HD, int NT, typename T, bool CL>
__global__ void __launch_bounds__(kThreads + 32, NT == 1 ? 3 : 2)
    kv4_attn_kernel(const __grid_constant__ Kv4AttnParams p) {
  using Tile = Kv4Tile<HD>;
  using Sm = Smem<HD, NT>;
  constexpr int GR = HD / 64;               // groups of 64 dims
  constexpr int S = Sm::kStages, NC = Sm::kCols;
  extern __shared__ __align__(128) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + Sm::kBar);
  uint64_t* empty = full + S;
  volatile unsigned* came = reinterpret_cast<unsigned*>(sm + Sm::kCame);
  float* so = reinterpret_cast<float*>(sm + Sm::kO);
  float2* sml = reinterpret_cast<float2*>(sm + Sm::kMl);
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  Place at;
  if constexpr (CL) {
    const int unit = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    at.b = unit / (p.c.kvh * p.CB);
    at.item = unit % (p.c.kvh * p.CB);
    at.len = kv4_seq_len(p, at.b);
    at.T = blocks_of(at.len);
    const int per = (at.T + p.cluster - 1) / p.cluster;
    at.t = rank * per;
    at.rem = min(per, max(0, at.T - at.t));
    if (threadIdx.x < NC) reinterpret_cast<float2*>(sm + Sm::kOwn)[threadIdx.x] = make_float2(kNone, 0.f);
    __syncthreads();
  } else {
    const long long quota = line_quota(p, lane);
    const long long from = quota * blockIdx.x;
    long long start;
    if (quota == 0 || !line_find(p, lane, from, at.b, at.len, start)) return;  // every warp of the CTA alike
    at.T = blocks_of(at.len);
    const long long off = from - start;
    at.item = static_cast<int>(quotient(off, at.T));
    at.t = static_cast<int>(off - static_cast<long long>(at.item) * at.T);
    at.rem = quota;
  }
  // where the blocks end that some column of the item's column block sees
  auto seen = [&](const Place& w) {
    const int last = min(p.n - 1, (w.item % p.CB * NC + NC - 1) / p.G);
    const int keys = w.len - p.n + last + 1;
    return keys > 0 ? min(w.end(), blocks_of(keys)) : 0;
  };

  if (warp == kWarps) {  // the copies: lane x looks after tile x of each block
    const int tiles_page = p.c.page >> 4;
    unsigned uses = 0;
    int stage = 0;
    bool dead = false;
    for (Place w = at; w.rem > 0 && !dead; w.next(p)) {
      const int tiles = (w.len + 15) >> 4, end = seen(w);
      const int32_t* row = p.table + static_cast<long long>(w.b) * p.table_ld;
      for (int blk = w.t; blk < end; ++blk) {
        const int tile = blk * (kBlock / 16) + lane;
        const bool mine = lane < kBlock / 16 && tile < tiles;
        const int page = mine ? __ldg(row + tile / tiles_page) : -1;
        const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(p.c.pages);
        if (mine && !ok) atomicOr(p.err, kErrBadPos);
        const unsigned mask = __ballot_sync(0xffffffffu, ok);
        if (uses >= S && !mbar_wait_quiet_warp(&empty[stage], uses / S - 1 & 1, p.err)) {
          dead = true;
          break;
        }
        if (lane == 0) {
          came[stage] = mask;
          mbar_arrive_expect_tx(&full[stage], __popc(mask) * Tile::kBytes);
        }
        __syncwarp();
        if (ok)
          bulk_g2s(sm + stage * Sm::kStage + lane * Tile::kBytes, Tile::ptr(p.c, page, w.item / p.CB, tile % tiles_page),
                   Tile::kBytes, &full[stage]);
        stage = stage + 1 == S ? 0 : stage + 1;
        ++uses;
      }
    }
    // every copy lands before the CTA's memory is another's
    for (unsigned x = uses < S ? 0 : uses - S; x < uses; ++x) mbar_wait_quiet_warp(&full[x % S], x / S & 1, p.err);
    if constexpr (!CL) return;
    at.rem = 0;
  }
  const int cl_item = at.item, cl_b = at.b;

  bool dead = false;                        // a wait of the warp gave up: the error word says so, nothing more is computed
  int slot = 0, phase = 0;
  while (at.rem > 0) {
    const int j = at.item / p.CB, col0 = at.item % p.CB * NC, cols = min(NC, p.n * p.G - col0);
    // q as B fragments: word w of a lane's 8 or 16 bytes of codes holds dims 8w .. 8w + 7 of its chunk, and its four
    // masks give dims (0, 4), (1, 5) 2^4, (2, 6), (3, 7) 2^4
    uint32_t qf[NT][GR][2][4];
    float unq[NT][2], qsum[NT][GR][2];      // of columns 2c, 2c + 1: 2^24 over q's factor, and sum(q_g) / unq
    int lim[NT][2];                         // keys a column sees
    int least = 0x7fffffff, most = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + r;
      float f[GR][16], mx = 0.f;
      const bool live = col < cols;
      const int i = (col0 + col) / p.G;
      const T* src = static_cast<const T*>(p.q) +
                     ((static_cast<long long>(at.b) * p.n + i) * p.H + j * p.G + (col0 + col) % p.G) * HD + 16 * c;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        const uint4 u0 = live ? *reinterpret_cast<const uint4*>(src + 64 * g) : make_uint4(0, 0, 0, 0);
        const uint4 u1 = live ? *reinterpret_cast<const uint4*>(src + 64 * g + 8) : make_uint4(0, 0, 0, 0);
        unpack8(u0, f[g], static_cast<const T*>(nullptr));
        unpack8(u1, f[g] + 8, static_cast<const T*>(nullptr));
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fabsf(f[g][e]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^x with x = 8 - floor(log2 max): the largest |q| becomes 2^8 .. 2^9
      const int ex = mx > 1e-35f ? static_cast<int>(__float_as_uint(mx) >> 23) : 127;
      const float up = __uint_as_float(static_cast<uint32_t>(min(max(262 - ex, 30), 230)) << 23);
      const float down = 16777216.f / up;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += f[g][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum /= down;
        qsum[nt][g][0] = __shfl_sync(0xffffffffu, sum, 8 * c);
        qsum[nt][g][1] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const float* h = f[g] + 8 * w;
          qf[nt][g][w][0] = half2_bits(h[0] * up, h[4] * up);
          qf[nt][g][w][1] = half2_bits(h[1] * up * 0.0625f, h[5] * up * 0.0625f);
          qf[nt][g][w][2] = half2_bits(h[2] * up, h[6] * up);
          qf[nt][g][w][3] = half2_bits(h[3] * up * 0.0625f, h[7] * up * 0.0625f);
        }
      }
      unq[nt][0] = __shfl_sync(0xffffffffu, down, 8 * c);
      unq[nt][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int cc = nt * 8 + 2 * c + e;
        lim[nt][e] = cc < cols ? max(0, at.len - p.n + (col0 + cc) / p.G + 1) : 0;
      }
    }
    // keys that every (any) column of the block sees
    least = max(0, at.len - p.n + col0 / p.G + 1);
    most = max(0, at.len - p.n + (col0 + cols - 1) / p.G + 1);

    float o[NT][GR][4][4], m[NT][2], l[NT][2], bt[NT][GR][2], sref[GR], isref[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) sref[g] = 5.9604645e-8f, isref[g] = 16777216.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = 0.f;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        bt[nt][g][0] = bt[nt][g][1] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][g][k][0] = o[nt][g][k][1] = o[nt][g][k][2] = o[nt][g][k][3] = 0.f;
      }
    }

    const int end = seen(at);
    bool fresh = true;                       // no key yet: m is set, up or down, by the first ones
    for (int blk = at.t; blk < end; ++blk) {
      if (!dead && !mbar_wait_warp(&full[slot], phase, p.err)) dead = true;
      if (dead) continue;
      const unsigned mask = came[slot] >> (2 * warp) & 3u;
      const uint8_t* st = sm + slot * Sm::kStage + warp * 2 * Tile::kBytes;
      const int key0 = blk * kBlock + warp * 32;
      if (mask != 0u) {
      float y[2][NT][4];                     // log2 of the weights of (key r, columns 2c, 2c + 1), (key r + 8, the same)
      uint32_t ve[2][2][GR];                 // V's {scale, bias} of keys r, r + 8
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* tl = st + h * Tile::kBytes;
        // K words and entries of keys r and r + 8
        uint32_t kw[2][2 * GR], ke[2][GR];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (GR == 2) {
            const uint4 k4 = *reinterpret_cast<const uint4*>(tl + i * 512 + lane * 16);
            kw[i][0] = k4.x; kw[i][1] = k4.y; kw[i][2] = k4.z; kw[i][3] = k4.w;
            const uint4 e4 = *reinterpret_cast<const uint4*>(tl + Tile::kSb + (r + 8 * i) * 16);
            ke[i][0] = e4.x; ke[i][1] = e4.y; ve[h][i][0] = e4.z; ve[h][i][1] = e4.w;
          } else {
            const uint2 k2 = *reinterpret_cast<const uint2*>(tl + i * 256 + lane * 8);
            kw[i][0] = k2.x; kw[i][1] = k2.y;
            const uint2 e2 = *reinterpret_cast<const uint2*>(tl + Tile::kSb + (r + 8 * i) * 8);
            ke[i][0] = e2.x; ve[h][i][0] = e2.y;
          }
        }
        float d[NT][GR][4];
        // the groups' chains of four in turn, so that an MMA does not wait for the one before it
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int up = 0; up < 2; ++up)
#pragma unroll
            for (int g = 0; g < GR; ++g) {
              const uint32_t a = kw[0][2 * g + w] >> (8 * up), b = kw[1][2 * g + w] >> (8 * up);
              const uint32_t f0 = a & 0x000f000fu, f1 = b & 0x000f000fu, f2 = a & 0x00f000f0u, f3 = b & 0x00f000f0u;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float* x = d[nt][g];
                if (w + up == 0) mma_zero(x, f0, f1, f2, f3, qf[nt][g][0]);
                else mma(x, f0, f1, f2, f3, qf[nt][g][w] + 2 * up);
              }
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 sb[GR];
#pragma unroll
          for (int g = 0; g < GR; ++g) sb[g] = bits_float2(ke[i][g]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = sb[0].y * qsum[nt][0][e];
              if (GR == 2) v = fmaf(sb[GR - 1].y, qsum[nt][GR - 1][e], v);
#pragma unroll
              for (int g = 0; g < GR; ++g) v = fmaf(sb[g].x, d[nt][g][2 * i + e], v);
              y[h][nt][2 * i + e] = fmaf(v, unq[nt][e], -m[nt][e]);
            }
        }
      }
      if (key0 + 32 > least || mask != 3u) {  // the mask's edge: an unseen key weighs nothing, whatever its bytes hold
        bool odd = false;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = mask >> h & 1 ? key0 + h * 16 + r + 8 * i : 0x7fffffff;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (key >= lim[nt][e]) y[h][nt][2 * i + e] = -INFINITY;
            if (key >= most) {
#pragma unroll
              for (int g = 0; g < GR; ++g) ve[h][i][g] = 0u;
            }
#pragma unroll
            for (int g = 0; g < GR; ++g) odd |= !finite_pair(ve[h][i][g]);
          }
        // A V that is not finite, of a key that only some of the rows see: it counts here, for the columns that see it,
        // because a weight of zero times it would not be zero for the others.
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int g = 0; g < GR; ++g) {
                if (finite_pair(ve[h][i][g])) continue;
                ve[h][i][g] = 0u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (key0 + h * 16 + r + 8 * i < lim[nt][e]) bt[nt][g][e] = NAN;
              }
        }
      }
      // Has a weight or a scale outgrown its reference? The weights' sums of this lane's keys tell of the first (over
      // 4,096 where one passes 2^12), each lane looks at the scales of one key for the second.
      float pw[2][NT][4], ps[NT][2];
      auto weigh = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x) pw[h][nt][x] = ex2(y[h][nt][x]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            ps[nt][e] = (pw[0][nt][e] + pw[0][nt][2 + e]) + (pw[1][nt][e] + pw[1][nt][2 + e]);
        }
      };
      weigh();
      float big[GR];
      {
        const uint8_t* en = st + (lane >> 4) * Tile::kBytes + Tile::kSb + (lane & 15) * Tile::kEntry + 4 * GR;
        const bool in = key0 + lane < most && (mask >> (lane >> 4) & 1u);
#pragma unroll
        for (int g = 0; g < GR; ++g)
          big[g] = in ? fabsf(__half2float(*reinterpret_cast<const __half*>(en + 4 * g))) : 0.f;
      }
      bool move = fresh;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) move |= fmaxf(ps[nt][0], ps[nt][1]) > 4096.f;
#pragma unroll
      for (int g = 0; g < GR; ++g) move |= big[g] > 8.f * sref[g];
      if (__any_sync(0xffffffffu, move)) {
        float fg[GR];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const uint32_t top = __float_as_uint(warp_max(finite_abs(big[g])));
          const float up = fmaxf(sref[g], __uint_as_float((top + 0x7fffffu) & 0x7f800000u));
          fg[g] = sref[g] / up;
          sref[g] = up;
          isref[g] = 1.f / up;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(y[0][nt][e], y[0][nt][2 + e]), fmaxf(y[1][nt][e], y[1][nt][2 + e]));
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            // the reference goes up by this much; a column that sees none of the first keys sees no later ones
            const float by = fresh ? (mx > -INFINITY ? mx - 8.f : 0.f) : fmaxf(0.f, mx - 8.f);
            const float f = fresh ? 1.f : ex2(-by);
            m[nt][e] += by;
            l[nt][e] *= f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              y[h][nt][e] -= by;
              y[h][nt][2 + e] -= by;
            }
#pragma unroll
            for (int g = 0; g < GR; ++g) {
              bt[nt][g][e] *= f;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][g][k][e] *= f * fg[g];
                o[nt][g][k][2 + e] *= f * fg[g];
              }
            }
          }
        weigh();
      }
      fresh = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        l[nt][0] += ps[nt][0];
        l[nt][1] += ps[nt][1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // weights: P operands, the sum, and the bias term
        uint32_t pf[NT][GR][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float s1[GR], b8[GR];
#pragma unroll
          for (int g = 0; g < GR; ++g) {
            const float2 e2 = bits_float2(ve[h][i][g]);
            s1[g] = e2.x * isref[g];
            b8[g] = fmaf(8.f, e2.x, e2.y);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float p0 = pw[h][nt][2 * i], p1 = pw[h][nt][2 * i + 1];
#pragma unroll
            for (int g = 0; g < GR; ++g) {
              bt[nt][g][0] = fmaf(p0, b8[g], bt[nt][g][0]);
              bt[nt][g][1] = fmaf(p1, b8[g], bt[nt][g][1]);
              pf[nt][g][i] = transpose8(half2_bits(p0 * s1[g], p1 * s1[g]));
            }
          }
        }
        // values of keys 2c, 2c + 1, 2c + 8, 2c + 9: rows r hold the even nibbles, rows r + 8 the odd ones (2^4 larger)
        const uint8_t* tl = st + h * Tile::kBytes + Tile::kCodes;
        uint32_t vw[4][GR];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (GR == 2) {
            const uint4 v4 = *reinterpret_cast<const uint4*>(tl + i * 512 + lane * 16);
            vw[2 * i][0] = v4.x; vw[2 * i][1] = v4.y; vw[2 * i + 1][0] = v4.z; vw[2 * i + 1][1] = v4.w;
          } else {
            const uint2 v2 = *reinterpret_cast<const uint2*>(tl + i * 256 + lane * 8);
            vw[2 * i][0] = v2.x; vw[2 * i + 1][0] = v2.y;
          }
        }
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const uint32_t xa = prmt(vw[0][g], vw[1][g], 0x5410u), xb = prmt(vw[2][g], vw[3][g], 0x5410u);
          const uint32_t ya = prmt(vw[0][g], vw[1][g], 0x7632u), yb = prmt(vw[2][g], vw[3][g], 0x7632u);
          const uint32_t a[4] = {xa, xa >> 8, ya, ya >> 8}, b[4] = {xb, xb >> 8, yb, yb >> 8};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a0 = about8(a[k], 0), a1 = about8(a[k], 1), a2 = about8(b[k], 0), a3 = about8(b[k], 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(o[nt][g][k], a0, a1, a2, a3, pf[nt][g]);
          }
        }
      }
      }
      __syncwarp();                        // every lane has read its keys: the next copy may overwrite them
      if (lane == 0) mbar_arrive(&empty[slot]);
      slot = slot + 1 == S ? 0 : slot + 1;
      if (slot == 0) phase ^= 1;
    }

    // the warp's result: a lane holds dims 64 g + 8 r + (0 .. 7) of columns 2c, 2c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = nt * 8 + 2 * c + e;
        float sum = l[nt][e];
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (r == 0) sml[warp * NC + col] = make_float2(sum != 0.f ? m[nt][e] : kNone, sum);
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          float bias = bt[nt][g][e];
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) bias += __shfl_xor_sync(0xffffffffu, bias, x);
          const float f0 = 16777216.f * sref[g], f1 = 1048576.f * sref[g];
          float* dst = so + (warp * NC + col) * Sm::kRow + 64 * g + 8 * r;
          *reinterpret_cast<float4*>(dst) =
              make_float4(fmaf(o[nt][g][0][e], f0, bias), fmaf(o[nt][g][0][2 + e], f1, bias),
                          fmaf(o[nt][g][1][e], f0, bias), fmaf(o[nt][g][1][2 + e], f1, bias));
          *reinterpret_cast<float4*>(dst + 4) =
              make_float4(fmaf(o[nt][g][2][e], f0, bias), fmaf(o[nt][g][2][2 + e], f1, bias),
                          fmaf(o[nt][g][3][e], f0, bias), fmaf(o[nt][g][3][2 + e], f1, bias));
        }
      }
    warps_sync();
    // the four warps joined; whole items are written out, pieces go to the workspace
    const bool whole = !CL && at.t == 0 && at.end() == at.T;
    const int piece = 2 * blockIdx.x + (at.t == 0 ? 1 : 0);
    for (int u = threadIdx.x; u < cols * (HD / 8); u += kThreads) {
      const int col = u / (HD / 8), d = u % (HD / 8) * 8;
      float2 ml[kWarps];
      float mx = kNone, sum = 0.f, v[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ml[w] = sml[w * NC + col];
        mx = fmaxf(mx, ml[w].x);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(ml[w].x - mx);
        sum += f * ml[w].y;
        const float* src = so + (w * NC + col) * Sm::kRow + d;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(f, src[e], v[e]);
      }
      if (whole) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv;
        kv4_write8<HD, T>(p, at.b, j, col0 + col, d, v);
      } else if (CL) {                       // this thread's own place among the first warp's results
        float* dst = so + col * Sm::kRow + d;
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (d == 0) reinterpret_cast<float2*>(sm + Sm::kOwn)[col] = make_float2(mx, sum);
      } else {
        float* ml_out = p.part + (static_cast<long long>(piece) * NC + col) * 2;
        float* dst = p.part + static_cast<long long>(p.ctas) * 2 * NC * 2 + (static_cast<long long>(piece) * NC + col) * HD + d;
        if (d == 0) *reinterpret_cast<float2*>(ml_out) = make_float2(mx, sum);
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
    if constexpr (CL) break;
    warps_sync();
    at.next(p);
  }
  if constexpr (CL) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int rank = blockIdx.x % p.cluster, j = cl_item / p.CB, col0 = cl_item % p.CB * NC;
    const int units = min(NC, p.n * p.G - col0) * (HD / 8);
    // a lane for each CTA's piece, so that a warp takes 32 / cluster units of eight dims at once (with sixteen lanes a unit
    // whatever the cluster's size, one block of 16 columns in a cluster of one took 27 us; it takes 8)
    const int lg = 31 - __clz(p.cluster), step = 32 >> lg;
    for (int u0 = (rank * kWarps + warp) * step; warp < kWarps && u0 < units; u0 += p.cluster * kWarps * step) {
      const int u = min(u0 + (lane >> lg), units - 1), col = u / (HD / 8), d = u % (HD / 8) * 8, x = lane & (p.cluster - 1);
      float v[8] = {};
      const float2 ml = *cluster.map_shared_rank(reinterpret_cast<float2*>(sm + Sm::kOwn) + col, x);
      if (ml.y != 0.f) {
        const float4* src = reinterpret_cast<const float4*>(cluster.map_shared_rank(so + col * Sm::kRow + d, x));
        const float4 a = src[0], e = src[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = e.x; v[5] = e.y; v[6] = e.z; v[7] = e.w;
      }
      join_lanes(p.cluster, ml.x, ml.y, v);
      if (x == 0 && u0 + (lane >> lg) < units) kv4_write8<HD, T>(p, cl_b, j, col0 + col, d, v);
    }
    cluster.sync();                          // the neighbours' shared memory stays until all have read it
  }
}

// One CTA an item: joins the pieces that the CTAs of kv4_attn_kernel left of it, in their order; writes zeros for a
// sequence of no tokens. Its few threads of 64 registers fit on an SM beside the first kernel's CTAs, so that it has
// found its pieces when they end.
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(64 * NT, 16 / NT) kv4_join_kernel(const __grid_constant__ Kv4AttnParams p) {
  constexpr int NC = 8 * NT, kJoin = 64 * NT;
  const int lane = threadIdx.x & 31;
  const int items = p.c.kvh * p.CB, b = blockIdx.x / items, item = blockIdx.x % items;
  // The lengths may be read before the first kernel is done: it let this one start after its own wait. What follows in
  // the stream may start to start: it waits for this kernel's end.
  pdl_launch_dependents();
  const int blocks = blocks_of(kv4_seq_len(p, b));
  const int j = item / p.CB, col0 = item % p.CB * NC, cols = min(NC, p.n * p.G - col0);
  long long c0 = 0, c1 = 0;
  if (blocks) {
    const long long quota = line_quota(p, lane);
    long long before = 0;
    for (int x = lane; x < b; x += 32) before += blocks_of(kv4_seq_len(p, x));
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) before += __shfl_xor_sync(0xffffffffu, before, m);
    const long long start = before * items + static_cast<long long>(item) * blocks;
    c0 = quotient(start, quota);
    c1 = quotient(start + blocks - 1, quota);
  }
  pdl_wait();
  if (blocks && c0 == c1) return;           // one CTA had all of it
  const float* ml = p.part;
  const float* val = p.part + static_cast<long long>(p.ctas) * 2 * NC * 2;
  const int units = cols * (HD / 8);
  struct Sum {  // pieces of one column's eight dims, taken in one after another
    float m = kNone, sum = 0.f, v[8] = {};
    __device__ void add(const float* ml, const float* val, long long k, int d) {
      const float2 q = __ldcg(reinterpret_cast<const float2*>(ml) + k);
      const float4 a = __ldcg(reinterpret_cast<const float4*>(val + k * HD + d));
      const float4 e = __ldcg(reinterpret_cast<const float4*>(val + k * HD + d + 4));
      const float nm = fmaxf(m, q.x), f = ex2(m - nm), g = ex2(q.x - nm);
      m = nm;
      sum = fmaf(f, sum, g * q.y);
      v[0] = fmaf(f, v[0], g * a.x); v[1] = fmaf(f, v[1], g * a.y); v[2] = fmaf(f, v[2], g * a.z);
      v[3] = fmaf(f, v[3], g * a.w); v[4] = fmaf(f, v[4], g * e.x); v[5] = fmaf(f, v[5], g * e.y);
      v[6] = fmaf(f, v[6], g * e.z); v[7] = fmaf(f, v[7], g * e.w);
    }
  };
  if (c1 - c0 < 8) {  // few pieces: a thread a (column, eight dims)
    for (int u = threadIdx.x; u < units; u += kJoin) {
      const int col = u / (HD / 8), d = u % (HD / 8) * 8;
      Sum t;
      if (blocks) {
#pragma unroll 4
        for (long long x = c0; x <= c1; ++x) t.add(ml, val, (2 * x + (x == c0)) * NC + col, d);
      }
      const float inv = t.sum != 0.f ? 1.f / t.sum : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) t.v[e] *= inv;
      kv4_write8<HD, T>(p, b, j, col0 + col, d, t.v);
    }
    return;
  }
  // many: sixteen lanes, a piece each in turn
  for (int u0 = (threadIdx.x >> 5) * 2; u0 < units; u0 += kJoin / 32 * 2) {
    const int u = min(u0 + (lane >> 4), units - 1), col = u / (HD / 8), d = u % (HD / 8) * 8;
    Sum t;
    for (long long x = c0 + (lane & 15); x <= c1; x += 16) t.add(ml, val, (2 * x + (x == c0)) * NC + col, d);
    join_lanes(16, t.m, t.sum, t.v);
    if ((lane & 15) == 0 && u0 + (lane >> 4) < units) kv4_write8<HD, T>(p, b, j, col0 + col, d, t.v);
  }
}

int attn_check(const agxc_kv4_attention_args* a) {
  if (!a) return fail(AGXC_EINVAL, "kv4_attention: null argument");
  if (int rc = kv4_check(&a->cache, "kv4_attention")) return rc;
  if (a->dtype != AGXC_F16 && a->dtype != AGXC_BF16) return fail(AGXC_EINVAL, "kv4_attention: q fp16 or bf16");
  if (a->batch < 0 || a->rows < 0) return fail(AGXC_EINVAL, "kv4_attention: batch and rows >= 0");
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return fail(AGXC_EINVAL, "kv4_attention: heads a positive multiple of kv_heads");
  if (a->max_pages < 0 || a->table_ld < a->max_pages)
    return fail(AGXC_EINVAL, "kv4_attention: 0 <= max_pages <= table_ld");
  if (static_cast<int64_t>(a->max_pages) * a->cache.page_size > 0x7fffff00)
    return fail(AGXC_EINVAL, "kv4_attention: max_pages * page_size must stay below 2^31");
  if (static_cast<int64_t>(a->batch) * a->rows * a->heads > 0x7fffffff)
    return fail(AGXC_EINVAL, "kv4_attention: too many query rows for one call");
  return 0;
}

// A kernel's attributes, set once a device; the device, or a negative error.
template <int HD, int NT, typename T, bool CL>
int attn_device() {
  static std::atomic<bool> allowed[64] = {};
  int dev = 0;
  AGXC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return fail(AGXC_EINVAL, "kv4_attention: device index below 64");
  if (!allowed[dev]) {
    auto* kernel = kv4_attn_kernel<HD, NT, T, CL>;
    AGXC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, NT>::kBytes));
    if (CL) AGXC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    allowed[dev] = true;
  }
  return dev;
}

template <int HD, int NT>
cudaLaunchConfig_t attn_config(int ctas, int cluster, cudaStream_t s, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads + 32);
  cfg.dynamicSmemBytes = Smem<HD, NT>::kBytes;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// How many clusters of 2^log2 CTAs run at once, as the runtime says it; negative on an error.
template <int HD, int NT, typename T>
int attn_fit(int log2) {
  static std::atomic<int> fit[64][5] = {};  // one more than the clusters, 0 = not asked yet
  const int dev = attn_device<HD, NT, T, true>();
  if (dev < 0) return dev;
  int n = fit[dev][log2];
  if (!n) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = attn_config<HD, NT>(1 << log2, 1 << log2, nullptr, attr);
    cfg.numAttrs = 1;
    AGXC_CUDA(cudaOccupancyMaxActiveClusters(&n, kv4_attn_kernel<HD, NT, T, true>, &cfg));
    fit[dev][log2] = ++n;
  }
  return n - 1;
}

// The launch's shape: 16 columns a block where one row's heads do not fill 8. Where clusters of four CTAs (or of as many
// as the longest sequence possible has blocks) run for all items at once: a cluster an item, of as many CTAs as do, 16 at
// most. Clusters of two where these are three quarters of the CTAs that the GPU holds. More items than that: the line, over
// all CTAs that the GPU holds at once, or, from 64 columns a KV head on (33 where no sequence is longer than a block), the
// kernel of many rows.
//   1 x 1,792 tokens, 8 items of 8 columns: 6.7 us as clusters, 12.4 as a line. 64 items of 8 columns, 8 x 1,807: 12.8 as
//   clusters, 13.7 as a line; ragged 11.8 and 14.7; 8 x 8,192: 31.3 and 27.8. The line balances unequal lengths, but is two
//   launches, and its join has few CTAs where there are few items (8 x 64 blocks: 10.2 as clusters, 21.7 as a line).
//   Clusters of two, items of 16 columns, 256 of 296 CTAs: 8 x 1,807 x 16 rows ragged 22.9, as a line 26.7; 8 x 8,192 66.0
//   and 70.8; items of 8 columns, 256 of 444 CTAs: 16 x 8,192 55.0 and 43.9; 384 of 444: 24 x 1,807 16.4 and 21.5. One
//   cluster more than run at once costs a second wave: 16 items of 16 columns took 22.4 us in clusters of 16, 14.5 of 8.
//   8 x 1,807 ragged of 8 KV heads, columns a head: 32 as clusters of two 22.9, in the other kernel 31.2; 64 as a line 41.6,
//   there 32.0; 128: 62.8 and 33.8. 1 x 1,807 as clusters here and there: 64 columns (32 items) 14.0 and 20.9, 128 17.0 and 23.
//   60 sequences of at most 40 tokens, 128 columns a head: 118 as clusters of one, 45 there; 91 of 16, 48 columns: 66 and
//   59; 235 of 6, 20 columns: 109 and 148.
struct Shape {
  int nt, cb, ctas, cluster;
  bool chunk;
  int64_t bytes(int hd) const { return cluster || chunk ? 0 : static_cast<int64_t>(ctas) * 2 * (8 * nt) * (hd + 2) * 4; }
};

template <int HD, int NT, typename T>
int attn_cluster(const agxc_ctx* ctx, bool many, int64_t items, int64_t longest, int64_t full, int& size) {
  size = 0;
  for (int x = 0; x <= 4 && 1 << x <= ctx->max_cluster && (x == 0 || (1 << x) < 2 * longest); ++x) {
    const bool any = longest <= 1 && !many;  // an item is one block: CTAs in turn, without the line's second launch
    if (!any && items << x > 4 * ctx->num_sms) break;  // no more than four CTAs an SM: not asked for
    const int most = any ? 0x7fffffff : attn_fit<HD, NT, T>(x);
    if (most < 0) return most;
    if (items > most) break;
    size = 1 << x;
  }
  const bool fills = size == 2 && !many && items * 8 >= full * 3;
  if (size < 4 && size < longest && !fills) size = 0;
  return 0;
}

int attn_shape(const agxc_ctx* ctx, const agxc_kv4_attention_args* a, Shape& s) {
  const int64_t cols = static_cast<int64_t>(a->rows) * (a->heads / a->cache.kv_heads);
  s.nt = cols > 8 ? 2 : 1;
  s.cb = static_cast<int>((cols + 8 * s.nt - 1) / (8 * s.nt));
  const int64_t items = static_cast<int64_t>(a->batch) * a->cache.kv_heads * s.cb;
  const int64_t most = static_cast<int64_t>(a->max_pages) * a->cache.page_size;
  const int64_t longest = (most + kBlock - 1) / kBlock, full = static_cast<int64_t>(ctx->num_sms) * (s.nt == 1 ? 3 : 2);
  s.chunk = false;
  s.ctas = 0;
  const bool bf16 = a->dtype == AGXC_BF16, many = cols >= (longest <= 1 ? 33 : 64);
  int rc;
  if (a->cache.head_dim == 128)
    rc = s.nt == 1 ? bf16 ? attn_cluster<128, 1, __nv_bfloat16>(ctx, many, items, longest, full, s.cluster)
                          : attn_cluster<128, 1, __half>(ctx, many, items, longest, full, s.cluster)
                   : bf16 ? attn_cluster<128, 2, __nv_bfloat16>(ctx, many, items, longest, full, s.cluster)
                          : attn_cluster<128, 2, __half>(ctx, many, items, longest, full, s.cluster);
  else
    rc = s.nt == 1 ? bf16 ? attn_cluster<64, 1, __nv_bfloat16>(ctx, many, items, longest, full, s.cluster)
                          : attn_cluster<64, 1, __half>(ctx, many, items, longest, full, s.cluster)
                   : bf16 ? attn_cluster<64, 2, __nv_bfloat16>(ctx, many, items, longest, full, s.cluster)
                          : attn_cluster<64, 2, __half>(ctx, many, items, longest, full, s.cluster);
  if (rc) return rc;
  if (s.cluster) {
    s.ctas = static_cast<int>(items * s.cluster);
    return 0;
  }
  s.chunk = many;
  if (s.chunk) return 0;
  const int64_t blocks = items * longest;
  s.ctas = static_cast<int>(blocks < full ? blocks : full);
  return 0;
}

template <int HD, int NT, typename T, bool CL>
int attn_launch(const Kv4AttnParams& p, cudaStream_t s) {
  if (const int dev = attn_device<HD, NT, T, CL>(); dev < 0) return dev;
  auto* kernel = kv4_attn_kernel<HD, NT, T, CL>;
  if (CL) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = attn_config<HD, NT>(p.ctas, p.cluster, s, attr);
    AGXC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return 0;
  }
  if (int rc = launch_ex(kernel, dim3(p.ctas), dim3(kThreads + 32), Smem<HD, NT>::kBytes, s, 1, p)) return rc;
  return launch_ex(kv4_join_kernel<HD, NT, T>, dim3(static_cast<unsigned>(p.B) * p.c.kvh * p.CB), dim3(64 * NT), 0, s, 1,
                   p);
}

template <int HD, typename T>
int attn_launch_shape(const Kv4AttnParams& p, const Shape& sh, cudaStream_t s) {
  if (sh.cluster) return sh.nt == 1 ? attn_launch<HD, 1, T, true>(p, s) : attn_launch<HD, 2, T, true>(p, s);
  return sh.nt == 1 ? attn_launch<HD, 1, T, false>(p, s) : attn_launch<HD, 2, T, false>(p, s);
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" {

AGXC_API int64_t agxc_kv4_attention_workspace(agxc_ctx* ctx, const agxc_kv4_attention_args* a) {
  if (!ctx) return fail(AGXC_EINVAL, "kv4_attention: null context");
  if (attn_check(a)) return -1;
  if (a->batch == 0 || a->rows == 0) return 0;
  const OnDevice on(ctx->device);
  if (on.rc()) return -1;
  Shape sh;
  if (attn_shape(ctx, a, sh)) return -1;
  return sh.bytes(a->cache.head_dim);
}

AGXC_API int agxc_kv4_attention_dev(agxc_ctx* ctx, const agxc_kv4_attention_args* a, void* stream) {
  if (!ctx) return fail(AGXC_EINVAL, "kv4_attention: null context");
  if (int rc = attn_check(a)) return rc;
  if (a->batch == 0 || a->rows == 0) return 0;
  if (!a->q_dev || !a->out_dev || !a->lengths_dev || (a->max_pages && !a->page_table_dev))
    return fail(AGXC_EINVAL, "kv4_attention: null buffer");
  if (reinterpret_cast<uintptr_t>(a->q_dev) % 16 || reinterpret_cast<uintptr_t>(a->out_dev) % 16)
    return fail(AGXC_EINVAL, "kv4_attention: q and out must be 16-byte aligned");
  const OnDevice on(ctx->device);
  if (on.rc()) return on.rc();
  Shape sh;
  if (int rc = attn_shape(ctx, a, sh)) return rc;
  const int64_t need = sh.bytes(a->cache.head_dim);
  if (need && (a->workspace_bytes < need || !a->workspace_dev || reinterpret_cast<uintptr_t>(a->workspace_dev) % 16))
    return fail(AGXC_EINVAL, "kv4_attention: a 16-byte aligned workspace of agxc_kv4_attention_workspace bytes");
  Kv4AttnParams p;
  p.c = kv4_of(a->cache);
  p.q = a->q_dev; p.out = a->out_dev; p.B = a->batch; p.n = a->rows; p.H = a->heads;
  p.G = a->heads / a->cache.kv_heads; p.CB = sh.cb; p.ctas = sh.ctas; p.cluster = sh.cluster;
  p.table_ld = a->table_ld; p.max_pages = a->max_pages; p.table = a->page_table_dev; p.lengths = a->lengths_dev;
  p.part = static_cast<float*>(a->workspace_dev); p.err = ctx->err_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const bool bf16 = a->dtype == AGXC_BF16;
  if (sh.chunk) return launch_kv4_chunk(ctx, p, a->cache.head_dim, bf16, s);
  if (a->cache.head_dim == 128)
    return bf16 ? attn_launch_shape<128, __nv_bfloat16>(p, sh, s) : attn_launch_shape<128, __half>(p, sh, s);
  return bf16 ? attn_launch_shape<64, __nv_bfloat16>(p, sh, s) : attn_launch_shape<64, __half>(p, sh, s);
}

}  // extern "C"
