// kv4_chunk.cu — attention over the paged 4-bit KV cache for many query rows a sequence (prompt chunks), on the fifth
// generation tensor cores. The mathematics is kv4_attention.cu's: codes meet the tensor cores as they are (about 8), the
// scales and biases are applied to the scores and weights in fp32, out = (sum_t p_t s_t (code_t - 8) + sum_t p_t (b_t +
// 8 s_t)) / sum_t p_t per group of 64 dims.
//
// A CTA takes 128 columns (a column = one (row, head) of a KV head) against the keys of its share, 64 at a time:
//   copy warp      a bulk copy a tile into three raw stages
//   dequant warps  (four) the tiles' codes as fp16 into 128-byte-swizzled operands, K [key][dim] and V [dim][key], and the
//                  keys' scales and biases into a table of floats. K's dims lie in the order the fields come out of a
//                  word ((0, 4), (1, 5) 16-fold, (2, 6), (3, 7) 16-fold of each eight) and q's are stored to match
//   MMA warp       D_g[column][key] = q_g (code_g - 8) for each group g (tcgen05.mma, M 128, N 64, q and K from shared
//                  memory), and O_g[column][dim] += P_g (code_g - 8) with P from tensor memory
//   softmax warps  two groups of four that take blocks in turn, each with sums and an O of its own, so that one computes
//                  while the tensor core works for the other. One thread a column: scores from D, weights, P_g = p s_g /
//                  sref_g in fp16 to tensor memory over D; no reduction crosses threads. The references m and sref move
//                  as rarely as there, and then this thread's row of O is rescaled in tensor memory
// Tensor memory: two O, two D (and P): 512 columns, one CTA an SM. Few items: a cluster of CTAs shares the keys of one
// item and joins through distributed shared memory.
//
// 256 rows of 32 heads over 8 KV heads, 2,304 keys of 128 dims (9.1 GFLOP, 5.5 us at the measured peak): 41.4 us; the
// kernel of single tokens, whose mma.sync dequantises each key once per 16 columns, takes 81.5. 512 rows over 8,192 keys:
// 218 us, 1.7 us a block of 64 keys and 128 columns, 0.97 at 64 dims. What bounds it is the shared memory pipe, busy for 80
// of 100 cycles on the SMs that work: each softmax warp reads every key's scales and biases (1,020 of a block's 2,060
// wavefronts; a read of 16 bytes by all lanes costs two), the dequantised operands are written (390) and the tensor core reads
// them (500). Tried and not kept: P through shared memory instead of tensor memory (49 us), scores fetched 16 keys at a
// time with a wait each (42.3). Not done: scales multiplied into K by the dequant warps. One fp16 product would round K to
// 11 bits, and at 8,192 keys more error than fp32 arithmetic leaves; the exact product takes two operands a key.
#include <cooperative_groups.h>

#include <atomic>

#include "kv4_attention.cuh"

namespace agxc {
namespace {

namespace cg = cooperative_groups;

constexpr int kRows = 128, kKeys = 64;
// Warps 0 .. 7 softmax, 8 .. 11 dequant, 12 copies, 13 MMAs, 14 and 15 only give up registers: 512 threads of 128, of which
// the softmax warps take 160 and the others keep 96 (256 x 160 + 256 x 96 = 65,536).
constexpr int kDeq = 8, kDeqWarps = 4, kCopy = 12, kMma = 13, kWarps = 16, kThreads = 32 * kWarps;
constexpr int kMoreRegs = 160, kFewerRegs = 96;
constexpr int kRaw = 3, kSt = 3;                                // raw stages, operand stages
constexpr int kTmemCols = 512, kD = 256;
constexpr float kNone = -1e30f;
constexpr unsigned kOdd = 16u;                                  // some V of the block is not finite
constexpr int kMaxShare = 8;                                    // CTAs an item: what a portable cluster has

template <int HD>
struct ChunkSmem {
  static constexpr int GR = HD / 64;
  static constexpr int kTile = Kv4Tile<HD>::kBytes;
  static constexpr int kQ = 1024;                                 // [group][128 rows][128 B]
  static constexpr int kK = kQ + GR * kRows * 128;                // kSt stages of [group][64 keys][128 B]
  static constexpr int kV = kK + kSt * GR * kKeys * 128;            // kSt stages of [HD dims][128 B]
  static constexpr int kRawAt = kV + kSt * HD * 128;                // three stages of four tiles
  static constexpr int kTable = kRawAt + kRaw * 4 * kTile;        // kSt stages of [two keys]{K s0 s1 b0 b1, V s0 s1 b0 b1}[2]
  static constexpr int kMl = kTable + kSt * kKeys * 32;             // {m, sum} of the rows, for the cluster
  static constexpr int kStat = kMl + kRows * 8;                   // {1 / q's factor, q's sums} of the rows
  static constexpr int kEnd = kStat + kRows * 16;
  static constexpr int kRow = HD + 4;                             // the rows' results over K, V and the raw stages
  static_assert(kRows * kRow * 4 <= kTable - kK, "the results fit");
  static constexpr int kBytes = kEnd + 1024;                      // and the 1,024-byte alignment
};

// barriers and words in the first 1,024 bytes
struct Bars {
  uint64_t raw_full[kRaw], raw_empty[kRaw], kv_full[kSt], kv_done[kSt], s_full[2], p_full[2], pv_done[2], drained;
  uint32_t tmem;
  volatile int dead;
  volatile unsigned came_raw[kRaw], came[kSt];   // bits 0 .. 3: the tiles that were copied; kOdd
  volatile unsigned odd[kSt][2][2];              // [group][half of the keys] whose V is not finite, where kOdd is set
  volatile float sref[kSt][2];
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
  // K-major, 128-byte swizzle: start >> 4, leading offset 16 B, 1,024 B between eight-row atoms, version 1, layout 2
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// fp32 accumulator, fp16 operands, both K-major, N 64, M 128
constexpr uint32_t kIdesc = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, bool acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
               "l"(a), "l"(b), "r"(kIdesc), "r"(static_cast<uint32_t>(acc))
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, bool acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
               "r"(a), "l"(b), "r"(kIdesc), "r"(static_cast<uint32_t>(acc))
               : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this thread's lane, there when this returns (the wait is in the same statement as the load)
__device__ __forceinline__ void tmem_ld32(uint32_t a, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(a)
      : "memory");
}
// 8 columns on their way: they are there after tmem_wait8 of the same values
__device__ __forceinline__ void tmem_begin8(uint32_t a, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void tmem_wait8(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// code - 8 of the even or 16 (code - 8) of the odd nibble in the low byte of each half of x, times 2^-24: an exact
// difference of fp16 subnormals, which the tensor core takes as they are
__device__ __forceinline__ uint32_t about8(uint32_t x, int odd) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x & (odd ? 0x00f000f0u : 0x000f000fu)), "r"(odd ? 0x00800080u : 0x00080008u));
  return d;
}
constexpr float kUnit = 16777216.f;  // 2^24

// two fp32 operations an instruction
using f2 = uint64_t;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void apart(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

struct ChunkParams {
  Kv4AttnParams a;
  int RB, S;  // blocks of 128 columns an item row, CTAs (a cluster) an item
};

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1) kv4_chunk_kernel(const __grid_constant__ ChunkParams cp) {
  using Tile = Kv4Tile<HD>;
  using Sm = ChunkSmem<HD>;
  constexpr int GR = Sm::GR;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* sm = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  Bars& br = *reinterpret_cast<Bars*>(sm);
  static_assert(sizeof(Bars) <= 1024);
  const Kv4AttnParams& p = cp.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&br.raw_full[i], 1);
      mbar_init(&br.raw_empty[i], kDeqWarps);
    }
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&br.kv_full[i], kDeqWarps);
      mbar_init(&br.kv_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&br.s_full[i], 1);
      mbar_init(&br.p_full[i], 4);
      mbar_init(&br.pv_done[i], 1);
    }
    mbar_init(&br.drained, 1);
    br.dead = 0;
    fence_mbar_init();
  }
  // Tensor memory is taken only now that the kernels before are done: a CTA that holds it waits for no other's.
  pdl_wait();
  pdl_launch_dependents();
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&br.tmem)), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = br.tmem;

  // the CTA's item and its share of the keys that some column sees
  const int unit = blockIdx.x / cp.S, rank = blockIdx.x % cp.S;
  const int b = unit / (p.c.kvh * cp.RB), j = unit / cp.RB % p.c.kvh, col0 = unit % cp.RB * kRows;
  const int cols = min(kRows, p.n * p.G - col0);
  const int len = kv4_seq_len(p, b);
  const int least = max(0, len - p.n + col0 / p.G + 1), most = max(0, len - p.n + (col0 + cols - 1) / p.G + 1);
  const int blocks = (most + kKeys - 1) / kKeys, per = (blocks + cp.S - 1) / cp.S;
  const int first = min(blocks, rank * per), count = min(blocks, first + per) - first;
  uint8_t* sk = sm + Sm::kK;
  uint8_t* sv = sm + Sm::kV;
  const auto ok_all = [&](bool ok) {  // a warp leaves together
    if (__all_sync(0xffffffffu, ok)) return true;
    br.dead = 1;
    return false;
  };

  if (warp >= kCopy) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewerRegs));
    if (warp == kCopy) {
    // ---- copies
    const int tiles_page = p.c.page >> 4, tiles = (len + 15) >> 4;
    const int32_t* row = p.table + static_cast<long long>(b) * p.table_ld;
    int issued = 0;
    for (; issued < count; ++issued) {
      const int st = issued % kRaw, tile = (first + issued) * 4 + lane;
      const bool mine = lane < 4 && tile < tiles;
      const int page = mine ? __ldg(row + tile / tiles_page) : -1;
      const bool ok = static_cast<unsigned>(page) < static_cast<unsigned>(p.c.pages);
      if (mine && !ok) atomicOr(p.err, kErrBadPos);
      const unsigned mask = __ballot_sync(0xffffffffu, ok);
      if (!ok_all(!br.dead && (issued < kRaw || mbar_wait_quiet(&br.raw_empty[st], issued / kRaw - 1 & 1, p.err)))) break;
      if (lane == 0) {
        br.came_raw[st] = mask;
        mbar_arrive_expect_tx(&br.raw_full[st], __popc(mask) * Tile::kBytes);
      }
      __syncwarp();
      if (ok)
        bulk_g2s(sm + Sm::kRawAt + (st * 4 + lane) * Tile::kBytes, Tile::ptr(p.c, page, j, tile % tiles_page), Tile::kBytes,
                 &br.raw_full[st]);
    }
    // every copy lands before the memory is used otherwise
    for (int x = max(0, issued - kRaw); x < issued; ++x) mbar_wait_quiet_warp(&br.raw_full[x % kRaw], x / kRaw & 1, p.err);
  } else if (warp == kMma) {
    // ---- MMAs: the values of block i, then the scores of block i + 2 over the same buffer
    const uint64_t qd = desc_sw128(smem_u32(sm + Sm::kQ)), kd = desc_sw128(smem_u32(sk)), vd = desc_sw128(smem_u32(sv));
    const bool leader = lane == 0;
    asm volatile("bar.sync 2, 288;" ::: "memory");  // q is in place
    auto scores = [&](int i) {
      const int st = i % kSt;
      if (!ok_all(!br.dead && mbar_wait_bounded(&br.kv_full[st], i / kSt & 1, p.err))) return false;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ss(tmem + kD + (i & 1) * 128 + g * 64, qd + ((g * kRows * 128) >> 4) + 2 * k,
                   kd + ((st * GR + g) * kKeys * 128 >> 4) + 2 * k, k > 0);
        tc_commit(&br.s_full[i & 1]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    for (int i = 0; i < 2 && i < count && ok; ++i) ok = scores(i);
    for (int i = 0; i < count && ok; ++i) {
      if (!ok_all(!br.dead && mbar_wait_bounded(&br.p_full[i & 1], i >> 1 & 1, p.err))) break;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(tmem + (i & 1) * 128 + g * 64, tmem + kD + (i & 1) * 128 + g * 32 + 8 * k,
                   vd + ((i % kSt * HD + g * 64) * 128 >> 4) + 2 * k, i > 1 || k > 0);
        tc_commit(&br.pv_done[i & 1]);
        tc_commit(&br.kv_done[i % kSt]);
      }
      __syncwarp();
      if (i + 2 < count) {
        if (!ok_all(mbar_wait_bounded(&br.pv_done[i & 1], i >> 1 & 1, p.err))) break;
        ok = scores(i + 2);
      }
    }
    // whatever was begun ends before tensor memory is given back
    if (leader) tc_commit(&br.drained);
    __syncwarp();
    mbar_wait_quiet_warp(&br.drained, 0, p.err);
    }
  } else if (warp >= kDeq) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewerRegs));
    // ---- codes to operands
    const int w = warp - kDeq;
    float sref[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) sref[g] = 5.9604645e-8f;
    for (int i = 0; i < count; ++i) {
      const int rs = i % kRaw, st = i % kSt;
      if (!ok_all(!br.dead && mbar_wait_bounded(&br.raw_full[rs], i / kRaw & 1, p.err) &&
                  (i < kSt || mbar_wait_bounded(&br.kv_done[st], i / kSt - 1 & 1, p.err))))
        break;
      const uint8_t* raw = sm + Sm::kRawAt + rs * 4 * Tile::kBytes;
      const unsigned mask = br.came_raw[rs];
#pragma unroll
      for (int z = 0; z < 2; ++z) {  // K: a tile a warp, eight keys at a time, lane = 4 key + chunk of 16 dims
        const int t = lane >> 2, c = lane & 3, key = w * 16 + z * 8 + t;
        const uint8_t* src = raw + w * Tile::kBytes + z * 256 * GR + lane * 8 * GR;
        uint32_t x[2 * GR];
        if constexpr (GR == 2) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          x[0] = u.x; x[1] = u.y;
        }
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a = x[2 * g + h], a8 = a >> 8;
            *reinterpret_cast<uint4*>(sk + (st * GR + g) * kKeys * 128 + key * 128 + (((2 * c + h) ^ (key & 7)) << 4)) =
                make_uint4(about8(a, 0), about8(a, 1), about8(a8, 0), about8(a8, 1));
          }
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {  // V: eight dims of each group, lane = 8 tile + 4 (half of its keys) + pair of keys
        const int tile = lane >> 3, h = lane >> 2 & 1, c = lane & 3, r = w + 4 * z;
        const uint8_t* src = raw + tile * Tile::kBytes + Tile::kCodes + h * 256 * GR + (4 * r + c) * 8 * GR;
        uint32_t x[2][GR];  // [key of the pair][group]
        if constexpr (GR == 2) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          x[0][0] = u.x; x[0][1] = u.y; x[1][0] = u.z; x[1][1] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          x[0][0] = u.x; x[1][0] = u.y;
        }
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const uint32_t lo = prmt(x[0][g], x[1][g], 0x5410u), hi = prmt(x[0][g], x[1][g], 0x7632u);
          const uint32_t y[4] = {lo, lo >> 8, hi, hi >> 8};
#pragma unroll
          for (int d = 0; d < 8; ++d)
            *reinterpret_cast<uint32_t*>(sv + (st * HD + g * 64 + 8 * r + d) * 128 + (((2 * tile + h) ^ d) << 4) + 4 * c) =
                about8(y[d >> 1], d & 1);
        }
      }
      if (w == 0) {  // the table; a key that did not come counts as one of no weight (its scores are masked)
        float f[2][8] = {}, big[GR] = {};
        unsigned bad = 0u;  // V's entries that are not finite: bit 2 g + z
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int key = z * 32 + lane;
          const __half2* e = reinterpret_cast<const __half2*>(raw + (key >> 4) * Tile::kBytes + Tile::kSb + (key & 15) * Tile::kEntry);
          const bool in = (mask >> (key >> 4) & 1u) && (first + i) * kKeys + key < most;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int g = 0; g < GR; ++g) {
              const uint32_t u = *reinterpret_cast<const uint32_t*>(e + kv * GR + g);
              const bool fine = kv == 0 || finite_pair(u);
              const float2 sb = bits_float2(u);
              if (in && !fine) bad |= 1u << (2 * g + z);
              f[z][4 * kv + g] = in && fine ? sb.x : 0.f;
              f[z][4 * kv + 2 + g] = in && fine ? fmaf(8.f, sb.x, sb.y) : 0.f;
            }
#pragma unroll
          for (int g = 0; g < GR; ++g) big[g] = fmaxf(big[g], fabsf(f[z][4 + g]));
        }
        // V's scales are kept beside the running power of two above them, which moves when one is 8 times as large
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          big[g] = warp_max(big[g]);
          if (big[g] > 8.f * sref[g]) sref[g] = __uint_as_float((__float_as_uint(big[g]) + 0x7fffffu) & 0x7f800000u);
        }
        float* t = reinterpret_cast<float*>(sm + Sm::kTable) + st * kKeys * 8 + (lane >> 1) * 16 + (lane & 1);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int g = 0; g < GR; ++g) {
            float* to = t + 256 * z + 2 * g;
            to[0] = f[z][g] * kUnit;
            to[4] = f[z][2 + g];
            to[8] = f[z][4 + g] / sref[g];
            to[12] = f[z][6 + g];
          }
        // They go into the sums of the columns that see them, not into the table: a weight of zero times one of them would
        // not be zero for the columns that do not.
        const bool odd = __any_sync(0xffffffffu, bad != 0u);
        if (odd) {
#pragma unroll
          for (int x = 0; x < 2 * GR; ++x) {
            const unsigned keys = __ballot_sync(0xffffffffu, bad >> x & 1u);
            if (lane == 0) br.odd[st][x >> 1][x & 1] = keys;
          }
        }
        if (lane == 0) {
          br.came[st] = odd ? mask | kOdd : mask;
          br.sref[st][0] = sref[0];
          br.sref[st][1] = sref[GR - 1];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&br.raw_empty[rs]);
        mbar_arrive(&br.kv_full[st]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    // ---- softmax: thread = column of the block (tensor memory lane 32 (warp % 4) + lane)
    const int q4 = warp & 3, row = 32 * q4 + lane, col = col0 + row, grp = warp >> 2;
    const bool live = row < cols;
    const uint32_t tl = tmem + (static_cast<uint32_t>(32 * q4) << 16) + grp * 128;  // O; D and P kD columns on
    // q: scaled to 2^8 .. 2^9 by a power of two a row, in K's order of dims; its sums a group. A row's eights of dims lie
    // over HD / 8 lanes, sixteen rows a warp.
    {
      constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes, kTurns = 16 / kAtOnce;
      const int x = lane % kLanes;
      uint4 u[kTurns];
#pragma unroll
      for (int z = 0; z < kTurns; ++z) {
        const int r = warp * 16 + z * kAtOnce + lane / kLanes, c = col0 + r;
        const T* src = static_cast<const T*>(p.q) +
                       ((static_cast<long long>(b) * p.n + c / p.G) * p.H + j * p.G + c % p.G) * HD + 8 * x;
        u[z] = r < cols ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int z = 0; z < kTurns; ++z) {
        const int r = warp * 16 + z * kAtOnce + lane / kLanes;
        float f[8], mx = 0.f, sum = 0.f;
        unpack8(u[z], f, static_cast<const T*>(nullptr));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          mx = fmaxf(mx, fabsf(f[e]));
          sum += f[e];
        }
#pragma unroll
        for (int k = 1; k < kLanes; k <<= 1) {
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
          if (k < 8) sum += __shfl_xor_sync(0xffffffffu, sum, k);  // eight lanes a group of 64 dims
        }
        const int ex = mx > 1e-35f ? static_cast<int>(__float_as_uint(mx) >> 23) : 127;
        const float up = __uint_as_float(static_cast<uint32_t>(min(max(262 - ex, 30), 230)) << 23), u16 = up * 0.0625f;
        *reinterpret_cast<uint4*>(sm + Sm::kQ + (x / 8) * kRows * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4)) =
            make_uint4(half2_bits(f[0] * up, f[4] * up), half2_bits(f[1] * u16, f[5] * u16),
                       half2_bits(f[2] * up, f[6] * up), half2_bits(f[3] * u16, f[7] * u16));
        float* stat = reinterpret_cast<float*>(sm + Sm::kStat) + 4 * r;
        if (x == 0) stat[0] = 1.f / up;
        if ((x & 7) == 0) stat[1 + x / 8] = sum * up;
      }
      fence_proxy_async();
      asm volatile("bar.sync 2, 288;" ::: "memory");
    }
    const float unq = reinterpret_cast<const float*>(sm + Sm::kStat)[4 * row];
    f2 qs[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const float q = reinterpret_cast<const float*>(sm + Sm::kStat)[4 * row + 1 + g];
      qs[g] = pair(q, q);
    }
    const int lim = live ? max(0, len - p.n + col / p.G + 1) : 0;
    float m = 0.f, sref[GR];
    f2 l2 = 0, bt2[GR] = {};                 // of even and odd keys
    const f2 unq2 = pair(unq, unq);
#pragma unroll
    for (int g = 0; g < GR; ++g) sref[g] = 5.9604645e-8f;
    bool fresh = true;
    for (int i = grp; i < count; i += 2) {
      const int st = i % kSt;
      if (!ok_all(!br.dead && mbar_wait_bounded(&br.kv_full[st], i / kSt & 1, p.err) &&
                  mbar_wait_bounded(&br.s_full[grp], i >> 1 & 1, p.err)))
        break;
      tc_fence_after();
      const ulonglong2* table = reinterpret_cast<const ulonglong2*>(sm + Sm::kTable) + st * kKeys * 2;
      const unsigned came = br.came[st], mask = came & 0xFu;
      const int key0 = (first + i) * kKeys;
      float y[kKeys], mx = -INFINITY;
      const f2 minus_m = pair(-m, -m);
      // eight keys' scores are worked on while the next eight's are on their way
      float d[2][GR][8];
#pragma unroll
      for (int g = 0; g < GR; ++g) tmem_begin8(tl + kD + 64 * g, d[0][g]);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
#pragma unroll
        for (int g = 0; g < GR; ++g) tmem_wait8(d[h & 1][g]);
        if (h < 7) {
#pragma unroll
          for (int g = 0; g < GR; ++g) tmem_begin8(tl + kD + 64 * g + 8 * (h + 1), d[h + 1 & 1][g]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const ulonglong2 sc = table[4 * (4 * h + k)], bi = table[4 * (4 * h + k) + 1];
          const float(&e)[GR][8] = d[h & 1];
          f2 v = mul2(bi.x, qs[0]);
          if (GR == 2) v = fma2(bi.y, qs[GR - 1], v);
          v = fma2(sc.x, pair(e[0][2 * k], e[0][2 * k + 1]), v);
          if (GR == 2) v = fma2(sc.y, pair(e[GR - 1][2 * k], e[GR - 1][2 * k + 1]), v);
          apart(fma2(v, unq2, minus_m), y[8 * h + 2 * k], y[8 * h + 2 * k + 1]);
        }
      }
      if (key0 + kKeys > least || mask != 0xFu) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k)
          if (key0 + k >= lim || !(mask >> (k >> 4) & 1u)) y[k] = -INFINITY;
      }
      if (came & kOdd) {
        const int keys = lim - key0;  // that the column sees
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll
          for (int z = 0; z < 2; ++z)
            if (keys > 32 * z && (br.odd[st][g][z] & (keys >= 32 * z + 32 ? 0xffffffffu : (1u << (keys - 32 * z)) - 1u)))
              bt2[g] = pair(NAN, NAN);
      }
#pragma unroll
      for (int k = 0; k < kKeys; ++k) mx = fmaxf(mx, y[k]);
      float fo[GR];
      bool move = fresh || mx > 12.f;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        const float up = br.sref[st][g];
        fo[g] = sref[g] / up;
        move |= up != sref[g];
        sref[g] = up;
      }
      if (__any_sync(0xffffffffu, move)) {
        // a column that sees none of the first keys sees no later ones
        const float by = fresh ? (mx > -INFINITY ? mx - 8.f : 0.f) : fmaxf(0.f, mx - 8.f);
        const float f = fresh ? 1.f : ex2(-by);
        m += by;
        const f2 ff = pair(f, f);
        l2 = mul2(l2, ff);
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          fo[g] *= f;
          bt2[g] = mul2(bt2[g], ff);
        }
#pragma unroll
        for (int k = 0; k < kKeys; ++k) y[k] -= by;
        if (i > 1) {  // this row of O: the group's last block had been added before these scores were computed
#pragma unroll
          for (int x = 0; x < HD / 32; ++x) {
            float o[32];
            tmem_ld32(tl + 32 * x, o);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t u[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[16 * h + e] * fo[x / 2]);
              tmem_st16(tl + 32 * x + 16 * h, u);
            }
          }
          tc_wait_st();
        }
      }
      if (mask != 0u) fresh = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[GR][16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const ulonglong2 sc = table[4 * (16 * h + k) + 2], bi = table[4 * (16 * h + k) + 3];
          const f2 pp = pair(ex2(y[32 * h + 2 * k]), ex2(y[32 * h + 2 * k + 1]));
          l2 = add2(l2, pp);
          float a, c;
          apart(mul2(pp, sc.x), a, c);
          w[0][k] = half2_bits(a, c);
          bt2[0] = fma2(pp, bi.x, bt2[0]);
          if (GR == 2) {
            apart(mul2(pp, sc.y), a, c);
            w[GR - 1][k] = half2_bits(a, c);
            bt2[GR - 1] = fma2(pp, bi.y, bt2[GR - 1]);
          }
        }
#pragma unroll
        for (int g = 0; g < GR; ++g) tmem_st16(tl + kD + g * 32 + 16 * h, w[g]);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&br.p_full[grp]);
    }
    // ---- the rows' results: the first group's in shared memory (K, V and the raw stages are free by then), the second
    // joins its own to them
    float l, bt[GR];
    {
      float a, c;
      apart(l2, a, c);
      l = a + c;
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        apart(bt2[g], a, c);
        bt[g] = a + c;
      }
    }
    const int mine = (count - grp + 1) / 2;  // blocks of the group
    bool done = mine > 0 && !br.dead;
    if (done) done = ok_all(mbar_wait_bounded(&br.pv_done[grp], mine - 1 & 1, p.err));
    if (grp == 0 && count > 1 && done) done = ok_all(mbar_wait_bounded(&br.pv_done[1], count / 2 - 1 & 1, p.err));
    tc_fence_after();
    if (!done) l = 0.f;
    float* out = reinterpret_cast<float*>(sk) + row * Sm::kRow;
    float2* ml = reinterpret_cast<float2*>(sm + Sm::kMl) + row;
    if (grp == 0) {
      *ml = make_float2(l != 0.f ? m : kNone, l);
      if (done)
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) {
          float o[32];
          tmem_ld32(tl + 32 * x, o);
          const float a = kUnit * sref[x / 2], c = a * 0.0625f, z = bt[x / 2];
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(out + 32 * x + e) =
                make_float4(fmaf(o[e], a, z), fmaf(o[e + 1], c, z), fmaf(o[e + 2], a, z), fmaf(o[e + 3], c, z));
        }
    }
    asm volatile("bar.sync 3, 256;" ::: "memory");
    if (grp == 1) {
      const float2 other = *ml;
      const float mm = fmaxf(l != 0.f ? m : kNone, other.x);  // a sum that is NaN goes along
      float f1 = l != 0.f ? ex2(m - mm) : 0.f, f0 = other.y != 0.f ? ex2(other.x - mm) : 0.f;
      const float sum = f1 * l + f0 * other.y;
      if (cp.S == 1) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        f0 *= inv;
        f1 *= inv;
      } else {
        *ml = make_float2(mm, sum);
      }
#pragma unroll
      for (int x = 0; x < HD / 32; ++x) {
        float o[32] = {};
        if (done) {
          tmem_ld32(tl + 32 * x, o);
        }
        const float a = kUnit * sref[x / 2] * f1, c = a * 0.0625f, z = bt[x / 2] * f1;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float v[8];
#pragma unroll
          for (int y = 0; y < 8; ++y) v[y] = f1 != 0.f ? fmaf(o[e + y], y & 1 ? c : a, z) : 0.f;
          if (f0 != 0.f) {
#pragma unroll
            for (int y = 0; y < 8; y += 4) {
              const float4 u = *reinterpret_cast<const float4*>(out + 32 * x + e + y);
              v[y] = fmaf(f0, u.x, v[y]);
              v[y + 1] = fmaf(f0, u.y, v[y + 1]);
              v[y + 2] = fmaf(f0, u.z, v[y + 2]);
              v[y + 3] = fmaf(f0, u.w, v[y + 3]);
            }
          }
          if (cp.S == 1) {
            if (live) kv4_write8<HD, T>(p, b, j, col, 32 * x + e, v);
          } else {
            *reinterpret_cast<float4*>(out + 32 * x + e) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(out + 32 * x + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  if (cp.S > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int u = rank * kThreads + tid; u < cols * (HD / 8); u += cp.S * kThreads) {
      const int r = u / (HD / 8), d = u % (HD / 8) * 8;
      float mx = kNone, sum = 0.f, v[8] = {};
      float2 ml[kMaxShare];
#pragma unroll
      for (int x = 0; x < kMaxShare; ++x) {
        ml[x] = x < cp.S ? *cluster.map_shared_rank(reinterpret_cast<float2*>(sm + Sm::kMl) + r, x) : make_float2(kNone, 0.f);
        mx = fmaxf(mx, ml[x].x);
      }
#pragma unroll
      for (int x = 0; x < kMaxShare; ++x)
        if (ml[x].y != 0.f) {
          const float f = ex2(ml[x].x - mx);
          const float4* src = reinterpret_cast<const float4*>(
              cluster.map_shared_rank(reinterpret_cast<float*>(sk) + r * Sm::kRow + d, x));
          const float4 a = src[0], e = src[1];
          sum = fmaf(f, ml[x].y, sum);
          v[0] = fmaf(f, a.x, v[0]); v[1] = fmaf(f, a.y, v[1]); v[2] = fmaf(f, a.z, v[2]); v[3] = fmaf(f, a.w, v[3]);
          v[4] = fmaf(f, e.x, v[4]); v[5] = fmaf(f, e.y, v[5]); v[6] = fmaf(f, e.z, v[6]); v[7] = fmaf(f, e.w, v[7]);
        }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inv;
      kv4_write8<HD, T>(p, b, j, col0 + r, d, v);
    }
    cluster.sync();  // the neighbours' shared memory stays until all have read it
  }
}

template <int HD, typename T>
int chunk_launch(const agxc_ctx* ctx, ChunkParams cp, cudaStream_t s) {
  constexpr int smem = ChunkSmem<HD>::kBytes;
  static std::atomic<int> fit[64][kMaxShare + 1] = {};  // clusters of x CTAs that run at once, 0 = not asked yet
  int dev = 0;
  AGXC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return fail(AGXC_EINVAL, "kv4_attention: device index below 64");
  auto* kernel = kv4_chunk_kernel<HD, T>;
  if (!fit[dev][1]) {
    AGXC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    fit[dev][1] = ctx->num_sms;
  }
  const Kv4AttnParams& p = cp.a;
  cp.RB = (p.n * p.G + kRows - 1) / kRows;
  const int64_t items = static_cast<int64_t>(p.B) * p.c.kvh * cp.RB;
  const int64_t longest = (static_cast<int64_t>(p.max_pages) * p.c.page + kKeys - 1) / kKeys;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // The largest share of CTAs an item with which all items run at once, each CTA with two blocks of keys at least. The
  // runtime says how many clusters fit: GPCs differ in SMs, and 16 clusters of 8, one more than fit, took 37.6 us where
  // 24.2 as clusters of 7.
  int share = 1;
  for (int x = 2; x <= kMaxShare && x <= ctx->max_cluster && 2 * x <= longest && items * x <= ctx->num_sms; ++x) {
    int most = fit[dev][x];
    if (!most) {
      attr[0].val.clusterDim.x = x;
      cfg.gridDim = dim3(x);
      cfg.numAttrs = 1;
      AGXC_CUDA(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg));
      fit[dev][x] = most = most > 0 ? most : -1;
    }
    if (items <= most) share = x;
  }
  cp.S = share;
  attr[0].val.clusterDim.x = share;
  cfg.numAttrs = 2;
  cfg.gridDim = dim3(static_cast<unsigned>(items * share));
  AGXC_CUDA(cudaLaunchKernelEx(&cfg, kernel, cp));
  return 0;
}

}  // namespace

int launch_kv4_chunk(const agxc_ctx* ctx, const Kv4AttnParams& p, int hd, bool bf16, cudaStream_t s) {
  ChunkParams cp;
  cp.a = p;
  if (hd == 128) return bf16 ? chunk_launch<128, __nv_bfloat16>(ctx, cp, s) : chunk_launch<128, __half>(ctx, cp, s);
  return bf16 ? chunk_launch<64, __nv_bfloat16>(ctx, cp, s) : chunk_launch<64, __half>(ctx, cp, s);
}

}  // namespace agxc
