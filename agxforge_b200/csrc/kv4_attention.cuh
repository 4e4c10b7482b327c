// kv4_attention.cuh — what the two kernels of the attention over the 4-bit cache share: a call's arguments and the small
// conversions.
#pragma once

#include "kv4.cuh"

namespace agxc {

struct Kv4AttnParams {
  Kv4 c;
  const void* q;
  void* out;
  int B, n, H, G, CB;                   // G = q heads a KV head, CB = column blocks an item row
  int table_ld, max_pages;
  int ctas, cluster;                    // cluster = CTAs an item, 0 = the line
  const int32_t* table;
  const int32_t* lengths;
  float* part;                          // [2 ctas][columns]{max, sum}, then [2 ctas][columns][hd]
  unsigned* err;
};

__device__ __forceinline__ int kv4_seq_len(const Kv4AttnParams& p, int b) {
  const int len = p.lengths[b];
  const int most = p.max_pages * p.c.page;
  if (len < 0 || len > most) {
    atomicOr(p.err, kErrBadPos);
    return len < 0 ? 0 : most;
  }
  return len;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the size of an fp16 scale, 0 where it is not finite: the running power of two above the scales is every row's
__device__ __forceinline__ float finite_abs(float s) { return fabsf(s) <= 65504.f ? fabsf(s) : 0.f; }

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ float2 bits_float2(uint32_t u) { return __half22float2(as_half2(u)); }

// are an entry's scale and bias finite?
__device__ __forceinline__ bool finite_pair(uint32_t u) {
  const float2 v = bits_float2(u);
  return fabsf(v.x) + fabsf(v.y) <= 131008.f;
}

__device__ __forceinline__ void unpack8(const uint4& u, float* f, const __half*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = bits_float2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ void unpack8(const uint4& u, float* f, const __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f);
template <>
__device__ __forceinline__ uint4 pack8<__half>(const float* f) {
  return make_uint4(half2_bits(f[0], f[1]), half2_bits(f[2], f[3]), half2_bits(f[4], f[5]), half2_bits(f[6], f[7]));
}
template <>
__device__ __forceinline__ uint4 pack8<__nv_bfloat16>(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int HD, typename T>
__device__ __forceinline__ void kv4_write8(const Kv4AttnParams& p, int b, int j, int col, int d, const float* v) {
  T* dst = static_cast<T*>(p.out) +
           ((static_cast<long long>(b) * p.n + col / p.G) * p.H + j * p.G + col % p.G) * HD + d;
  *reinterpret_cast<uint4*>(dst) = pack8<T>(v);
}

// The attention of many columns a KV head (kv4_chunk.cu).
int launch_kv4_chunk(const agxc_ctx* ctx, const Kv4AttnParams& p, int hd, bool bf16, cudaStream_t s);

}  // namespace agxc
