// 16-byte vectors of fp32 / bf16 elements as floats, and sums over a CTA, for the bandwidth-bound kernels.
#pragma once

#include "common.cuh"

namespace jpb {

template <typename T> struct Vec;  // 16-byte vector of T
template <> struct Vec<float> {
  static constexpr int N = 4;
  float4 raw;
  __device__ __forceinline__ void load(const float* p) { raw = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = raw; }
  __device__ __forceinline__ void to_float(float (&f)[4]) const { f[0] = raw.x; f[1] = raw.y; f[2] = raw.z; f[3] = raw.w; }
  __device__ __forceinline__ void from_float(const float (&f)[4]) { raw = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ __forceinline__ void to_float(float (&f)[8]) const {
    float2 a = unpack_bf16(raw.x), b = unpack_bf16(raw.y), c = unpack_bf16(raw.z), d = unpack_bf16(raw.w);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
  __device__ __forceinline__ void from_float(const float (&f)[8]) {
    raw.x = pack_bf16(f[0], f[1]); raw.y = pack_bf16(f[2], f[3]); raw.z = pack_bf16(f[4], f[5]); raw.w = pack_bf16(f[6], f[7]);
  }
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Pairs of fp32 values: one instruction for both (half the issue slots of a kernel that is bound by them).
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ float lo() const { return __uint_as_float(uint32_t(v)); }
  __device__ __forceinline__ float hi() const { return __uint_as_float(uint32_t(v >> 32)); }
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// 16 bytes from shared memory by its 32-bit address: a pointer that went through a structure is loaded from as a generic one.
__device__ __forceinline__ void lds_vec(Vec<float>& v, uint32_t addr) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.raw.x), "=f"(v.raw.y), "=f"(v.raw.z), "=f"(v.raw.w) : "r"(addr));
}
__device__ __forceinline__ void lds_vec(Vec<__nv_bfloat16>& v, uint32_t addr) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.raw.x), "=r"(v.raw.y), "=r"(v.raw.z), "=r"(v.raw.w) : "r"(addr));
}
// 16 bytes of T as pairs, and back.
__device__ __forceinline__ void to_pairs(const Vec<float>& v, F2 (&f)[2]) {
  f[0] = f2(v.raw.x, v.raw.y);
  f[1] = f2(v.raw.z, v.raw.w);
}
__device__ __forceinline__ void to_pairs(const Vec<__nv_bfloat16>& v, F2 (&f)[4]) {
  const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void from_pairs(Vec<float>& v, const F2 (&f)[2]) { v.raw = make_float4(f[0].lo(), f[0].hi(), f[1].lo(), f[1].hi()); }
__device__ __forceinline__ void from_pairs(Vec<__nv_bfloat16>& v, const F2 (&f)[4]) {
  v.raw = make_uint4(pack_bf16(f[0].lo(), f[0].hi()), pack_bf16(f[1].lo(), f[1].hi()), pack_bf16(f[2].lo(), f[2].hi()),
                     pack_bf16(f[3].lo(), f[3].hi()));
}

// Sum (and optionally a second sum) over a CTA; result broadcast to all threads.
template <int NV>
__device__ __forceinline__ void block_sum(float (&v)[NV], float* scratch /* >= NV*32 floats */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = warp_sum(v[i]);
  __syncthreads();  // scratch may still be read from a previous call
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) scratch[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float x = lane < nwarps ? scratch[i * 32 + lane] : 0.f;
    v[i] = warp_sum(x);
  }
}

}  // namespace jpb
