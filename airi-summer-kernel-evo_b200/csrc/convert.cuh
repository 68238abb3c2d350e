// Loads and stores of four neighbouring elements of any element type of the C ABI, as f32.
// Plain (coherent) accesses: operators that may run in place use them.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b2f {

// Four elements as they lie in memory, for loads that are issued long before their use.
template <int DT>
struct Raw4 {
  uint2 v;
};
template <>
struct Raw4<kF32> {
  float4 v;
};
template <>
struct Raw4<kE4M3> {
  uint32_t v;
};

template <int DT>
__device__ __forceinline__ Raw4<DT> load_raw4(const char* base, long long off) {
  constexpr int kBytes = DT == kF32 ? 4 : DT == kE4M3 ? 1 : 2;
  return *reinterpret_cast<const Raw4<DT>*>(base + off * kBytes);
}

template <int DT>
__device__ __forceinline__ void unpack4(const Raw4<DT>& r, float* x) {
  if constexpr (DT == kF32) {
    x[0] = r.v.x; x[1] = r.v.y; x[2] = r.v.z; x[3] = r.v.w;
  } else if constexpr (DT == kE4M3) {
    const float2 a = e4m3x2_to_f32x2(uint16_t(r.v)), b = e4m3x2_to_f32x2(uint16_t(r.v >> 16));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  } else {
    const float2 a = DT == kBF16 ? unpack_bf16x2(r.v.x) : unpack_f16x2(r.v.x);
    const float2 b = DT == kBF16 ? unpack_bf16x2(r.v.y) : unpack_f16x2(r.v.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
}

template <int DT>
__device__ __forceinline__ void load4(const char* base, long long off, float* x) {
  unpack4<DT>(load_raw4<DT>(base, off), x);
}

// Sixteen elements (16-byte aligned) as they lie in memory.
template <int DT>
struct Raw16 {
  static constexpr int kVecs = DT == kF32 ? 4 : DT == kE4M3 ? 1 : 2;
  uint4 v[kVecs];
};

template <int DT>
__device__ __forceinline__ Raw16<DT> load_raw16(const char* base, long long off) {
  Raw16<DT> r;
  const uint4* p = reinterpret_cast<const uint4*>(base + off * Raw16<DT>::kVecs);
#pragma unroll
  for (int i = 0; i < Raw16<DT>::kVecs; ++i) r.v[i] = p[i];
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack16(const Raw16<DT>& r, float* x) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    Raw4<DT> q;
    if constexpr (DT == kF32)
      q.v = make_float4(__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]), __uint_as_float(w[4 * i + 2]),
                        __uint_as_float(w[4 * i + 3]));
    else if constexpr (DT == kE4M3)
      q.v = w[i];
    else
      q.v = make_uint2(w[2 * i], w[2 * i + 1]);
    unpack4<DT>(q, x + 4 * i);
  }
}

// Sixteen elements to f32, bf16 or f16, 16-byte aligned.
template <int DT>
__device__ __forceinline__ void store16(char* base, long long off, const float* x) {
  if constexpr (DT == kF32) {
    float4* p = reinterpret_cast<float4*>(base + off * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
    uint4* p = reinterpret_cast<uint4*>(base + off * 2);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i] = DT == kBF16 ? pack_bf16x2(x[2 * i], x[2 * i + 1]) : pack_f16x2(x[2 * i], x[2 * i + 1]);
    p[0] = make_uint4(w[0], w[1], w[2], w[3]);
    p[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Round-to-nearest-even; e4m3 saturates.
template <int DT>
__device__ __forceinline__ void store4(char* base, long long off, const float* x) {
  if (DT == kF32) {
    *reinterpret_cast<float4*>(base + off * 4) = make_float4(x[0], x[1], x[2], x[3]);
  } else if (DT == kE4M3) {
    *reinterpret_cast<uint32_t*>(base + off) =
        uint32_t(f32x2_to_e4m3x2(x[0], x[1])) | (uint32_t(f32x2_to_e4m3x2(x[2], x[3])) << 16);
  } else {
    uint2 v;
    v.x = DT == kBF16 ? pack_bf16x2(x[0], x[1]) : pack_f16x2(x[0], x[1]);
    v.y = DT == kBF16 ? pack_bf16x2(x[2], x[3]) : pack_f16x2(x[2], x[3]);
    *reinterpret_cast<uint2*>(base + off * 2) = v;
  }
}

// Eight e2m1 codes (a byte holds two, the first in its low nibble) as four f16 pairs: exact.
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t w, uint32_t (&f)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3])
      : "r"(w));
}

}  // namespace b2f
