// Helpers of the kernels that work on rows of values (norms, losses): loads and stores of 16 bytes
// at any address in every element type, and sums and maxima over the lanes that share a row.
#pragma once

#include "ow_device.h"

namespace ow {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Element types as rows hold them: kVec values are 16 bytes.
template <class Ty>
struct Row {  // BF16, F16
  typedef uint16_t Elem;
  typedef u32x4 Raw;  // a vector as memory holds it
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to_f32(Elem e) { return Ty::to_f32(e); }
  static __device__ __forceinline__ Elem from_f32(float f) { return Ty::from_f32(f); }
  static __device__ __forceinline__ Raw raw(const Elem* p) { return *reinterpret_cast<const u32x4_any*>(p); }
  static __device__ __forceinline__ Raw zero() { return u32x4{0u, 0u, 0u, 0u}; }
  static __device__ __forceinline__ void set(Raw& w, int j, Elem e) { w[j >> 1] |= static_cast<uint32_t>(e) << (16 * (j & 1)); }
  static __device__ __forceinline__ void widen(const Raw& w, float (&v)[kVec]) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = Ty::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
  }
  static __device__ __forceinline__ void load(const Elem* p, float (&v)[kVec]) { widen(raw(p), v); }
  static __device__ __forceinline__ void store(Elem* p, const float (&v)[kVec]) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) w[j] = Ty::pack2(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<u32x4_any*>(p) = w;
  }
};

struct F32;
template <>
struct Row<F32> {
  typedef float Elem;
  typedef f32x4 Raw;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float to_f32(Elem e) { return e; }
  static __device__ __forceinline__ Elem from_f32(float f) { return f; }
  static __device__ __forceinline__ Raw raw(const Elem* p) { return *reinterpret_cast<const f32x4_any*>(p); }
  static __device__ __forceinline__ Raw zero() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ void set(Raw& w, int j, Elem e) { w[j] = e; }
  static __device__ __forceinline__ void widen(const Raw& w, float (&v)[kVec]) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = w[j];
  }
  static __device__ __forceinline__ void load(const Elem* p, float (&v)[kVec]) { widen(raw(p), v); }
  static __device__ __forceinline__ void store(Elem* p, const float (&v)[kVec]) {
    *reinterpret_cast<f32x4_any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  }
};

// Value i of a tensor of a type known at run time (OW_DTYPE_*).
__device__ __forceinline__ float load_any(const void* p, int32_t dtype, int64_t i) {
  if (dtype == OW_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return dtype == OW_DTYPE_BF16 ? BF16::to_f32(u) : F16::to_f32(u);
}
__device__ __forceinline__ void store_any(void* p, int32_t dtype, int64_t i, float v) {
  if (dtype == OW_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = dtype == OW_DTYPE_BF16 ? BF16::from_f32(v) : F16::from_f32(v);
}

// Values i .. i + N - 1 of a tensor of a type known at run time (N = 4 or 8), at any address: the
// type is looked at once, so that the loads are in flight together.
template <int N>
__device__ __forceinline__ void load_any_vec(const void* p, int32_t dtype, int64_t i, float (&v)[N]) {
  if (dtype == OW_DTYPE_F32) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const f32x4 w = *reinterpret_cast<const f32x4_any*>(static_cast<const float*>(p) + i + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * h + j] = w[j];
    }
    return;
  }
  typedef u32x2 __attribute__((aligned(2))) u32x2_any;
  uint32_t w[N / 2];
#pragma unroll
  for (int h = 0; h < N / 4; ++h) {
    const u32x2 u = *reinterpret_cast<const u32x2_any*>(static_cast<const uint16_t*>(p) + i + 4 * h);
    w[2 * h] = u.x, w[2 * h + 1] = u.y;
  }
  if (dtype == OW_DTYPE_BF16) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = BF16::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = F16::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
  }
}

struct AddOp {
  static __device__ __forceinline__ float apply(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float apply(float a, float b) { return fmaxf(a, b); }
};

struct MaxUintOp {
  static __device__ __forceinline__ uint32_t apply(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// Op over aligned groups of T lanes (8, 16, 32 or 64); every lane gets the result.  Mirrors within a row of
// 16 lanes, then gfx950's row and half swaps: of two copies of v, permlane16_swap leaves the even
// rows in one and the odd rows in the other (permlane32_swap: the halves).
template <class Op, int T, class V>
__device__ __forceinline__ V lanes_reduce(V v) {
  static_assert((T == 8 || T == 16 || T == 32 || T == 64) && sizeof(V) == 4, "lanes of a row");
  auto bits = [](V x) { return __builtin_bit_cast(uint32_t, x); };
  auto value = [](uint32_t x) { return __builtin_bit_cast(V, x); };
  auto dpp = [&](V x, auto ctrl) {
    return value(__builtin_amdgcn_update_dpp(0u, bits(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v = Op::apply(v, dpp(v, std::integral_constant<int, 0xb1>{}));   // quad_perm 1,0,3,2
  v = Op::apply(v, dpp(v, std::integral_constant<int, 0x4e>{}));   // quad_perm 2,3,0,1
  v = Op::apply(v, dpp(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  if constexpr (T >= 16) v = Op::apply(v, dpp(v, std::integral_constant<int, 0x140>{}));  // row_mirror
  if constexpr (T >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
    v = Op::apply(value(s[0]), value(s[1]));
  }
  if constexpr (T >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    v = Op::apply(value(s[0]), value(s[1]));
  }
  return v;
}

// N <= kRowSums sums over the T threads that share a row (T > 64: whole waves, which meet in `red`,
// [2][kRowSums * waves of the workgroup]; `turn` picks the half, so that one barrier a call suffices:
// a half is written again only after the barrier of the call between).  Every thread of the workgroup
// calls it.
constexpr int kRowSums = 2;
template <int T, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_reduce<AddOp, (T > 64 ? 64 : T)>(v[i]);
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
    static_assert(N <= kRowSums, "sums of a call");
    float* half = red + turn * kRowSums * waves;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) half[i * waves + wave] = v[i];
    }
    __syncthreads();
    const int first = wave / W * W;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float sum = half[i * waves + first];
#pragma unroll
      for (int w = 1; w < W; ++w) sum += half[i * waves + first + w];
      v[i] = sum;
    }
  }
}

}  // namespace ow
