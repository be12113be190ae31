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

// Op over aligned groups of T lanes (a power of two up to 64); every lane gets the result.  Mirrors within a row of
// 16 lanes, then gfx950's row and half swaps: of two copies of v, permlane16_swap leaves the even
// rows in one and the odd rows in the other (permlane32_swap: the halves).
template <class Op, int T, class V>
__device__ __forceinline__ V lanes_reduce(V v) {
  static_assert(T >= 1 && T <= 64 && (T & (T - 1)) == 0 && sizeof(V) == 4, "lanes of a row");
  auto bits = [](V x) { return __builtin_bit_cast(uint32_t, x); };
  auto value = [](uint32_t x) { return __builtin_bit_cast(V, x); };
  auto dpp = [&](V x, auto ctrl) {
    return value(__builtin_amdgcn_update_dpp(0u, bits(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  if constexpr (T >= 2) v = Op::apply(v, dpp(v, std::integral_constant<int, 0xb1>{}));   // quad_perm 1,0,3,2
  if constexpr (T >= 4) v = Op::apply(v, dpp(v, std::integral_constant<int, 0x4e>{}));   // quad_perm 2,3,0,1
  if constexpr (T >= 8) v = Op::apply(v, dpp(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
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
constexpr int kRowSums = 3;
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

// ---------------------------------------------------------------------------------------
// Rows that stay in registers: T threads a row, K vectors each

template <int T>
constexpr int kThreads = T > 256 ? T : 256;

// Which channels a thread holds.
template <class R, int T, int K, bool RAGGED>
struct Place {
  static constexpr int V = R::kVec;
  int col[K];  // first channel; -1: none
  int dup[K];  // values at its start that another lane counts
  int n;       // values of a vector (less than V only for rows shorter than a vector)
  __device__ __forceinline__ Place(int t, int c) {
    n = RAGGED && c < V ? c : V;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int want = V * (t + T * k);
      col[k] = want < c ? want : -1;
      dup[k] = 0;
      if (RAGGED && want < c && want + V > c) {
        col[k] = c < V ? 0 : c - V;
        dup[k] = want - col[k];
      }
    }
  }
  // Whether a value counts in sums over the row.
  __device__ __forceinline__ bool counts(int k, int j) const { return col[k] >= 0 && j >= dup[k] && j < n; }
  __device__ __forceinline__ typename R::Raw load(const typename R::Elem* row, int k, bool valid) const {
    if (!valid || col[k] < 0) return R::zero();
    if (RAGGED && n < V) {
      typename R::Raw w = R::zero();
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) R::set(w, j, row[j]);
      return w;
    }
    return R::raw(row + col[k]);
  }
  __device__ __forceinline__ void store(typename R::Elem* row, int k, bool valid, const float (&v)[V]) const {
    if (!valid || col[k] < 0) return;
    if (RAGGED && n < V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) row[j] = R::from_f32(v[j]);
    } else {
      R::store(row + col[k], v);
    }
  }
  // A vector of channels of a weight, `absent` where there is no weight.
  __device__ __forceinline__ void weight(const void* p, int32_t dtype, int64_t base, int k, float absent,
                                         float (&v)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = absent;
    if (p == nullptr || col[k] < 0) return;
    if (RAGGED && n < V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) v[j] = load_any(p, dtype, base + j);
    } else {
      load_any_vec<V>(p, dtype, base + col[k], v);
    }
  }
};

// A value as it enters its row's sums, 0 where another lane counts it (whole vectors need no mask).  Chosen, not
// multiplied by 0 or 1: 0 times an infinity would make the whole row NaN.
template <bool RAGGED>
__device__ __forceinline__ float counted(float a, bool counts) { return !RAGGED || counts ? a : 0.f; }

}  // namespace ow
