// One AdamW step over many tensors, with states in 32 or 8 bits, and the norm of their gradients.
//
//   g <- g min(1, max_norm / (norm + 1e-6))             (where the caller gives partial norms)
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: every value of p, g, m and v is read once and every updated one written once (28 bytes
// a parameter in fp32, 16 with 8-bit states).  A launch covers as many tensors as fit in the 4 KB of a
// kernel's arguments, so that no table is uploaded, and a workgroup takes 4,096 values (a chunk) of one of
// them.  Measured: 90 million parameters, fp32 with 8-bit states, in tensors of two launches 278 us (1.44 GB,
// 5.2 TB/s, above a copy's rate at that size); with one vector of a thread in flight after the other 297, with
// four times the threads and one vector each 357.  10.2 million in fp32: 65 us in two launches (4.4 TB/s);
// 1 million: 8.5, the latency of a launch.
//
// Steps are counted on the device, so that a captured step counts and a skipped one does not: one
// counter per chunk, all of a tensor's equal, so that no workgroup waits for another's read before it
// writes.
//
// 8-bit states: 256 consecutive values (one wave's vectors) share an fp32 scale, their largest magnitude
// over 448; a value is held as the nearest e4m3fn number of its ratio to the scale.  The second moment is
// held as its square root: e4m3fn reaches 2^-18 of the block's largest value, so v has 2^-36.  A root
// that is not zero is never held as zero, since m / (0 + eps) would be a step of m / eps.  The nearest code is
// also the format's limit: half a code's step is 3 to 6%, a step moves a root by (1 - b2) / 2 = 0.05%, so what a
// value's root does beside its block's largest one is not followed unless a gradient exceeds some 8 roots (the
// scale follows what the block has in common).  The update
// itself uses the unrounded m and v.  Arithmetic is not contracted to fused multiply-adds: rounding
// after each operation is what the states' definition says, and a value next to a border of two codes
// then falls on the same side everywhere.  The update's quotient (and a root that is not stored, of normal
// numbers) is the hardware's, within a unit in the last place; 1 - b^t is formed as -expm1(t ln b), which keeps its relative
// precision where b^t is near one.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_rows.h"

namespace ow {
namespace {

constexpr int kChunk = OW_ADAMW_CHUNK;  // values of a workgroup
constexpr int kBlock = OW_ADAMW_BLOCK;  // values that share a scale: 64 lanes x 4
constexpr int kThreads = 256;
constexpr int kIters = kChunk / (4 * kThreads);
constexpr int kGroups = 6;              // hyperparameter sets of a launch
constexpr int kArgBytes = 4096 - 64;    // of the tensor and hyperparameter tables
constexpr float kFp8Most = 448.f;
constexpr float kFp8Least = 0x1p-9f;    // the least e4m3fn number above zero
constexpr float kLeastNormal = 0x1p-126f;  // a scale below it is held as zero, and its block of zeros
static_assert(kBlock == 4 * 64 && kIters == 4, "a wave's vector is a block, and its blocks' scales a vector");

struct Hyper {
  const float* lr_device;  // NULL: lr
  float ln_b1, ln_b2, lr, decay, b1, c1, b2, c2, eps, unused;
};

enum { kParam, kGrad, kM, kV, kStep, kMScale, kVScale, kPtrs8, kPtrs32 = kMScale };

// Tensors of a launch: what fits beside the hyperparameters.
template <int PTRS>
constexpr int kTensors = (kArgBytes - kGroups * static_cast<int>(sizeof(Hyper))) / (8 * PTRS + 7);

template <int PTRS>
struct Table {
  static constexpr int N = kTensors<PTRS>;
  void* ptr[PTRS][N];
  Hyper hyper[kGroups];
  uint32_t first[N];  // first chunk
  uint16_t last[N];   // values of the last chunk, less one
  uint8_t group[N];
};

// Tensor of chunk c, the last one whose first chunk is not past c: every lane looks at one of them (a
// bisection would wait for one argument after the other).
template <int N, class T>
__device__ __forceinline__ int tensor_of(const T& t, int count, uint32_t c) {
  const int lane = threadIdx.x & 63;
  int found = 0;
#pragma unroll
  for (int base = 0; base < N; base += 64) {
    const int i = base + lane;
    const bool before = i < count && t.first[i < N ? i : 0] <= c;
    found += __popcll(__ballot(before));
  }
  return __builtin_amdgcn_readfirstlane(found) - 1;
}

typedef uint32_t __attribute__((aligned(1))) u32_any;
typedef u32x2 __attribute__((aligned(2))) u32x2_any2;

// Four consecutive values, or the first n of them (others: 0).
template <class Ty>
__device__ __forceinline__ void load4(const void* base, int64_t i, int n, float (&v)[4]) {
  const typename Row<Ty>::Elem* p = static_cast<const typename Row<Ty>::Elem*>(base) + i;
  if (n >= 4) {
    if constexpr (Row<Ty>::kVec == 4) {
      Row<Ty>::load(p, v);
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2_any2*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = Ty::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = j < n ? Row<Ty>::to_f32(p[j]) : 0.f;
}
template <class Ty>
__device__ __forceinline__ void store4(void* base, int64_t i, int n, const float (&v)[4]) {
  typename Row<Ty>::Elem* p = static_cast<typename Row<Ty>::Elem*>(base) + i;
  if (n >= 4) {
    if constexpr (Row<Ty>::kVec == 4) {
      Row<Ty>::store(p, v);
    } else {
      *reinterpret_cast<u32x2_any2*>(p) = u32x2{Ty::pack2(v[0], v[1]), Ty::pack2(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) p[j] = Row<Ty>::from_f32(v[j]);
}
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t i, int n) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + i;
  if (n >= 4) return *reinterpret_cast<const u32_any*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < n) w |= static_cast<uint32_t>(p[j]) << (8 * j);
  return w;
}
__device__ __forceinline__ void store_codes(void* base, int64_t i, int n, uint32_t w) {
  uint8_t* p = static_cast<uint8_t*>(base) + i;
  if (n >= 4) {
    *reinterpret_cast<u32_any*>(p) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < n) p[j] = static_cast<uint8_t>(w >> (8 * j));
}
__device__ __forceinline__ void decode4(uint32_t w, float scale, float (&v)[4]) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0) * scale;
  v[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 1) * scale;
  v[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 2) * scale;
  v[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 3) * scale;
}
// Codes of four values and the scale of their block (all 64 lanes); ROOT: values from zero up, of which
// none above zero becomes zero.  A ratio exceeds 448 by its rounding at most, which the conversion
// rounds back.  Magnitudes are compared as integers: a NaN is the largest, so that its block's scale and with it
// the block are none.
template <bool ROOT>
__device__ __forceinline__ uint32_t encode4(const float (&v)[4], float& scale) {
#pragma clang fp contract(off)
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t u = ROOT ? __float_as_uint(v[j]) : __float_as_uint(v[j]) & 0x7fffffffu;
    most = u > most ? u : most;
  }
  most = lanes_reduce<MaxUintOp, 64>(most);
  scale = __uint_as_float(most) * (1.f / kFp8Most);
  if (scale < kLeastNormal) scale = 0.f;
  const float inv = scale != 0.f ? 1.f / scale : 0.f;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = v[j] * inv;
    if (ROOT) y[j] = v[j] > 0.f && y[j] < kFp8Least ? kFp8Least : y[j];
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
}

// Sum over a workgroup of WAVES waves; every thread gets it.
template <int WAVES>
__device__ __forceinline__ double workgroup_sum(double sum, double* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) sum += lds[w];
  return sum;
}

template <int PTRS>
struct StepArgs {
  Table<PTRS> t;
  const double* partials;
  float* norm_out;
  double max_norm;
  int32_t n_partials, count;
};

template <class Ty, int BITS, bool MASTER>
constexpr int kPtrsOf = (BITS == 8 ? kPtrs8 : kPtrs32) + (MASTER ? 1 : 0);

template <class Ty, int BITS, bool MASTER>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(StepArgs<kPtrsOf<Ty, BITS, MASTER>> a) {
#pragma clang fp contract(off)
  constexpr int PTRS = kPtrsOf<Ty, BITS, MASTER>;
  __shared__ double lds[kThreads / 64];
  const uint32_t chunk = blockIdx.x;
  const int i = tensor_of<Table<PTRS>::N>(a.t, a.count, chunk);
  const uint32_t local = chunk - a.t.first[i];
  const uint32_t next = i + 1 < a.count ? a.t.first[i + 1] : gridDim.x;
  const int n = chunk + 1 == next ? a.t.last[i] + 1 : kChunk;  // values of this chunk
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t base = static_cast<int64_t>(local) * kChunk;

  // Everything is read before anything is written: a vector's loads do not wait for the stores of the
  // one before it, nor for the counter and the norm.  A wave has four blocks in a row, whose scales are one
  // vector.
  float p[kIters][4], g[kIters][4], m[kIters][4], v[kIters][4];
  uint32_t mw[kIters], vw[kIters];
  float ms[kIters], vs[kIters];
#pragma unroll
  for (int k = 0; k < kIters; ++k) {
    const int at = (wave * kIters + k) * kBlock + 4 * lane;
    const int left = n - at;
    const int64_t idx = base + at;
    if constexpr (MASTER) load4<F32>(a.t.ptr[PTRS - 1][i], idx, left, p[k]);
    else load4<Ty>(a.t.ptr[kParam][i], idx, left, p[k]);
    load4<Ty>(a.t.ptr[kGrad][i], idx, left, g[k]);
    if constexpr (BITS == 8) {
      mw[k] = load_codes(a.t.ptr[kM][i], idx, left);
      vw[k] = load_codes(a.t.ptr[kV][i], idx, left);
    } else {
      load4<F32>(a.t.ptr[kM][i], idx, left, m[k]);
      load4<F32>(a.t.ptr[kV][i], idx, left, v[k]);
    }
  }
  const int64_t block0 = static_cast<int64_t>(local) * (kChunk / kBlock) + wave * kIters;
  const int blocks = (n + kBlock - 1) / kBlock - wave * kIters;  // of this wave, where below kIters
  if constexpr (BITS == 8) {
    load4<F32>(a.t.ptr[kMScale][i], block0, blocks, ms);
    load4<F32>(a.t.ptr[kVScale][i], block0, blocks, vs);
  }

  float coef = 1.f;
  if (a.partials != nullptr) {
    double sum = 0.0;  // in a fixed order, every workgroup alike
    for (int k = threadIdx.x; k < a.n_partials; k += 8 * kThreads) {  // eight loads in flight, not one
      double part[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) part[u] = k + u * kThreads < a.n_partials ? a.partials[k + u * kThreads] : 0.0;
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += part[u];
    }
    const float norm = static_cast<float>(sqrt(workgroup_sum<kThreads / 64>(sum, lds)));
    if (chunk == 0 && threadIdx.x == 0 && a.norm_out != nullptr) *a.norm_out = norm;
    if (!(norm < __builtin_inff())) return;  // the step is skipped
    coef = fminf(static_cast<float>(a.max_norm) / (norm + 1e-6f), 1.f);
  }
  const Hyper& h = a.t.hyper[a.t.group[i]];
  int32_t* counter = static_cast<int32_t*>(a.t.ptr[kStep][i]) + local;
  const int32_t steps = *counter + 1;
  const float t = static_cast<float>(steps);
  const float lr = h.lr_device != nullptr ? *h.lr_device : h.lr;
  const float step = lr / -expm1f(t * h.ln_b1);
  const float unbias = 1.f / sqrtf(-expm1f(t * h.ln_b2));
  const float keep = 1.f - lr * h.decay;
  __syncthreads();  // every thread has read the counter
  if (threadIdx.x == 0) *counter = steps;

#pragma unroll
  for (int k = 0; k < kIters; ++k) {
    if (k >= blocks) break;  // wave-uniform
    const int at = (wave * kIters + k) * kBlock + 4 * lane;
    const int left = n - at;
    const int64_t idx = base + at;
    if constexpr (BITS == 8) {
      decode4(mw[k], ms[k], m[k]);
      decode4(vw[k], vs[k], v[k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = v[k][j] * v[k][j];
    }
    float root[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = g[k][j] * coef;
      m[k][j] = m[k][j] * h.b1 + gj * h.c1;
      v[k][j] = v[k][j] * h.b2 + gj * gj * h.c2;
      // A root that is stored is rounded correctly, as m and v are: its code is then the definition's.
      root[j] = BITS == 8 ? sqrtf(v[k][j]) : __builtin_amdgcn_sqrtf(v[k][j]);
    }
    // The hardware's root takes subnormal numbers for zero, which a small eps would not hide.
    if (BITS != 8 && fminf(fminf(v[k][0], v[k][1]), fminf(v[k][2], v[k][3])) < kLeastNormal) {
#pragma unroll
      for (int j = 0; j < 4; ++j) root[j] = sqrtf(v[k][j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      p[k][j] = p[k][j] * keep - step * (m[k][j] * __builtin_amdgcn_rcpf(root[j] * unbias + h.eps));
    if constexpr (MASTER) store4<F32>(a.t.ptr[PTRS - 1][i], idx, left, p[k]);
    store4<Ty>(a.t.ptr[kParam][i], idx, left, p[k]);
    if constexpr (BITS == 8) {
      mw[k] = encode4<false>(m[k], ms[k]);
      vw[k] = encode4<true>(root, vs[k]);
      store_codes(a.t.ptr[kM][i], idx, left, mw[k]);
      store_codes(a.t.ptr[kV][i], idx, left, vw[k]);
    } else {
      store4<F32>(a.t.ptr[kM][i], idx, left, m[k]);
      store4<F32>(a.t.ptr[kV][i], idx, left, v[k]);
    }
  }
  if (BITS == 8 && lane == 0) {
    store4<F32>(a.t.ptr[kMScale][i], block0, blocks, ms);
    store4<F32>(a.t.ptr[kVScale][i], block0, blocks, vs);
  }
}

// Sums of squares of gradients, in fp64 (no square of an fp32 value overflows): one partial a workgroup.
struct NormArgs {
  static constexpr int N = (4096 - 256) / 14;
  const void* grad[N];
  uint32_t first[N];
  uint16_t last[N];
  double* partials;
  uint32_t chunks;
  int32_t count;
};

// A workgroup takes a range of chunks and walks the tensors that they are of, so that it looks a tensor up
// once and has four vectors of 16 bytes a thread in flight.
template <class Ty>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(NormArgs a) {
  typedef Row<Ty> R;
  constexpr int V = R::kVec, U = 4;
  __shared__ double lds[kThreads / 64];
  double sum = 0.0;
  uint32_t chunk = static_cast<uint32_t>(static_cast<uint64_t>(a.chunks) * blockIdx.x / gridDim.x);
  const uint32_t stop = static_cast<uint32_t>(static_cast<uint64_t>(a.chunks) * (blockIdx.x + 1) / gridDim.x);
  int i = chunk < stop ? tensor_of<NormArgs::N>(a, a.count, chunk) : 0;
  for (; chunk < stop; ++i) {
    const uint32_t first = a.first[i], next = i + 1 < a.count ? a.first[i + 1] : a.chunks;
    const int64_t numel = static_cast<int64_t>(next - first - 1) * kChunk + a.last[i] + 1;
    const uint32_t until = next < stop ? next : stop;
    const int64_t limit = static_cast<int64_t>(until - first) * kChunk, end = limit < numel ? limit : numel;
    const typename R::Elem* g = static_cast<const typename R::Elem*>(a.grad[i]);
    auto add = [&](const float (&v)[V]) {
#pragma unroll
      for (int j = 0; j < V; ++j) sum += static_cast<double>(v[j]) * v[j];
    };
    int64_t at = static_cast<int64_t>(chunk - first) * kChunk + threadIdx.x * V;
    for (; at + (U - 1) * kThreads * V + V <= end; at += U * kThreads * V) {
      typename R::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = R::raw(g + at + u * kThreads * V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[V];
        R::widen(raw[u], v);
        add(v);
      }
    }
    for (; at < end; at += kThreads * V) {
      float v[V];
      if (at + V <= end) {
        R::load(g + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = at + j < end ? R::to_f32(g[at + j]) : 0.f;
      }
      add(v);
    }
    chunk = until;
  }
  sum = workgroup_sum<kThreads / 64>(sum, lds);
  if (threadIdx.x == 0) a.partials[blockIdx.x] = sum;
}

int64_t chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

int check_tensors(const OwAdamwTensor* t, int32_t count, int32_t dtype) {
  OW_CHECK_ARG(count >= 0, "negative count %d", count);
  OW_CHECK_SUPPORTED(dtype == OW_DTYPE_F32 || dtype == OW_DTYPE_BF16 || dtype == OW_DTYPE_F16,
                     "adamw: dtype %d; expected f32, bf16 or f16", dtype);
  OW_CHECK_ARG(count == 0 || t != nullptr, "tensor list is NULL");
  for (int32_t i = 0; i < count; ++i) {
    OW_CHECK_ARG(t[i].numel > 0 && t[i].grad != nullptr, "tensor %d: %lld values, gradient %p", i,
                 static_cast<long long>(t[i].numel), t[i].grad);
    OW_CHECK_SUPPORTED(t[i].numel <= (int64_t(1) << 40), "tensor %d: %lld values; at most 2^40 are supported", i,
                       static_cast<long long>(t[i].numel));
  }
  return OW_OK;
}

template <class Ty, int BITS, bool MASTER>
int launch_step(const OwAdamwTensor* t, int32_t count, const OwAdamwGroup* groups, const double* partials,
                int32_t n_partials, double max_norm, float* norm_out, hipStream_t s) {
  constexpr int PTRS = kPtrsOf<Ty, BITS, MASTER>;
  static_assert(sizeof(StepArgs<PTRS>) <= 4096, "kernel arguments");
  int32_t at = 0;
  while (at < count) {
    StepArgs<PTRS> a{};
    a.partials = partials;
    a.n_partials = n_partials;
    a.max_norm = max_norm;
    a.norm_out = at == 0 ? norm_out : nullptr;
    int64_t chunks = 0;
    int64_t of[kGroups];
    int n_groups = 0;
    while (at < count && a.count < Table<PTRS>::N && (a.count == 0 || chunks + chunks_of(t[at].numel) < (int64_t(1) << 31))) {
      const OwAdamwTensor& x = t[at];
      int g = 0;
      while (g < n_groups && of[g] != x.group) ++g;
      if (g == n_groups) {
        if (n_groups == kGroups) break;
        of[n_groups++] = x.group;
        const OwAdamwGroup& y = groups[x.group];
        Hyper& h = a.t.hyper[g];
        h.lr_device = y.lr_device;
        h.ln_b1 = static_cast<float>(log(y.beta1));
        h.ln_b2 = static_cast<float>(log(y.beta2));
        h.lr = static_cast<float>(y.lr);
        h.decay = static_cast<float>(y.weight_decay);
        h.b1 = static_cast<float>(y.beta1);
        h.c1 = static_cast<float>(1.0 - y.beta1);
        h.b2 = static_cast<float>(y.beta2);
        h.c2 = static_cast<float>(1.0 - y.beta2);
        h.eps = static_cast<float>(y.eps);
      }
      const int i = a.count++;
      a.t.ptr[kParam][i] = x.param;
      a.t.ptr[kGrad][i] = const_cast<void*>(x.grad);
      a.t.ptr[kM][i] = x.exp_avg;
      a.t.ptr[kV][i] = x.exp_avg_sq;
      a.t.ptr[kStep][i] = x.step;
      if constexpr (BITS == 8) {
        a.t.ptr[kMScale][i] = x.exp_avg_scale;
        a.t.ptr[kVScale][i] = x.exp_avg_sq_scale;
      }
      if constexpr (MASTER) a.t.ptr[PTRS - 1][i] = x.master;
      a.t.first[i] = static_cast<uint32_t>(chunks);
      a.t.last[i] = static_cast<uint16_t>((x.numel - 1) % kChunk);
      a.t.group[i] = static_cast<uint8_t>(g);
      chunks += chunks_of(x.numel);
      ++at;
    }
    hipLaunchKernelGGL((adamw_kernel<Ty, BITS, MASTER>), dim3(static_cast<unsigned>(chunks)), dim3(kThreads), 0, s, a);
    if (int rc = hip_status(hipGetLastError(), "adamw_kernel launch")) return rc;
  }
  return OW_OK;
}

template <class Ty>
int launch_norm(const OwAdamwTensor* t, int32_t count, double* partials, hipStream_t s) {
  static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");
  for (int32_t at = 0; at < count;) {
    NormArgs a{};
    int64_t chunks = 0;
    while (at < count && a.count < NormArgs::N && (a.count == 0 || chunks + chunks_of(t[at].numel) < (int64_t(1) << 31))) {
      const int i = a.count++;
      a.grad[i] = t[at].grad;
      a.first[i] = static_cast<uint32_t>(chunks);
      a.last[i] = static_cast<uint16_t>((t[at].numel - 1) % kChunk);
      chunks += chunks_of(t[at].numel);
      ++at;
    }
    a.chunks = static_cast<uint32_t>(chunks);
    a.partials = partials;
    partials += OW_GRAD_NORM_PARTIALS;
    hipLaunchKernelGGL((grad_norm_kernel<Ty>), dim3(OW_GRAD_NORM_PARTIALS), dim3(kThreads), 0, s, a);
    if (int rc = hip_status(hipGetLastError(), "grad_norm_kernel launch")) return rc;
  }
  return OW_OK;
}

template <class Ty>
int step_of(const OwAdamwTensor* t, int32_t count, const OwAdamwGroup* groups, int32_t bits, bool master,
            const double* partials, int32_t n_partials, double max_norm, float* norm_out, hipStream_t s) {
  if (bits == 8)
    return master ? launch_step<Ty, 8, true>(t, count, groups, partials, n_partials, max_norm, norm_out, s)
                  : launch_step<Ty, 8, false>(t, count, groups, partials, n_partials, max_norm, norm_out, s);
  return master ? launch_step<Ty, 32, true>(t, count, groups, partials, n_partials, max_norm, norm_out, s)
                : launch_step<Ty, 32, false>(t, count, groups, partials, n_partials, max_norm, norm_out, s);
}

}  // namespace
}  // namespace ow

extern "C" {

int64_t ow_grad_norm_partials(const OwAdamwTensor* tensors, int32_t count) {
  if (tensors == nullptr || count <= 0) return 0;
  int64_t launches = 0;
  for (int32_t at = 0; at < count; ++launches) {
    int64_t chunks = 0;
    int n = 0;
    while (at < count && n < ow::NormArgs::N &&
           (n == 0 || chunks + ow::chunks_of(tensors[at].numel) < (int64_t(1) << 31))) {
      chunks += ow::chunks_of(tensors[at].numel);
      ++n, ++at;
    }
  }
  return launches * OW_GRAD_NORM_PARTIALS;
}

int ow_grad_norm(const OwAdamwTensor* tensors, int32_t count, int32_t dtype, double* partials, int64_t n_partials,
                 void* stream) {
  if (int rc = ow::check_tensors(tensors, count, dtype)) return rc;
  const int64_t need = ow_grad_norm_partials(tensors, count);
  OW_CHECK_ARG(n_partials >= need && (need == 0 || partials != nullptr), "%lld partial sums; %lld are needed",
               static_cast<long long>(n_partials), static_cast<long long>(need));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = dtype == OW_DTYPE_F32    ? ow::launch_norm<ow::F32>(tensors, count, partials, s)
                 : dtype == OW_DTYPE_BF16 ? ow::launch_norm<ow::BF16>(tensors, count, partials, s)
                                          : ow::launch_norm<ow::F16>(tensors, count, partials, s);
  if (rc == OW_OK) ow::clear_error();
  return rc;
}

int ow_adamw_step(const OwAdamwTensor* tensors, int32_t count, const OwAdamwGroup* groups, int32_t n_groups,
                  int32_t dtype, int32_t state_bits, int32_t use_master, const double* partials, int64_t n_partials,
                  double max_norm, float* norm_out, void* stream) {
  if (int rc = ow::check_tensors(tensors, count, dtype)) return rc;
  OW_CHECK_SUPPORTED(state_bits == 8 || state_bits == 32, "adamw: states of %d bits; expected 8 or 32", state_bits);
  OW_CHECK_SUPPORTED(!use_master || dtype != OW_DTYPE_F32, "adamw: master weights are for bf16 and f16 parameters");
  OW_CHECK_ARG(count == 0 || (groups != nullptr && n_groups > 0), "no hyperparameters");
  OW_CHECK_ARG(partials == nullptr || (n_partials > 0 && n_partials < (int64_t(1) << 31) && max_norm > 0.0),
               "clipping: %lld partial sums, largest norm %g", static_cast<long long>(n_partials), max_norm);
  for (int32_t i = 0; i < count; ++i) {
    const OwAdamwTensor& t = tensors[i];
    OW_CHECK_ARG(t.param && t.exp_avg && t.exp_avg_sq && t.step, "tensor %d: a pointer is NULL", i);
    OW_CHECK_ARG(state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale), "tensor %d: 8-bit states need scales", i);
    OW_CHECK_ARG(!use_master || t.master, "tensor %d: no master weights", i);
    OW_CHECK_ARG(t.group >= 0 && t.group < n_groups, "tensor %d: group %lld of %d", i, static_cast<long long>(t.group),
                 n_groups);
  }
  for (int32_t i = 0; i < n_groups && count > 0; ++i) {
    const OwAdamwGroup& g = groups[i];
    OW_CHECK_ARG(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0,
                 "group %d: beta1 %g, beta2 %g, eps %g", i, g.beta1, g.beta2, g.eps);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int32_t n = static_cast<int32_t>(n_partials);
  const bool m = use_master != 0;
  int rc;
  if (dtype == OW_DTYPE_F32) {
    rc = state_bits == 8
             ? ow::launch_step<ow::F32, 8, false>(tensors, count, groups, partials, n, max_norm, norm_out, s)
             : ow::launch_step<ow::F32, 32, false>(tensors, count, groups, partials, n, max_norm, norm_out, s);
  } else if (dtype == OW_DTYPE_BF16) {
    rc = ow::step_of<ow::BF16>(tensors, count, groups, state_bits, m, partials, n, max_norm, norm_out, s);
  } else {
    rc = ow::step_of<ow::F16>(tensors, count, groups, state_bits, m, partials, n, max_norm, norm_out, s);
  }
  if (rc == OW_OK) ow::clear_error();
  return rc;
}

}  // extern "C"
