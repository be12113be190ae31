// What the losses over rows of logits share (cross-entropy, distillation): one pass over a row with the running
// maximum and the sum of exponentials below it, the joining of such numbers, the sum of the rows' losses, and how rows
// are given to threads and workgroups.
//
// Exponentials are powers of two of (x - m) times a factor: log2(e), or less for a softmax at a temperature.  The
// factor is a type, so that the plain one is a constant in the code.
#pragma once

#include "ow_rows.h"

namespace ow {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLong = 4096;  // most logits of a row that a wave takes
constexpr int kShort = 1024; // a wave takes them even where rows are too few to fill the chip with waves
constexpr int kPart = 4096;  // least logits of a part
constexpr int kSumThreads = 1024, kSumLanes = 16;
// More rows than these: workgroups take several, and sum their losses (401,408 rows: the sum over rows by one
// workgroup took 62 us, over workgroups 4).
constexpr int64_t kManyRows = 8192;
constexpr int kFwdVectors = 8, kBwdVectors = 2;  // vectors of a row that a lane takes, where rows are many

struct Log2e {
  __device__ __forceinline__ float value() const { return kLog2e; }
};
struct Log2eOver {  // a temperature
  float of;
  __device__ __forceinline__ float value() const { return of; }
};

// What a workgroup sums where it takes many rows.
struct LossPartial {
  double sum;
  int64_t count;
};

// exp(x - m), 0 where both are -inf (nothing has been seen yet).
template <class F>
__device__ __forceinline__ float exp_below(F f, float x, float m) { return x == m ? 1.f : __builtin_amdgcn_exp2f((x - m) * f.value()); }

template <class F>
__device__ __forceinline__ void join(F f, float& m, float& z, float m2, float z2) {
  const float top = fmaxf(m, m2);
  z = z * exp_below(f, m, top) + z2 * exp_below(f, m2, top);
  m = top;
}

template <int T, class F>
__device__ __forceinline__ void join_lanes(F f, float& m, float& z, float& total) {
  const float top = lanes_reduce<MaxOp, T>(m);
  z = lanes_reduce<AddOp, T>(z * exp_below(f, m, top));
  total = lanes_reduce<AddOp, T>(total);
  m = top;
}

// Numbers of logits begin .. end - 1 of a row that a thread takes, T of them apart by a vector.
template <class F>
struct Numbers {
  F f;
  __device__ __forceinline__ explicit Numbers(F factor) : f(factor) {}
  static constexpr int U = 4;  // vectors of a block
  float m = -__builtin_inff(), z = 0.f, total = 0.f;
  // Vectors u < count (WHOLE: all).
  template <class R, bool WHOLE>
  __device__ __forceinline__ void add(const typename R::Raw (&raw)[U], int count) {
    constexpr int V = R::kVec;
    float v[U][V], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      R::widen(raw[u], v[u]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!WHOLE && u >= count) v[u][j] = -__builtin_inff();
        else total += v[u][j];
        top = fmaxf(top, v[u][j]);
      }
    }
    scale_to(top);
    // Blocks that are not whole, a row's last ones, are left early (200,000 rows of 1,000 bf16: 88.5 us, 92.9 without;
    // whole ones, 4,096 of 21,841, lose 0.3 by it).
    if (!WHOLE && top == -__builtin_inff()) {
      if (total != total) z = total;
      return;
    }
    const float from = WHOLE ? floor_of(top) : top;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) z += __builtin_amdgcn_exp2f((v[u][j] - from) * f.value());
  }
  __device__ __forceinline__ void scale_to(float top) {
    z *= exp_below(f, m, top);
    m = top;
  }
  // What is subtracted from a logit before its exponential is added to z: the maximum, and the lowest finite number
  // while nothing above -inf has been seen: -inf then adds 0, and a NaN, which a maximum passes over, is in z all
  // the same.  (`total` is NaN then, too, and only then: it is a sum of -inf otherwise.)  Every join keeps a NaN z,
  // and the row's loss and gradient get it from there.
  static __device__ __forceinline__ float floor_of(float m) { return fmaxf(m, -3.402823466e38f); }
  template <class R, int T>
  __device__ __forceinline__ void scan(const typename R::Elem* x, int64_t begin, int64_t end, int t) {
    constexpr int V = R::kVec;
    x += begin;
    // Vectors of a long row begin at 16 bytes: the values before and behind them are taken one by one.
    const int64_t n = end - begin;
    int head = 0;
    if (T > 64) {
      head = static_cast<int>((0 - reinterpret_cast<uintptr_t>(x)) % 16 / sizeof(typename R::Elem));
      head = head < n ? head : static_cast<int>(n);
    }
    const typename R::Elem* body = x + head;
    const int64_t vectors = (n - head) / V;
    // Vectors of this thread: t, t + T, ...
    typename R::Raw next[U];
    auto load = [&](int64_t at) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = at + u * T < vectors ? R::raw(body + (at + u * T) * V) : R::zero();
    };
    // A long row's next block is read while one is computed; a wave's short rows have few blocks, and more
    // waves instead (30,000 rows of 300 fp32: 22.3 us with, 18.5 without).
    constexpr bool AHEAD = T > 64;
    if (AHEAD) load(t);
    for (int64_t at = t; at < vectors; at += U * T) {
      if (!AHEAD) load(at);
      typename R::Raw raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
      if (AHEAD) load(at + U * T);
      const int left = static_cast<int>((vectors - at + T - 1) / T);
      if (left >= U) add<R, true>(raw, U);
      else add<R, false>(raw, left);
    }
    // What fills no vector, a value each (fewer than V before and behind: 2 V <= T where both may be).
    const int64_t i = t < head ? t : vectors * V + t;
    if (t < head + V && i < n) {
      const float v = R::to_f32(x[i]);
      total += v;
      const float top = fmaxf(m, v);
      scale_to(top);
      z += __builtin_amdgcn_exp2f((v - floor_of(top)) * f.value());
    }
  }
  template <int T>
  __device__ __forceinline__ void join_row() { join_lanes<T>(f, m, z, total); }
};

// Sum of a workgroup's values, in a fixed order; thread 0 gets it.
template <int WAVES>
__device__ __forceinline__ LossPartial workgroup_sum(double sum, int64_t count) {
  __shared__ LossPartial wave_sums[WAVES];
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    sum += __shfl_xor(sum, k);
    count += __shfl_xor(count, k);
  }
  if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = LossPartial{sum, count};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < WAVES; ++w) sum += wave_sums[w].sum, count += wave_sums[w].count;
  }
  return LossPartial{sum, count};
}

// Rows of logits as the launches see them.
struct LogitRows {
  int64_t rows, classes;
  int32_t dtype;
};

// How rows are cut: `parts` of `len` logits each, enough of them for two workgroups a compute unit.  The
// parts' join costs 0.7 us and 1.3 more for every 64 rows, a row read by one workgroup 0.09 us for every 1,000
// logits; cut against not, forward of bf16 rows with their mean: 8 x 8,192 6.8 / 6.2 us, 8 x 21,841 6.8 / 8.0,
// 64 x 50,000 8.6 / 10.4, 160 x 50,000 11.9 / 10.6, 128 x 200,000 18.8 / 29.2, 300 x 200,000 36.2 / 34.8.
inline void cut(const LogitRows& c, int32_t* parts, int32_t* len) {
  int64_t n = 1;
  if (c.rows < device_cus() && c.classes > 4 * kPart && c.classes > 400 * c.rows) {
    const int64_t want = (2 * static_cast<int64_t>(device_cus()) + c.rows - 1) / c.rows;
    const int64_t most = (c.classes + kPart - 1) / kPart;
    n = want < most ? want : most;
  }
  const int64_t each = ((c.classes + n - 1) / n + 7) / 8 * 8;
  *parts = static_cast<int32_t>((c.classes + each - 1) / each);
  *len = static_cast<int32_t>(each);
}

// Logits of a workgroup of the backward: 4 vectors a thread (8 for fp32), or one (2) where that leaves
// compute units without work (64 x 21,841 bf16: 14.1 us with the forward at 4 vectors, 12.9 at one;
// 4,096 x 21,841: 102 and 117).
inline int backward_part(const LogitRows& c) {
  const int64_t workgroups = c.rows * ((c.classes + 2 * kPart - 1) / (2 * kPart));
  return workgroups < device_cus() ? kPart / 2 : 2 * kPart;
}

// Whether a row belongs to a wave or to a workgroup (700 rows of 4,096 fp32: forward 6.8 and backward 10.8 us
// a wave, 5.5 and 6.1 a workgroup; 5,249 rows of 1,641 bf16: 11.0 and 10.5 a wave, 17.5 and 12.4 a workgroup).
inline bool wave_rows(const LogitRows& c) {
  return c.classes <= kShort || (c.classes <= kLong && c.rows >= 8 * static_cast<int64_t>(device_cus()));
}

// Whether one workgroup takes all rows with their sum, a wave each: a second launch costs more there than the
// rows gain from more workgroups (bf16, one launch against two: 8 x 1,000 4.7 / 5.6 us, 16 x 2,048 5.6 / 6.2,
// 8 x 4,096 5.7 / 6.1, but 16 x 4,096 7.5 / 6.3 and 32 x 1,000 8.2 / 5.8).
inline bool few_rows(const LogitRows& c, bool reduced) {
  return reduced && c.rows <= kSumThreads / 64 && c.classes <= kLong && c.rows * c.classes <= 8 * kLong;
}

// Threads of a row (or of a part of one): a wave or a workgroup, and as few as have `vectors` vectors of it each
// where rows are many, for a wave's instructions serve all its rows (401,408 rows of 100 bf16: forward 271 us
// with a wave a row, 38 with 8 threads; backward 165 and 43).
inline int threads_of(const LogitRows& c, int vectors) {
  if (!wave_rows(c)) return 256;
  const int vec = c.dtype == OW_DTYPE_F32 ? 4 : 8;
  int t = c.rows >= 8 * static_cast<int64_t>(device_cus()) ? 8 : 64;
  while (t < 64 && t * vec * vectors < c.classes) t *= 2;
  return t;
}

// Workgroups of a launch: one for every 256 / t units; where rows are many and short, twice as many as run at
// once, which take the units in turn (200,000 rows of 1,000 bf16, forward: 128, 125, 108 and 103 us with 4, 8, 16
// and 64 a compute unit; 401,408 of 21, with gradient: 61.5 with 16, 67.5 with 64).  Never more threads than a
// launch may have.
inline unsigned workgroups(const LogitRows& c, int64_t units, int t) {
  const int64_t groups = (units + 256 / t - 1) / (256 / t);
  const int64_t most = c.rows > kManyRows && t <= 64 ? 16 * static_cast<int64_t>(device_cus()) : int64_t(1) << 23;
  return static_cast<unsigned>(groups < most ? groups : most);
}

// A forward's launch: its kernel's threads of a row, its workgroups, and whether those sum the losses.
struct LogitPlan {
  int32_t n_parts, part_len, t;
  unsigned groups;
  bool sums;
  size_t workspace;
};
inline LogitPlan plan_of(const LogitRows& c, bool reduced) {
  LogitPlan p;
  cut(c, &p.n_parts, &p.part_len);
  p.t = threads_of(c, kFwdVectors);
  p.groups = workgroups(c, c.rows * p.n_parts, p.t);
  p.sums = c.rows > kManyRows && reduced;
  p.workspace = p.n_parts > 1 ? static_cast<size_t>(c.rows) * p.n_parts * 3 * sizeof(float)
                : p.sums      ? p.groups * sizeof(LossPartial)
                              : 0;
  return p;
}

}  // namespace ow
