// Softmax cross-entropy of rows of logits with its gradient: one label a row or two weighted ones (the
// labels of a mixed image), label smoothing, rows that are left out.
//
//   m, z = max_k x_k, sum_k exp(x_k - m)
//   loss = (1 - s) (l (m - x_a) + (1 - l) (m - x_b) + ln z) + s (m - mean_k x_k + ln z)   (one label: l = 1)
//   dx_k = w (exp(x_k - m) / z - (1 - s) (l [k = a] + (1 - l) [k = b]) - s / K)
//
// with w the upstream gradient, divided by the number of counted rows for their mean, and 0 for rows
// left out.  Forward and backward read the logits once each; they are bound by memory where there are many
// and by the launches where there are few.  A thread of the forward keeps a running maximum, the sum of
// exponentials below it and the sum of the logits, four vectors at a time, so a row of any length is one
// pass; a row belongs to a wave, or to a workgroup where it is long, and where rows are too few to fill the
// chip each is cut into parts whose numbers the second kernel joins.  That kernel also sums the rows' losses,
// in a fixed order.  The backward needs m and z of a row alone, so it is cut into workgroups at will.  m and
// z are kept apart: x - m has the rounding of the difference, x - (m + ln z) would have that of x.
// Exponentials, sums and losses are fp32 (the sum of losses fp64); the gradient is rounded once.
//
// Measured: 4,096 x 21,841 bf16 forward 54 us (3.3 TB/s; 47.5 us where every row starts at 16 bytes, and
// 44.4 for the read alone), backward 61 us (5.9 TB/s); 1,024 x 1,000 fp32 4.9 + 4.0 (the sum) and 5.0 us;
// 8 x 1,000 bf16 4.4 and 3.3 us, where a call costs its caller 48 us.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_rows.h"

namespace ow {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLong = 4096;  // most logits of a row that a wave takes
constexpr int kShort = 1024; // a wave takes them even where rows are too few to fill the chip with waves
constexpr int kPart = 4096;  // least logits of a part
constexpr int kSumThreads = 1024, kSumLanes = 16;

struct XentArgs {
  OwCrossEntropy c;
  float* parts;  // [rows][n_parts][3]: m, z, sum of logits
  float* stats;  // [rows][2]: m, 1 / z
  float* losses; // [rows], 0 for rows left out
  float* loss;   // [1] their sum or mean; NULL: the losses are the result
  float* weight; // [1] a row's weight in it
  int32_t n_parts, part_len;  // part_len: whole vectors
};

// exp(x - m), 0 where both are -inf (nothing has been seen yet).
__device__ __forceinline__ float exp_below(float x, float m) { return x == m ? 1.f : __builtin_amdgcn_exp2f((x - m) * kLog2e); }

__device__ __forceinline__ void join(float& m, float& z, float m2, float z2) {
  const float top = fmaxf(m, m2);
  z = z * exp_below(m, top) + z2 * exp_below(m2, top);
  m = top;
}

template <int T>
__device__ __forceinline__ void join_lanes(float& m, float& z, float& total) {
  const float top = lanes_reduce<MaxOp, T>(m);
  z = lanes_reduce<AddOp, T>(z * exp_below(m, top));
  total = lanes_reduce<AddOp, T>(total);
  m = top;
}

// A row's labels and their logits, which a row's kernel asks for before it reads the row.
struct Labels {
  float l, x_a, x_b;
  bool counted, known;
  __device__ __forceinline__ Labels() {}
  __device__ __forceinline__ Labels(const XentArgs& a, int64_t row) {
    const int64_t la = a.c.target[row], k = a.c.classes, off = row * a.c.row_stride;
    l = a.c.target_b == nullptr ? 1.f : a.c.mix != nullptr ? a.c.mix[row] : a.c.mix_value;
    const int64_t lb = a.c.target_b != nullptr && l != 1.f ? a.c.target_b[row] : la;
    counted = la != a.c.ignore_index;
    known = la >= 0 && la < k && lb >= 0 && lb < k;
    x_a = known ? load_any(a.c.logits, a.c.dtype, off + la) : 0.f;
    x_b = known ? load_any(a.c.logits, a.c.dtype, off + lb) : 0.f;
  }
};

// Writes a row's statistics and loss.
__device__ __forceinline__ void finish_row(const XentArgs& a, int64_t row, const Labels& y, float m, float z, float total) {
  a.stats[2 * row] = m;
  a.stats[2 * row + 1] = 1.f / z;
  float loss = 0.f;
  if (y.counted) {
    const float ln_z = logf(z), s = a.c.smoothing;
    if (s != 1.f) {  // a term of weight zero is left out, whatever its logit
      float picked = 0.f;
      if (y.l != 0.f) picked += y.l * (m - y.x_a);
      if (y.l != 1.f) picked += (1.f - y.l) * (m - y.x_b);
      loss = (1.f - s) * (picked + ln_z);
    }
    if (s != 0.f) loss += s * (m - total / static_cast<float>(a.c.classes) + ln_z);
    if (!y.known) loss = __builtin_nanf("");  // no such class
  }
  a.losses[row] = loss;
}

// Numbers of logits begin .. end - 1 of a row that a thread takes, T of them apart by a vector.
struct Numbers {
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
    if (top == -__builtin_inff()) return;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) z += __builtin_amdgcn_exp2f((v[u][j] - top) * kLog2e);
  }
  __device__ __forceinline__ void scale_to(float top) {
    z *= exp_below(m, top);
    m = top;
  }
  template <class R, int T>
  __device__ __forceinline__ void scan(const typename R::Elem* x, int64_t begin, int64_t end, int t) {
    constexpr int V = R::kVec;
    const int64_t vectors = (end - begin) / V;
    x += begin;
    // Vectors of this thread: t, t + T, ...
    typename R::Raw next[U];
    auto load = [&](int64_t at) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = at + u * T < vectors ? R::raw(x + (at + u * T) * V) : R::zero();
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
    // What fills no vector, a value each.
    const int64_t i = vectors * V + t;
    if (t < V && begin + i < end) {
      const float v = R::to_f32(x[i]);
      total += v;
      const float top = fmaxf(m, v);
      scale_to(top);
      if (top != -__builtin_inff()) z += __builtin_amdgcn_exp2f((v - top) * kLog2e);
    }
  }
  __device__ __forceinline__ void join_wave() { join_lanes<64>(m, z, total); }
};

// T threads a (row, part).
template <class Ty, int T>
__global__ void __launch_bounds__(256) xent_fwd_kernel(XentArgs a) {
  typedef Row<Ty> R;
  constexpr int UNITS = 256 / T;
  const int t = threadIdx.x % T;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * UNITS + threadIdx.x / T;
  const int64_t row = unit / a.n_parts;
  const int part = static_cast<int>(unit % a.n_parts);
  const bool valid = row < a.c.rows;  // uniform over a unit
  Labels y;
  if (valid && t == 0 && a.n_parts == 1) y = Labels(a, row);
  Numbers s;
  if (valid) {
    const int64_t begin = static_cast<int64_t>(part) * a.part_len, stop = begin + a.part_len;
    s.scan<R, T>(static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride, begin,
                 stop < a.c.classes ? stop : a.c.classes, t);
  }
  s.join_wave();
  if constexpr (T == 256) {
    __shared__ float lds[3][4];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[0][wave] = s.m, lds[1][wave] = s.z, lds[2][wave] = s.total;
    __syncthreads();
    s.m = lds[0][0], s.z = lds[1][0], s.total = lds[2][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      join(s.m, s.z, lds[0][w], lds[1][w]);
      s.total += lds[2][w];
    }
  }
  if (t != 0 || !valid) return;
  if (a.n_parts == 1) {
    finish_row(a, row, y, s.m, s.z, s.total);
  } else {
    float* p = a.parts + unit * 3;
    p[0] = s.m, p[1] = s.z, p[2] = s.total;
  }
}

// The rows' losses, which this workgroup's threads see, as their sum or mean.
__device__ __forceinline__ void sum_rows(const XentArgs& a) {
  __shared__ double sums[kSumThreads / 64];
  __shared__ int64_t counts[kSumThreads / 64];
  double sum = 0.0;
  int64_t count = 0;
#pragma unroll 4
  for (int64_t row = threadIdx.x; row < a.c.rows; row += kSumThreads) {
    sum += a.losses[row];
    count += a.c.target[row] != a.c.ignore_index;
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    sum += __shfl_xor(sum, k);
    count += __shfl_xor(count, k);
  }
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum, counts[threadIdx.x >> 6] = count;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSumThreads / 64; ++w) sum += sums[w], count += counts[w];
    const double weight = a.c.reduction == OW_REDUCE_MEAN ? 1.0 / static_cast<double>(count) : 1.0;
    *a.loss = static_cast<float>(count ? sum * weight : a.c.reduction == OW_REDUCE_MEAN ? __builtin_nan("") : 0.0);
    *a.weight = static_cast<float>(weight);
  }
}

// Few short rows and their sum in one launch: one workgroup, a wave a row.
template <class Ty>
__global__ void __launch_bounds__(kSumThreads) xent_few_kernel(XentArgs a) {
  typedef Row<Ty> R;
  const int lane = threadIdx.x & 63;
  const int64_t row = threadIdx.x >> 6;
  if (row < a.c.rows) {
    Labels y;
    if (lane == 0) y = Labels(a, row);
    Numbers s;
    s.scan<R, 64>(static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride, 0, a.c.classes, lane);
    s.join_wave();
    if (lane == 0) finish_row(a, row, y, s.m, s.z, s.total);
  }
  __syncthreads();
  sum_rows(a);
}

// Joins the parts of rows, 16 lanes a row (n_parts > 1), and sums the losses (one workgroup then).
__global__ void __launch_bounds__(kSumThreads) xent_sum_kernel(XentArgs a) {
  constexpr int ROWS = kSumThreads / kSumLanes;
  if (a.n_parts > 1) {
    const int lane = threadIdx.x % kSumLanes;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.c.rows; base += static_cast<int64_t>(gridDim.x) * ROWS) {
      const int64_t row = base + threadIdx.x / kSumLanes;
      float m = -__builtin_inff(), z = 0.f, total = 0.f;
      Labels y;
      if (row < a.c.rows) {
        if (lane == 0) y = Labels(a, row);
        const float* p = a.parts + row * a.n_parts * 3;
        for (int i = lane; i < a.n_parts; i += kSumLanes) {
          join(m, z, p[3 * i], p[3 * i + 1]);
          total += p[3 * i + 2];
        }
      }
      join_lanes<kSumLanes>(m, z, total);
      if (lane == 0 && row < a.c.rows) finish_row(a, row, y, m, z, total);
    }
    __syncthreads();  // the losses of this workgroup's rows, which are all rows where they are summed
  }
  if (a.loss != nullptr) sum_rows(a);
}

struct XentBwdArgs {
  OwCrossEntropy c;
  const float* stats;
  const float* weight;    // a row's weight; NULL: 1
  const float* upstream;  // [1], or [rows] without reduction
  void* grad;             // [rows][classes]
  int32_t n_parts, part_len;
};

template <class Ty, int T>
__global__ void __launch_bounds__(256) xent_bwd_kernel(XentBwdArgs a) {
  typedef Row<Ty> R;
  constexpr int V = R::kVec, UNITS = 256 / T;
  const int t = threadIdx.x % T;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * UNITS + threadIdx.x / T;
  const int64_t row = unit / a.n_parts;
  if (row >= a.c.rows) return;
  const int64_t k = a.c.classes, la = a.c.target[row];
  const bool counted = la != a.c.ignore_index;
  const typename R::Elem* x = static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride;
  typename R::Elem* out = static_cast<typename R::Elem*>(a.grad) + row * k;
  const float l = a.c.target_b == nullptr ? 1.f : a.c.mix != nullptr ? a.c.mix[row] : a.c.mix_value;
  const int64_t lb = a.c.target_b != nullptr && l != 1.f ? a.c.target_b[row] : la;
  float w = a.upstream[a.c.reduction == OW_REDUCE_NONE ? row : 0];
  if (a.weight != nullptr) w *= *a.weight;
  if (la < 0 || la >= k || lb < 0 || lb >= k) w = __builtin_nanf("");  // no such class
  const float m = a.stats[2 * row], p = w * a.stats[2 * row + 1];
  const float flat = w * (a.c.smoothing / static_cast<float>(k));
  const float hit_a = w * ((1.f - a.c.smoothing) * l), hit_b = w * ((1.f - a.c.smoothing) * (1.f - l));
  const int64_t begin = unit % a.n_parts * a.part_len, stop = begin + a.part_len, end = stop < k ? stop : k;
  for (int64_t i = begin + t * V; i < end; i += T * V) {
    float v[V];
    const int n = end - i < V ? static_cast<int>(end - i) : V;
    if (!counted) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.f;
    } else {
      if (n == V) {
        R::load(x + i, v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < n ? R::to_f32(x[i + j]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = p * __builtin_amdgcn_exp2f((v[j] - m) * kLog2e) - flat;
      if (static_cast<uint64_t>(la - i) < V || static_cast<uint64_t>(lb - i) < V) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (i + j == la) v[j] -= hit_a;
          if (i + j == lb && l != 1.f) v[j] -= hit_b;
        }
      }
    }
    if (n == V) {
      R::store(out + i, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) out[i + j] = R::from_f32(v[j]);
    }
  }
}

// How rows are cut: `parts` of `len` logits each, enough of them for two workgroups a compute unit.  The
// parts' join costs 0.7 us and 1.3 more for every 64 rows, a row read by one workgroup 0.09 us for every 1,000
// logits; cut against not, forward of bf16 rows with their mean: 8 x 8,192 6.8 / 6.2 us, 8 x 21,841 6.8 / 8.0,
// 64 x 50,000 8.6 / 10.4, 160 x 50,000 11.9 / 10.6, 128 x 200,000 18.8 / 29.2, 300 x 200,000 36.2 / 34.8.
void cut(const OwCrossEntropy& c, int32_t* parts, int32_t* len) {
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
int backward_part(const OwCrossEntropy& c) {
  const int64_t workgroups = c.rows * ((c.classes + 2 * kPart - 1) / (2 * kPart));
  return workgroups < device_cus() ? kPart / 2 : 2 * kPart;
}

// Whether a row belongs to a wave or to a workgroup (700 rows of 4,096 fp32: forward 6.8 and backward 10.8 us
// a wave, 5.5 and 6.1 a workgroup; 5,249 rows of 1,641 bf16: 11.0 and 10.5 a wave, 17.5 and 12.4 a workgroup).
bool wave_rows(const OwCrossEntropy& c) {
  return c.classes <= kShort || (c.classes <= kLong && c.rows >= 8 * static_cast<int64_t>(device_cus()));
}

int check(const OwCrossEntropy* c) {
  OW_CHECK_ARG(c != nullptr, "cross-entropy descriptor is NULL");
  OW_CHECK_SUPPORTED(c->dtype == OW_DTYPE_F32 || c->dtype == OW_DTYPE_BF16 || c->dtype == OW_DTYPE_F16,
                     "cross-entropy: dtype %d; expected f32, bf16 or f16", c->dtype);
  OW_CHECK_ARG(c->reduction == OW_REDUCE_NONE || c->reduction == OW_REDUCE_SUM || c->reduction == OW_REDUCE_MEAN,
               "unknown reduction %d", c->reduction);
  OW_CHECK_ARG(c->rows >= 0 && c->classes >= 1, "%lld rows of %lld classes", static_cast<long long>(c->rows),
               static_cast<long long>(c->classes));
  OW_CHECK_SUPPORTED(c->rows < (int64_t(1) << 31) && c->classes < (int64_t(1) << 30),
                     "%lld rows of %lld classes; fewer than 2^31 and 2^30 are supported",
                     static_cast<long long>(c->rows), static_cast<long long>(c->classes));
  OW_CHECK_ARG(c->rows == 0 || (c->logits != nullptr && c->target != nullptr), "logits or target is NULL");
  OW_CHECK_ARG(c->smoothing >= 0.f && c->smoothing <= 1.f, "label smoothing %g is not in [0, 1]", c->smoothing);
  return OW_OK;
}

// Whether one workgroup takes all rows with their sum, a wave each: a second launch costs more there than the
// rows gain from more workgroups (bf16, one launch against two: 8 x 1,000 4.7 / 5.6 us, 16 x 2,048 5.6 / 6.2,
// 8 x 4,096 5.7 / 6.1, but 16 x 4,096 7.5 / 6.3 and 32 x 1,000 8.2 / 5.8).
bool few_rows(const XentArgs& a) {
  return a.loss != nullptr && a.c.rows <= kSumThreads / 64 && a.c.classes <= kLong && a.c.rows * a.c.classes <= 8 * kLong;
}

template <class Ty>
void launch_fwd(const XentArgs& a, hipStream_t s) {
  const int64_t units = a.c.rows * a.n_parts;
  if (few_rows(a))
    hipLaunchKernelGGL((xent_few_kernel<Ty>), dim3(1), dim3(kSumThreads), 0, s, a);
  else if (wave_rows(a.c))
    hipLaunchKernelGGL((xent_fwd_kernel<Ty, 64>), dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((xent_fwd_kernel<Ty, 256>), dim3(static_cast<unsigned>(units)), dim3(256), 0, s, a);
}

template <class Ty>
void launch_bwd(const XentBwdArgs& a, hipStream_t s) {
  const int64_t units = a.c.rows * a.n_parts;
  if (wave_rows(a.c))
    hipLaunchKernelGGL((xent_bwd_kernel<Ty, 64>), dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((xent_bwd_kernel<Ty, 256>), dim3(static_cast<unsigned>(units)), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace ow

extern "C" {

size_t ow_cross_entropy_workspace(const OwCrossEntropy* ce) {
  if (ce == nullptr || ce->rows <= 0 || ce->classes <= 0) return 0;
  int32_t parts = 0, len = 0;
  ow::cut(*ce, &parts, &len);
  return parts > 1 ? static_cast<size_t>(ce->rows) * parts * 3 * sizeof(float) : 0;
}

int ow_cross_entropy_fwd(const OwCrossEntropy* ce, float* stats, float* losses, float* loss, float* weight, void* workspace,
                         size_t workspace_bytes, void* stream) {
  if (int rc = ow::check(ce)) return rc;
  const bool reduced = ce->reduction != OW_REDUCE_NONE;
  OW_CHECK_ARG(ce->rows == 0 || (stats != nullptr && losses != nullptr), "stats or losses is NULL");
  OW_CHECK_ARG(!reduced || (loss != nullptr && weight != nullptr), "loss or weight is NULL");
  if (ce->rows == 0 && !reduced) {
    ow::clear_error();
    return OW_OK;
  }
  ow::XentArgs a{};
  a.c = *ce;
  a.stats = stats;
  a.losses = losses;
  a.loss = reduced ? loss : nullptr;
  a.weight = weight;
  a.n_parts = 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ce->rows > 0) {
    ow::cut(*ce, &a.n_parts, &a.part_len);
    const size_t need = ow_cross_entropy_workspace(ce);
    OW_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                               reinterpret_cast<uintptr_t>(workspace) % 4 == 0),
                 "workspace of %zu bytes; %zu are needed", workspace_bytes, need);
    OW_CHECK_SUPPORTED(ce->rows * a.n_parts < (int64_t(1) << 31), "too many rows");
    a.parts = static_cast<float*>(workspace);
    if (ce->dtype == OW_DTYPE_F32) ow::launch_fwd<ow::F32>(a, s);
    else if (ce->dtype == OW_DTYPE_BF16) ow::launch_fwd<ow::BF16>(a, s);
    else ow::launch_fwd<ow::F16>(a, s);
    if (int rc = ow::hip_status(hipGetLastError(), "xent_fwd_kernel launch")) return rc;
  }
  if ((reduced && (ce->rows == 0 || !ow::few_rows(a))) || a.n_parts > 1) {
    const int64_t rows_at_once = ow::kSumThreads / ow::kSumLanes;
    const int64_t groups = reduced ? 1 : (ce->rows + rows_at_once - 1) / rows_at_once;
    hipLaunchKernelGGL(ow::xent_sum_kernel, dim3(static_cast<unsigned>(groups)), dim3(ow::kSumThreads), 0, s, a);
    if (int rc = ow::hip_status(hipGetLastError(), "xent_sum_kernel launch")) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

int ow_cross_entropy_bwd(const OwCrossEntropy* ce, const float* stats, const float* weight, const float* upstream,
                         void* grad, void* stream) {
  if (int rc = ow::check(ce)) return rc;
  if (ce->rows == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG(stats && upstream && grad, "a pointer is NULL");
  ow::XentBwdArgs a{};
  a.c = *ce;
  a.stats = stats;
  a.weight = weight;
  a.upstream = upstream;
  a.grad = grad;
  a.part_len = ow::wave_rows(*ce) ? static_cast<int32_t>((ce->classes + 7) / 8 * 8) : ow::backward_part(*ce);
  a.n_parts = static_cast<int32_t>((ce->classes + a.part_len - 1) / a.part_len);
  OW_CHECK_SUPPORTED(ce->rows * a.n_parts < (int64_t(1) << 31), "too many rows");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ce->dtype == OW_DTYPE_F32) ow::launch_bwd<ow::F32>(a, s);
  else if (ce->dtype == OW_DTYPE_BF16) ow::launch_bwd<ow::BF16>(a, s);
  else ow::launch_bwd<ow::F16>(a, s);
  if (int rc = ow::hip_status(hipGetLastError(), "xent_bwd_kernel launch")) return rc;
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
