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
// chip each is cut into parts whose numbers the second kernel joins; many short rows share a wave.  The second
// kernel also sums the rows' losses, in a fixed order.  The backward needs m and z of a row alone, so it is cut into workgroups at will.  m and
// z are kept apart: x - m has the rounding of the difference, x - (m + ln z) would have that of x.
// Exponentials, sums and losses are fp32 (the sum of losses fp64); the gradient is rounded once.
//
// Measured: 4,096 x 21,841 bf16 forward 50 us (179 MB; 55 where vectors began with the row, at any address),
// backward 61 us (358 MB, 5.9 TB/s); 1,024 x 1,000 fp32 4.9 + 4.0 (the sum) and 5.0 us; 8 x 1,000 bf16 4.4 and
// 3.3 us, where a call costs its caller 48 us.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_softmax.h"

namespace ow {
namespace {

struct XentArgs {
  OwCrossEntropy c;
  float* parts;  // [rows][n_parts][3]: m, z, sum of logits
  LossPartial* sums; // [n_sums], of the workgroups; NULL: the losses of rows are summed
  float* stats;  // [rows][2]: m, 1 / z
  float* losses; // [rows], 0 for rows left out
  float* loss;   // [1] their sum or mean; NULL: the losses are the result
  float* weight; // [1] a row's weight in it
  int32_t n_parts, part_len;  // part_len: whole vectors
  int32_t n_sums;
};

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

// Writes a row's statistics and loss, which it returns.
__device__ __forceinline__ float finish_row(const XentArgs& a, int64_t row, const Labels& y, float m, float z, float total) {
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
  return loss;
}

// T threads a (row, part); one part a row for T <= 64.
template <class Ty, int T>
__global__ void __launch_bounds__(256) xent_fwd_kernel(XentArgs a) {
  typedef Row<Ty> R;
  constexpr int UNITS = 256 / T;
  const int t = threadIdx.x % T;
  const int64_t units = a.c.rows * a.n_parts;
  double sum = 0.0;
  int64_t count = 0;
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * UNITS; base < units; base += static_cast<int64_t>(gridDim.x) * UNITS) {
    const int64_t unit = base + threadIdx.x / T;
    const bool valid = unit < units;  // uniform over a unit
    int64_t row = unit, begin = 0, end = a.c.classes;
    if (T > 64 && a.n_parts > 1) {
      row = unit / a.n_parts;
      begin = unit % a.n_parts * a.part_len;
      end = begin + a.part_len < end ? begin + a.part_len : end;
    }
    Labels y;
    if (valid && t == 0 && a.n_parts == 1) y = Labels(a, row);
    Numbers<Log2e> s{Log2e()};
    if (valid) s.scan<R, T>(static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride, begin, end, t);
    s.join_row<(T > 64 ? 64 : T)>();
    if constexpr (T == 256) {
      // One half a turn: it is written again only after the barrier of the turn between.
      __shared__ float lds[2][3][4];
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) lds[turn][0][wave] = s.m, lds[turn][1][wave] = s.z, lds[turn][2][wave] = s.total;
      __syncthreads();
      s.m = lds[turn][0][0], s.z = lds[turn][1][0], s.total = lds[turn][2][0];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        join(s.f, s.m, s.z, lds[turn][0][w], lds[turn][1][w]);
        s.total += lds[turn][2][w];
      }
      turn ^= 1;
    }
    if (t == 0 && valid) {
      if (a.n_parts == 1) {
        sum += finish_row(a, row, y, s.m, s.z, s.total);
        count += y.counted;
      } else {
        float* p = a.parts + unit * 3;
        p[0] = s.m, p[1] = s.z, p[2] = s.total;
      }
    }
  }
  if (a.sums != nullptr) {
    const LossPartial all = workgroup_sum<4>(sum, count);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = all;
  }
}

// The loss from what the workgroups summed, or from the rows' losses, which this workgroup's threads see.
__device__ __forceinline__ void sum_rows(const XentArgs& a) {
  double sum = 0.0;
  int64_t count = 0;
  if (a.sums != nullptr) {
    for (int i = threadIdx.x; i < a.n_sums; i += kSumThreads) sum += a.sums[i].sum, count += a.sums[i].count;
  } else {
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.c.rows; row += kSumThreads) {
      sum += a.losses[row];
      count += a.c.target[row] != a.c.ignore_index;
    }
  }
  const LossPartial all = workgroup_sum<kSumThreads / 64>(sum, count);
  if (threadIdx.x == 0) {
    const double weight = a.c.reduction == OW_REDUCE_MEAN ? 1.0 / static_cast<double>(all.count) : 1.0;
    *a.loss = static_cast<float>(all.count ? all.sum * weight : a.c.reduction == OW_REDUCE_MEAN ? __builtin_nan("") : 0.0);
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
    Numbers<Log2e> s{Log2e()};
    s.scan<R, 64>(static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride, 0, a.c.classes, lane);
    s.join_row<64>();
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
          join(Log2e(), m, z, p[3 * i], p[3 * i + 1]);
          total += p[3 * i + 2];
        }
      }
      join_lanes<kSumLanes>(Log2e(), m, z, total);
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

// T threads a (row, part); one part a row for T <= 64.
template <class Ty, int T>
__global__ void __launch_bounds__(256) xent_bwd_kernel(XentBwdArgs a) {
  typedef Row<Ty> R;
  constexpr int V = R::kVec, UNITS = 256 / T;
  const int t = threadIdx.x % T;
  const int64_t k = a.c.classes, units = a.c.rows * a.n_parts;
  const float row_weight = a.weight != nullptr ? *a.weight : 1.f;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * UNITS + threadIdx.x / T; unit < units;
       unit += static_cast<int64_t>(gridDim.x) * UNITS) {
    int64_t row = unit, begin = 0, end = k;
    if (T > 64) {
      row = unit / a.n_parts;
      begin = unit % a.n_parts * a.part_len;
      end = begin + a.part_len < k ? begin + a.part_len : k;
    }
    const int64_t la = a.c.target[row];
    const bool counted = la != a.c.ignore_index;
    const typename R::Elem* x = static_cast<const typename R::Elem*>(a.c.logits) + row * a.c.row_stride;
    typename R::Elem* out = static_cast<typename R::Elem*>(a.grad) + row * k;
    const float l = a.c.target_b == nullptr ? 1.f : a.c.mix != nullptr ? a.c.mix[row] : a.c.mix_value;
    const int64_t lb = a.c.target_b != nullptr && l != 1.f ? a.c.target_b[row] : la;
    float w = a.upstream[a.c.reduction == OW_REDUCE_NONE ? row : 0] * row_weight;
    if (la < 0 || la >= k || lb < 0 || lb >= k) w = __builtin_nanf("");  // no such class
    const float m = a.stats[2 * row], p = w * a.stats[2 * row + 1];
    const float flat = w * (a.c.smoothing / static_cast<float>(k));
    const float hit_a = w * ((1.f - a.c.smoothing) * l), hit_b = w * ((1.f - a.c.smoothing) * (1.f - l));
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

LogitRows shape(const OwCrossEntropy& c) { return LogitRows{c.rows, c.classes, c.dtype}; }

template <class Ty>
void launch_fwd(const XentArgs& a, int t, unsigned groups, hipStream_t s) {
  if (few_rows(shape(a.c), a.loss != nullptr)) hipLaunchKernelGGL((xent_few_kernel<Ty>), dim3(1), dim3(kSumThreads), 0, s, a);
  else if (t == 8) hipLaunchKernelGGL((xent_fwd_kernel<Ty, 8>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 16) hipLaunchKernelGGL((xent_fwd_kernel<Ty, 16>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 32) hipLaunchKernelGGL((xent_fwd_kernel<Ty, 32>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 64) hipLaunchKernelGGL((xent_fwd_kernel<Ty, 64>), dim3(groups), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((xent_fwd_kernel<Ty, 256>), dim3(groups), dim3(256), 0, s, a);
}

template <class Ty>
void launch_bwd(const XentBwdArgs& a, int t, hipStream_t s) {
  const unsigned groups = workgroups(shape(a.c), a.c.rows * a.n_parts, t);
  if (t == 8) hipLaunchKernelGGL((xent_bwd_kernel<Ty, 8>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 16) hipLaunchKernelGGL((xent_bwd_kernel<Ty, 16>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 32) hipLaunchKernelGGL((xent_bwd_kernel<Ty, 32>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 64) hipLaunchKernelGGL((xent_bwd_kernel<Ty, 64>), dim3(groups), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((xent_bwd_kernel<Ty, 256>), dim3(groups), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace ow

extern "C" {

size_t ow_cross_entropy_workspace(const OwCrossEntropy* ce) {
  if (ce == nullptr || ce->rows <= 0 || ce->classes <= 0) return 0;
  return ow::plan_of(ow::shape(*ce), ce->reduction != OW_REDUCE_NONE).workspace;
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
    const ow::LogitPlan p = ow::plan_of(ow::shape(*ce), reduced);
    OW_CHECK_ARG(p.workspace == 0 || (workspace != nullptr && workspace_bytes >= p.workspace &&
                                      reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
                 "workspace of %zu bytes; %zu are needed", workspace_bytes, p.workspace);
    a.n_parts = p.n_parts;
    a.part_len = p.part_len;
    if (p.n_parts > 1) a.parts = static_cast<float*>(workspace);
    else if (p.sums) a.sums = static_cast<ow::LossPartial*>(workspace), a.n_sums = static_cast<int32_t>(p.groups);
    if (ce->dtype == OW_DTYPE_F32) ow::launch_fwd<ow::F32>(a, p.t, p.groups, s);
    else if (ce->dtype == OW_DTYPE_BF16) ow::launch_fwd<ow::BF16>(a, p.t, p.groups, s);
    else ow::launch_fwd<ow::F16>(a, p.t, p.groups, s);
    if (int rc = ow::hip_status(hipGetLastError(), "xent_fwd_kernel launch")) return rc;
  }
  if ((reduced && (ce->rows == 0 || !ow::few_rows(ow::shape(*ce), reduced))) || a.n_parts > 1) {
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
  const int t = ow::threads_of(ow::shape(*ce), ow::kBwdVectors);
  a.part_len = ow::backward_part(ow::shape(*ce));
  a.n_parts = t > 64 ? static_cast<int32_t>((ce->classes + a.part_len - 1) / a.part_len) : 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ce->dtype == OW_DTYPE_F32) ow::launch_bwd<ow::F32>(a, t, s);
  else if (ce->dtype == OW_DTYPE_BF16) ow::launch_bwd<ow::BF16>(a, t, s);
  else ow::launch_bwd<ow::F16>(a, t, s);
  if (int rc = ow::hip_status(hipGetLastError(), "xent_bwd_kernel launch")) return rc;
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
