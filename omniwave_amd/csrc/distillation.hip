// Distillation from a teacher's top logits: rows of logits x against `top` entries a row, each a class i_j and the
// teacher's logit t_j for it, both as softmax at a temperature T, with the gradient.
//
//   q_j = exp((t_j - mt) / T) / zt    over the row's entries (mt their maximum, zt the sum)
//   p_v = exp((x_v - m) / T) / z      over all classes
//   loss = T^2 sum_j q_j (ln q_j - ln p_{i_j})
//        = T^2 (sum_j q_j ((t_j - mt) - (x_{i_j} - m)) / T  -  ln zt  +  ln z)
//   dx_v = w T (p_v - sum_{j: i_j = v} q_j)
//
// with w the upstream gradient, divided by the number of counted rows for their mean.  Entries whose class is
// ignore_index, or whose logit is -inf, are none; a row without entries is left out (loss and gradient 0, not
// counted).  A class outside the row, or a NaN among the entries, makes the row NaN, as a NaN logit does.
//
// Forward and backward read the logits once each, as the cross-entropy does (ow_softmax.h); a row's entries
// are read by the lanes that have its m and z.  Differences are taken from the maxima before anything is summed.  The loss
// of a student near its teacher keeps its digits where the list has all classes (near_row); a shorter list's loss is at least
// the student's share of the other classes, and is off by some 1e-7 T^2 (1,000 classes: 0.6 to 1.4e-7 in the mean square).
//
// The backward writes w T p for every class first, and then the classes that have an entry once more: the same threads write
// both, with a barrier between them, and a class is written by one entry only.  A bitmap of the part's classes in LDS finds
// classes that have several; then the first of these adds all of them up in their order, so results do not depend on timing.
// Exponentials, sums and losses are fp32 (the sum of losses fp64); the gradient is rounded once.
//
// Bound by memory for long rows (4,096 of 21,841 bf16 with 64 entries: forward 40.2 us and 4.6 for the sum, 179 MB;
// backward 69.7, 358 MB, a copy's time 73), by launches for few (8 of 1,000: 5.2 and 3.7; 1,024 of 1,000 fp32 with 100 entries
// 5.2 + 3.0 and 5.7).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_softmax.h"

namespace ow {
namespace {

struct DistillArgs {
  OwDistillation d;
  float scale;        // log2(e) / T
  float* parts;       // [rows][n_parts][3]: m, z, unused
  LossPartial* sums;  // [n_sums], of the workgroups; NULL: the losses of rows are summed
  float* stats;       // [rows][4]: m, 1 / z, mt, 1 / zt (0: the row is left out)
  float* losses;      // [rows], 0 for rows left out
  float* loss;        // [1] their sum or mean; NULL: the losses are the result
  float* weight;      // [1] a row's weight in it
  int32_t n_parts, part_len;  // part_len: whole vectors
  int32_t n_sums;
};

// Whether an entry is one, and that its class is in the row.
struct Entry {
  int64_t at;
  float t;
  bool given, known;
  __device__ __forceinline__ Entry(const OwDistillation& d, int64_t row, int j) {
    at = d.indices[row * d.top + j];
    t = load_any(d.teacher, d.teacher_dtype, row * d.top + j);
    given = at != d.ignore_index && t != -__builtin_inff();
    known = at >= 0 && at < d.classes;
  }
};

// e^d - 1 - d for |d| <= 1/2: the first eight terms, the next one is below 2^-28 of them.
__device__ __forceinline__ float power_rest(float d) {
  float s = 1.f / 40320.f + d * (1.f / 362880.f);
  s = 1.f / 5040.f + d * s;
  s = 1.f / 720.f + d * s;
  s = 1.f / 120.f + d * s;
  s = 1.f / 24.f + d * s;
  s = 1.f / 6.f + d * s;
  return d * d * (0.5f + d * s);
}

// The loss of a row, T^2 left out, whose entries are all classes, one each, by T lanes.  A student near its teacher has a
// small one, the rest of sums that cancel.  With d_j = ln(p_j / q_j) and both distributions over the same classes,
// sum_j (p_j - q_j) = 0, so
//   sum_j q_j (-d_j) = sum_j q_j (e^{d_j} - 1 - d_j)
// of which no term is negative, and an error of d that the entries have in common (ln of the sums) enters by its square:
// 1,000 classes, T = 4, logits 0.01 apart, a loss of 5e-5: 11% off as sum_j q_j (-d_j), 6e-8 this way.  Such entries are known by
// their number and their part of z, which is all of it within what rounding does to two sums; `loss` comes back for others.
// The row's entries are read twice more (8,192 x 1,000 fp32, every row near: 85 us forward without, 204 with).
template <int T>
__device__ __forceinline__ float near_row(const DistillArgs& a, int64_t row, float m, float z, float mt, float zt, int lane, int top, float loss) {
  const OwDistillation& d = a.d;
  float given = 0.f, part = 0.f;
  for (int j = lane; j < top; j += T) {
    const Entry e(d, row, j);
    if (!e.given || !e.known) continue;
    given += 1.f;
    part += __builtin_amdgcn_exp2f((load_any(d.logits, d.dtype, row * d.row_stride + e.at) - m) * a.scale);
  }
  given = lanes_reduce<AddOp, T>(given);
  part = lanes_reduce<AddOp, T>(part);
  const float k = static_cast<float>(d.classes);  // at most the entries of a row
  const bool all = given == k && fabsf(part - z) <= (128.f + k / 16.f) * 0x1p-24f * z;
  const float log_ratio = logf(part / zt), to_p = zt / part;
  float sum = 0.f;
  for (int j = all ? lane : top; j < top; j += T) {
    const Entry e(d, row, j);
    if (!e.given || !e.known) continue;  // more entries than classes: some are none
    const float x = load_any(d.logits, d.dtype, row * d.row_stride + e.at);
    const float q = __builtin_amdgcn_exp2f((e.t - mt) * a.scale);
    const double apart = (static_cast<double>(x) - m) - (static_cast<double>(e.t) - mt);  // four fp32 numbers that cancel
    const float diff = static_cast<float>(apart) / d.temperature - log_ratio;
    if (q > 0.f && fabsf(diff) < 0.5f) {
      sum += q * power_rest(diff);
    } else {
      sum += __builtin_amdgcn_exp2f((x - m) * a.scale) * to_p;
      if (q > 0.f) sum -= q + q * diff;
    }
  }
  sum = lanes_reduce<AddOp, T>(sum);
  return all ? sum / zt : loss;
}

// A row's teacher and loss, from its m and z, by T lanes of whole waves; all of them get the loss, and lane 0 writes.  ALL: lists
// may be as long as the classes (registers for near_row cost the others 5%, 200,000 rows of 100 bf16).
template <int T, bool ALL>
__device__ __forceinline__ float finish_row(const DistillArgs& a, int64_t row, float m, float z, int lane, bool valid, bool* counted) {
  const OwDistillation& d = a.d;
  const int top = valid ? d.top : 0;
  float mt = -__builtin_inff(), bad = 0.f;
  for (int j = lane; j < top; j += T) {
    const Entry e(d, row, j);
    if (!e.given) continue;
    mt = fmaxf(mt, e.t);
    if (!e.known || e.t != e.t) bad = 1.f;
  }
  mt = lanes_reduce<MaxOp, T>(mt);
  bad = lanes_reduce<MaxOp, T>(bad);
  float zt = 0.f, sum = 0.f;  // sum of q zt ((t - mt) - (x - m))
  for (int j = lane; j < top; j += T) {
    const Entry e(d, row, j);
    if (!e.given || !e.known) continue;
    const float q = __builtin_amdgcn_exp2f((e.t - mt) * a.scale);
    zt += q;
    if (q > 0.f) sum += q * ((e.t - mt) - (load_any(d.logits, d.dtype, row * d.row_stride + e.at) - m));
  }
  zt = lanes_reduce<AddOp, T>(zt);
  sum = lanes_reduce<AddOp, T>(sum);
  if (bad != 0.f) zt = __builtin_nanf("");
  *counted = zt != 0.f;  // a NaN counts
  float loss = 0.f;
  if (zt != 0.f) loss = sum / zt / d.temperature + logf(z / zt);
  // From 1/32 on a loss this way has five digits.
  if (ALL && d.top >= d.classes) {
    const bool near = zt > 0.f && loss < 0.03125f;
    if (__any(near)) loss = near_row<T>(a, row, m, z, mt, zt, lane, near ? top : 0, loss);
  }
  loss *= d.temperature * d.temperature;
  if (lane == 0 && valid) {
    float* s = a.stats + 4 * row;
    s[0] = m, s[1] = 1.f / z, s[2] = mt, s[3] = zt != 0.f ? 1.f / zt : 0.f;
    a.losses[row] = loss;
  }
  return loss;
}

// T threads a (row, part); one part a row for T <= 64.
template <class Ty, int T, bool ALL>
__global__ void __launch_bounds__(256) distill_fwd_kernel(DistillArgs a) {
  typedef Row<Ty> R;
  constexpr int UNITS = 256 / T;
  const int t = threadIdx.x % T;
  const int64_t units = a.d.rows * a.n_parts;
  double sum = 0.0;
  int64_t count = 0;
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * UNITS; base < units; base += static_cast<int64_t>(gridDim.x) * UNITS) {
    const int64_t unit = base + threadIdx.x / T;
    const bool valid = unit < units;  // uniform over a unit
    int64_t row = unit, begin = 0, end = a.d.classes;
    if (T > 64 && a.n_parts > 1) {
      row = unit / a.n_parts;
      begin = unit % a.n_parts * a.part_len;
      end = begin + a.part_len < end ? begin + a.part_len : end;
    }
    Numbers<Log2eOver> s{Log2eOver{a.scale}};
    if (valid) s.template scan<R, T>(static_cast<const typename R::Elem*>(a.d.logits) + row * a.d.row_stride, begin, end, t);
    s.template join_row<(T > 64 ? 64 : T)>();
    if constexpr (T == 256) {
      // One half a turn: it is written again only after the barrier of the turn between.
      __shared__ float lds[2][2][4];
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) lds[turn][0][wave] = s.m, lds[turn][1][wave] = s.z;
      __syncthreads();
      s.m = lds[turn][0][0], s.z = lds[turn][1][0];
#pragma unroll
      for (int w = 1; w < 4; ++w) join(s.f, s.m, s.z, lds[turn][0][w], lds[turn][1][w]);
      turn ^= 1;
    }
    if (a.n_parts > 1) {
      if (t == 0 && valid) {
        float* p = a.parts + unit * 3;
        p[0] = s.m, p[1] = s.z;
      }
    } else if (T <= 64 || t < 64) {  // whole waves
      bool counted = false;
      const float loss = finish_row<(T > 64 ? 64 : T), ALL>(a, row, s.m, s.z, t, valid, &counted);
      if (t == 0 && valid) sum += loss, count += counted;
    }
  }
  if (a.sums != nullptr) {
    const LossPartial all = workgroup_sum<4>(sum, count);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = all;
  }
}

// The loss from what the workgroups summed, or from the rows' losses, which this workgroup's threads see.
__device__ __forceinline__ void sum_rows(const DistillArgs& a) {
  double sum = 0.0;
  int64_t count = 0;
  if (a.sums != nullptr) {
    for (int i = threadIdx.x; i < a.n_sums; i += kSumThreads) sum += a.sums[i].sum, count += a.sums[i].count;
  } else {
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.d.rows; row += kSumThreads) {
      sum += a.losses[row];
      count += a.stats[4 * row + 3] != 0.f;
    }
  }
  const LossPartial all = workgroup_sum<kSumThreads / 64>(sum, count);
  if (threadIdx.x == 0) {
    const double weight = a.d.reduction == OW_REDUCE_MEAN ? 1.0 / static_cast<double>(all.count) : 1.0;
    *a.loss = static_cast<float>(all.count ? all.sum * weight : a.d.reduction == OW_REDUCE_MEAN ? __builtin_nan("") : 0.0);
    *a.weight = static_cast<float>(weight);
  }
}

// Few short rows and their sum in one launch: one workgroup, a wave a row.
template <class Ty>
__global__ void __launch_bounds__(kSumThreads) distill_few_kernel(DistillArgs a) {
  typedef Row<Ty> R;
  const int lane = threadIdx.x & 63;
  const int64_t row = threadIdx.x >> 6;
  if (row < a.d.rows) {
    Numbers<Log2eOver> s{Log2eOver{a.scale}};
    s.template scan<R, 64>(static_cast<const typename R::Elem*>(a.d.logits) + row * a.d.row_stride, 0, a.d.classes, lane);
    s.template join_row<64>();
    bool counted;
    finish_row<64, true>(a, row, s.m, s.z, lane, true, &counted);
  }
  __syncthreads();
  sum_rows(a);
}

// Joins the parts of rows, 16 lanes a row (n_parts > 1), and sums the losses (one workgroup then).
__global__ void __launch_bounds__(kSumThreads) distill_sum_kernel(DistillArgs a) {
  constexpr int ROWS = kSumThreads / kSumLanes;
  if (a.n_parts > 1) {
    const int lane = threadIdx.x % kSumLanes;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.d.rows; base += static_cast<int64_t>(gridDim.x) * ROWS) {
      const int64_t row = base + threadIdx.x / kSumLanes;
      const bool valid = row < a.d.rows;
      const Log2eOver f{a.scale};
      float m = -__builtin_inff(), z = 0.f, unused = 0.f;
      if (valid) {
        const float* p = a.parts + row * a.n_parts * 3;
        for (int i = lane; i < a.n_parts; i += kSumLanes) join(f, m, z, p[3 * i], p[3 * i + 1]);
      }
      join_lanes<kSumLanes>(f, m, z, unused);
      bool counted;
      finish_row<kSumLanes, true>(a, row, m, z, lane, valid, &counted);
    }
    __syncthreads();  // the losses of this workgroup's rows, which are all rows where they are summed
  }
  if (a.loss != nullptr) sum_rows(a);
}

struct DistillBwdArgs {
  OwDistillation d;
  float scale;
  const float* stats;
  const float* weight;    // a row's weight; NULL: 1
  const float* upstream;  // [1], or [rows] without reduction
  void* grad;             // [rows][classes]
  int32_t n_parts, part_len;
};

// What the T threads of a unit wrote is theirs to write again.
template <int T>
__device__ __forceinline__ void unit_sync() {
  if constexpr (T > 64) __syncthreads();
  else wave_lds_sync();
}

// T threads a (row, part); one part a row for T <= 64.
template <class Ty, int T>
__global__ void __launch_bounds__(256) distill_bwd_kernel(DistillBwdArgs a) {
  typedef Row<Ty> R;
  constexpr int V = R::kVec, UNITS = 256 / T;
  // Bits of a unit's classes: of a part, or of a whole row.
  constexpr int WORDS = (T == 256 ? 2 * kPart : T == 64 ? kLong : T * V * kBwdVectors) / 32;
  __shared__ uint32_t seen_of[UNITS][WORDS], again_of[UNITS][WORDS];
  uint32_t *seen = seen_of[threadIdx.x / T], *again = again_of[threadIdx.x / T];
  const int t = threadIdx.x % T;
  const int64_t k = a.d.classes, units = a.d.rows * a.n_parts;
  const float row_weight = a.weight != nullptr ? *a.weight : 1.f;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * UNITS; base < units; base += static_cast<int64_t>(gridDim.x) * UNITS) {
    const int64_t unit = base + threadIdx.x / T;
    const bool valid = unit < units;  // uniform over a unit
    int64_t row = valid ? unit : 0, begin = 0, end = k;
    if (T > 64) {
      row = unit / a.n_parts;
      begin = unit % a.n_parts * a.part_len;
      end = begin + a.part_len < k ? begin + a.part_len : k;
    }
    if (!valid) end = begin;
    const typename R::Elem* x = static_cast<const typename R::Elem*>(a.d.logits) + row * a.d.row_stride;
    typename R::Elem* out = static_cast<typename R::Elem*>(a.grad) + row * k;
    const float* s = a.stats + 4 * row;
    const float m = s[0], mt = s[2], inv_zt = s[3];
    const bool counted = inv_zt != 0.f;
    float w = a.upstream[a.d.reduction == OW_REDUCE_NONE ? row : 0] * row_weight * a.d.temperature;
    if (inv_zt != inv_zt) w = inv_zt;
    const float p = w * s[1];
    const int words = static_cast<int>((end - begin + 31) / 32);
    for (int i = t; i < words; i += T) seen[i] = again[i] = 0u;
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
        for (int j = 0; j < V; ++j) v[j] = p * __builtin_amdgcn_exp2f((v[j] - m) * a.scale);
      }
      if (n == V) {
        R::store(out + i, v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < n) out[i + j] = R::from_f32(v[j]);
      }
    }
    unit_sync<T>();  // the bits are clear, and the part is written
    const int top = counted && valid ? a.d.top : 0;
    auto q_of = [&](const Entry& e) { return __builtin_amdgcn_exp2f((e.t - mt) * a.scale) * inv_zt; };
    auto write = [&](int64_t at, float q) {
      out[at] = R::from_f32(p * __builtin_amdgcn_exp2f((R::to_f32(x[at]) - m) * a.scale) - w * q);
    };
    bool twice = false;
    for (int j = t; j < top; j += T) {
      const Entry e(a.d, row, j);
      if (!e.given || e.at < begin || e.at >= end) continue;
      const int bit = static_cast<int>(e.at - begin);
      if (atomicOr(&seen[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u) {
        atomicOr(&again[bit >> 5], 1u << (bit & 31));
        twice = true;
      } else {
        write(e.at, q_of(e));
      }
    }
    if (T <= 64) unit_sync<T>();
    // Rare: a class has several entries.  Only these look for the others, and only the first of them through all (64 rows
    // of 8,192 entries, forward and gradient: no class twice 120 us, one of them 450, every one eight times 4,900).
    if (T > 64 ? __syncthreads_or(twice) : __any(twice)) {
      for (int j = t; j < top; j += T) {
        const Entry e(a.d, row, j);
        if (!e.given || e.at < begin || e.at >= end) continue;
        const int bit = static_cast<int>(e.at - begin);
        if (!(again[bit >> 5] >> (bit & 31) & 1u)) continue;
        float q = 0.f;
        bool first = true;
        constexpr int U = 16;  // classes that are read together
        for (int o = 0; o < top && first; o += U) {
          int64_t at[U];
#pragma unroll
          for (int u = 0; u < U; ++u) at[u] = a.d.indices[row * a.d.top + (o + u < top ? o + u : top - 1)];
          uint32_t same = 0u;
#pragma unroll
          for (int u = 0; u < U; ++u) same |= (at[u] == e.at && o + u < top ? 1u : 0u) << u;
          for (; same != 0u && first; same &= same - 1u) {
            const int of = o + __builtin_ctz(same);
            const Entry f(a.d, row, of);
            if (!f.given) continue;
            first = of >= j;
            q += q_of(f);
          }
        }
        if (first) write(e.at, q);
      }
    }
    unit_sync<T>();  // before the bits are cleared again
  }
}

LogitRows shape(const OwDistillation& d) { return LogitRows{d.rows, d.classes, d.dtype}; }

template <class Ty, bool ALL>
void launch_fwd_rows(const DistillArgs& a, int t, unsigned groups, hipStream_t s) {
  if (t == 8) hipLaunchKernelGGL((distill_fwd_kernel<Ty, 8, ALL>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 16) hipLaunchKernelGGL((distill_fwd_kernel<Ty, 16, ALL>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 32) hipLaunchKernelGGL((distill_fwd_kernel<Ty, 32, ALL>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 64) hipLaunchKernelGGL((distill_fwd_kernel<Ty, 64, ALL>), dim3(groups), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((distill_fwd_kernel<Ty, 256, ALL>), dim3(groups), dim3(256), 0, s, a);
}

template <class Ty>
void launch_fwd(const DistillArgs& a, int t, unsigned groups, hipStream_t s) {
  if (few_rows(shape(a.d), a.loss != nullptr)) hipLaunchKernelGGL((distill_few_kernel<Ty>), dim3(1), dim3(kSumThreads), 0, s, a);
  else if (a.d.top >= a.d.classes) launch_fwd_rows<Ty, true>(a, t, groups, s);
  else launch_fwd_rows<Ty, false>(a, t, groups, s);
}

template <class Ty>
void launch_bwd(const DistillBwdArgs& a, int t, hipStream_t s) {
  const unsigned groups = workgroups(shape(a.d), a.d.rows * a.n_parts, t);
  if (t == 8) hipLaunchKernelGGL((distill_bwd_kernel<Ty, 8>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 16) hipLaunchKernelGGL((distill_bwd_kernel<Ty, 16>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 32) hipLaunchKernelGGL((distill_bwd_kernel<Ty, 32>), dim3(groups), dim3(256), 0, s, a);
  else if (t == 64) hipLaunchKernelGGL((distill_bwd_kernel<Ty, 64>), dim3(groups), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((distill_bwd_kernel<Ty, 256>), dim3(groups), dim3(256), 0, s, a);
}

constexpr int kMostEntries = 1 << 16;

bool dtype_ok(int32_t d) { return d == OW_DTYPE_F32 || d == OW_DTYPE_BF16 || d == OW_DTYPE_F16; }

int check(const OwDistillation* d) {
  OW_CHECK_ARG(d != nullptr, "distillation descriptor is NULL");
  OW_CHECK_SUPPORTED(dtype_ok(d->dtype) && dtype_ok(d->teacher_dtype), "distillation: dtypes %d and %d; expected f32, bf16 or f16",
                     d->dtype, d->teacher_dtype);
  OW_CHECK_ARG(d->reduction == OW_REDUCE_NONE || d->reduction == OW_REDUCE_SUM || d->reduction == OW_REDUCE_MEAN,
               "unknown reduction %d", d->reduction);
  OW_CHECK_ARG(d->rows >= 0 && d->classes >= 1 && d->top >= 0, "%lld rows of %lld classes, %d entries",
               static_cast<long long>(d->rows), static_cast<long long>(d->classes), d->top);
  OW_CHECK_SUPPORTED(d->rows < (int64_t(1) << 31) && d->classes < (int64_t(1) << 30) && d->top <= kMostEntries,
                     "%lld rows of %lld classes, %d entries; fewer than 2^31 and 2^30, and at most 2^16, are supported",
                     static_cast<long long>(d->rows), static_cast<long long>(d->classes), d->top);
  // Its square and log2(e) over it stay well inside fp32.
  OW_CHECK_ARG(d->temperature >= 0.99e-15f && d->temperature <= 1.01e15f, "temperature %g is not in [1e-15, 1e15]", d->temperature);
  OW_CHECK_ARG(d->rows == 0 || (d->logits != nullptr && (d->top == 0 || (d->teacher != nullptr && d->indices != nullptr))),
               "logits, teacher or indices is NULL");
  return OW_OK;
}

}  // namespace
}  // namespace ow

extern "C" {

size_t ow_distillation_workspace(const OwDistillation* d) {
  if (d == nullptr || d->rows <= 0 || d->classes <= 0) return 0;
  return ow::plan_of(ow::shape(*d), d->reduction != OW_REDUCE_NONE).workspace;
}

int ow_distillation_fwd(const OwDistillation* d, float* stats, float* losses, float* loss, float* weight, void* workspace,
                        size_t workspace_bytes, void* stream) {
  if (int rc = ow::check(d)) return rc;
  const bool reduced = d->reduction != OW_REDUCE_NONE;
  OW_CHECK_ARG(d->rows == 0 || (stats != nullptr && losses != nullptr), "stats or losses is NULL");
  OW_CHECK_ARG(!reduced || (loss != nullptr && weight != nullptr), "loss or weight is NULL");
  if (d->rows == 0 && !reduced) {
    ow::clear_error();
    return OW_OK;
  }
  ow::DistillArgs a{};
  a.d = *d;
  a.scale = ow::kLog2e / d->temperature;
  a.stats = stats;
  a.losses = losses;
  a.loss = reduced ? loss : nullptr;
  a.weight = weight;
  a.n_parts = 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->rows > 0) {
    const ow::LogitPlan p = ow::plan_of(ow::shape(*d), reduced);
    OW_CHECK_ARG(p.workspace == 0 || (workspace != nullptr && workspace_bytes >= p.workspace &&
                                      reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
                 "workspace of %zu bytes; %zu are needed", workspace_bytes, p.workspace);
    a.n_parts = p.n_parts;
    a.part_len = p.part_len;
    if (p.n_parts > 1) a.parts = static_cast<float*>(workspace);
    else if (p.sums) a.sums = static_cast<ow::LossPartial*>(workspace), a.n_sums = static_cast<int32_t>(p.groups);
    if (d->dtype == OW_DTYPE_F32) ow::launch_fwd<ow::F32>(a, p.t, p.groups, s);
    else if (d->dtype == OW_DTYPE_BF16) ow::launch_fwd<ow::BF16>(a, p.t, p.groups, s);
    else ow::launch_fwd<ow::F16>(a, p.t, p.groups, s);
    if (int rc = ow::hip_status(hipGetLastError(), "distill_fwd_kernel launch")) return rc;
  }
  if ((reduced && (d->rows == 0 || !ow::few_rows(ow::shape(*d), reduced))) || a.n_parts > 1) {
    const int64_t rows_at_once = ow::kSumThreads / ow::kSumLanes;
    const int64_t groups = reduced ? 1 : (d->rows + rows_at_once - 1) / rows_at_once;
    hipLaunchKernelGGL(ow::distill_sum_kernel, dim3(static_cast<unsigned>(groups)), dim3(ow::kSumThreads), 0, s, a);
    if (int rc = ow::hip_status(hipGetLastError(), "distill_sum_kernel launch")) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

int ow_distillation_bwd(const OwDistillation* d, const float* stats, const float* weight, const float* upstream, void* grad,
                        void* stream) {
  if (int rc = ow::check(d)) return rc;
  if (d->rows == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG(stats && upstream && grad, "a pointer is NULL");
  ow::DistillBwdArgs a{};
  a.d = *d;
  a.scale = ow::kLog2e / d->temperature;
  a.stats = stats;
  a.weight = weight;
  a.upstream = upstream;
  a.grad = grad;
  const int t = ow::threads_of(ow::shape(*d), ow::kBwdVectors);
  a.part_len = ow::backward_part(ow::shape(*d));
  a.n_parts = t > 64 ? static_cast<int32_t>((d->classes + a.part_len - 1) / a.part_len) : 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == OW_DTYPE_F32) ow::launch_bwd<ow::F32>(a, t, s);
  else if (d->dtype == OW_DTYPE_BF16) ow::launch_bwd<ow::BF16>(a, t, s);
  else ow::launch_bwd<ow::F16>(a, t, s);
  if (int rc = ow::hip_status(hipGetLastError(), "distill_bwd_kernel launch")) return rc;
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
