// Layer norm of rows, forward and backward:
//
//   mu = mean_c x    r = rsqrt(mean_c (x - mu)^2 + eps)    n = (x - mu) r    y = n weight + bias
//
// and, with an upstream gradient g, h = g weight:
//
//   dx = r (h - mean_c h - n mean_c(n h))    dweight = sum_rows g n    dbias = sum_rows g
//
// Both directions read every tensor once and are bound by memory; the backward forms mu and r again from x,
// which it reads anyway, so the forward stores no statistics.  Differences are taken from the rounded mean, and their own
// mean is taken off again with the variance: a mean far above the deviations costs no digits (a row of one large
// value times the rounded 1 / C would seem to vary).  All sums and intermediates are fp32 and each stored value is
// rounded once.
//
// Rows lie in registers, T threads a row, as in block_norms.hip (Place, ow_rows.h); a row shorter than 8 vectors
// takes as few threads as hold it.  A row takes two rounds of sums: the mean of x (backward: with that of h), then the
// differences, their squares (and their products with h).
//
// Measured: 401,408 rows of 128 bf16 forward 33 us (206 MB, what a copy moves in 42: part of it is still in the last
// cache); 25,088 of 512 bf16 forward 11.9, backward 19.5 and 3.9 for the column sums; 102,400 of 95 fp32, whose vectors lie
// at any 4 bytes, 14.2 and 24.0 + 4.1; one row 2.4, a launch and one read's latency.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_rows.h"

namespace ow {
namespace {

constexpr int kMaxChannels = 8192;

struct LayerNormArgs {
  OwLayerNorm n;
  void* y;
  const void* dy;
  int64_t dy_stride;
  void* dx;
  void* dweight;
  void* dbias;
  float* partial;  // [2][n_part][C]: dweight, dbias
  int32_t n_part;  // workgroups of the backward
  int32_t want;    // bits: dweight, dbias
  float inv_c;
};
constexpr int kWantWeight = 1, kWantBias = 2;

// Waves per SIMD that the kernels' registers leave room for (a workgroup of 1,024 threads is four): grids are as
// many workgroups as run at once.
constexpr int fwd_waves(int t) { return t == 1024 ? 4 : 8; }
constexpr int bwd_waves(int t) { return 4; }

// The inverse root of the variance of values whose mean is `off` and whose mean square is `square`.
__device__ __forceinline__ float inverse_root(float square, float off, float eps) {
  const float variance = square - off * off;
  return rsqrtf((variance < 0.f ? 0.f : variance) + eps);  // a NaN stays one
}

template <class Ty, int T, int K, bool RAGGED>
__global__ void __launch_bounds__(kThreads<T>, fwd_waves(T)) layer_norm_fwd_kernel(LayerNormArgs a) {
  typedef Row<Ty> R;
  typedef typename R::Elem Elem;
  constexpr int V = R::kVec, ROWS = kThreads<T> / T;
  __shared__ float red[2 * kRowSums * (kThreads<T> / 64)];
  int turn = 0;
  const int t = threadIdx.x % T, slot = threadIdx.x / T, c = a.n.channels;
  const Place<R, T, K, RAGGED> at(t, c);
  float weight[K][V], bias[K][V];
  bool mask[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at.weight(a.n.weight, a.n.weight_dtype, 0, k, 1.f, weight[k]);
    at.weight(a.n.bias, a.n.bias_dtype, 0, k, 0.f, bias[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) mask[k][j] = at.counts(k, j);
  }
  // A row is read while the one before it is computed.
  typename R::Raw next[K];
  auto read = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < K; ++k) next[k] = at.load(static_cast<const Elem*>(a.n.x) + row * a.n.x_stride, k, row < a.n.rows);
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  read(static_cast<int64_t>(blockIdx.x) * ROWS + slot);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.n.rows; base += step) {
    const int64_t row = base + slot;
    float x[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) R::widen(next[k], x[k]);
    read(row + step);
    float sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += counted<RAGGED>(x[k][j], mask[k][j]);
    row_sums<T>(sum, red, turn);
    const float mean = sum[0] * a.inv_c;
    float s2[2] = {0.f, 0.f};  // x - mean, its square
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] -= mean;
        const float w = at.col[k] < 0 ? 0.f : counted<RAGGED>(x[k][j], mask[k][j]);
        s2[0] += w;
        s2[1] += w * w;
      }
    row_sums<T>(s2, red, turn);
    const float off = s2[0] * a.inv_c;
    const float r = inverse_root(s2[1] * a.inv_c, off, a.n.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = (x[k][j] - off) * r * weight[k][j] + bias[k][j];
      at.store(static_cast<Elem*>(a.y) + row * c, k, row < a.n.rows, x[k]);
    }
  }
}

// One workgroup takes a contiguous share of the rows; its sums over them are partial sums that
// layer_norm_sum_kernel adds in a fixed order.
template <class Ty, int T, int K, bool RAGGED>
__global__ void __launch_bounds__(kThreads<T>, bwd_waves(T)) layer_norm_bwd_kernel(LayerNormArgs a) {
  typedef Row<Ty> R;
  typedef typename R::Elem Elem;
  constexpr int V = R::kVec, ROWS = kThreads<T> / T, COLS = T * K * V;
  __shared__ float red[2 * kRowSums * (kThreads<T> / 64)];
  __shared__ float sums[ROWS > 1 ? ROWS * COLS : 1];
  int turn = 0;
  const int t = threadIdx.x % T, slot = threadIdx.x / T, c = a.n.channels;
  const Place<R, T, K, RAGGED> at(t, c);
  float weight[K][V], s_weight[K][V], s_bias[K][V];
  bool mask[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at.weight(a.n.weight, a.n.weight_dtype, 0, k, 1.f, weight[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s_weight[k][j] = s_bias[k][j] = 0.f;
      mask[k][j] = at.counts(k, j);
    }
  }
  const int64_t groups = (a.n.rows + ROWS - 1) / ROWS;
  const int64_t first = groups * blockIdx.x / a.n_part * ROWS;
  const int64_t share_end = groups * (blockIdx.x + 1) / a.n_part * ROWS;
  const int64_t end = share_end < a.n.rows ? share_end : a.n.rows;

  typename R::Raw xn[K], gn[K];
  constexpr bool AHEAD = K == 1;  // the next row is read while one is computed, where the registers hold both
  auto read = [&](int64_t row) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xn[k] = at.load(static_cast<const Elem*>(a.n.x) + row * a.n.x_stride, k, row < end);
      gn[k] = at.load(static_cast<const Elem*>(a.dy) + row * a.dy_stride, k, row < end);
    }
  };
  if (AHEAD) read(first + slot);
  for (int64_t base = first; base < end; base += ROWS) {
    const int64_t row = base + slot;
    const bool valid = row < end;
    if (!AHEAD) read(row);
    float x[K][V], g[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      R::widen(xn[k], x[k]);
      R::widen(gn[k], g[k]);
    }
    if (AHEAD) read(row + ROWS);
    float s1[2] = {0.f, 0.f};  // x, h
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s1[0] += counted<RAGGED>(x[k][j], mask[k][j]);
        s1[1] += counted<RAGGED>(g[k][j] * weight[k][j], mask[k][j]);
      }
    row_sums<T>(s1, red, turn);
    const float mean = s1[0] * a.inv_c, mean_h = s1[1] * a.inv_c;
    float s2[3] = {0.f, 0.f, 0.f};  // x - mean, its square, its product with h
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] -= mean;
        const float w = at.col[k] < 0 ? 0.f : counted<RAGGED>(x[k][j], mask[k][j]);
        s2[0] += w;
        s2[1] += w * w;
        s2[2] += w * counted<RAGGED>(g[k][j] * weight[k][j], mask[k][j]);
      }
    row_sums<T>(s2, red, turn);
    const float off = s2[0] * a.inv_c;
    const float r = valid ? inverse_root(s2[1] * a.inv_c, off, a.n.eps) : 0.f;  // no row adds nothing, also where eps is 0
    const float back = r * r * (s2[2] * a.inv_c - off * mean_h);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] -= off;
        s_weight[k][j] += g[k][j] * (x[k][j] * r);
        s_bias[k][j] += g[k][j];
        x[k][j] = r * (g[k][j] * weight[k][j] - mean_h - x[k][j] * back);
      }
      if (a.dx != nullptr) at.store(static_cast<Elem*>(a.dx) + row * c, k, valid, x[k]);
    }
  }

  // The workgroup's row slots, added in order; one workgroup's sums are the gradients.
  auto each_sum = [&](const float (&s)[K][V], int which, void* dst, int32_t dtype) {
    if constexpr (ROWS > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) sums[slot * COLS + (k * V + j) * T + t] = s[k][j];
      __syncthreads();
    }
    if (slot != 0) return;
    float* partial = a.partial + (static_cast<int64_t>(which) * a.n_part + blockIdx.x) * c;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float sum = s[k][j];
        if constexpr (ROWS > 1) {
          for (int r = 1; r < ROWS; ++r) sum += sums[r * COLS + (k * V + j) * T + t];
        }
        if (!at.counts(k, j)) continue;
        if (a.n_part == 1) store_any(dst, dtype, at.col[k] + j, sum);
        else partial[at.col[k] + j] = sum;
      }
  };
  if (a.want & kWantWeight) each_sum(s_weight, 0, a.dweight, a.n.weight_dtype);
  if (a.want & kWantBias) each_sum(s_bias, 1, a.dbias, a.n.bias_dtype);
}

// Column sums of the partial rows: 32 columns and 32 slices of the rows a workgroup, every slice added in order.
// blockIdx.x: dweight, dbias.
struct SumArgs {
  const float* partial;  // [2][n_part][C]
  void* dst[2];
  int32_t dtype[2];
  int32_t channels, n_part;
};

__global__ void __launch_bounds__(1024) layer_norm_sum_kernel(SumArgs a) {
  __shared__ float part[32][33];
  const int which = blockIdx.x;
  if (a.dst[which] == nullptr) return;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.y * 32 + lane;
  const float* src = a.partial + static_cast<int64_t>(which) * a.n_part * a.channels;
  float sum = 0.f;
  if (col < a.channels) {
#pragma unroll 8
    for (int64_t r = slice; r < a.n_part; r += 32) sum += src[r * a.channels + col];
  }
  part[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && col < a.channels) {
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < 32; ++s) total += part[s][lane];
    store_any(a.dst[which], a.dtype[which], col, total);
  }
}

// Threads that share a row of `channels`: the smallest power of two whose vectors hold it.
int threads_of(int channels, int vec) {
  int t = 1;
  while (t < 1024 && t * vec < channels) t *= 2;
  return t;
}

int64_t at_once_of(int waves, int t) {
  return static_cast<int64_t>(device_cus()) * (waves * 256 / (t > 256 ? t : 256));
}

// Workgroups of the backward: as many as run at once, and none without a row group.
int backward_parts(const OwLayerNorm& n) {
  const int t = threads_of(n.channels, n.dtype == OW_DTYPE_F32 ? 4 : 8);
  const int64_t rows = t >= 256 ? 1 : 256 / t;
  const int64_t groups = (n.rows + rows - 1) / rows, most = at_once_of(bwd_waves(t), t);
  return static_cast<int>(groups < most ? groups : most);
}

template <class Ty, int T, int K, bool RAGGED>
void launch(const LayerNormArgs& a, bool backward, hipStream_t s) {
  constexpr int ROWS = kThreads<T> / T;
  if (backward) {
    hipLaunchKernelGGL((layer_norm_bwd_kernel<Ty, T, K, RAGGED>), dim3(a.n_part), dim3(kThreads<T>), 0, s, a);
    return;
  }
  const int64_t groups = (a.n.rows + ROWS - 1) / ROWS, most = at_once_of(fwd_waves(T), T);
  hipLaunchKernelGGL((layer_norm_fwd_kernel<Ty, T, K, RAGGED>), dim3(static_cast<unsigned>(groups < most ? groups : most)),
                     dim3(kThreads<T>), 0, s, a);
}

template <class Ty, bool RAGGED>
void launch_ty(const LayerNormArgs& a, bool backward, hipStream_t s) {
  constexpr int V = Row<Ty>::kVec;
  switch (threads_of(a.n.channels, V)) {
    case 1: return launch<Ty, 1, 1, RAGGED>(a, backward, s);
    case 2: return launch<Ty, 2, 1, RAGGED>(a, backward, s);
    case 4: return launch<Ty, 4, 1, RAGGED>(a, backward, s);
    case 8: return launch<Ty, 8, 1, RAGGED>(a, backward, s);
    case 16: return launch<Ty, 16, 1, RAGGED>(a, backward, s);
    case 32: return launch<Ty, 32, 1, RAGGED>(a, backward, s);
    case 64: return launch<Ty, 64, 1, RAGGED>(a, backward, s);
    case 128: return launch<Ty, 128, 1, RAGGED>(a, backward, s);
    case 256: return launch<Ty, 256, 1, RAGGED>(a, backward, s);
    case 512: return launch<Ty, 512, 1, RAGGED>(a, backward, s);
    default: break;
  }
  if constexpr (1024 * V < kMaxChannels) {
    if (a.n.channels > 1024 * V) return launch<Ty, 1024, 2, RAGGED>(a, backward, s);
  }
  return launch<Ty, 1024, 1, RAGGED>(a, backward, s);
}

void run(const LayerNormArgs& a, bool backward, hipStream_t s) {
  const bool ragged = a.n.channels % (a.n.dtype == OW_DTYPE_F32 ? 4 : 8) != 0;
  switch (a.n.dtype) {
    case OW_DTYPE_BF16: return ragged ? launch_ty<BF16, true>(a, backward, s) : launch_ty<BF16, false>(a, backward, s);
    case OW_DTYPE_F16: return ragged ? launch_ty<F16, true>(a, backward, s) : launch_ty<F16, false>(a, backward, s);
    default: return ragged ? launch_ty<F32, true>(a, backward, s) : launch_ty<F32, false>(a, backward, s);
  }
}

bool dtype_ok(int32_t d) { return d == OW_DTYPE_F32 || d == OW_DTYPE_BF16 || d == OW_DTYPE_F16; }

int check(const OwLayerNorm* n) {
  OW_CHECK_ARG(n != nullptr, "layer norm descriptor is NULL");
  OW_CHECK_SUPPORTED(dtype_ok(n->dtype), "layer norm: dtype %d; expected f32, bf16 or f16", n->dtype);
  OW_CHECK_ARG(n->rows >= 0 && n->channels >= 0, "negative size");
  if (n->rows == 0 || n->channels == 0) return OW_OK;
  OW_CHECK_SUPPORTED(n->channels <= kMaxChannels, "layer norm: %d channels; at most %d", n->channels, kMaxChannels);
  OW_CHECK_SUPPORTED(n->rows < (int64_t(1) << 31), "layer norm: %lld rows; fewer than 2^31 are supported",
                     static_cast<long long>(n->rows));
  OW_CHECK_ARG(n->x != nullptr, "x is NULL");
  OW_CHECK_ARG((!n->weight || dtype_ok(n->weight_dtype)) && (!n->bias || dtype_ok(n->bias_dtype)), "unknown weight dtype");
  return OW_OK;
}

}  // namespace
}  // namespace ow

extern "C" {

int ow_layer_norm_fwd(const OwLayerNorm* norm, void* y, void* stream) {
  if (int rc = ow::check(norm)) return rc;
  if (norm->rows == 0 || norm->channels == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG(y != nullptr, "y is NULL");
  ow::LayerNormArgs a{};
  a.n = *norm;
  a.y = y;
  a.inv_c = 1.f / static_cast<float>(norm->channels);
  ow::run(a, false, static_cast<hipStream_t>(stream));
  if (int rc = ow::hip_status(hipGetLastError(), "layer_norm_fwd_kernel launch")) return rc;
  ow::clear_error();
  return OW_OK;
}

size_t ow_layer_norm_bwd_workspace(const OwLayerNorm* norm) {
  if (norm == nullptr || norm->rows <= 0 || norm->channels <= 0) return 0;
  const int parts = ow::backward_parts(*norm);
  return parts > 1 ? static_cast<size_t>(2) * parts * norm->channels * sizeof(float) : 0;
}

int ow_layer_norm_bwd(const OwLayerNorm* norm, const void* dy, int64_t dy_stride, void* dx, void* dweight, void* dbias,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check(norm)) return rc;
  OW_CHECK_ARG(norm->rows > 0 && norm->channels > 0, "the backward of no rows has no kernel");
  OW_CHECK_ARG(dy != nullptr, "dy is NULL");
  OW_CHECK_ARG((!dweight || norm->weight) && (!dbias || norm->bias), "a gradient of an input that is not given");
  ow::LayerNormArgs a{};
  a.n = *norm;
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.dx = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  a.want = (dweight ? ow::kWantWeight : 0) | (dbias ? ow::kWantBias : 0);
  a.n_part = ow::backward_parts(*norm);
  a.partial = static_cast<float*>(workspace);
  a.inv_c = 1.f / static_cast<float>(norm->channels);
  const size_t need = a.want ? ow_layer_norm_bwd_workspace(norm) : 0;
  OW_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                             reinterpret_cast<uintptr_t>(workspace) % 4 == 0),
               "workspace of %zu bytes; %zu are needed", workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ow::run(a, true, s);
  if (int rc = ow::hip_status(hipGetLastError(), "layer_norm_bwd_kernel launch")) return rc;
  if (a.want != 0 && a.n_part > 1) {
    ow::SumArgs m{};
    m.partial = a.partial;
    m.dst[0] = dweight, m.dst[1] = dbias;
    m.dtype[0] = norm->weight_dtype, m.dtype[1] = norm->bias_dtype;
    m.channels = norm->channels;
    m.n_part = a.n_part;
    const unsigned cols = static_cast<unsigned>((norm->channels + 31) / 32);
    hipLaunchKernelGGL(ow::layer_norm_sum_kernel, dim3(2, cols), dim3(1024), 0, s, m);
    if (int rc = ow::hip_status(hipGetLastError(), "layer_norm_sum_kernel launch")) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
