// The norms around a block with its gate, residual scale and residual, forward and backward:
//
//   p    = delta r1 post          r1 = rsqrt(mean_c delta^2 + eps)      (without post: p = delta)
//   out  = x + scale_b gate p
//   next = out r2 next_weight     r2 = rsqrt(mean_c out^2 + eps)
//
// and, with upstream gradients dout and dnext, h = dnext next_weight:
//
//   dx     = dout + r2 h - out r2^3 mean_c(out h)          dnext_weight = sum_rows dnext out r2
//   e      = scale_b dx                                    dgate        = sum_rows e p
//   q      = e gate                                        dpost        = sum_rows q delta r1
//   ddelta = r1 q post - delta r1^3 mean_c(delta q post)   (without post: q)
//
// Both directions read every tensor once and are bound by memory.  The backward forms p, out, r1 and r2
// again from x and delta, which it reads anyway, so the forward stores no statistics.  All sums and every
// intermediate are fp32; each stored value is rounded once.
//
// A row is shared by T threads of one 16-byte vector each (two where 1,024 threads do not reach):
// T is the smallest power of two that holds the row, so a row's values stay in registers between the
// load, the sums and the stores, and a lane keeps its channels' weights (and, backward, the sums of
// their gradients) in registers over all its rows.  Channels that fill no whole vector: the last lane's
// vector ends at the row's end and its first `dup` values, which the lane before it holds too, are left
// out of the sums; both lanes store the same values there.
//
// A grid is as many workgroups as run at once, and a row group is read while the one before it is computed:
// without that 128 x 56 x 56 x 128 bf16 forward took 88.7 us, with it 76.5 (411 MB, 5.4 TB/s, a copy's rate);
// 128 x 14 x 14 x 512 bf16 forward 21.0 us (4.9 TB/s), backward 35.4 (154 MB, 4.4 TB/s; 61 without) and 4.0 for
// the sums of the weights' gradients over workgroups; 64 x 40 x 40 x 95 bf16, ragged, 18.4 and 38.4 us.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_rows.h"

namespace ow {
namespace {

constexpr int kMaxChannels = 8192;

struct NormsArgs {
  OwBlockNorms n;
  void* out;
  void* next;
  const void* dout;
  const void* dnext;
  int64_t dout_stride, dnext_stride;
  void* dx;
  void* ddelta;
  void* dgate;          // written here where a segment has one workgroup
  void* dpost;          // written here where there is one workgroup
  void* dnextw;
  float* partial;       // [3][n_part][C]: dpost, dnext_weight, dgate
  int32_t want;         // bits: dpost, dnext_weight, dgate
  int32_t n_part;       // workgroups
  int32_t seg_parts;    // workgroups of a segment (1: a workgroup may have several segments)
  int64_t segments;
  int64_t seg_rows;     // rows of a segment (an image where the gate is per image, else all)
  float inv_c;
};
constexpr int kWantPost = 1, kWantNext = 2, kWantGate = 4;

// Waves per SIMD that the kernels' registers leave room for (vectors of `vec` values, t threads a row; a
// workgroup of 1,024 threads is four): grids are as many workgroups as run at once.
constexpr int fwd_waves(int t) { return t == 1024 ? 4 : 6; }
constexpr int bwd_waves(int vec, int t) { return t == 1024 ? 4 : vec == 8 ? 3 : 4; }

template <class Ty, int T, int K, bool RAGGED>
__global__ void __launch_bounds__(kThreads<T>, fwd_waves(T)) block_norms_fwd_kernel(NormsArgs a) {
  typedef Row<Ty> R;
  typedef typename R::Elem Elem;
  constexpr int V = R::kVec, ROWS = kThreads<T> / T;
  __shared__ float red[2 * kRowSums * (kThreads<T> / 64)];
  int turn = 0;
  const int t = threadIdx.x % T, slot = threadIdx.x / T, c = a.n.channels;
  const Place<R, T, K, RAGGED> at(t, c);
  const bool has_delta = a.n.delta != nullptr, has_post = a.n.post_weight != nullptr, has_next = a.next != nullptr;
  const bool per_image = a.n.gate_per_image != 0;

  float post[K][V], gate[K][V], nextw[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at.weight(a.n.post_weight, a.n.post_dtype, 0, k, 1.f, post[k]);
    at.weight(per_image ? nullptr : a.n.gate, a.n.gate_dtype, 0, k, 1.f, gate[k]);
    at.weight(a.n.next_weight, a.n.next_dtype, 0, k, 1.f, nextw[k]);
  }
  bool mask[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) mask[k][j] = at.counts(k, j);

  // A row is read while the one before it is computed.
  typename R::Raw xn[K], dn[K];
  auto read = [&](int64_t row) {
    const bool valid = row < a.n.rows;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xn[k] = at.load(static_cast<const Elem*>(a.n.x) + row * a.n.x_stride, k, valid);
      dn[k] = at.load(static_cast<const Elem*>(a.n.delta) + row * a.n.delta_stride, k, valid && has_delta);
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  read(static_cast<int64_t>(blockIdx.x) * ROWS + slot);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * ROWS; base < a.n.rows; base += step) {
    const int64_t row = base + slot;
    const bool valid = row < a.n.rows;
    float x[K][V], d[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      R::widen(xn[k], x[k]);
      R::widen(dn[k], d[k]);
    }
    read(row + step);
    if (has_delta) {
      float f = 1.f;
      if (a.n.scale != nullptr || per_image) {
        const uint32_t image = valid ? static_cast<uint32_t>(row) / static_cast<uint32_t>(a.n.rows_per_image) : 0u;
        if (a.n.scale != nullptr) f = a.n.scale[image];
        if (per_image) {
#pragma unroll
          for (int k = 0; k < K; ++k) at.weight(a.n.gate, a.n.gate_dtype, static_cast<int64_t>(image) * c, k, 1.f, gate[k]);
        }
      }
      if (has_post) {
        float ss[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float w = counted<RAGGED>(d[k][j], mask[k][j]);
            ss[0] += w * w;
          }
        row_sums<T>(ss, red, turn);
        const float r1 = rsqrtf(ss[0] * a.inv_c + a.n.eps);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) d[k][j] *= r1 * post[k][j];
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k][j] += f * gate[k][j] * d[k][j];
        if (a.out != nullptr) at.store(static_cast<Elem*>(a.out) + row * c, k, valid, x[k]);
      }
    }
    if (has_next) {
      float ss[1] = {0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float w = counted<RAGGED>(x[k][j], mask[k][j]);
          ss[0] += w * w;
        }
      row_sums<T>(ss, red, turn);
      const float r2 = rsqrtf(ss[0] * a.inv_c + a.n.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[k][j] *= r2 * nextw[k][j];
        at.store(static_cast<Elem*>(a.next) + row * c, k, valid, x[k]);
      }
    }
  }
}

// One workgroup takes a contiguous share of a segment's rows, so its sums over rows are partial sums
// of that segment: norms_sum_kernel adds them in a fixed order.
template <class Ty, int T, int K, bool RAGGED>
__global__ void __launch_bounds__(kThreads<T>, bwd_waves(Row<Ty>::kVec, T)) block_norms_bwd_kernel(NormsArgs a) {
  typedef Row<Ty> R;
  typedef typename R::Elem Elem;
  constexpr int V = R::kVec, ROWS = kThreads<T> / T, COLS = T * K * V;
  __shared__ float red[2 * kRowSums * (kThreads<T> / 64)];
  __shared__ float sums[ROWS > 1 ? ROWS * COLS : 1];
  int turn = 0;
  const int t = threadIdx.x % T, slot = threadIdx.x / T, c = a.n.channels;
  const Place<R, T, K, RAGGED> at(t, c);
  const bool has_delta = a.n.delta != nullptr, has_post = a.n.post_weight != nullptr, has_next = a.dnext != nullptr;
  const bool parted = a.seg_parts > 1;
  const int part = parted ? blockIdx.x % a.seg_parts : 0;
  const int64_t groups = (a.seg_rows + ROWS - 1) / ROWS;  // of ROWS rows, in a segment
  // A workgroup has a share of one segment, or whole segments.
  const int64_t seg_first = parted ? blockIdx.x / a.seg_parts : static_cast<int64_t>(blockIdx.x) * a.segments / a.n_part;
  const int64_t seg_last = parted ? seg_first + 1 : (static_cast<int64_t>(blockIdx.x) + 1) * a.segments / a.n_part;

  float post[K][V], gate[K][V], nextw[K][V];
  float s_post[K][V], s_next[K][V], s_gate[K][V];
  bool mask[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at.weight(a.n.post_weight, a.n.post_dtype, 0, k, 1.f, post[k]);
    at.weight(a.n.next_weight, a.n.next_dtype, 0, k, 1.f, nextw[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s_post[k][j] = s_next[k][j] = 0.f;
      mask[k][j] = at.counts(k, j);
    }
  }
  // put(column, sum over the workgroup's rows) of a thread's sums.
  auto each_sum = [&](const float (&s)[K][V], auto&& put) {
    if constexpr (ROWS > 1) {  // the workgroup's row slots, added in order
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) sums[slot * COLS + (k * V + j) * T + t] = s[k][j];
      __syncthreads();
    }
    if (slot == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float sum = s[k][j];
          if constexpr (ROWS > 1) {
            for (int r = 1; r < ROWS; ++r) sum += sums[r * COLS + (k * V + j) * T + t];
          }
          if (at.counts(k, j)) put(at.col[k] + j, sum);
        }
    }
  };
  auto partial_row = [&](int which) { return a.partial + (static_cast<int64_t>(which) * a.n_part + blockIdx.x) * c; };

  for (int64_t seg = seg_first; seg < seg_last; ++seg) {
  const int64_t seg_end = (seg + 1) * a.seg_rows;
  const int64_t first = seg * a.seg_rows + groups * part / a.seg_parts * ROWS;
  const int64_t share_end = seg * a.seg_rows + groups * (part + 1) / a.seg_parts * ROWS;
  const int64_t end = share_end < seg_end ? share_end : seg_end;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    at.weight(a.n.gate, a.n.gate_dtype, a.n.gate_per_image ? seg * c : 0, k, 1.f, gate[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) s_gate[k][j] = 0.f;
  }
  typename R::Raw xn[K], dn[K], gn[K], hn[K];
  // While the row before it is computed, where the registers hold both rows (1,500 rows of 8,192 fp32, with it
  // 107, without 69 us).
  constexpr bool AHEAD = K == 1;
  auto read = [&](int64_t row) {
    const bool valid = row < end;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xn[k] = at.load(static_cast<const Elem*>(a.n.x) + row * a.n.x_stride, k, valid && has_next);
      dn[k] = at.load(static_cast<const Elem*>(a.n.delta) + row * a.n.delta_stride, k, valid && has_delta);
      gn[k] = at.load(static_cast<const Elem*>(a.dout) + row * a.dout_stride, k, valid && a.dout != nullptr);
      hn[k] = at.load(static_cast<const Elem*>(a.dnext) + row * a.dnext_stride, k, valid && has_next);
    }
  };
  if (AHEAD) read(first + slot);
  for (int64_t base = first; base < end; base += ROWS) {
    const int64_t row = base + slot;
    const bool valid = row < end;
    if (!AHEAD) read(row);
    float x[K][V], d[K][V], g[K][V], h[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      R::widen(xn[k], x[k]);
      R::widen(dn[k], d[k]);
      R::widen(gn[k], g[k]);
      R::widen(hn[k], h[k]);
    }
    if (AHEAD) read(row + ROWS);
    float f = 1.f, r1 = 1.f;
    if (has_delta) {
      if (a.n.scale != nullptr)
        f = valid ? a.n.scale[static_cast<uint32_t>(row) / static_cast<uint32_t>(a.n.rows_per_image)] : 0.f;
      if (has_post) {
        float ss[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float w = counted<RAGGED>(d[k][j], mask[k][j]);
            ss[0] += w * w;
          }
        row_sums<T>(ss, red, turn);
        r1 = valid ? rsqrtf(ss[0] * a.inv_c + a.n.eps) : 0.f;  // no row adds nothing, also where eps is 0
      }
    }
    if (has_next) {
      float ss[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (has_delta) x[k][j] += f * gate[k][j] * (d[k][j] * (r1 * post[k][j]));  // out
          const float w = counted<RAGGED>(x[k][j], mask[k][j]);
          ss[0] += w * w;
          ss[1] += w * counted<RAGGED>(h[k][j] * nextw[k][j], mask[k][j]);
        }
      row_sums<T>(ss, red, turn);
      const float r2 = valid ? rsqrtf(ss[0] * a.inv_c + a.n.eps) : 0.f;
      const float back = r2 * r2 * (ss[1] * a.inv_c);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s_next[k][j] += h[k][j] * (x[k][j] * r2);
          g[k][j] += r2 * (h[k][j] * nextw[k][j] - x[k][j] * back);
        }
    }
    if (a.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < K; ++k) at.store(static_cast<Elem*>(a.dx) + row * c, k, valid, g[k]);
    }
    if (has_delta) {
      float ss[1] = {0.f};
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float e = f * g[k][j], u = d[k][j] * r1;  // u: the norm's value before its weight
          s_gate[k][j] += e * (u * post[k][j]);
          const float q = e * gate[k][j];
          s_post[k][j] += q * u;
          g[k][j] = q * post[k][j];
          ss[0] += counted<RAGGED>(g[k][j] * d[k][j], mask[k][j]);
        }
      if (has_post) {
        row_sums<T>(ss, red, turn);
        const float back = r1 * r1 * (ss[0] * a.inv_c);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) g[k][j] = r1 * (g[k][j] - d[k][j] * back);
      }
      if (a.ddelta != nullptr) {
#pragma unroll
        for (int k = 0; k < K; ++k) at.store(static_cast<Elem*>(a.ddelta) + row * c, k, valid, g[k]);
      }
    }
  }

  if (a.want & kWantGate) {
    if (parted) {
      float* dst = partial_row(2);
      each_sum(s_gate, [&](int col, float sum) { dst[col] = sum; });
    } else {
      each_sum(s_gate, [&](int col, float sum) { store_any(a.dgate, a.n.gate_dtype, seg * c + col, sum); });
    }
  }
  }
  const bool alone = a.n_part == 1;  // these sums are the gradients
  if (a.want & kWantPost) {
    float* dst = partial_row(0);
    each_sum(s_post, [&](int col, float sum) {
      if (alone) store_any(a.dpost, a.n.post_dtype, col, sum);
      else dst[col] = sum;
    });
  }
  if (a.want & kWantNext) {
    float* dst = partial_row(1);
    each_sum(s_next, [&](int col, float sum) {
      if (alone) store_any(a.dnextw, a.n.next_dtype, col, sum);
      else dst[col] = sum;
    });
  }
}

// Column sums of the backward's partial rows: 32 columns and 32 slices of the rows a workgroup, every
// slice added in order.  blockIdx.x: dpost, dnext_weight, then one dgate row per segment.
struct SumArgs {
  const float* partial;  // [3][n_part][C]
  void* dst[3];
  int32_t dtype[3];
  int32_t channels, n_part, seg_parts, want;
};

__global__ void __launch_bounds__(1024) norms_sum_kernel(SumArgs a) {
  __shared__ float part[32][33];
  const int which = blockIdx.x < 2 ? blockIdx.x : 2, seg = blockIdx.x < 2 ? 0 : blockIdx.x - 2;
  if (!(a.want >> which & 1)) return;
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.y * 32 + lane;
  const int64_t rows = which == 2 ? a.seg_parts : a.n_part;
  const float* src = a.partial + (static_cast<int64_t>(which) * a.n_part + static_cast<int64_t>(seg) * a.seg_parts) * a.channels;
  float sum = 0.f;
  if (col < a.channels) {
#pragma unroll 8
    for (int64_t r = slice; r < rows; r += 32) sum += src[r * a.channels + col];
  }
  part[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && col < a.channels) {
    float total = 0.f;
#pragma unroll
    for (int s = 0; s < 32; ++s) total += part[s][lane];
    store_any(a.dst[which], a.dtype[which], static_cast<int64_t>(seg) * a.channels + col, total);
  }
}

// Threads that share a row of `channels`: the smallest power of two whose vectors hold it.
int threads_of(int channels, int vec) {
  int t = 8;
  while (t < 1024 && t * vec < channels) t *= 2;
  return t;
}

int rows_at_once(int channels, int vec) {
  const int t = threads_of(channels, vec);
  return t >= 256 ? 1 : 256 / t;
}

// Workgroups of T threads a row that run at once: whole ones on each compute unit (4,096 channels bf16, backward:
// one of 512 threads, not one and a half).
int64_t at_once_of(int waves, int t) {
  return static_cast<int64_t>(device_cus()) * (waves * 256 / (t > 256 ? t : 256));
}

struct Parts {
  int64_t segments, seg_rows;
  int32_t seg_parts, n_part;
};

// How the backward's rows are shared out: segments (images where the gate is per image, else one), each
// to seg_parts workgroups, as many in all as run at once and none without a row group; more segments
// than that go several to a workgroup.  One workgroup writes the weights' gradients itself, but rows are not
// kept in one to save the second launch: it costs less than the second group of rows (forward and backward
// of 4 x 1,024 bf16: 11.6 us in one workgroup, 10.7 in two; 16 x 1,024: 21.3 and 10.9).
Parts backward_parts(const OwBlockNorms& n) {
  const int vec = n.dtype == OW_DTYPE_F32 ? 4 : 8, threads = threads_of(n.channels, vec);
  const int at_once = rows_at_once(n.channels, vec);
  const int64_t most = at_once_of(bwd_waves(vec, threads), threads);
  Parts p;
  p.segments = n.gate != nullptr && n.gate_per_image ? n.rows / n.rows_per_image : 1;
  p.seg_rows = n.rows / p.segments;
  const int64_t groups = (p.seg_rows + at_once - 1) / at_once, parts = most / p.segments;
  p.seg_parts = static_cast<int32_t>(parts < 1 ? 1 : parts < groups ? parts : groups);
  p.n_part = static_cast<int32_t>(p.segments < most ? p.segments * p.seg_parts : most);
  return p;
}

template <class Ty, int T, int K, bool RAGGED>
void launch(const NormsArgs& a, bool backward, hipStream_t s) {
  constexpr int ROWS = kThreads<T> / T;
  if (backward) {
    hipLaunchKernelGGL((block_norms_bwd_kernel<Ty, T, K, RAGGED>), dim3(a.n_part), dim3(kThreads<T>), 0, s, a);
    return;
  }
  const int64_t groups = (a.n.rows + ROWS - 1) / ROWS;
  const int64_t most = at_once_of(fwd_waves(T), T);
  hipLaunchKernelGGL((block_norms_fwd_kernel<Ty, T, K, RAGGED>), dim3(static_cast<unsigned>(groups < most ? groups : most)),
                     dim3(kThreads<T>), 0, s, a);
}

template <class Ty, bool RAGGED>
void launch_ty(const NormsArgs& a, bool backward, hipStream_t s) {
  constexpr int V = Row<Ty>::kVec;
  switch (threads_of(a.n.channels, V)) {
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

void run(const NormsArgs& a, bool backward, hipStream_t s) {
  const bool ragged = a.n.channels % (a.n.dtype == OW_DTYPE_F32 ? 4 : 8) != 0;
  switch (a.n.dtype) {
    case OW_DTYPE_BF16: return ragged ? launch_ty<BF16, true>(a, backward, s) : launch_ty<BF16, false>(a, backward, s);
    case OW_DTYPE_F16: return ragged ? launch_ty<F16, true>(a, backward, s) : launch_ty<F16, false>(a, backward, s);
    default: return ragged ? launch_ty<F32, true>(a, backward, s) : launch_ty<F32, false>(a, backward, s);
  }
}

bool dtype_ok(int32_t d) { return d == OW_DTYPE_F32 || d == OW_DTYPE_BF16 || d == OW_DTYPE_F16; }

int check(const OwBlockNorms* n) {
  OW_CHECK_ARG(n != nullptr, "norms descriptor is NULL");
  OW_CHECK_SUPPORTED(dtype_ok(n->dtype), "norms: dtype %d; expected f32, bf16 or f16", n->dtype);
  OW_CHECK_ARG(n->rows >= 0 && n->rows_per_image >= 0 && n->channels >= 0, "negative size");
  if (n->rows == 0 || n->channels == 0) return OW_OK;
  OW_CHECK_SUPPORTED(n->channels <= kMaxChannels, "norms: %d channels; at most %d", n->channels, kMaxChannels);
  OW_CHECK_SUPPORTED(n->rows < (int64_t(1) << 31), "norms: %lld rows; fewer than 2^31 are supported",
                     static_cast<long long>(n->rows));
  OW_CHECK_ARG(n->rows_per_image > 0 && n->rows % n->rows_per_image == 0,
               "rows %lld are not whole images of %lld", static_cast<long long>(n->rows),
               static_cast<long long>(n->rows_per_image));
  OW_CHECK_ARG(n->x != nullptr, "x is NULL");
  OW_CHECK_ARG(n->delta != nullptr || (!n->post_weight && !n->gate && !n->scale),
               "post_weight, gate and scale need delta");
  OW_CHECK_ARG((!n->post_weight || dtype_ok(n->post_dtype)) && (!n->gate || dtype_ok(n->gate_dtype)) &&
                   (!n->next_weight || dtype_ok(n->next_dtype)),
               "unknown weight dtype");
  return OW_OK;
}

}  // namespace
}  // namespace ow

extern "C" {

int ow_block_norms_fwd(const OwBlockNorms* norms, void* out, void* next, void* stream) {
  if (int rc = ow::check(norms)) return rc;
  if (norms->rows == 0 || norms->channels == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG((out != nullptr) == (norms->delta != nullptr), "out is written with delta, and only then");
  OW_CHECK_ARG((next != nullptr) == (norms->next_weight != nullptr), "next is written with next_weight, and only then");
  OW_CHECK_ARG(out != nullptr || next != nullptr, "neither delta nor next_weight is given");
  ow::NormsArgs a{};
  a.n = *norms;
  a.out = out;
  a.next = next;
  a.inv_c = 1.f / static_cast<float>(norms->channels);
  ow::run(a, false, static_cast<hipStream_t>(stream));
  if (int rc = ow::hip_status(hipGetLastError(), "block_norms_fwd_kernel launch")) return rc;
  ow::clear_error();
  return OW_OK;
}

size_t ow_block_norms_bwd_workspace(const OwBlockNorms* norms) {
  if (norms == nullptr || norms->rows <= 0 || norms->channels <= 0 || norms->rows_per_image <= 0) return 0;
  const int32_t parts = ow::backward_parts(*norms).n_part;
  return parts > 1 ? static_cast<size_t>(3) * parts * norms->channels * sizeof(float) : 0;
}

int ow_block_norms_bwd(const OwBlockNorms* norms, const void* dout, int64_t dout_stride, const void* dnext,
                       int64_t dnext_stride, void* dx, void* ddelta, void* dpost_weight, void* dgate,
                       void* dnext_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check(norms)) return rc;
  OW_CHECK_ARG(norms->rows > 0 && norms->channels > 0, "the backward of no rows has no kernel");
  OW_CHECK_ARG(dnext == nullptr || norms->next_weight != nullptr, "dnext needs next_weight");
  OW_CHECK_ARG(dout != nullptr || dnext != nullptr, "no upstream gradient");
  OW_CHECK_ARG((!ddelta || norms->delta) && (!dpost_weight || norms->post_weight) && (!dgate || norms->gate) &&
                   (!dnext_weight || dnext),
               "a gradient of an input that is not given");
  ow::NormsArgs a{};
  a.n = *norms;
  a.dout = dout;
  a.dnext = dnext;
  a.dout_stride = dout_stride;
  a.dnext_stride = dnext_stride;
  a.dx = dx;
  a.ddelta = ddelta;
  a.want = (dpost_weight ? ow::kWantPost : 0) | (dnext_weight ? ow::kWantNext : 0) | (dgate ? ow::kWantGate : 0);
  a.inv_c = 1.f / static_cast<float>(norms->channels);
  a.dgate = dgate;
  a.dpost = dpost_weight;
  a.dnextw = dnext_weight;
  const ow::Parts p = ow::backward_parts(*norms);
  a.segments = p.segments;
  a.seg_rows = p.seg_rows;
  a.seg_parts = p.seg_parts;
  a.n_part = p.n_part;
  a.partial = static_cast<float*>(workspace);
  const size_t need = a.want ? ow_block_norms_bwd_workspace(norms) : 0;
  OW_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                             reinterpret_cast<uintptr_t>(workspace) % 4 == 0),
               "workspace of %zu bytes; %zu are needed", workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ow::run(a, true, s);
  if (int rc = ow::hip_status(hipGetLastError(), "block_norms_bwd_kernel launch")) return rc;
  const bool gate_sums = dgate != nullptr && a.seg_parts > 1;  // else the kernel wrote dgate
  if (gate_sums || ((dpost_weight || dnext_weight) && a.n_part > 1)) {
    ow::SumArgs m{};
    m.partial = a.partial;
    m.dst[0] = dpost_weight, m.dst[1] = dnext_weight, m.dst[2] = dgate;
    m.dtype[0] = norms->post_dtype, m.dtype[1] = norms->next_dtype, m.dtype[2] = norms->gate_dtype;
    m.channels = norms->channels;
    m.n_part = a.n_part;
    m.seg_parts = a.seg_parts;
    m.want = gate_sums ? a.want : a.want & ~ow::kWantGate;
    const unsigned cols = static_cast<unsigned>((norms->channels + 31) / 32);
    hipLaunchKernelGGL(ow::norms_sum_kernel, dim3(2 + static_cast<unsigned>(gate_sums ? p.segments : 0), cols), dim3(1024), 0, s, m);
    if (int rc = ow::hip_status(hipGetLastError(), "norms_sum_kernel launch")) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
