// The backward of the gated feed-forward products (gated_linear.hip), s = 1 / (1 + e^-G), dh the upstream gradient:
//
//   dU = dh G s    dG = dh U s (1 + G (1 - s))    dx = dG Wg + dU Wu    dWg = dG^T x    dWu = dU^T x
//
// Three products on the tiles of ow_gated.h: G and U are formed again from x and become dG and dU in the same kernel, or
// gated_gates_kernel reads what the forward kept of them (ow_gated_linear_kept); dx is one product over both halves; the weights' gradients are
// products over the tokens.  dG and dU are rounded to x's type, the operands of the other two.
//
// Where an output has fewer tiles than the chip has compute units, k is cut into parts, whose fp32 sums
// gated_sum_kernel adds in their order.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_gated.h"

namespace ow {

int check_gated(const OwGatedLinear* d);
GatedArgs gated_args(const OwGatedLinear& d);
bool gated_x_direct(const GatedArgs& a, int64_t size);
bool gated_w_direct(const GatedArgs& a, int64_t size);
void apply_plan(GatedArgs& a, const GatedPlan& p);

namespace {

struct GatedSumArgs {
  const float* partial;  // [splits][sets][n]
  void* out[2];
  int64_t n;
  int32_t splits, sets, dtype;
};

__global__ void __launch_bounds__(256) gated_sum_kernel(GatedSumArgs a) {
  const int set = blockIdx.y;
  if (a.out[set] == nullptr) return;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= a.n) return;
  const float* p = a.partial + set * a.n + i;
  const int64_t step = a.sets * a.n;
  if (i + 4 <= a.n) {
    f32x4 sum = *reinterpret_cast<const f32x4_any*>(p);
#pragma unroll 4
    for (int s = 1; s < a.splits; ++s) sum += *reinterpret_cast<const f32x4_any*>(p + s * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) store_any(a.out[set], a.dtype, i + j, sum[j]);
  } else {
    for (int j = 0; i + j < a.n; ++j) {
      float sum = p[j];
      for (int s = 1; s < a.splits; ++s) sum += p[s * step + j];
      store_any(a.out[set], a.dtype, i + j, sum);
    }
  }
}

int sum_parts(const GatedArgs& a, int64_t n, int sets, int dtype, hipStream_t s) {
  GatedSumArgs m{};
  m.partial = a.partial;
  m.out[0] = a.out[0], m.out[1] = a.out[1];
  m.n = n;
  m.splits = a.splits;
  m.sets = sets;
  m.dtype = dtype;
  hipLaunchKernelGGL(gated_sum_kernel, dim3(static_cast<unsigned>(ceil_div(n, 1024)), sets), dim3(256), 0, s, m);
  return hip_status(hipGetLastError(), "gated_sum_kernel launch");
}

// dG and dU from kept products, a piece of 16 bytes of a row a thread; pieces behind `hidden` are zeros.
template <class Ty>
__global__ void __launch_bounds__(256) gated_gates_kernel(GatedArgs a) {
  constexpr int S = Elem<Ty>::kSize, V = Elem<Ty>::kPiece;
  typedef Row<Ty> R;
  const uint32_t pieces = static_cast<uint32_t>(a.ld_gu / V);
  const int64_t all = a.rows * pieces, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += step) {
    const int64_t row = i / pieces;
    const int c = static_cast<int>(i - row * pieces) * V, n = a.hidden - c;
    const float *g = a.kept + row * a.hidden + c, *u = g + a.rows * a.hidden;
    float dh[V], dg[V], du[V];
    R::widen(__builtin_bit_cast(typename R::Raw, load_piece<S>(a.dh + row * a.dh_ld + c * S, n)), dh);
    u32x4 gw[V / 4], uw[V / 4];
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      gw[k] = load_piece<4>(reinterpret_cast<const char*>(g + 4 * k), n - 4 * k);
      uw[k] = load_piece<4>(reinterpret_cast<const char*>(u + 4 * k), n - 4 * k);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float gj = __uint_as_float(gw[j / 4][j % 4]), uj = __uint_as_float(uw[j / 4][j % 4]), s = sigmoid(gj);
      du[j] = dh[j] * (gj * s);
      dg[j] = dh[j] * uj * (s * (1.f + gj * (1.f - s)));
    }
    const int64_t at = row * a.ld_gu + c;
    R::store(static_cast<typename R::Elem*>(a.out[0]) + at, dg);
    R::store(static_cast<typename R::Elem*>(a.out[1]) + at, du);
  }
}

int gates_of_kept(const GatedArgs& a, int dtype, hipStream_t s) {
  const int64_t all = a.rows * (a.ld_gu / (dtype == OW_DTYPE_F32 ? 4 : 8)), most = 16 * static_cast<int64_t>(device_cus());
  const int64_t groups = ceil_div(all, 256);
  const dim3 grid(static_cast<unsigned>(groups < most ? groups : most));
  if (dtype == OW_DTYPE_BF16) hipLaunchKernelGGL((gated_gates_kernel<BF16>), grid, dim3(256), 0, s, a);
  else if (dtype == OW_DTYPE_F16) hipLaunchKernelGGL((gated_gates_kernel<F16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gated_gates_kernel<F32>), grid, dim3(256), 0, s, a);
  return hip_status(hipGetLastError(), "gated_gates_kernel launch");
}

GatedPlan plan_gates(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.rows, 2 * static_cast<int64_t>(d.hidden), ceil_div(d.channels * size, 128), 1, false, size == 4);
}
GatedPlan plan_dx(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.rows, d.channels, 2 * ceil_div(d.hidden * size, 128), 1, true, size == 4);
}
GatedPlan plan_dw(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.hidden, d.channels, ceil_div(d.rows * size, 128), 2, true, size == 4);
}

// Bytes of dG and dU (each), and of the parts of dx or the weights' gradients.
struct Space {
  size_t gu, parts;
};
Space space_of(const OwGatedLinear& d) {
  const int64_t size = d.dtype == OW_DTYPE_F32 ? 4 : 2;
  const GatedPlan x = plan_dx(d, size), w = plan_dw(d, size);
  const size_t px = x.splits > 1 ? static_cast<size_t>(x.splits) * d.rows * d.channels * 4 : 0;
  const size_t pw = w.splits > 1 ? static_cast<size_t>(w.splits) * 2 * d.hidden * d.channels * 4 : 0;
  const GatedArgs a = gated_args(d);
  return Space{(static_cast<size_t>(d.rows) * a.ld_gu * size + 255) / 256 * 256, px > pw ? px : pw};
}

}  // namespace
}  // namespace ow

extern "C" {

size_t ow_gated_linear_bwd_workspace(const OwGatedLinear* d) {
  if (d == nullptr || d->rows <= 0 || d->channels <= 0 || d->hidden <= 0) return 0;
  const ow::Space s = ow::space_of(*d);
  return 2 * s.gu + s.parts;
}

int ow_gated_linear_bwd(const OwGatedLinear* d, const void* kept, const void* dh, int64_t dh_stride, void* dx, void* dgate_weight,
                        void* dup_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check_gated(d)) return rc;
  OW_CHECK_ARG(d->rows > 0 && d->channels > 0 && d->hidden > 0, "the backward of empty products has no kernel");
  const int64_t size = d->dtype == OW_DTYPE_F32 ? 4 : 2;
  OW_CHECK_ARG(dh != nullptr && reinterpret_cast<uintptr_t>(dh) % size == 0, "dh is NULL or not aligned to its values");
  OW_CHECK_ARG(reinterpret_cast<uintptr_t>(kept) % 4 == 0, "the kept products are not aligned to fp32 values");
  const size_t need = ow_gated_linear_bwd_workspace(d);
  OW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "workspace of %zu bytes; %zu are needed, 16-byte aligned", workspace_bytes, need);
  const ow::GatedPlan gates = ow::plan_gates(*d, size), to_x = ow::plan_dx(*d, size), to_w = ow::plan_dw(*d, size);
  for (const ow::GatedPlan& p : {gates, to_x, to_w})
    OW_CHECK_SUPPORTED(p.tiles_r * p.tiles_c * p.splits < (int64_t(1) << 31), "gated linear: too many tiles for a launch");
  const ow::Space space = ow::space_of(*d);
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ow::GatedArgs a = ow::gated_args(*d);
  const bool x_direct = ow::gated_x_direct(a, size), w_direct = ow::gated_w_direct(a, size);
  a.dh = static_cast<const char*>(dh);
  a.dh_ld = dh_stride * size;
  a.dgu[0] = ws;
  a.dgu[1] = ws + space.gu;
  a.partial = reinterpret_cast<float*>(ws + 2 * space.gu);
  a.out[0] = ws;
  a.out[1] = ws + space.gu;
  if (kept != nullptr) {
    a.kept = static_cast<float*>(const_cast<void*>(kept));
    if (int rc = ow::gates_of_kept(a, d->dtype, s)) return rc;
  } else {
    ow::apply_plan(a, gates);
    ow::launch_gated_mode<ow::kGatedGates>(a, gates.size, d->dtype, x_direct && w_direct, s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
  }
  if (dx != nullptr) {
    a.out[0] = dx;
    a.out[1] = nullptr;
    ow::apply_plan(a, to_x);
    ow::launch_gated_mode<ow::kGatedDx>(a, to_x.size, d->dtype, w_direct, s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
    if (a.splits > 1)
      if (int rc = ow::sum_parts(a, d->rows * d->channels, 1, d->dtype, s)) return rc;
  }
  if (dgate_weight != nullptr || dup_weight != nullptr) {
    a.out[0] = dgate_weight;
    a.out[1] = dup_weight;
    ow::apply_plan(a, to_w);
    ow::launch_gated_mode<ow::kGatedDw>(a, to_w.size, d->dtype, x_direct, s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
    if (a.splits > 1)
      if (int rc = ow::sum_parts(a, static_cast<int64_t>(d->hidden) * d->channels, 2, d->dtype, s)) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
