// The backward of the gated feed-forward products (gated_linear.hip), s = 1 / (1 + e^-G), dh the upstream gradient:
//
//   dU = dh G s    dG = dh U s (1 + G (1 - s))    dx = dG Wg + dU Wu    dWg = dG^T x    dWu = dU^T x
//
// Three products on the tiles of ow_gated.h: G and U are formed again from x (the forward keeps nothing but its
// inputs) and become dG and dU in the same kernel; dx is one product over both halves; the weights' gradients are
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

GatedPlan plan_gates(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.rows, 2 * static_cast<int64_t>(d.hidden), ceil_div(d.channels * size, 128), 1, false);
}
GatedPlan plan_dx(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.rows, d.channels, 2 * ceil_div(d.hidden * size, 128), 1, true);
}
GatedPlan plan_dw(const OwGatedLinear& d, int64_t size) {
  return gated_plan(d.hidden, d.channels, ceil_div(d.rows * size, 128), 2, true);
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

int ow_gated_linear_bwd(const OwGatedLinear* d, const void* dh, int64_t dh_stride, void* dx, void* dgate_weight,
                        void* dup_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check_gated(d)) return rc;
  OW_CHECK_ARG(d->rows > 0 && d->channels > 0 && d->hidden > 0, "the backward of empty products has no kernel");
  const int64_t size = d->dtype == OW_DTYPE_F32 ? 4 : 2;
  OW_CHECK_ARG(dh != nullptr && reinterpret_cast<uintptr_t>(dh) % size == 0, "dh is NULL or not aligned to its values");
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
  ow::apply_plan(a, gates);
  ow::launch_gated_mode<ow::kGatedGates>(a, gates.size, d->dtype, x_direct && w_direct, s);
  if (int rc = ow::hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
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
