// The backward of the gated feed-forward products (gated_linear.hip), s = 1 / (1 + e^-G), dh the upstream gradient:
//
//   dU = dh G s    dG = dh U s (1 + G (1 - s))    dx = dG Wg + dU Wu    dWg = dG^T x    dWu = dU^T x
//
// Three products on the tiles of ow_gated.h: G and U are formed again from x and become dG and dU in the same kernel, or
// gated_gates_kernel reads what the forward kept of them (ow_gated_linear_kept); dx is one product over both halves; the weights'
// gradients are products over the tokens.  dG and dU are rounded to x's type, the operands of the other two.
//
// 6,272 tokens of 4,096 to 8,192 bf16: gates from kept products 139 us, dx 780 to 838 + 23 to join (1,005 to 1,079 TFLOP/s), the
// weights' gradients 719 to 781: bound by the matrix cores at the clock that the card holds.  401,408 tokens of 128 to 256
// bf16: gates with the products formed again 197, dx 117, the weights' gradients 106 + 13: bound by writing dG and dU once
// and reading them twice.  25,088 tokens of 256 to 512 fp32: copies into planes 16, gates 55, dx 107 + 16, the weights' 84 + 12.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_gated.h"

namespace ow {

int check_gated(const OwGatedLinear* d);
size_t gated_operand_bytes(const OwGatedLinear& d);
int gated_operands(const OwGatedLinear& d, char* workspace, GatedArgs* a, hipStream_t s);
bool gated_few(const OwGatedLinear& d);
GatedPlan gated_plan_forward(const OwGatedLinear& d);

namespace {

// dG and dU from kept products, a piece of 8 values of a row a thread; values behind `hidden` are zeros.
template <class Ty, class Out>
__global__ void __launch_bounds__(256) gated_gates_kernel(GatedArgs a) {
  constexpr bool kWide = std::is_same<Out, F32>::value;
  constexpr int S = kWide ? 4 : 2, V = 16 / S;
  typedef Row<Out> R;
  const uint32_t pieces = static_cast<uint32_t>(a.gu[0].ld / 16);
  const int64_t all = a.rows * pieces, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += step) {
    const int64_t row = i / pieces;
    const int c = static_cast<int>(i - row * pieces) * 8, n = a.hidden - c;
    const char* g = reinterpret_cast<const char*>(a.kept + row * a.hidden + c);
    const char* u = g + a.rows * a.hidden * 4;
    float dh[8], d[2][8];
#pragma unroll
    for (int k = 0; k < 8 / V; ++k) {
      float v[V];
      R::widen(__builtin_bit_cast(typename R::Raw, load_piece<S>(a.dh + row * a.dh_ld + (c + k * V) * S, n - k * V)), v);
#pragma unroll
      for (int j = 0; j < V; ++j) dh[k * V + j] = v[j];
    }
    u32x4 gw[2], uw[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      gw[k] = load_piece<4>(g + 16 * k, n - 4 * k);
      uw[k] = load_piece<4>(u + 16 * k, n - 4 * k);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) gates(dh[j], __uint_as_float(gw[j / 4][j % 4]), __uint_as_float(uw[j / 4][j % 4]), d[0][j], d[1][j]);
    const int64_t at = row * a.gu[0].ld + c * 2;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      char* out = static_cast<char*>(a.out[o]) + at;
      if constexpr (kWide) {
        const X3 parts = x3_split8([&](int j) { return d[o][j]; });
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>(out + p * a.gu[0].plane) = parts.p[p];
      } else {
        R::store(reinterpret_cast<typename R::Elem*>(out), d[o]);
      }
    }
  }
}

int gates_of_kept(const GatedArgs& a, int dtype, hipStream_t s) {
  const int64_t groups = ceil_div(a.rows * (a.gu[0].ld / 16), 256), most = 16 * static_cast<int64_t>(device_cus());
  const dim3 grid(static_cast<unsigned>(groups < most ? groups : most));
  if (dtype == OW_DTYPE_BF16) hipLaunchKernelGGL((gated_gates_kernel<BF16, BF16>), grid, dim3(256), 0, s, a);
  else if (dtype == OW_DTYPE_F16) hipLaunchKernelGGL((gated_gates_kernel<F16, F16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gated_gates_kernel<BF16, F32>), grid, dim3(256), 0, s, a);
  return hip_status(hipGetLastError(), "gated_gates_kernel launch");
}

GatedPlan plan_gates(const OwGatedLinear& d) {
  return gated_plan(d.rows, 2 * static_cast<int64_t>(d.hidden), gated_k_tiles(d.channels, d.dtype), 1, true, false);
}
GatedPlan plan_dx(const OwGatedLinear& d) { return gated_plan(d.rows, d.channels, 2 * gated_k_tiles(d.hidden, d.dtype), 1, false, true); }
GatedPlan plan_dw(const OwGatedLinear& d) { return gated_plan(d.hidden, d.channels, gated_k_tiles(d.rows, d.dtype), 2, false, true); }

// Bytes of x and the weights where they are copied, of a plane of dG and dU, and of the parts of dx or the weights' gradients.
struct Space {
  size_t operands, ld, plane, parts;
  int planes;
  size_t all() const { return operands + 2 * planes * plane + parts; }
};
Space space_of(const OwGatedLinear& d) {
  const size_t x = gated_partial_bytes(plan_dx(d)), w = gated_partial_bytes(plan_dw(d));
  Space s;
  s.operands = gated_operand_bytes(d);
  s.ld = static_cast<size_t>(ceil_div(d.hidden, 8)) * 16;
  s.plane = (static_cast<size_t>(d.rows) * s.ld + 255) / 256 * 256;
  s.parts = x > w ? x : w;
  s.planes = d.dtype == OW_DTYPE_F32 ? 3 : 1;
  return s;
}

}  // namespace
}  // namespace ow

extern "C" {

size_t ow_gated_linear_bwd_workspace(const OwGatedLinear* d) {
  if (d == nullptr || d->rows <= 0 || d->channels <= 0 || d->hidden <= 0) return 0;
  return ow::space_of(*d).all();
}

int ow_gated_linear_plan(const OwGatedLinear* d, int32_t product, OwGatedPlan* plan) {
  if (int rc = ow::check_gated(d)) return rc;
  OW_CHECK_ARG(plan != nullptr, "plan is NULL");
  OW_CHECK_ARG(product >= OW_GATED_FORWARD && product <= OW_GATED_DW, "unknown product %d", product);
  OW_CHECK_ARG(d->rows > 0 && d->channels > 0 && d->hidden > 0, "empty products have no plan");
  *plan = OwGatedPlan{};
  if (product != OW_GATED_FORWARD || !ow::gated_few(*d)) {
    const ow::GatedPlan p = product == OW_GATED_FORWARD ? ow::gated_plan_forward(*d)
                            : product == OW_GATED_GATES ? ow::plan_gates(*d)
                            : product == OW_GATED_DX    ? ow::plan_dx(*d)
                                                        : ow::plan_dw(*d);
    plan->tile_rows = ow::gated_tile_rows(p.size);
    plan->tile_cols = ow::gated_tile_cols(p.size);
    plan->parts = p.parts;
    plan->whole = p.whole;
    plan->cut = p.tiles_r * p.tiles_c - p.whole;
  }
  ow::clear_error();
  return OW_OK;
}

int ow_gated_linear_bwd(const OwGatedLinear* d, const void* kept, const void* dh, int64_t dh_stride, void* dx,
                        void* dgate_weight, void* dup_weight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check_gated(d)) return rc;
  OW_CHECK_ARG(d->rows > 0 && d->channels > 0 && d->hidden > 0, "the backward of empty products has no kernel");
  const int64_t size = d->dtype == OW_DTYPE_F32 ? 4 : 2;
  OW_CHECK_ARG(dh != nullptr && reinterpret_cast<uintptr_t>(dh) % size == 0, "dh is NULL or not aligned to its values");
  OW_CHECK_ARG(kept == nullptr || (ow_gated_linear_kept(d) != 0 && reinterpret_cast<uintptr_t>(kept) % 4 == 0),
               "the products of these sizes are not kept, or are not aligned to fp32 values");
  const ow::Space space = ow::space_of(*d);
  const size_t need = space.all();
  OW_CHECK_ARG(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "workspace of %zu bytes; %zu are needed, 16-byte aligned", workspace_bytes, need);
  const ow::GatedPlan gates = ow::plan_gates(*d), to_x = ow::plan_dx(*d), to_w = ow::plan_dw(*d);
  for (const ow::GatedPlan& p : {gates, to_x, to_w})
    OW_CHECK_SUPPORTED(p.units < (int64_t(1) << 31), "gated linear: too many tiles for a launch");
  hipStream_t s = static_cast<hipStream_t>(stream);
  ow::GatedArgs a{};
  char* ws = static_cast<char*>(workspace);
  if (int rc = ow::gated_operands(*d, ws, &a, s)) return rc;
  ws += space.operands;
  for (int i = 0; i < 2; ++i) {
    a.gu[i] = ow::GatedPlanes{ws, static_cast<int64_t>(space.ld), static_cast<int64_t>(space.plane)};
    a.out[i] = ws;
    ws += space.planes * space.plane;
  }
  float* partial = reinterpret_cast<float*>(ws);
  a.dh = static_cast<const char*>(dh);
  a.dh_ld = dh_stride * size;
  if (kept != nullptr) {
    a.kept = static_cast<float*>(const_cast<void*>(kept));
    if (int rc = ow::gates_of_kept(a, d->dtype, s)) return rc;
  } else {
    if (int rc = ow::launch_gated_mode<ow::kGatedGates>(a, gates, d->dtype, d->channels, partial, s)) return rc;
  }
  if (dx != nullptr) {
    a.out[0] = dx;
    if (int rc = ow::launch_gated_mode<ow::kGatedDx>(a, to_x, d->dtype, d->hidden, partial, s)) return rc;
  }
  if (dgate_weight != nullptr || dup_weight != nullptr) {
    a.out[0] = dgate_weight;
    a.out[1] = dup_weight;
    if (int rc = ow::launch_gated_mode<ow::kGatedDw>(a, to_w, d->dtype, d->rows, partial, s)) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
