// The gated feed-forward block's first half: both projections of rows of tokens, SiLU of the one and their product
// in one kernel (the backward: gated_linear_bwd.hip).
//
//   G = x Wg^T    U = x Wu^T    h = silu(G) U,  silu(g) = g / (1 + e^-g)
//
// Tokens enough for tiles go through gated_tile_kernel (ow_gated.h): a tile's columns are 32 of the gate beside the same
// 32 of the other projection, so that a lane has both values of an output.  G and U are never stored; they are fp32 until
// h is rounded.
//
// Up to 64 tokens take gated_few_kernel, which is bound by reading the weights: a workgroup has 16 columns of both,
// its 8 waves take k in turns of 64 bytes a column and go from memory to the matrix cores without LDS; their sums meet there.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_gated.h"

namespace ow {
namespace {

constexpr int kFewRows = 64, kFewWaves = 8;

template <class Ty>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) { return Ty::mma16k32(a, b, c); }
template <>
__device__ __forceinline__ f32x4 mma16<F32>(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  return c;
}

// TG: groups of 16 tokens.
template <class Ty, int TG>
__global__ void __launch_bounds__(kFewWaves * 64, 2) gated_few_kernel(GatedArgs a) {
  constexpr int S = Elem<Ty>::kSize, V = Elem<Ty>::kPiece, KS = 4 * V;  // k of a step
  __shared__ f32x4 part[kFewWaves][2 * TG][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, h = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  // Columns and tokens behind the last one are the last one; nobody stores them.
  const int64_t n = n0 + l16 < a.hidden ? n0 + l16 : a.hidden - 1, ld = static_cast<int64_t>(a.channels) * S;
  const char* w[2] = {a.w[0] + n * ld + h * 16, a.w[1] + n * ld + h * 16};
  const char* x[TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) x[g] = a.x + (16 * g + l16 < a.rows ? 16 * g + l16 : a.rows - 1) * a.x_ld + h * 16;
  f32x4 acc[2][TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) acc[0][g] = acc[1][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int whole = a.channels / KS;
  // Four steps' loads are in flight together.
  constexpr int U = 4;
  for (int s = wave; s < whole; s += U * kFewWaves) {
    u32x4 wg[U], wu[U], v[U][TG];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int step = s + u * kFewWaves;
      const int64_t at = static_cast<int64_t>(step) * 64;
      if (step < whole) {
        wg[u] = *reinterpret_cast<const u32x4_any*>(w[0] + at), wu[u] = *reinterpret_cast<const u32x4_any*>(w[1] + at);
#pragma unroll
        for (int g = 0; g < TG; ++g) v[u][g] = *reinterpret_cast<const u32x4_any*>(x[g] + at);
      } else {
        wg[u] = wu[u] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int g = 0; g < TG; ++g) v[u][g] = u32x4{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < TG; ++g) {
        acc[0][g] = mma16<Ty>(wg[u], v[u][g], acc[0][g]);
        acc[1][g] = mma16<Ty>(wu[u], v[u][g], acc[1][g]);
      }
  }
  if (whole * KS < a.channels && wave == whole % kFewWaves) {
    const int64_t at = static_cast<int64_t>(whole) * 64, left = a.channels - whole * KS - h * V;
    const u32x4 wg = load_piece<S>(w[0] + at, left), wu = load_piece<S>(w[1] + at, left);
#pragma unroll
    for (int g = 0; g < TG; ++g) {
      const u32x4 v = load_piece<S>(x[g] + at, left);
      acc[0][g] = mma16<Ty>(wg, v, acc[0][g]);
      acc[1][g] = mma16<Ty>(wu, v, acc[1][g]);
    }
  }
  mfma_drain();
#pragma unroll
  for (int g = 0; g < TG; ++g) part[wave][g][lane] = acc[0][g], part[wave][TG + g][lane] = acc[1][g];
  __syncthreads();
  // A thread has one output: value e of lane `at` of a group, column 4 (at / 16) + e of token at % 16.
  for (int i = threadIdx.x; i < 256 * TG; i += kFewWaves * 64) {
    const int g = i >> 8, at = (i & 255) >> 2, e = i & 3;
    float G = 0.f, U = 0.f;
#pragma unroll
    for (int k = 0; k < kFewWaves; ++k) G += part[k][g][at][e], U += part[k][TG + g][at][e];
    const int64_t row = 16 * g + (at & 15), col = n0 + 4 * (at >> 4) + e;
    if (row >= a.rows || col >= a.hidden) continue;
    static_cast<typename Row<Ty>::Elem*>(a.out[0])[row * a.hidden + col] = Row<Ty>::from_f32(G * U * sigmoid(G));
  }
}

template <class Ty>
void launch_few(const GatedArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.hidden, 16))), block(kFewWaves * 64);
  if (a.rows <= 16) hipLaunchKernelGGL((gated_few_kernel<Ty, 1>), grid, block, 0, s, a);
  else if (a.rows <= 32) hipLaunchKernelGGL((gated_few_kernel<Ty, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gated_few_kernel<Ty, 4>), grid, block, 0, s, a);
}

}  // namespace

int check_gated(const OwGatedLinear* d) {
  OW_CHECK_ARG(d != nullptr, "gated linear descriptor is NULL");
  OW_CHECK_SUPPORTED(d->dtype == OW_DTYPE_F32 || d->dtype == OW_DTYPE_BF16 || d->dtype == OW_DTYPE_F16,
                     "gated linear: dtype %d; expected f32, bf16 or f16", d->dtype);
  OW_CHECK_ARG(d->rows >= 0 && d->channels >= 0 && d->hidden >= 0, "negative size");
  OW_CHECK_SUPPORTED(d->channels <= kGatedMost && d->hidden <= kGatedMost, "gated linear: %d channels, %d hidden; at most %d",
                     d->channels, d->hidden, kGatedMost);
  OW_CHECK_SUPPORTED(d->rows < (int64_t(1) << 31), "gated linear: %lld rows; fewer than 2^31 are supported",
                     static_cast<long long>(d->rows));
  if (d->rows == 0 || d->hidden == 0 || d->channels == 0) return OW_OK;
  OW_CHECK_ARG(d->x != nullptr && d->gate_weight != nullptr && d->up_weight != nullptr, "x or a weight is NULL");
  const int64_t size = d->dtype == OW_DTYPE_F32 ? 4 : 2;
  OW_CHECK_ARG(reinterpret_cast<uintptr_t>(d->x) % size == 0 && reinterpret_cast<uintptr_t>(d->gate_weight) % size == 0 &&
                   reinterpret_cast<uintptr_t>(d->up_weight) % size == 0,
               "x or a weight is not aligned to its values");
  return OW_OK;
}

GatedArgs gated_args(const OwGatedLinear& d) {
  GatedArgs a{};
  const int64_t size = d.dtype == OW_DTYPE_F32 ? 4 : 2, piece = 16 / size;
  a.x = static_cast<const char*>(d.x);
  a.w[0] = static_cast<const char*>(d.gate_weight);
  a.w[1] = static_cast<const char*>(d.up_weight);
  a.x_ld = d.x_stride * size;
  a.rows = d.rows;
  a.channels = d.channels;
  a.hidden = d.hidden;
  a.ld_gu = static_cast<int32_t>(ceil_div(d.hidden, piece) * piece);
  return a;
}

// Whether x, or both weights, lie in whole pieces of 16 bytes; offsets inside a tile of 256 rows have 31 bits.
bool gated_x_direct(const GatedArgs& a, int64_t size) {
  return reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_ld % 16 == 0 && a.x_ld >= 0 && a.x_ld < (int64_t(1) << 22) &&
         a.channels * size % 16 == 0;
}
bool gated_w_direct(const GatedArgs& a, int64_t size) {
  return (reinterpret_cast<uintptr_t>(a.w[0]) | reinterpret_cast<uintptr_t>(a.w[1])) % 16 == 0 && a.channels * size % 16 == 0;
}

void apply_plan(GatedArgs& a, const GatedPlan& p) {
  a.tiles_r = p.tiles_r;
  a.tiles_c = p.tiles_c;
  a.splits = p.splits;
  a.k_tiles = p.k_tiles;
  a.k_split = p.k_split;
  // (Numbers past 2^31 are refused before a launch.)
  a.by_tiles = Divisor::of(static_cast<uint32_t>(p.tiles_r * p.tiles_c));
  a.by_group = Divisor::of(8 * static_cast<uint32_t>(p.tiles_c));
}

}  // namespace ow

extern "C" {

// The products are kept where forming them again (4 K operations a value) would take longer than to write and read them (16 bytes).
size_t ow_gated_linear_kept(const OwGatedLinear* d) {
  if (d == nullptr || d->rows <= ow::kFewRows || d->channels <= 0 || d->hidden <= 0) return 0;
  const int32_t from = d->dtype == OW_DTYPE_F32 ? 128 : 1536;
  return d->channels >= from ? static_cast<size_t>(2) * d->rows * d->hidden * sizeof(float) : 0;
}

int ow_gated_linear_fwd(const OwGatedLinear* d, void* h, void* kept, void* stream) {
  if (int rc = ow::check_gated(d)) return rc;
  if (d->rows == 0 || d->hidden == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG(d->channels > 0, "products over no channels have no kernel");
  OW_CHECK_ARG(h != nullptr, "h is NULL");
  OW_CHECK_ARG(kept == nullptr || (ow_gated_linear_kept(d) != 0 && reinterpret_cast<uintptr_t>(kept) % 4 == 0),
               "the products of these sizes are not kept, or have no place for fp32 values");
  ow::GatedArgs a = ow::gated_args(*d);
  a.out[0] = h;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->rows <= ow::kFewRows) {
    if (d->dtype == OW_DTYPE_BF16) ow::launch_few<ow::BF16>(a, s);
    else if (d->dtype == OW_DTYPE_F16) ow::launch_few<ow::F16>(a, s);
    else ow::launch_few<ow::F32>(a, s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_few_kernel launch")) return rc;
  } else {
    const int64_t size = d->dtype == OW_DTYPE_F32 ? 4 : 2;
    const ow::GatedPlan p = ow::gated_plan(d->rows, 2 * static_cast<int64_t>(d->hidden), ow::ceil_div(d->channels * size, 128), 1, false, size == 4);
    OW_CHECK_SUPPORTED(p.tiles_r * p.tiles_c < (int64_t(1) << 31), "gated linear: too many tiles for a launch");
    ow::apply_plan(a, p);
    a.kept = static_cast<float*>(kept);
    const bool direct = ow::gated_x_direct(a, size) && ow::gated_w_direct(a, size);
    if (kept != nullptr) ow::launch_gated_mode<ow::kGatedKeep>(a, p.size, d->dtype, direct, s);
    else ow::launch_gated_mode<ow::kGatedForward>(a, p.size, d->dtype, direct, s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
