// The gated feed-forward block's first half: both projections of rows of tokens, SiLU of the one and their product
// in one kernel (the backward: gated_linear_bwd.hip).
//
//   G = x Wg^T    U = x Wu^T    h = silu(G) U,  silu(g) = g / (1 + e^-g)
//
// Many tokens go through gated_tile_kernel (ow_gated.h): a tile's columns are 32 of the gate beside the same
// 32 of the other projection, so that a lane has both values of an output.  G and U are fp32 until h is rounded; for a
// backward to come they are stored as they are where that costs less than forming them again.
//
// Few tokens take gated_few_kernel, which is bound by reading the weights: a workgroup has 16 columns of both and up to 64
// tokens, its 8 waves take k in turns of 64 bytes a column and go from memory to the matrix cores without LDS; their sums meet there.
// One token of 1,024 to 2,048 f16: 4.8 us, 49 tokens bf16 6.6 (8.4 MB of weights, a copy's time 1.7: the rest is a launch,
// the latency of the first reads and the meeting of the waves); one token of 4,096 to 8,192 bf16 28.8, 4.7 TB/s.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "ow_gated.h"

namespace ow {
namespace {

constexpr int kFewRows = 64, kFewWaves = 8;

// Values of 16 bytes, of the few tokens' kernel, which takes fp32 as it is.
template <class Ty>
struct Elem {
  static constexpr int kSize = 2, kPiece = 8;
};
template <>
struct Elem<F32> {
  static constexpr int kSize = 4, kPiece = 4;
};

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
__global__ void __launch_bounds__(kFewWaves * 64, 2) gated_few_kernel(OwGatedLinear d, void* h_out, float* kept) {
  constexpr int S = Elem<Ty>::kSize, V = Elem<Ty>::kPiece, KS = 4 * V;  // k of a step
  __shared__ f32x4 part[kFewWaves][2 * TG][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, h = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, first = static_cast<int64_t>(blockIdx.y) * 16 * TG;  // token
  // Columns and tokens behind the last one are the last one; nobody stores them.
  const int64_t n = n0 + l16 < d.hidden ? n0 + l16 : d.hidden - 1, at_w = n * d.channels * S + h * 16;
  const char* w[2] = {static_cast<const char*>(d.gate_weight) + at_w, static_cast<const char*>(d.up_weight) + at_w};
  const char* x[TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) {
    const int64_t token = first + 16 * g + l16 < d.rows ? first + 16 * g + l16 : d.rows - 1;
    x[g] = static_cast<const char*>(d.x) + token * d.x_stride * S + h * 16;
  }
  f32x4 acc[2][TG];
#pragma unroll
  for (int g = 0; g < TG; ++g) acc[0][g] = acc[1][g] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int whole = d.channels / KS;
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
  if (whole * KS < d.channels && wave == whole % kFewWaves) {
    const int64_t at = static_cast<int64_t>(whole) * 64, left = d.channels - whole * KS - h * V;
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
    const int64_t row = first + 16 * g + (at & 15), col = n0 + 4 * (at >> 4) + e;
    if (row >= d.rows || col >= d.hidden) continue;
    if (kept != nullptr) kept[row * d.hidden + col] = G, kept[(d.rows + row) * d.hidden + col] = U;
    static_cast<typename Row<Ty>::Elem*>(h_out)[row * d.hidden + col] = Row<Ty>::from_f32(gated(G, U));
  }
}

template <class Ty>
void launch_few(const OwGatedLinear& d, void* h, float* kept, hipStream_t s) {
  // Fewer tokens a workgroup, where compute units would else be idle: each workgroup reads the weights' columns anew, but
  // less of x (49 tokens bf16: 1,024 to 2,048 in 64s 7.9 us, in 32s 6.6, in 16s, which is two rounds, 8.4; 2,048 to 1,024 in 64s
  // 12.6, in 16s 8.3; fp32 31 and 15).
  const int64_t columns = ceil_div(d.hidden, 16);
  int tokens = d.rows <= 16 ? 16 : d.rows <= 32 ? 32 : kFewRows;
  while (tokens > 16 && columns * ceil_div(d.rows, tokens / 2) <= device_cus()) tokens /= 2;
  const dim3 grid(static_cast<unsigned>(columns), static_cast<unsigned>(ceil_div(d.rows, tokens))), block(kFewWaves * 64);
  if (tokens == 16) hipLaunchKernelGGL((gated_few_kernel<Ty, 1>), grid, block, 0, s, d, h, kept);
  else if (tokens == 32) hipLaunchKernelGGL((gated_few_kernel<Ty, 2>), grid, block, 0, s, d, h, kept);
  else hipLaunchKernelGGL((gated_few_kernel<Ty, 4>), grid, block, 0, s, d, h, kept);
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

namespace {

// Rows of values, of any alignment, to planes of rows of whole pieces with zeros behind them: a copy of 16-bit values, or fp32
// ones in three bf16 parts.  A thread has a piece of 8 values; x and the weights go in one launch (blockIdx.y).
struct PackArgs {
  const char* src[3];
  int64_t src_ld[3], rows[3], plane[3];
  char* dst[3];
  int64_t ld;
  int32_t values;
};

template <bool WIDE>
__global__ void __launch_bounds__(256) gated_pack_kernel(PackArgs a) {
  const int o = blockIdx.y;
  const char* const src = a.src[o];
  const int64_t src_ld = a.src_ld[o], plane = a.plane[o];
  const uint32_t pieces = static_cast<uint32_t>(a.ld / 16);
  const int64_t all = a.rows[o] * pieces, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += step) {
    const int64_t row = i / pieces;
    const int c = static_cast<int>(i - row * pieces) * 8, n = a.values - c;
    char* out = a.dst[o] + row * a.ld + c * 2;
    if constexpr (WIDE) {
      const char* in = src + row * src_ld + static_cast<int64_t>(c) * 4;
      const u32x4 lo = load_piece<4>(in, n), hi = load_piece<4>(in + 16, n - 4);
      const X3 parts = x3_split8<true>([&](int j) { return __uint_as_float(j < 4 ? lo[j] : hi[j - 4]); });
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>(out + p * plane) = parts.p[p];
    } else {
      *reinterpret_cast<u32x4*>(out) = load_piece<2>(src + row * src_ld + static_cast<int64_t>(c) * 2, n);
    }
  }
}

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

int64_t row_bytes(int32_t values) { return ceil_div(values, 8) * 16; }

// Whether x, or both weights, can be read as they lie: 16-bit values in whole pieces, offsets inside a tile of 256 rows of 31 bits.
bool x_direct(const OwGatedLinear& d) {
  return d.dtype != OW_DTYPE_F32 && reinterpret_cast<uintptr_t>(d.x) % 16 == 0 && d.x_stride % 8 == 0 && d.x_stride >= 0 &&
         d.x_stride < (int64_t(1) << 21) && d.channels % 8 == 0;
}
bool w_direct(const OwGatedLinear& d) {
  return d.dtype != OW_DTYPE_F32 && d.channels % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(d.gate_weight) | reinterpret_cast<uintptr_t>(d.up_weight)) % 16 == 0;
}

}  // namespace

size_t gated_operand_bytes(const OwGatedLinear& d) {
  const size_t planes = d.dtype == OW_DTYPE_F32 ? 3 : 1, row = static_cast<size_t>(row_bytes(d.channels));
  return (x_direct(d) ? 0 : aligned(planes * d.rows * row)) + (w_direct(d) ? 0 : 2 * aligned(planes * d.hidden * row));
}

int gated_operands(const OwGatedLinear& d, char* workspace, GatedArgs* a, hipStream_t s) {
  const bool wide = d.dtype == OW_DTYPE_F32;
  const int64_t size = wide ? 4 : 2, ld = row_bytes(d.channels);
  a->rows = d.rows;
  a->channels = d.channels;
  a->hidden = d.hidden;
  a->x = GatedPlanes{static_cast<const char*>(d.x), d.x_stride * 2, 0};
  const void* weights[2] = {d.gate_weight, d.up_weight};
  for (int i = 0; i < 2; ++i) a->w[i] = GatedPlanes{static_cast<const char*>(weights[i]), d.channels * 2, 0};
  PackArgs pack{};
  int n = 0;
  const auto copy = [&](GatedPlanes* to, const void* src, int64_t src_ld, int64_t rows) {
    *to = GatedPlanes{workspace, ld, rows * ld};
    pack.src[n] = static_cast<const char*>(src);
    pack.src_ld[n] = src_ld;
    pack.rows[n] = rows;
    pack.plane[n] = rows * ld;
    pack.dst[n++] = workspace;
    workspace += aligned((wide ? 3 : 1) * rows * ld);
  };
  if (!x_direct(d)) copy(&a->x, d.x, d.x_stride * size, d.rows);
  if (!w_direct(d)) {
    for (int i = 0; i < 2; ++i) copy(&a->w[i], weights[i], d.channels * size, d.hidden);
  }
  if (n == 0) return OW_OK;
  pack.ld = ld;
  pack.values = d.channels;
  int64_t rows = 0;
  for (int i = 0; i < n; ++i) rows = pack.rows[i] > rows ? pack.rows[i] : rows;
  const int64_t groups = ceil_div(rows * (ld / 16), 256);
  const int64_t most = 16 * static_cast<int64_t>(device_cus());
  const dim3 grid(static_cast<unsigned>(groups < most ? groups : most), n);
  if (wide) hipLaunchKernelGGL((gated_pack_kernel<true>), grid, dim3(256), 0, s, pack);
  else hipLaunchKernelGGL((gated_pack_kernel<false>), grid, dim3(256), 0, s, pack);
  return hip_status(hipGetLastError(), "gated_pack_kernel launch");
}

// Whether gated_few_kernel takes the tokens (no workspace): 64 at most, or more where its workgroups, of 64 tokens and
// 16 columns, are one round of a GPU's 256 (bf16, 128 tokens of 1,024 to 2,048: 8.6 us, 9.8 in tiles; 192: 15.0 and 9.9), and fp32
// up to 128, which it takes without splitting the operands (2,048 to 4,096: 74 us, 78 in tiles; 192: 107 and 96).
bool gated_few(const OwGatedLinear& d) {
  if (d.rows <= kFewRows || (d.dtype == OW_DTYPE_F32 && d.rows <= 2 * kFewRows)) return true;
  return d.channels <= (d.dtype == OW_DTYPE_F32 ? 2048 : 1024) && ceil_div(d.hidden, 16) * ceil_div(d.rows, kFewRows) <= 256;
}

GatedPlan gated_plan_forward(const OwGatedLinear& d) {
  return gated_plan(d.rows, 2 * static_cast<int64_t>(d.hidden), gated_k_tiles(d.channels, d.dtype), 1, true, true);
}

}  // namespace ow

extern "C" {

// The products are kept where forming them again (4 K operations a value, six times as many for fp32) would take longer than
// to write and read them (16 bytes).  With few tokens, too: forward and backward of 49 tokens of 2,048 to 4,096 fp32 233 us
// with the products formed again, 130 with them kept; below those widths a call's host hides it.
size_t ow_gated_linear_kept(const OwGatedLinear* d) {
  if (d == nullptr || d->rows <= 0 || d->channels <= 0 || d->hidden <= 0) return 0;
  const int32_t from = d->dtype == OW_DTYPE_F32 ? 128 : 1536;
  return d->channels >= from ? static_cast<size_t>(2) * d->rows * d->hidden * sizeof(float) : 0;
}

size_t ow_gated_linear_fwd_workspace(const OwGatedLinear* d) {
  if (d == nullptr || ow::gated_few(*d) || d->channels <= 0 || d->hidden <= 0) return 0;
  return ow::gated_operand_bytes(*d) + ow::gated_partial_bytes(ow::gated_plan_forward(*d));
}

int ow_gated_linear_fwd(const OwGatedLinear* d, void* h, void* kept, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = ow::check_gated(d)) return rc;
  if (d->rows == 0 || d->hidden == 0) {
    ow::clear_error();
    return OW_OK;
  }
  OW_CHECK_ARG(d->channels > 0, "products over no channels have no kernel");
  OW_CHECK_ARG(h != nullptr, "h is NULL");
  OW_CHECK_ARG(kept == nullptr || (ow_gated_linear_kept(d) != 0 && reinterpret_cast<uintptr_t>(kept) % 4 == 0),
               "the products of these sizes are not kept, or have no place for fp32 values");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ow::gated_few(*d)) {
    if (d->dtype == OW_DTYPE_BF16) ow::launch_few<ow::BF16>(*d, h, static_cast<float*>(kept), s);
    else if (d->dtype == OW_DTYPE_F16) ow::launch_few<ow::F16>(*d, h, static_cast<float*>(kept), s);
    else ow::launch_few<ow::F32>(*d, h, static_cast<float*>(kept), s);
    if (int rc = ow::hip_status(hipGetLastError(), "gated_few_kernel launch")) return rc;
  } else {
    const ow::GatedPlan p = ow::gated_plan_forward(*d);
    OW_CHECK_SUPPORTED(p.units < (int64_t(1) << 31), "gated linear: too many tiles for a launch");
    const size_t need = ow_gated_linear_fwd_workspace(d), operands = ow::gated_operand_bytes(*d);
    OW_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "workspace of %zu bytes; %zu are needed, 16-byte aligned", workspace_bytes, need);
    ow::GatedArgs a{};
    char* ws = static_cast<char*>(workspace);
    if (int rc = ow::gated_operands(*d, ws, &a, s)) return rc;
    a.out[0] = h;
    a.kept = static_cast<float*>(kept);
    float* partial = reinterpret_cast<float*>(ws + operands);
    if (kept != nullptr) {
      if (int rc = ow::launch_gated_mode<ow::kGatedKeep>(a, p, d->dtype, d->channels, partial, s)) return rc;
    } else {
      if (int rc = ow::launch_gated_mode<ow::kGatedForward>(a, p, d->dtype, d->channels, partial, s)) return rc;
    }
  }
  ow::clear_error();
  return OW_OK;
}

}  // extern "C"
