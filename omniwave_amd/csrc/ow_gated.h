// Tiles of the gated feed-forward products (gated_linear.hip, gated_linear_bwd.hip): one matrix product kernel in which
// an output tile O[r][c] = sum_k R[r][k] C[c][k] is formed by MFMA from tiles of both operands in LDS.
//
// An operand lies in memory with its contraction index contiguous (kAlongK: x and the weights forward, the gates'
// gradients in dx) or with its output index contiguous (kAcrossK: the weights in dx, every operand of the weights'
// gradients).  The tile in LDS keeps that order, in pieces of 16 bytes:
//
//   kAlongK    rows of 128 bytes (64 values of 16 bits, 32 of fp32); piece p of row r at slot p ^ (r & 7), so that eight
//              rows' pieces of one column fall in eight bank windows; a lane reads its 16 bytes of k at once
//   kAcrossK   a row for each k; 16-bit values are read transposed (ds_read_b64_tr_b16: 4 k of 16 output indexes by
//              16 lanes), 32-byte pairs of row k at pair ^ (k & 7), fp32 values one by one, rows with k & 4 moved by 128 bytes
//
// A step takes 16 bytes of k from each half of the wave: one 32x32x16 MFMA for 16-bit types, four 32x32x2 for fp32.  Its A operand is
// C, its B operand R: a lane then has 16 values of one row r, in runs of 4 along c, and two halves exchange runs
// (permlane32_swap) to store 16 bytes.
//
// Tiles come by direct copies into LDS (16 bytes a lane; what lies outside the matrix reads as zeros), one tile ahead
// of the products: 128 KB for both stages of 256 x 256, one workgroup of 8 waves a compute unit.  Operands that do not lie in whole 16-byte
// pieces come through registers instead, value by value at the ends of rows.
#pragma once

#include "ow_rows.h"

namespace ow {

constexpr int kGatedMost = 1 << 20;  // channels, hidden

enum GatedMode {
  kGatedForward,  // h = silu(x Wg^T) (x Wu^T)
  kGatedGates,    // dG and dU, with both products formed again
  kGatedDx,       // dG Wg + dU Wu
  kGatedDw,       // dG^T x, dU^T x
};

struct GatedArgs {
  const char* x;
  const char* w[2];   // gate, up
  const char* dh;
  const char* dgu[2]; // dG, dU: [rows][ld_gu]
  int64_t x_ld, dh_ld;  // bytes
  void* out[2];       // h; dG, dU; dx; dgate, dup
  float* partial;     // [splits][outputs], fp32; used where splits > 1
  int64_t rows;
  int32_t channels, hidden, ld_gu;  // ld_gu: hidden, up to whole 16-byte pieces
  int64_t tiles_r;
  int32_t tiles_c, splits;
  int64_t k_tiles, k_split;  // tiles of k in all, and of a split
};

// Geometry of a tile: WR x WC waves, each RI x CI products of 32 x 32.
template <int WR_, int WC_, int RI_, int CI_>
struct Tile {
  static constexpr int WR = WR_, WC = WC_, RI = RI_, CI = CI_;
  static constexpr int BR = WR * RI * 32, BC = WC * CI * 32, kWaves = WR * WC, kThreads = kWaves * 64;
  static constexpr int kBytesR = BR * 128, kBytesC = BC * 128;  // of one stage
};
typedef Tile<2, 4, 4, 2> TileL;  // 256 x 256
typedef Tile<2, 2, 2, 2> TileM;  // 128 x 128
typedef Tile<2, 2, 1, 2> TileS;  // 64 x 128

// Element types: K values of a 128-byte row, values of a 16-byte piece, one step's product.
template <class Ty>
struct Elem {  // BF16, F16
  static constexpr int kSize = 2, kPiece = 8, kTile = 64, kProducts = 1;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) { return Ty::mma32(a, b, c); }
};
template <>
struct Elem<F32> {
  static constexpr int kSize = 4, kPiece = 4, kTile = 32, kProducts = 4;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
};

// Up to n values of `size` bytes at p as 16 bytes, zeros behind them; p may have any alignment that a value may have.
template <int SIZE>
__device__ __forceinline__ u32x4 load_piece(const char* p, int64_t n) {
  constexpr int V = 16 / SIZE;
  if (n >= V) return *reinterpret_cast<const u32x4_any*>(p);
  u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j >= n) break;
    if constexpr (SIZE == 2) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (16 * (j & 1));
    else w[j] = reinterpret_cast<const uint32_t*>(p)[j];
  }
  return w;
}

// A lane's pieces of an operand on their way to LDS.  DIRECT: `off` is each one's offset from the tile's base, kOffOut where
// its index is outside the matrix; else offsets of any size, and what has been loaded.
template <int COPIES, bool DIRECT>
struct Pieces {
  uint32_t off[COPIES];
};
template <int COPIES>
struct Pieces<COPIES, false> {
  int64_t off[COPIES];
  int left[COPIES];  // values that are in the matrix
  u32x4 held[COPIES];
};
__device__ __forceinline__ void put_piece(uint32_t lds, int lane, u32x4 v) {
  *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(static_cast<uintptr_t>(lds + 16 * lane)) = v;
}

// A tile of N output indexes, 128 bytes of k each: 1 KB (8 rows) an instruction.  PAIR: 32 of one matrix and 32 of the
// other in turn.
template <int N, int WAVES, int SIZE, bool DIRECT, bool PAIR>
struct AlongK {
  static constexpr int kCopies = N / 8 / WAVES, kReads = 1, V = 16 / SIZE;
  static_assert(kCopies * 8 * WAVES == N && (!PAIR || 32 % (8 * WAVES) == 0 || 8 * WAVES == 64), "whole copies of one matrix");
  Pieces<kCopies, DIRECT> at;
  int piece;  // of a row
  static __device__ __forceinline__ int part(int i, int wave) { return PAIR ? ((8 * (i * WAVES + wave)) >> 5) & 1 : 0; }
  // extent: indexes from the tile's first one on.
  __device__ __forceinline__ void init(int64_t extent, int64_t ld, int wave, int lane) {
    piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int q = 8 * (i * WAVES + wave), index = (PAIR ? (q >> 6) * 32 + (q & 31) : q) + (lane >> 3);
      if constexpr (DIRECT) {
        at.off[i] = index < extent ? static_cast<uint32_t>(index * ld) + piece * 16 : kOffOut;
      } else {
        at.off[i] = index * ld + piece * 16;
        at.left[i] = index < extent;
      }
    }
  }
  // base: the tile's first index of each matrix at the tile's k; k_left: values of k that are there, up to a tile's.
  __device__ __forceinline__ void fetch(const char* base, const char* other, int k_left, uint32_t lds, int wave) {
    if constexpr (DIRECT) {
      const auto r0 = buffer_rsrc(base, 0x7fffffffu), r1 = buffer_rsrc(PAIR ? other : base, 0x7fffffffu);
      const bool there = piece * V < k_left;
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        tile_copy(part(i, wave) ? r1 : r0, there ? at.off[i] : kOffOut, lds + 8 * (i * WAVES + wave) * 128);
    } else {
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        at.held[i] = load_piece<SIZE>((part(i, wave) ? other : base) + at.off[i], at.left[i] ? k_left - piece * V : 0);
    }
  }
  __device__ __forceinline__ void put(uint32_t lds, int wave, int lane) const {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) put_piece(lds + 8 * (i * WAVES + wave) * 128, lane, at.held[i]);
    }
  }
  template <class Ty>
  static __device__ __forceinline__ u32x4 read(uint32_t lds, int first, int step, int lane) {
    const int l32 = lane & 31, hh = lane >> 5;
    const uint32_t at = lds + (first + l32) * 128 + (((2 * step + hh) ^ (l32 & 7)) << 4);
    return *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(static_cast<uintptr_t>(at));
  }
};

// A tile of 128 / SIZE values of k, N output indexes each.
template <int N, int WAVES, int SIZE, bool DIRECT>
struct AcrossK {
  static constexpr int kRow = N * SIZE, kPieces = kRow / 16;   // of a k
  static constexpr int kRowsOfCopy = 64 / kPieces > 0 ? 64 / kPieces : 1;
  static constexpr int kCopies = N / 8 / WAVES, kReads = SIZE, V = 16 / SIZE;
  static_assert(kRow <= 1024 && kCopies * 8 * WAVES == N, "whole copies");
  Pieces<kCopies, DIRECT> at;
  int in;  // the lane's k of a copy
  static constexpr int kPairs = kPieces / 2 < 8 ? kPieces / 2 : 8;
  static __device__ __forceinline__ int slot(int p, int k) {
    if constexpr (SIZE == 2) return p ^ ((k & (kPairs - 1)) << 1);
    else return p ^ ((k & 4) << 1);
  }
  // n_out: output indexes from the tile's first one on.
  __device__ __forceinline__ void init(int64_t n_out, int64_t ld, int wave, int lane) {
    in = lane / kPieces;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int k = (i * WAVES + wave) * kRowsOfCopy + in, p = slot(lane % kPieces, k);
      if constexpr (DIRECT) {
        at.off[i] = p * V < n_out ? static_cast<uint32_t>(k * ld) + p * 16 : kOffOut;
      } else {
        at.off[i] = k * ld + p * 16;
        at.left[i] = n_out - p * V < V ? static_cast<int>(n_out - p * V) : V;
      }
    }
  }
  // base: the first output index at the tile's k; k_left: values of k that are there, up to a tile's.
  __device__ __forceinline__ void fetch(const char* base, int k_left, uint32_t lds, int wave) {
    const auto r = buffer_rsrc(base, 0x7fffffffu);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int copy = i * WAVES + wave;
      const bool there = in < k_left - copy * kRowsOfCopy;
      if constexpr (DIRECT) tile_copy(r, there ? at.off[i] : kOffOut, lds + copy * 1024);
      else at.held[i] = load_piece<SIZE>(base + at.off[i], there ? at.left[i] : 0);
    }
  }
  __device__ __forceinline__ void put(uint32_t lds, int wave, int lane) const {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) put_piece(lds + (i * WAVES + wave) * 1024, lane, at.held[i]);
    }
  }
  template <class Ty>
  static __device__ __forceinline__ u32x4 read(uint32_t lds, int first, int step, int lane) {
    const int l32 = lane & 31, hh = lane >> 5, l16 = lane & 15;
    if constexpr (SIZE == 2) {
      const int c = first + 16 * ((lane >> 4) & 1) + 4 * (l16 & 3);
      const int k = 16 * step + 8 * hh + (l16 >> 2);
      const auto at = [&](int kk) { return lds + kk * kRow + (slot(c >> 3, kk) << 4) + ((c & 4) << 1); };
      const u32x2 a = lds_read_tr16(at(k)), b = lds_read_tr16(at(k + 4));
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 8 * step + 4 * hh + j, c = first + l32;
        const uint32_t at = lds + k * kRow + (slot(c >> 2, k) << 4) + ((c & 3) << 2);
        v[j] = *reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(static_cast<uintptr_t>(at));
      }
      return v;
    }
  }
};

// Runs of 4 values along c of one row, as a product's lane has them, stored as 16 bytes a lane: run g of lane (l32, hh)
// is c0 + 8 g + 4 hh.
template <class Ty>
struct RunStore {  // BF16, F16
  // row: the row's first value; n: its values from c0 on
  static __device__ __forceinline__ void store(void* row, int64_t c0, int64_t n, const float (&v)[16], int hh) {
    uint16_t* out = static_cast<uint16_t*>(row) + c0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const auto s = __builtin_amdgcn_permlane32_swap(Ty::pack2(v[8 * p + 2 * j], v[8 * p + 2 * j + 1]),
                                                        Ty::pack2(v[8 * p + 4 + 2 * j], v[8 * p + 5 + 2 * j]), false, false);
        w[j] = s[0], w[2 + j] = s[1];
      }
      const int c = 16 * p + 8 * hh;
      if (c + 8 <= n) {
        *reinterpret_cast<u32x4_any*>(out + c) = u32x4{w[0], w[1], w[2], w[3]};
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < n) out[c + j] = j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]);
      }
    }
  }
};
template <>
struct RunStore<F32> {
  static __device__ __forceinline__ void store(void* row, int64_t c0, int64_t n, const float (&v)[16], int hh) {
    float* out = static_cast<float*>(row) + c0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 8 * g + 4 * hh;
      if (c + 4 <= n) {
        *reinterpret_cast<f32x4_any*>(out + c) = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < n) out[c + j] = v[4 * g + j];
      }
    }
  }
};

// Runs of a row as RunStore has them, zeros outside.
template <class Ty>
__device__ __forceinline__ void load_runs(const char* row, int64_t c0, int64_t n, int hh, float (&v)[16]) {
  constexpr int S = Elem<Ty>::kSize;
  typedef u32x2 __attribute__((aligned(2))) u32x2_any;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int c = 8 * g + 4 * hh;
    const char* p = row + (c0 + c) * S;
    if constexpr (S == 4) {
      const u32x4 w = load_piece<4>(p, n - c);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * g + j] = __uint_as_float(w[j]);
    } else if (c + 4 <= n) {
      const u32x2 w = *reinterpret_cast<const u32x2_any*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * g + j] = Ty::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * g + j] = c + j < n ? Ty::to_f32(reinterpret_cast<const uint16_t*>(p)[j]) : 0.f;
    }
  }
}

// silu(g) u = g u / (1 + e^-g)
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(kNegLog2e * g)); }

// Workgroups of an XCD take neighbouring tiles (round-robin dispatch), in groups of 8 rows of tiles.
__device__ __forceinline__ int64_t xcd_tile(int64_t id, int64_t n) {
  const int64_t xcd = id & 7, at = id >> 3, per = n >> 3, rem = n & 7;
  return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + at;
}

template <class Ty, int MODE, class T, bool DIRECT>
__global__ void __launch_bounds__(T::kThreads, 2) gated_tile_kernel(GatedArgs a) {
  constexpr int S = Elem<Ty>::kSize, KT = Elem<Ty>::kTile, W = T::kWaves;
  constexpr bool kPair = MODE == kGatedForward || MODE == kGatedGates;  // columns: 32 of the gate, 32 of the other
  constexpr int kCols = kPair ? T::BC / 2 : T::BC;                      // output columns of a tile
  typedef typename std::conditional<MODE == kGatedDw, AcrossK<T::BR, W, S, DIRECT>, AlongK<T::BR, W, S, DIRECT, false>>::type OpR;
  typedef typename std::conditional<kPair, AlongK<T::BC, W, S, DIRECT, true>, AcrossK<T::BC, W, S, DIRECT>>::type OpC;
  __shared__ __attribute__((aligned(1024))) char lds[2][T::kBytesR + T::kBytesC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hh = lane >> 5;

  const int64_t tiles = a.tiles_r * a.tiles_c;
  const int64_t id = xcd_tile(blockIdx.x, tiles * a.splits);
  const int64_t split = id / tiles, tile = id % tiles;
  constexpr int kGroup = 8;
  const int64_t group = tile / (kGroup * static_cast<int64_t>(a.tiles_c)), in = tile % (kGroup * static_cast<int64_t>(a.tiles_c));
  const int64_t left = a.tiles_r - group * kGroup, high = left < kGroup ? left : kGroup;
  const int64_t tile_r = group * kGroup + in % high;
  const int tile_c = static_cast<int>(in / high);
  // The weights' gradients: the first half of the rows of tiles is the gate's.
  const int64_t half_r = a.tiles_r / 2;
  const int which = MODE == kGatedDw && tile_r >= half_r ? 1 : 0;
  const int64_t r0 = (MODE == kGatedDw ? tile_r - which * half_r : tile_r) * T::BR;
  const int64_t c0 = static_cast<int64_t>(tile_c) * kCols;

  const int64_t kt_begin = split * a.k_split;
  const int64_t kt_end = kt_begin + a.k_split < a.k_tiles ? kt_begin + a.k_split : a.k_tiles;

  OpR op_r;
  OpC op_c;
  const int64_t ld_w = static_cast<int64_t>(a.channels) * S, ld_gu = static_cast<int64_t>(a.ld_gu) * S;
  if constexpr (kPair) {
    op_r.init(a.rows - r0, a.x_ld, wave, lane);
    op_c.init(a.hidden - c0, ld_w, wave, lane);
  } else if constexpr (MODE == kGatedDx) {
    op_r.init(a.rows - r0, ld_gu, wave, lane);
    op_c.init(a.channels - c0, ld_w, wave, lane);
  } else {
    op_r.init(a.ld_gu - r0, ld_gu, wave, lane);
    op_c.init(a.channels - c0, a.x_ld, wave, lane);
  }
  // Tiles behind the last one read as zeros (nobody uses them: the loop needs no branch).
  auto fetch = [&](int64_t kt, int stage) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
    const auto left = [&](int64_t k) { return kt >= kt_end ? 0 : k < KT ? static_cast<int>(k) : KT; };
    if constexpr (kPair) {
      const int k_left = left(a.channels - kt * KT);
      op_r.fetch(a.x + r0 * a.x_ld + kt * 128, nullptr, k_left, at_r, wave);
      op_c.fetch(a.w[0] + c0 * ld_w + kt * 128, a.w[1] + c0 * ld_w + kt * 128, k_left, at_c, wave);
    } else if constexpr (MODE == kGatedDx) {
      const int64_t each = a.k_tiles / 2;
      const int w = kt >= each;
      const int64_t k0 = (kt - w * each) * KT;
      op_r.fetch(a.dgu[w] + r0 * ld_gu + k0 * S, nullptr, left(a.ld_gu - k0), at_r, wave);
      op_c.fetch(a.w[w] + k0 * ld_w + c0 * S, left(a.hidden - k0), at_c, wave);
    } else {
      const int64_t k0 = kt * KT;
      const int k_left = left(a.rows - k0);
      op_r.fetch(a.dgu[which] + k0 * ld_gu + r0 * S, k_left, at_r, wave);
      op_c.fetch(a.x + k0 * a.x_ld + c0 * S, k_left, at_c, wave);
    }
  };
  auto put = [&](int stage) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
    op_r.put(at_r, wave, lane);
    op_c.put(at_c, wave, lane);
  };

  f32x16 acc[T::CI][T::RI];
#pragma unroll
  for (int i = 0; i < T::CI; ++i)
#pragma unroll
    for (int j = 0; j < T::RI; ++j) acc[i][j] = f32x16{};
  const int wr = wave / T::WC * (T::RI * 32), wc = wave % T::WC * (T::CI * 32);

  u32x4 fr[2][T::RI], fc[2][T::CI];
  auto read = [&](int stage, int s, int buf) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
#pragma unroll
    for (int i = 0; i < T::CI; ++i) fc[buf][i] = OpC::template read<Ty>(at_c, wc + 32 * i, s, lane);
#pragma unroll
    for (int j = 0; j < T::RI; ++j) fr[buf][j] = OpR::template read<Ty>(at_r, wr + 32 * j, s, lane);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int j = 0; j < T::RI; ++j)
#pragma unroll
      for (int i = 0; i < T::CI; ++i) acc[i][j] = Elem<Ty>::mma(fc[buf][i], fr[buf][j], acc[i][j]);
  };
  constexpr int kCopies = OpR::kCopies + OpC::kCopies;
  // A step's reads go between its products, one after each; left alone, the compiler puts them right before their use.
  constexpr int kReads = T::CI * OpC::kReads + T::RI * OpR::kReads, kProducts = T::CI * T::RI * Elem<Ty>::kProducts;
  auto interleave = [&]() {
    constexpr int kEach = kProducts / kReads > 0 ? kProducts / kReads : 1;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read of LDS
      __builtin_amdgcn_sched_group_barrier(0x8, kEach, 0);  // products
    }
    if constexpr (kProducts > kReads * kEach) __builtin_amdgcn_sched_group_barrier(0x8, kProducts - kReads * kEach, 0);
    __builtin_amdgcn_sched_barrier(0);
  };

  // Operands of a step are read while the step before it is multiplied, those of a tile's first step during the
  // last one of the tile before: at that point the next tile has arrived, all of this one is in registers, and
  // the tile after the next takes its place.
  fetch(kt_begin, 0);
  if constexpr (DIRECT) {
    fetch(kt_begin + 1, 1);
    wait_vmcnt<kCopies>();
  } else {
    put(0);
    fetch(kt_begin + 1, 1);
  }
  __syncthreads();
  read(0, 0, 0);
  for (int64_t kt = kt_begin; kt < kt_end; ++kt) {
    const int stage = static_cast<int>((kt - kt_begin) & 1);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      read(stage, s + 1, (s + 1) & 1);
      multiply(s & 1);
      interleave();
    }
    if constexpr (DIRECT) wait_vmcnt<0>();
    else put(stage ^ 1);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    read(stage ^ 1, 0, 0);
    fetch(kt + 2, stage);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }
  // No copy may still be on its way when the workgroup ends.
  wait_vmcnt<0>();
  mfma_drain();

  if constexpr (kPair) {
    const int64_t c = c0 + (wc >> 1), n = (MODE == kGatedGates ? a.ld_gu : a.hidden) - c;
#pragma unroll
    for (int j = 0; j < T::RI; ++j) {
      const int64_t r = r0 + wr + 32 * j + l32;
      const bool there = r < a.rows;
      if constexpr (MODE == kGatedForward) {
        float h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = acc[0][j][i] * acc[1][j][i] * sigmoid(acc[0][j][i]);
        RunStore<Ty>::store(static_cast<char*>(a.out[0]) + r * a.hidden * S, c, there ? n : 0, h, hh);
      } else {
        // Columns up to a whole piece are written: there both products are 0.  The gradients of G and U are
        // rounded to the operands' type here, as the products that take them need it (fp32 stays fp32).
        float dh[16], dg[16], du[16];
        load_runs<Ty>(a.dh + r * a.dh_ld, c, there ? a.hidden - c : 0, hh, dh);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float g = acc[0][j][i], u = acc[1][j][i], s = sigmoid(g);
          du[i] = dh[i] * (g * s);
          dg[i] = dh[i] * u * (s * (1.f + g * (1.f - s)));
        }
        const int64_t at = r * a.ld_gu * S;
        RunStore<Ty>::store(static_cast<char*>(a.out[0]) + at, c, there ? n : 0, dg, hh);
        RunStore<Ty>::store(static_cast<char*>(a.out[1]) + at, c, there ? n : 0, du, hh);
      }
    }
  } else {
    const int64_t n_r = MODE == kGatedDw ? a.hidden : a.rows;
#pragma unroll
    for (int j = 0; j < T::RI; ++j) {
      const int64_t r = r0 + wr + 32 * j + l32;
#pragma unroll
      for (int i = 0; i < T::CI; ++i) {
        const int64_t c = c0 + wc + 32 * i, n = r < n_r ? a.channels - c : 0;
        if (a.splits == 1 && a.out[which] == nullptr) continue;  // one weight's gradient is not asked for
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
        if (a.splits > 1) {
          const int64_t at = ((split * (MODE == kGatedDw ? 2 : 1) + which) * n_r + r) * a.channels;
          RunStore<F32>::store(a.partial + at, c, n, v, hh);
        } else {
          RunStore<Ty>::store(static_cast<char*>(a.out[which]) + r * a.channels * S, c, n, v, hh);
        }
      }
    }
  }
}

// Tiles of a launch.
struct GatedPlan {
  int size;  // 0: TileL, 1: TileM, 2: TileS
  int64_t tiles_r;
  int32_t tiles_c, splits;
  int64_t k_tiles, k_split;
};

template <class Ty, int MODE, bool DIRECT>
void launch_gated(const GatedArgs& a, int size, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.tiles_r * a.tiles_c * a.splits));
  if (size == 0) hipLaunchKernelGGL((gated_tile_kernel<Ty, MODE, TileL, DIRECT>), grid, dim3(TileL::kThreads), 0, s, a);
  else if (size == 1) hipLaunchKernelGGL((gated_tile_kernel<Ty, MODE, TileM, DIRECT>), grid, dim3(TileM::kThreads), 0, s, a);
  else hipLaunchKernelGGL((gated_tile_kernel<Ty, MODE, TileS, DIRECT>), grid, dim3(TileS::kThreads), 0, s, a);
}

template <int MODE>
void launch_gated_mode(const GatedArgs& a, int size, int dtype, bool direct, hipStream_t s) {
  if (dtype == OW_DTYPE_BF16) return direct ? launch_gated<BF16, MODE, true>(a, size, s) : launch_gated<BF16, MODE, false>(a, size, s);
  if (dtype == OW_DTYPE_F16) return direct ? launch_gated<F16, MODE, true>(a, size, s) : launch_gated<F16, MODE, false>(a, size, s);
  return direct ? launch_gated<F32, MODE, true>(a, size, s) : launch_gated<F32, MODE, false>(a, size, s);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows and columns of a tile's operands (gate and up columns together).
inline int gated_tile_rows(int size) { return size == 0 ? TileL::BR : size == 1 ? TileM::BR : TileS::BR; }
inline int gated_tile_cols(int size) { return size == 0 ? TileL::BC : size == 1 ? TileM::BC : TileS::BC; }

// The largest tile that still gives every compute unit one; `rows` x `cols` outputs (cols: gate and up together), and
// where even the smallest leave compute units without work, a k that is cut into `most` parts at most.
inline GatedPlan gated_plan(int64_t rows, int64_t cols, int64_t k_tiles, int row_sets, bool can_split) {
  const int64_t cus = device_cus();
  GatedPlan p;
  for (p.size = 0; p.size < 2; ++p.size)
    if (ceil_div(rows, gated_tile_rows(p.size)) * row_sets * ceil_div(cols, gated_tile_cols(p.size)) >= cus) break;
  if (can_split && p.size == 2) p.size = 1;
  p.tiles_r = ceil_div(rows, gated_tile_rows(p.size)) * row_sets;
  p.tiles_c = static_cast<int32_t>(ceil_div(cols, gated_tile_cols(p.size)));
  p.k_tiles = k_tiles;
  int64_t splits = 1;
  const int64_t tiles = p.tiles_r * p.tiles_c;
  if (can_split && tiles < 2 * cus) {
    splits = 2 * cus / tiles;
    const int64_t most = ceil_div(k_tiles, 8);  // 8 tiles of k at least
    splits = splits < most ? splits : most;
    splits = splits < 1 ? 1 : splits;
  }
  p.k_split = ceil_div(k_tiles, splits);
  p.splits = static_cast<int32_t>(ceil_div(k_tiles, p.k_split));
  return p;
}

}  // namespace ow
