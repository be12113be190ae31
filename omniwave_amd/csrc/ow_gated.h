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
// C, its B operand R: a lane then has 16 values of one row r, in runs of 4 along c, which go through LDS to be stored
// in whole rows of the wave's tile (Turn).
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
  kGatedKeep,     // the same, and both products stored in fp32
  kGatedGates,    // dG and dU, with both products formed again
  kGatedDx,       // dG Wg + dU Wu
  kGatedDw,       // dG^T x, dU^T x
};

// Division of numbers below 2^31 by one that the host knows: n / d = n mul >> shift.
struct Divisor {
  uint32_t mul, shift;
  __host__ static Divisor of(uint32_t d) {
    uint32_t log = 0;
    while ((uint64_t(1) << log) < d) ++log;
    return Divisor{static_cast<uint32_t>((uint64_t(1) << (31 + log)) / d + 1), 31 + log};
  }
  __device__ __forceinline__ uint32_t divide(uint32_t n) const { return static_cast<uint32_t>(static_cast<uint64_t>(n) * mul >> shift); }
};

struct GatedArgs {
  const char* x;
  const char* w[2];   // gate, up
  const char* dh;
  const char* dgu[2]; // dG, dU: [rows][ld_gu]
  int64_t x_ld, dh_ld;  // bytes
  void* out[2];       // h; dG, dU; dx; dgate, dup
  float* partial;     // [splits][outputs], fp32; used where splits > 1
  float* kept;        // [2][rows][hidden]: G and U, for kGatedKeep
  int64_t rows;
  int32_t channels, hidden, ld_gu;  // ld_gu: hidden, up to whole 16-byte pieces
  int64_t tiles_r;
  int32_t tiles_c, splits;
  int64_t k_tiles, k_split;  // tiles of k in all, and of a split
  Divisor by_tiles, by_group;  // tiles_r tiles_c, 8 tiles_c
};

// Geometry of a tile: WR x WC waves, each RI x CI products of 32 x 32.
template <int WR_, int WC_, int RI_, int CI_>
struct Tile {
  static constexpr int WR = WR_, WC = WC_, RI = RI_, CI = CI_;
  static constexpr int BR = WR * RI * 32, BC = WC * CI * 32, kWaves = WR * WC, kThreads = kWaves * 64;
  static constexpr int kBytesR = BR * 128, kBytesC = BC * 128;  // of one stage
  static constexpr bool kTurns = kWaves == 4;  // a workgroup takes several units (a larger one has no registers left for that)
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
        at.off[i] = index < extent ? static_cast<uint32_t>(index) * static_cast<uint32_t>(ld) + piece * 16 : kOffOut;
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
        at.off[i] = p * V < n_out ? static_cast<uint32_t>(k) * static_cast<uint32_t>(ld) + p * 16 : kOffOut;
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

// A wave's own 4 KB of LDS, in which outputs change from a product's layout (a lane has a row: runs of 4 values, run g at column
// 8 g + 4 hh) to that of memory (neighbouring lanes have neighbouring pieces): stores of 32 bytes to each of 32 rows reached
// 1.6 TB/s, whole rows of the tile are stored at more than twice that.  32 rows of PITCH bytes, pieces of a row
// permuted by it.
template <int PITCH>
struct Turn {
  static constexpr int kPieces = PITCH / 16, kRows = 64 / kPieces, kCopies = 32 / kRows;  // rows of an instruction, instructions
  static __device__ __forceinline__ uint32_t at(uint32_t lds, int row, int piece) {
    return lds + row * PITCH + ((piece ^ (PITCH == 128 ? row & 7 : row >> 1 & 3)) << 4);
  }
  typedef __attribute__((address_space(3))) u32x4 Whole;
  typedef __attribute__((address_space(3))) u32x2 Half;
  static __device__ __forceinline__ Whole* whole(uint32_t at) { return reinterpret_cast<Whole*>(static_cast<uintptr_t>(at)); }
  static __device__ __forceinline__ Half* half(uint32_t at) { return reinterpret_cast<Half*>(static_cast<uintptr_t>(at)); }
  // A product's values of 32 columns, the first of them at piece `first`.
  template <class Ty>
  static __device__ __forceinline__ void put(uint32_t lds, int first, const float (&v)[16], int lane) {
    const int row = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if constexpr (std::is_same<Ty, F32>::value) {
        *whole(at(lds, row, first + 2 * g + hh)) = u32x4{__float_as_uint(v[4 * g]), __float_as_uint(v[4 * g + 1]),
                                                         __float_as_uint(v[4 * g + 2]), __float_as_uint(v[4 * g + 3])};
      } else {
        *half(at(lds, row, first + g) + 8 * hh) = u32x2{Ty::pack2(v[4 * g], v[4 * g + 1]), Ty::pack2(v[4 * g + 2], v[4 * g + 3])};
      }
    }
  }
  template <class Ty>
  static __device__ __forceinline__ void get(uint32_t lds, float (&v)[16], int lane) {
    const int row = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if constexpr (std::is_same<Ty, F32>::value) {
        const u32x4 w = *whole(at(lds, row, 2 * g + hh));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * g + j] = __uint_as_float(w[j]);
      } else {
        const u32x2 w = *half(at(lds, row, g) + 8 * hh);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * g + j] = Ty::to_f32(j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]));
      }
    }
  }
  // Rows to memory: `out` is the tile's first value, `rows` and `cols` what there is of it from there on.
  template <int SIZE>
  static __device__ __forceinline__ void store(uint32_t lds, char* out, int64_t ld, int64_t rows, int64_t cols, int lane) {
    constexpr int V = 16 / SIZE;
    const int piece = lane % kPieces, c = piece * V;
    out += lane / kPieces * ld + piece * 16;
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int row = i * kRows + lane / kPieces;
      const u32x4 w = *whole(at(lds, row, piece));
      if (row < rows) {
        if (c + V <= cols) {
          *reinterpret_cast<u32x4_any*>(out) = w;
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c + j < cols) {
              if constexpr (SIZE == 2) reinterpret_cast<uint16_t*>(out)[j] = j & 1 ? hi16(w[j >> 1]) : lo16(w[j >> 1]);
              else reinterpret_cast<uint32_t*>(out)[j] = w[j];
            }
        }
      }
      out += kRows * ld;
    }
    wave_lds_sync();
  }
  // Rows from memory, zeros outside; `keep` brings them to LDS.
  template <int SIZE>
  static __device__ __forceinline__ void load(u32x4 (&w)[kCopies], const char* in, int64_t ld, int64_t rows, int64_t cols, int lane) {
    const int piece = lane % kPieces;
    in += lane / kPieces * ld + piece * 16;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) w[i] = load_piece<SIZE>(in + i * kRows * ld, i * kRows + lane / kPieces < rows ? cols - piece * (16 / SIZE) : 0);
  }
  static __device__ __forceinline__ void keep(uint32_t lds, const u32x4 (&w)[kCopies], int lane) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) *whole(at(lds, i * kRows + lane / kPieces, lane % kPieces)) = w[i];
    wave_lds_sync();
  }
};

// silu(g) u = g u / (1 + e^-g)
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(kNegLog2e * g)); }

// Workgroups of an XCD take neighbouring tiles (round-robin dispatch), in groups of 8 rows of tiles.
__device__ __forceinline__ uint32_t xcd_tile(uint32_t id, uint32_t n) {
  const uint32_t xcd = id & 7, at = id >> 3, per = n >> 3, rem = n & 7;
  return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + at;
}

template <class Ty, int MODE, class T, bool DIRECT>
__global__ void __launch_bounds__(T::kThreads, 2) gated_tile_kernel(GatedArgs a) {
  constexpr int S = Elem<Ty>::kSize, KT = Elem<Ty>::kTile, W = T::kWaves;
  constexpr bool kPair = MODE == kGatedForward || MODE == kGatedKeep || MODE == kGatedGates;  // columns: 32 of the gate, 32 of the other
  constexpr int kCols = kPair ? T::BC / 2 : T::BC;                      // output columns of a tile
  typedef typename std::conditional<MODE == kGatedDw, AcrossK<T::BR, W, S, DIRECT>, AlongK<T::BR, W, S, DIRECT, false>>::type OpR;
  typedef typename std::conditional<kPair, AlongK<T::BC, W, S, DIRECT, true>, AcrossK<T::BC, W, S, DIRECT>>::type OpC;
  __shared__ __attribute__((aligned(1024))) char lds[2][T::kBytesR + T::kBytesC];
  __shared__ __attribute__((aligned(1024))) char turns[W][4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hh = lane >> 5;

  // A workgroup takes units (a tile, or a part of its k) in turn, and their tiles of k as one sequence: a unit's first
  // operands are on their way while the one before it is stored.
  struct Unit {
    int64_t r0, c0, kt, kt_end;
    int which, split;
  };
  const uint32_t tiles = static_cast<uint32_t>(a.tiles_r) * a.tiles_c, units = tiles * a.splits;
  auto unit_at = [&](uint32_t index) {
    const uint32_t id = xcd_tile(index, units), split = a.by_tiles.divide(id), tile = id - split * tiles;
    constexpr uint32_t kGroup = 8;
    const uint32_t group = a.by_group.divide(tile), in = tile - group * kGroup * a.tiles_c;
    const uint32_t high = static_cast<uint32_t>(a.tiles_r) - group * kGroup;
    const uint32_t tile_c = high >= kGroup ? in / kGroup : in / high;
    const uint32_t tile_r = group * kGroup + (high >= kGroup ? in % kGroup : in - tile_c * high);
    // The weights' gradients: the first half of the rows of tiles is the gate's.
    const uint32_t half_r = static_cast<uint32_t>(a.tiles_r) / 2;
    Unit u;
    u.split = static_cast<int>(split);
    u.which = MODE == kGatedDw && tile_r >= half_r ? 1 : 0;
    u.r0 = static_cast<int64_t>(MODE == kGatedDw && u.which ? tile_r - half_r : tile_r) * T::BR;
    u.c0 = static_cast<int64_t>(tile_c) * kCols;
    u.kt = static_cast<int64_t>(split) * a.k_split;
    u.kt_end = u.kt + a.k_split < a.k_tiles ? u.kt + a.k_split : a.k_tiles;
    return u;
  };

  OpR op_r;
  OpC op_c;
  const int64_t ld_w = static_cast<int64_t>(a.channels) * S, ld_gu = static_cast<int64_t>(a.ld_gu) * S;
  uint32_t next = blockIdx.x;  // the unit that is fetched
  Unit f = unit_at(next);
  auto init = [&]() {
    if constexpr (kPair) {
      op_r.init(a.rows - f.r0, a.x_ld, wave, lane);
      op_c.init(a.hidden - f.c0, ld_w, wave, lane);
    } else if constexpr (MODE == kGatedDx) {
      op_r.init(a.rows - f.r0, ld_gu, wave, lane);
      op_c.init(a.channels - f.c0, ld_w, wave, lane);
    } else {
      op_r.init(a.ld_gu - f.r0, ld_gu, wave, lane);
      op_c.init(a.channels - f.c0, a.x_ld, wave, lane);
    }
  };
  // To the next unit, where this one's tiles have all been asked for; behind the last unit tiles read as zeros that
  // nobody uses.
  auto turn = [&]() {
    if (!T::kTurns || f.kt < f.kt_end || next >= units) return;
    next += gridDim.x;
    if (next >= units) return;
    f = unit_at(next);
    init();
  };
  auto fetch = [&](int stage) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
    const auto left = [&](int64_t k) { return f.kt >= f.kt_end ? 0 : k < KT ? static_cast<int>(k) : KT; };
    const int64_t kt = f.kt;
    if constexpr (kPair) {
      const int k_left = left(a.channels - kt * KT);
      op_r.fetch(a.x + f.r0 * a.x_ld + kt * 128, nullptr, k_left, at_r, wave);
      op_c.fetch(a.w[0] + f.c0 * ld_w + kt * 128, a.w[1] + f.c0 * ld_w + kt * 128, k_left, at_c, wave);
    } else if constexpr (MODE == kGatedDx) {
      const int64_t each = a.k_tiles / 2;
      const int w = kt >= each;
      const int64_t k0 = (kt - w * each) * KT;
      op_r.fetch(a.dgu[w] + f.r0 * ld_gu + k0 * S, nullptr, left(a.ld_gu - k0), at_r, wave);
      op_c.fetch(a.w[w] + k0 * ld_w + f.c0 * S, left(a.hidden - k0), at_c, wave);
    } else {
      const int64_t k0 = kt * KT;
      const int k_left = left(a.rows - k0);
      op_r.fetch(a.dgu[f.which] + k0 * ld_gu + f.r0 * S, k_left, at_r, wave);
      op_c.fetch(a.x + k0 * a.x_ld + f.c0 * S, k_left, at_c, wave);
    }
    f.kt += f.kt < f.kt_end;
  };
  auto put = [&](int stage) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
    op_r.put(at_r, wave, lane);
    op_c.put(at_c, wave, lane);
  };

  f32x16 acc[T::CI][T::RI];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < T::CI; ++i)
#pragma unroll
      for (int j = 0; j < T::RI; ++j) acc[i][j] = f32x16{};
  };
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
  Unit u = f;  // the unit that is multiplied
  init();
  fetch(0);
  turn();
  if constexpr (DIRECT) {
    fetch(1);
    wait_vmcnt<kCopies>();
  } else {
    put(0);
    fetch(1);
  }
  __syncthreads();
  read(0, 0, 0);
  clear();
  int stage = 0;
  for (uint32_t index = blockIdx.x;;) {
    turn();
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
    fetch(stage);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
    stage ^= 1;
    if (++u.kt < u.kt_end) continue;
    mfma_drain();
    const uint32_t own = lds_addr(turns[wave]);
    if constexpr (kPair) {
      typedef Turn<32 * S> Tn;
      const int64_t c = u.c0 + (wc >> 1), r = u.r0 + wr;
      if constexpr (MODE != kGatedGates) {
#pragma unroll
        for (int j = 0; j < T::RI; ++j) {
          if constexpr (MODE == kGatedKeep) {
            const int64_t ld = static_cast<int64_t>(a.hidden) * 4, row = r + 32 * j;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float v[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
              Turn<128>::put<F32>(own, 0, v, lane);
              Turn<128>::store<4>(own, reinterpret_cast<char*>(a.kept) + (i * a.rows + row) * ld + c * 4, ld, a.rows - row, a.hidden - c, lane);
            }
          }
          float h[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) h[i] = acc[0][j][i] * acc[1][j][i] * sigmoid(acc[0][j][i]);
          Tn::template put<Ty>(own, 0, h, lane);
          const int64_t ld = static_cast<int64_t>(a.hidden) * S, row = r + 32 * j;
          Tn::template store<S>(own, static_cast<char*>(a.out[0]) + row * ld + c * S, ld, a.rows - row, a.hidden - c, lane);
        }
      } else {
        // Columns up to a whole piece are written: there both products are 0.  The gradients of G and U are
        // rounded to the operands' type here, as the products that take them need it (fp32 stays fp32).
        u32x4 w[T::RI][Tn::kCopies];
#pragma unroll
        for (int j = 0; j < T::RI; ++j) {
          const int64_t row = r + 32 * j;
          Tn::template load<S>(w[j], a.dh + row * a.dh_ld + c * S, a.dh_ld, a.rows - row, a.hidden - c, lane);
        }
#pragma unroll
        for (int j = 0; j < T::RI; ++j) {
          const int64_t row = r + 32 * j, at = row * ld_gu + c * S;
          float dh[16], dg[16], du[16];
          Tn::keep(own, w[j], lane);
          Tn::template get<Ty>(own, dh, lane);
          wave_lds_sync();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float g = acc[0][j][i], up = acc[1][j][i], s = sigmoid(g);
            du[i] = dh[i] * (g * s);
            dg[i] = dh[i] * up * (s * (1.f + g * (1.f - s)));
          }
          Tn::template put<Ty>(own, 0, dg, lane);
          Tn::template store<S>(own, static_cast<char*>(a.out[0]) + at, ld_gu, a.rows - row, a.ld_gu - c, lane);
          Tn::template put<Ty>(own, 0, du, lane);
          Tn::template store<S>(own, static_cast<char*>(a.out[1]) + at, ld_gu, a.rows - row, a.ld_gu - c, lane);
        }
      }
    } else {
      const int64_t n_r = MODE == kGatedDw ? a.hidden : a.rows;
#pragma unroll
      for (int j = 0; j < T::RI; ++j) {
        const int64_t row = u.r0 + wr + 32 * j, c = u.c0 + wc;
        if (a.splits > 1 || S == 4) {  // fp32: 32 columns at a time
          if (a.splits == 1 && a.out[u.which] == nullptr) continue;  // one weight's gradient is not asked for
          const int64_t ld = static_cast<int64_t>(a.channels) * 4;
          char* out = a.splits > 1 ? reinterpret_cast<char*>(a.partial) +
                                         (static_cast<int64_t>(u.split) * (MODE == kGatedDw ? 2 : 1) + u.which) * n_r * ld
                                   : static_cast<char*>(a.out[u.which]);
#pragma unroll
          for (int i = 0; i < T::CI; ++i) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
            Turn<128>::put<F32>(own, 0, v, lane);
            Turn<128>::store<4>(own, out + row * ld + (c + 32 * i) * 4, ld, n_r - row, a.channels - c - 32 * i, lane);
          }
        } else if constexpr (S == 2) {
          if (a.out[u.which] == nullptr) continue;
          static_assert(T::CI == 2, "64 columns of a wave");
#pragma unroll
          for (int i = 0; i < T::CI; ++i) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
            Turn<128>::put<Ty>(own, 4 * i, v, lane);
          }
          Turn<128>::store<2>(own, static_cast<char*>(a.out[u.which]) + row * ld_w + c * 2, ld_w, n_r - row, a.channels - c, lane);
        }
      }
    }
    index += gridDim.x;
    if (!T::kTurns || index >= units) break;
    if (index == next) {
      u = f;
      u.kt = static_cast<int64_t>(u.split) * a.k_split;
    } else {
      u = unit_at(index);
    }
    clear();
    read(stage, 0, 0);  // once more: nothing is kept in registers over the stores
  }
  // No copy may still be on its way when the workgroup ends.
  wait_vmcnt<0>();
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
  // As many workgroups as run at once (by the LDS of their two stages, two of TileM and three of TileS on a compute
  // unit), which take units in turn; TileL takes one each.
  const int64_t units = a.tiles_r * a.tiles_c * a.splits, most = static_cast<int64_t>(device_cus()) * 2;
  const dim3 grid(static_cast<unsigned>(size == 0 || units < most ? units : most));
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

// How an output of `rows` x `cols` (cols: gate and up together; `row_sets` of them) is cut.  TileL where k is long and every
// compute unit gets one (16-bit types, 6,272 tokens, 4,096 to 8,192: forward 738 us, 860 with TileM; 25,088 tokens, 512 to 1,024:
// 72 and 66; fp32, 5,728 tokens, 1,024 to 2,048: 527 and 438); else TileM, and TileS where that leaves compute units without
// work, or where k may be cut (can_split) TileM with k in parts (6,272 tokens, 1,024 to 2,048, the weights' gradients: 63 us and 9 for
// the sum of the parts; TileL 68 and 23).
inline GatedPlan gated_plan(int64_t rows, int64_t cols, int64_t k_tiles, int row_sets, bool can_split, bool wide) {
  const int64_t cus = device_cus();
  GatedPlan p;
  const auto tiles_of = [&](int size) {
    return ceil_div(rows, gated_tile_rows(size)) * row_sets * ceil_div(cols, gated_tile_cols(size));
  };
  p.size = !wide && k_tiles >= 16 && tiles_of(0) >= cus ? 0 : can_split || tiles_of(1) >= cus ? 1 : 2;
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
