// Tiles of the gated feed-forward products (gated_linear.hip, gated_linear_bwd.hip): one matrix product kernel in which
// an output tile O[r][c] = sum_k R[r][k] C[c][k] is formed by MFMA from tiles of both operands in LDS.
//
// Operands are of 16 bits.  fp32 ones are three bf16 planes each (ow_x3.h), and a product of two is the six products of
// planes whose weight is above 2^-24, one after the other along k: to the kernel, k is six times as long.  (fp32 MFMAs have a
// sixteenth of the bf16 ones' rate; 25,088 tokens, 256 to 512: forward 141 us by them, 104 and 16 for the copies by planes.)
//
// An operand lies in memory with its contraction index contiguous (AlongK: x and the weights forward, the gates'
// gradients in dx) or with its output index contiguous (AcrossK: the weights in dx, every operand of the weights'
// gradients), in rows of whole 16-byte pieces: what does not lie so is copied first (gated_pack_kernel).  The tile in LDS
// keeps that order:
//
//   AlongK     rows of 128 bytes (64 values), of which a lane reads 16 bytes of k at once; piece p of row r at slot
//              p ^ (r / 2 & 7), so that 16 rows' pieces of one column fill the 256 bytes of all banks
//   AcrossK    a row for each k, read transposed (ds_read_b64_tr_b16: 4 k of 16 output indexes by 16 lanes); piece p of row k
//              at p ^ 4 (k & 3), so that 4 rows' 64 bytes fill them
//
// A step is one 32x32x16 MFMA for each product of a wave.  Its A operand is C, its B operand R: a lane then has 16 values of
// one row r, in runs of 4 along c, which go through LDS to be stored in whole rows of the wave's tile (Turn).
//
// Tiles come by direct copies into LDS (16 bytes a lane; what lies outside the matrix reads as zeros), a tile ahead of
// the products, and a step's operands are read during the step before it.  6,272 tokens of 4,096 to 8,192 bf16: 738 us
// forward (1,140 TFLOP/s; the library's product of that size 719 us), the weights' gradients 719.  Small k is bound by what
// surrounds a unit's two to four steps: 401,408 tokens of 128 to 256 bf16 take 123 us forward, where its bytes would take 63.
#pragma once

#include "ow_rows.h"
#include "ow_x3.h"

namespace ow {

constexpr int kGatedMost = 1 << 20;  // channels, hidden

enum GatedMode {
  kGatedForward,  // h = silu(x Wg^T) (x Wu^T)
  kGatedKeep,     // the same, and both products stored in fp32
  kGatedGates,    // dG and dU, with both products formed again
  kGatedDx,       // dG Wg + dU Wu
  kGatedDw,       // dG^T x, dU^T x
};
constexpr bool gated_pair(int mode) { return mode == kGatedForward || mode == kGatedKeep || mode == kGatedGates; }

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

// An operand's planes, rows of `ld` bytes, whole pieces.
struct GatedPlanes {
  const char* at;
  int64_t ld, plane;
};

// How a product is cut: a unit is a tile with its whole k (the first `whole` of them), or one of `parts` parts of the k of one of
// the other tiles.
struct GatedPlan {
  int size;  // 0: TileL, 1: TileM, 2: TileS
  int64_t tiles_r;
  int32_t tiles_c, parts;
  int64_t whole, units;
  int64_t k_tiles, k_part;  // tiles of k (64 values) in all, and of a part
};

struct GatedArgs {
  GatedPlanes x, w[2], gu[2];  // w: gate, up; gu: dG, dU
  const char* dh;
  int64_t dh_ld;       // bytes
  void* out[2];        // h; dG, dU; dx; dgate, dup
  float* kept;         // [2][rows][hidden]: G and U
  float* partial;      // [units - whole][tile rows][tile columns]
  int64_t rows;
  int32_t channels, hidden;
  int32_t k_each;      // tiles of k of one product of planes
  GatedPlan p;
  Divisor by_group, by_split, by_each;  // 8 tiles_c; tiles that are cut; k_each
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

// A tile of N output indexes, 64 values of k each: 1 KB (8 rows) an instruction.  PAIR: 32 of one matrix and 32 of the
// other in turn.  `off`: a lane's offsets from the tile's first byte, kOffOut where the index is outside the matrix.
template <int N, int WAVES, bool PAIR>
struct AlongK {
  static constexpr int kCopies = N / 8 / WAVES, kReads = 1;
  static_assert(kCopies * 8 * WAVES == N && (!PAIR || 32 % (8 * WAVES) == 0 || 8 * WAVES == 64), "whole copies of one matrix");
  uint32_t off[kCopies];
  int piece;  // of a row
  static __device__ __forceinline__ int slot_of(int row) { return row >> 1 & 7; }
  static __device__ __forceinline__ int part(int i, int wave) { return PAIR ? ((8 * (i * WAVES + wave)) >> 5) & 1 : 0; }
  // extent: indexes from the tile's first one on.
  __device__ __forceinline__ void init(int64_t extent, int64_t ld, int wave, int lane) {
    static_assert(WAVES % 2 == 0, "copies of a wave begin at the same row of 16");
    piece = (lane & 7) ^ slot_of(8 * wave + (lane >> 3));
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int q = 8 * (i * WAVES + wave), index = (PAIR ? (q >> 6) * 32 + (q & 31) : q) + (lane >> 3);
      off[i] = index < extent ? static_cast<uint32_t>(index) * static_cast<uint32_t>(ld) + piece * 16 : kOffOut;
    }
  }
  // Copy i.  r0, r1: from the tile's first index of each matrix at the tile's k; k_left: values of k that are there, up to a tile's.
  __device__ __forceinline__ void copy(int i, __amdgpu_buffer_rsrc_t r0, __amdgpu_buffer_rsrc_t r1, int k_left, uint32_t lds, int wave) const {
    tile_copy(part(i, wave) ? r1 : r0, piece * 8 < k_left ? off[i] : kOffOut, lds + 8 * (i * WAVES + wave) * 128);
  }
  // A lane's address for the wave's first index, of step 0; a step's pieces are a XOR away, further indexes an offset.
  static __device__ __forceinline__ uint32_t lane_at(uint32_t lds, int first, int lane) {
    const int l32 = lane & 31, hh = lane >> 5;
    return lds + (first + l32) * 128 + ((hh ^ slot_of(l32)) << 4);
  }
  static __device__ __forceinline__ u32x4 read(uint32_t lane_at, uint32_t stage, int i, int step) {
    const uint32_t at = (lane_at ^ (step << 5)) + stage + i * 4096;
    return *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(static_cast<uintptr_t>(at));
  }
};

// A tile of 64 values of k, N output indexes each.
template <int N, int WAVES>
struct AcrossK {
  static constexpr int kRow = N * 2, kPieces = kRow / 16;   // of a k
  static constexpr int kRowsOfCopy = 64 / kPieces;
  static constexpr int kCopies = N / 8 / WAVES, kReads = 2;
  static_assert(kRow <= 1024 && kCopies * 8 * WAVES == N, "whole copies");
  uint32_t off[kCopies];
  int in;  // the lane's k of a copy
  static __device__ __forceinline__ int slot(int p, int k) { return p ^ (kRow >= 256 ? (k & 3) << 2 : (k & 2) << 1); }
  // n_out: output indexes from the tile's first one on.
  __device__ __forceinline__ void init(int64_t n_out, int64_t ld, int wave, int lane) {
    in = lane / kPieces;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int k = (i * WAVES + wave) * kRowsOfCopy + in, p = slot(lane % kPieces, k);
      off[i] = p * 8 < n_out ? static_cast<uint32_t>(k) * static_cast<uint32_t>(ld) + p * 16 : kOffOut;
    }
  }
  // Copy i.  r: from the first output index at the tile's k; k_left: values of k that are there, up to a tile's.
  __device__ __forceinline__ void copy(int i, __amdgpu_buffer_rsrc_t r, __amdgpu_buffer_rsrc_t, int k_left, uint32_t lds, int wave) const {
    const int copy = i * WAVES + wave;
    tile_copy(r, in < k_left - copy * kRowsOfCopy ? off[i] : kOffOut, lds + copy * 1024);
  }
  // A lane's address for the wave's first index, of step 0; the next 32 indexes are a XOR away (the wave's first is a
  // multiple of what it has of them), steps an offset.
  static __device__ __forceinline__ uint32_t lane_at(uint32_t lds, int first, int lane) {
    const int l16 = lane & 15, k = 8 * (lane >> 5) + (l16 >> 2);
    const int c = first + 16 * ((lane >> 4) & 1) + 4 * (l16 & 3);
    return lds + k * kRow + (slot(c >> 3, k) << 4) + ((c & 4) << 1);
  }
  static __device__ __forceinline__ u32x4 read(uint32_t lane_at, uint32_t stage, int i, int step) {
    const uint32_t at = (lane_at ^ (i << 6)) + stage + step * 16 * kRow;
    const u32x2 a = lds_read_tr16(at), b = lds_read_tr16(at + 4 * kRow);
    return u32x4{a[0], a[1], b[0], b[1]};
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
        } else {  // the last piece of ragged rows, from LDS value by value
          typedef typename std::conditional<SIZE == 2, uint16_t, uint32_t>::type Value;
          const auto* from = reinterpret_cast<__attribute__((address_space(3))) Value*>(static_cast<uintptr_t>(at(lds, row, piece)));
#pragma unroll 1
          for (int j = 0; c + j < cols; ++j) reinterpret_cast<Value*>(out)[j] = from[j];
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

__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(kNegLog2e * g)); }

// silu(g) u.  The sigmoid meets g before u does: g u may leave fp32's range where the gate is closed (-1e20 and 1e20: 0).
__device__ __forceinline__ float gated(float g, float u) { return g * sigmoid(g) * u; }

// dG and dU of a value; the gate's factors come first here, too.
__device__ __forceinline__ void gates(float dh, float g, float u, float& dg, float& du) {
  const float s = sigmoid(g);
  du = dh * (g * s);
  dg = dh * (u * (s * (1.f + g * (1.f - s))));
}

// Workgroups of an XCD take neighbouring tiles (round-robin dispatch).
__device__ __forceinline__ uint32_t xcd_tile(uint32_t id, uint32_t n) {
  const uint32_t xcd = id & 7, at = id >> 3, per = n >> 3, rem = n & 7;
  return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + at;
}

// Where a tile lies: groups of 8 rows of tiles, column by column.
struct TilePlace {
  int64_t r0;
  int64_t c0;
  int which;  // the weights' gradients: the first half of the rows of tiles is the gate's
};
template <int MODE, class T>
__device__ __forceinline__ TilePlace tile_place(const GatedArgs& a, uint32_t tile) {
  constexpr uint32_t kGroup = 8;
  const uint32_t group = a.by_group.divide(tile), in = tile - group * kGroup * a.p.tiles_c;
  const uint32_t high = static_cast<uint32_t>(a.p.tiles_r) - group * kGroup;
  const uint32_t tile_c = high >= kGroup ? in / kGroup : in / high;
  const uint32_t tile_r = group * kGroup + (high >= kGroup ? in % kGroup : in - tile_c * high);
  const uint32_t half_r = static_cast<uint32_t>(a.p.tiles_r) / 2;
  TilePlace t;
  t.which = MODE == kGatedDw && tile_r >= half_r ? 1 : 0;
  t.r0 = static_cast<int64_t>(t.which ? tile_r - half_r : tile_r) * T::BR;
  t.c0 = static_cast<int64_t>(tile_c) * (gated_pair(MODE) ? T::BC / 2 : T::BC);
  return t;
}

// Ty: the operands' type; Out: x's and the outputs' (F32: three planes of bf16 operands).
template <class Ty, class Out, int MODE, class T>
__global__ void __launch_bounds__(T::kThreads, 2) gated_tile_kernel(GatedArgs a) {
  constexpr bool kWide = std::is_same<Out, F32>::value, kPair = gated_pair(MODE);
  constexpr int W = T::kWaves, S = kWide ? 4 : 2;  // S: bytes of an output
  constexpr int kProducts = kWide ? 6 : 1;         // of planes
  typedef typename std::conditional<MODE == kGatedDw, AcrossK<T::BR, W>, AlongK<T::BR, W, false>>::type OpR;
  typedef typename std::conditional<kPair, AlongK<T::BC, W, true>, AcrossK<T::BC, W>>::type OpC;
  __shared__ __attribute__((aligned(1024))) char lds[2][T::kBytesR + T::kBytesC];
  __shared__ __attribute__((aligned(1024))) char turns[W][4096];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // A workgroup takes units in turn, and their tiles of k as one sequence: a unit's first operands are on their way while the
  // one before it is stored.
  struct Unit {
    TilePlace at;
    uint32_t kt, kt_end, product, k_in;  // tiles of k; the product of planes of the next one, and its place there
    int part;                            // of the tile; -1: whole
  };
  const uint32_t units = static_cast<uint32_t>(a.p.units), whole = static_cast<uint32_t>(a.p.whole);
  auto unit_at = [&](uint32_t index) {
    Unit u;
    uint32_t tile;
    u.kt = 0;
    u.kt_end = static_cast<uint32_t>(a.p.k_tiles);
    if (index < whole) {
      tile = xcd_tile(index, whole);
      u.part = -1;
      u.product = u.k_in = 0;
    } else {
      // Parts with the same k lie side by side: they share rows of an operand.
      const uint32_t id = xcd_tile(index - whole, units - whole), part = a.by_split.divide(id);
      tile = whole + id - part * (static_cast<uint32_t>(a.p.tiles_r) * a.p.tiles_c - whole);
      u.part = static_cast<int>(part);
      u.kt = part * static_cast<uint32_t>(a.p.k_part);
      const uint32_t end = u.kt + static_cast<uint32_t>(a.p.k_part);
      u.kt_end = end < u.kt_end ? end : u.kt_end;
      u.product = a.by_each.divide(u.kt);
      u.k_in = u.kt - u.product * a.k_each;
    }
    u.at = tile_place<MODE, T>(a, tile);
    return u;
  };

  OpR op_r;
  OpC op_c;
  uint32_t next = blockIdx.x;  // the unit that is fetched
  Unit f = unit_at(next);
  auto init = [&]() {
    if constexpr (kPair) {
      op_r.init(a.rows - f.at.r0, a.x.ld, wave, lane);
      op_c.init(a.hidden - f.at.c0, a.w[0].ld, wave, lane);
    } else if constexpr (MODE == kGatedDx) {
      op_r.init(a.rows - f.at.r0, a.gu[0].ld, wave, lane);
      op_c.init(a.channels - f.at.c0, a.w[0].ld, wave, lane);
    } else {
      op_r.init(a.hidden - f.at.r0, a.gu[0].ld, wave, lane);
      op_c.init(a.channels - f.at.c0, a.x.ld, wave, lane);
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
  // Where the next tile of k is, and to the one after it.
  struct Source {
    __amdgpu_buffer_rsrc_t r, c, other;
    int k_left;
  };
  auto source = [&]() {
    // Products of planes, the smallest first: (2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0).  In dx all of dG's come before dU's.
    const uint32_t which = MODE == kGatedDx && f.product >= kProducts ? 1 : 0, pair = f.product - which * kProducts;
    const int plane_r = kWide ? (0x001012 >> (4 * pair)) & 3 : 0, plane_c = kWide ? (0x010210 >> (4 * pair)) & 3 : 0;
    const int64_t k0 = static_cast<int64_t>(f.k_in) * 64;
    const char *r, *c, *other;
    int64_t left;
    if constexpr (kPair) {
      left = a.channels - k0;
      r = a.x.at + plane_r * a.x.plane + f.at.r0 * a.x.ld + k0 * 2;
      const int64_t at = plane_c * a.w[0].plane + f.at.c0 * a.w[0].ld + k0 * 2;
      c = a.w[0].at + at, other = a.w[1].at + at;
    } else if constexpr (MODE == kGatedDx) {
      left = a.hidden - k0;
      r = a.gu[which].at + plane_r * a.gu[0].plane + f.at.r0 * a.gu[0].ld + k0 * 2;
      c = other = a.w[which].at + plane_c * a.w[0].plane + k0 * a.w[0].ld + f.at.c0 * 2;
    } else {
      left = a.rows - k0;
      r = a.gu[f.at.which].at + plane_r * a.gu[0].plane + k0 * a.gu[0].ld + f.at.r0 * 2;
      c = other = a.x.at + plane_c * a.x.plane + k0 * a.x.ld + f.at.c0 * 2;
    }
    Source s{buffer_rsrc(r, 0x7fffffffu), buffer_rsrc(c, 0x7fffffffu), buffer_rsrc(other, 0x7fffffffu),
             f.kt >= f.kt_end ? 0 : left < 64 ? static_cast<int>(left) : 64};
    if (f.kt < f.kt_end) {
      ++f.kt;
      if (++f.k_in == static_cast<uint32_t>(a.k_each)) f.k_in = 0, ++f.product;
    }
    return s;
  };
  constexpr int kCopies = OpR::kCopies + OpC::kCopies;
  auto copy = [&](const Source& s, int stage, int i) {
    const uint32_t at_r = lds_addr(lds[stage]), at_c = at_r + T::kBytesR;
    if (i < OpR::kCopies) op_r.copy(i, s.r, s.r, s.k_left, at_r, wave);
    else op_c.copy(i - OpR::kCopies, s.c, s.other, s.k_left, at_c, wave);
  };
  auto fetch = [&](int stage) {
    const Source s = source();
#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy(s, stage, i);
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
  const uint32_t lane_r = OpR::lane_at(lds_addr(lds[0]), wr, lane), lane_c = OpC::lane_at(lds_addr(lds[0]) + T::kBytesR, wc, lane);
  auto read = [&](int stage, int s, int buf) {
    const uint32_t from = stage * (T::kBytesR + T::kBytesC);
#pragma unroll
    for (int i = 0; i < T::CI; ++i) fc[buf][i] = OpC::read(lane_c, from, i, s);
#pragma unroll
    for (int j = 0; j < T::RI; ++j) fr[buf][j] = OpR::read(lane_r, from, j, s);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int j = 0; j < T::RI; ++j)
#pragma unroll
      for (int i = 0; i < T::CI; ++i) acc[i][j] = Ty::mma32(fc[buf][i], fr[buf][j], acc[i][j]);
  };
  // A step's reads go between its products, one after each; left alone, the compiler puts them right before their use.
  constexpr int kReads = T::CI * OpC::kReads + T::RI * OpR::kReads, kMfma = T::CI * T::RI;
  auto interleave = [&]() {
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read of LDS
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product
    }
    if constexpr (kMfma > kReads) __builtin_amdgcn_sched_group_barrier(0x8, kMfma - kReads, 0);
    __builtin_amdgcn_sched_barrier(0);
  };

  // Operands of a step are read while the step before it is multiplied, those of a tile's first step during the
  // last one of the tile before: at that point the next tile has arrived, all of this one is in registers, and
  // the tile after the next takes its place.
  Unit u = f;  // the unit that is multiplied
  init();
  fetch(0);
  turn();
  fetch(1);
  wait_vmcnt<kCopies>();
  __syncthreads();
  read(0, 0, 0);
  clear();
  int stage = 0;
  for (uint32_t index = blockIdx.x;;) {
    turn();
    const Source tile = source();
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      read(stage, s + 1, (s + 1) & 1);
      multiply(s & 1);
      interleave();
    }
    wait_vmcnt<0>();
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    // The copies go between this step's products.
    read(stage ^ 1, 0, 0);
#pragma unroll
    for (int m = 0; m < kMfma; ++m) {
      const int i = m % T::CI, j = m / T::CI;
      acc[i][j] = Ty::mma32(fc[1][i], fr[1][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = kCopies * m / kMfma; n < kCopies * (m + 1) / kMfma; ++n) copy(tile, stage, n);
      __builtin_amdgcn_sched_barrier(0);
    }
    stage ^= 1;
    if (++u.kt < u.kt_end) continue;
    mfma_drain();

    const uint32_t own = lds_addr(turns[wave]);
    // What the stores compute of the lane stays behind the loop: hoisted, it takes registers that the loop needs.
    int out_lane = lane;
    asm volatile("" : "+v"(out_lane));
    auto values = [&](int i, int j, float (&v)[16]) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[i][j][e];
    };
    if (u.part >= 0) {
      // Fewer tiles are cut than there are units, so this is the part's place among all units that are no whole tile.
      constexpr int64_t kLd = T::BC * 4;
      const uint32_t id = xcd_tile(index - whole, units - whole);
      char* out = reinterpret_cast<char*>(a.partial) + static_cast<int64_t>(id) * T::BR * kLd + wr * kLd + wc * 4;
#pragma unroll
      for (int j = 0; j < T::RI; ++j)
#pragma unroll
        for (int i = 0; i < T::CI; ++i) {
          float v[16];
          values(i, j, v);
          Turn<128>::put<F32>(own, 0, v, out_lane);
          Turn<128>::store<4>(own, out + 32 * j * kLd + 32 * i * 4, kLd, 32, 32, out_lane);
        }
    } else if constexpr (kPair) {
      typedef Turn<32 * S> Tn;
      const int64_t c = u.at.c0 + (wc >> 1), r = u.at.r0 + wr;
      if constexpr (MODE != kGatedGates) {
#pragma unroll
        for (int j = 0; j < T::RI; ++j) {
          const int64_t row = r + 32 * j, ld = static_cast<int64_t>(a.hidden) * S;
          if constexpr (MODE == kGatedKeep) {
            const int64_t ld_kept = static_cast<int64_t>(a.hidden) * 4;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float v[16];
              values(i, j, v);
              Turn<128>::put<F32>(own, 0, v, out_lane);
              Turn<128>::store<4>(own, reinterpret_cast<char*>(a.kept) + (i * a.rows + row) * ld_kept + c * 4, ld_kept, a.rows - row,
                                  a.hidden - c, out_lane);
            }
          }
          float h[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) h[i] = gated(acc[0][j][i], acc[1][j][i]);
          Tn::template put<Out>(own, 0, h, out_lane);
          Tn::template store<S>(own, static_cast<char*>(a.out[0]) + row * ld + c * S, ld, a.rows - row, a.hidden - c, out_lane);
        }
      } else {
        // Columns up to a whole piece are written: there both products are 0.  The gradients of G and U are
        // rounded to the operands' type here, as the products that take them need it (fp32: to its three planes).
        constexpr int kAhead = T::RI <= 2 ? T::RI : 1;  // rows of products whose upstream gradients are read at once
        u32x4 w[kAhead][Tn::kCopies];
        auto upstream = [&](int j) {
          const int64_t row = r + 32 * j;
          Tn::template load<S>(w[j % kAhead], a.dh + row * a.dh_ld + c * S, a.dh_ld, a.rows - row, a.hidden - c, out_lane);
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j) upstream(j);
#pragma unroll
        for (int j = 0; j < T::RI; ++j) {
          const int64_t row = r + 32 * j, at = row * a.gu[0].ld + c * 2;
          float dh[16], d[2][16];
          if (j >= kAhead) upstream(j);
          Tn::keep(own, w[j % kAhead], out_lane);
          Tn::template get<Out>(own, dh, out_lane);
          wave_lds_sync();
#pragma unroll
          for (int i = 0; i < 16; ++i) gates(dh[i], acc[0][j][i], acc[1][j][i], d[0][i], d[1][i]);
#pragma unroll
          for (int o = 0; o < 2; ++o) {
#pragma unroll
            for (int plane = 0; plane < (kWide ? 3 : 1); ++plane) {
              Turn<64>::put<Ty>(own, 0, d[o], out_lane);
              Turn<64>::store<2>(own, static_cast<char*>(a.out[o]) + plane * a.gu[0].plane + at, a.gu[0].ld, a.rows - row,
                                 a.gu[0].ld / 2 - c, out_lane);
              if constexpr (kWide) {
#pragma unroll
                for (int i = 0; i < 16; ++i) d[o][i] -= BF16::to_f32(BF16::from_f32(d[o][i]));
              }
            }
          }
        }
      }
    } else if (a.out[u.at.which] != nullptr) {  // NULL: one weight's gradient is not asked for
      const int64_t n_r = MODE == kGatedDw ? a.hidden : a.rows, ld = static_cast<int64_t>(a.channels) * S;
      char* out = static_cast<char*>(a.out[u.at.which]);
#pragma unroll
      for (int j = 0; j < T::RI; ++j) {
        const int64_t row = u.at.r0 + wr + 32 * j, c = u.at.c0 + wc;
        static_assert(T::CI == 2, "64 columns of a wave");
#pragma unroll
        for (int i = 0; i < T::CI; ++i) {
          float v[16];
          values(i, j, v);
          if constexpr (kWide) {  // 32 columns at a time
            Turn<128>::put<F32>(own, 0, v, out_lane);
            Turn<128>::store<4>(own, out + row * ld + (c + 32 * i) * 4, ld, n_r - row, a.channels - c - 32 * i, out_lane);
          } else {
            Turn<128>::put<Ty>(own, 4 * i, v, out_lane);
          }
        }
        if constexpr (!kWide) Turn<128>::store<2>(own, out + row * ld + c * 2, ld, n_r - row, a.channels - c, out_lane);
      }
    }
    index += gridDim.x;
    if (!T::kTurns || index >= units) break;
    if (index == next) {
      u = f;
      u.kt = u.part < 0 ? 0 : u.part * static_cast<uint32_t>(a.p.k_part);
    } else {
      u = unit_at(index);
    }
    clear();
    read(stage, 0, 0);  // once more: nothing is kept in registers over the stores
  }
  // No copy may still be on its way when the workgroup ends.
  wait_vmcnt<0>();
}

// The outputs of tiles whose k was cut: parts are added in their order.  A thread has 4 columns of a row, of the gate and of the other
// projection where there are both.
template <class Out, int MODE, class T>
__global__ void __launch_bounds__(256) gated_join_kernel(GatedArgs a) {
  constexpr bool kPair = gated_pair(MODE);
  constexpr int kRuns = (kPair ? T::BC / 2 : T::BC) / 4;
  typedef Row<Out> R;
  const uint32_t cut = static_cast<uint32_t>(a.p.tiles_r) * a.p.tiles_c - static_cast<uint32_t>(a.p.whole);
  const uint32_t per_tile = T::BR * kRuns / 256, t = blockIdx.x / per_tile, in = blockIdx.x % per_tile * 256 + threadIdx.x;
  const int row_in = in / kRuns, run = in % kRuns;
  const TilePlace at = tile_place<MODE, T>(a, static_cast<uint32_t>(a.p.whole) + t);
  const int64_t row = at.r0 + row_in, c = at.c0 + run * 4;
  const int64_t n_r = MODE == kGatedDw ? a.hidden : a.rows, n_c = kPair ? a.hidden : a.channels;
  void* const out = a.out[MODE == kGatedDw ? at.which : 0];
  if (row >= n_r || c >= n_c || out == nullptr) return;
  const int q = kPair ? run / 8 * 64 + run % 8 * 4 : run * 4;  // columns of the tile
  const float* p = a.partial + (static_cast<int64_t>(t) * T::BR + row_in) * T::BC + q;
  const int64_t step = static_cast<int64_t>(cut) * T::BR * T::BC;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f}, other = sum;
#pragma unroll 4
  for (int s = 0; s < a.p.parts; ++s) {
    sum += *reinterpret_cast<const f32x4*>(p + s * step);
    if constexpr (kPair) other += *reinterpret_cast<const f32x4*>(p + s * step + 32);
  }
  typename R::Elem* o = static_cast<typename R::Elem*>(out) + row * n_c + c;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c + j >= n_c) break;
    if constexpr (kPair) {
      if constexpr (MODE == kGatedKeep) {
        a.kept[row * n_c + c + j] = sum[j];
        a.kept[(a.rows + row) * n_c + c + j] = other[j];
      }
      o[j] = R::from_f32(gated(sum[j], other[j]));
    } else {
      o[j] = R::from_f32(sum[j]);
    }
  }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows and columns of a tile's operands (gate and up columns together).
inline int gated_tile_rows(int size) { return size == 0 ? TileL::BR : size == 1 ? TileM::BR : TileS::BR; }
inline int gated_tile_cols(int size) { return size == 0 ? TileL::BC : size == 1 ? TileM::BC : TileS::BC; }
// Units that run at once (the LDS of two stages and Turn: one workgroup a compute unit of TileL, two of the others).
inline int64_t gated_at_once(int size) { return static_cast<int64_t>(device_cus()) * (size == 0 ? 1 : 2); }

// How an output of `rows` x `cols` (cols: gate and up together; `row_sets` of them) is cut: the tile, and the parts of k of those tiles
// that fill no whole round of what runs at once, by their time.  A unit takes kStep us for a tile of k, more where an
// operand is read across k, and kBesides us for its beginning and its outputs (measured: 6,272 tokens, 4,096 to 8,192: 738, 860 and 995 us
// forward for TileL, M and S; 25,088 tokens, 512 to 1,024: 72, 66 and 72; the weights' gradients of 6,272 tokens, 1,024 to 2,048: 68, 63
// and 86 and, for L and M, 23 and 9 to join parts).  Parts are written and read at 0.4 us a MB, and joined by a launch
// of 6 us.
inline GatedPlan gated_plan(int64_t rows, int64_t cols, int64_t k_tiles, int row_sets, bool pair, bool may_cut) {
  constexpr double kSteps[2][3] = {{1.88, 1.3, 0.87}, {1.6, 0.98, 0.58}}, kBesides[3] = {7.0, 3.1, 2.0};
  const double(&kStep)[3] = kSteps[pair];
  GatedPlan best{};
  double least = 0.0;
  for (int size = 0; size < 3; ++size) {
    GatedPlan p{};
    p.size = size;
    p.tiles_r = ceil_div(rows, gated_tile_rows(size)) * row_sets;
    p.tiles_c = static_cast<int32_t>(ceil_div(cols, gated_tile_cols(size)));
    p.k_tiles = k_tiles;
    const int64_t tiles = p.tiles_r * p.tiles_c, slots = gated_at_once(size);
    const int64_t whole = tiles / slots * slots, rest = tiles - whole;
    const double unit = k_tiles * kStep[size] + kBesides[size];
    const double tile_mb = gated_tile_rows(size) * gated_tile_cols(size) * 4e-6;
    const auto consider = [&](int64_t parts) {
      if (parts < 1 || (parts > 1 && (!may_cut || rest == 0 || ceil_div(k_tiles, parts) < 4 || rest * parts > (1 << 24)))) return;
      const int64_t k_part = ceil_div(k_tiles, parts);
      parts = ceil_div(k_tiles, k_part);
      double time = static_cast<double>(whole / slots) * unit;
      if (rest > 0) time += static_cast<double>(ceil_div(rest * parts, slots)) * (k_part * kStep[size] + kBesides[size]);
      if (parts > 1) time += 6.0 + 0.4 * static_cast<double>(rest * parts) * tile_mb;
      if (best.k_tiles != 0 && time >= least) return;
      least = time;
      best = p;
      best.parts = static_cast<int32_t>(parts);
      best.k_part = k_part;
      best.whole = parts > 1 ? whole : tiles;
      best.units = parts > 1 ? whole + rest * parts : tiles;
    };
    for (int64_t parts = 1; parts <= 8; ++parts) consider(parts);
    for (int64_t rounds = 1; rounds <= 4 && rest > 0; ++rounds) consider(rounds * slots / rest);
  }
  return best;
}

inline size_t gated_partial_bytes(const GatedPlan& p) {
  return static_cast<size_t>(p.units - p.whole) * gated_tile_rows(p.size) * gated_tile_cols(p.size) * (p.parts > 1 ? 4 : 0);
}

template <class Ty, class Out, int MODE, class T>
int launch_gated_tile(const GatedArgs& a, hipStream_t s) {
  const int64_t most = T::kTurns ? gated_at_once(a.p.size) : a.p.units;
  const unsigned grid = static_cast<unsigned>(a.p.units < most ? a.p.units : most);
  hipLaunchKernelGGL((gated_tile_kernel<Ty, Out, MODE, T>), dim3(grid), dim3(T::kThreads), 0, s, a);
  if (int rc = hip_status(hipGetLastError(), "gated_tile_kernel launch")) return rc;
  if constexpr (MODE != kGatedGates) {
    if (a.p.parts > 1) {
      constexpr int64_t kPerTile = T::BR * (gated_pair(MODE) ? T::BC / 2 : T::BC) / 4 / 256;
      const int64_t cut = a.p.tiles_r * a.p.tiles_c - a.p.whole;
      hipLaunchKernelGGL((gated_join_kernel<Out, MODE, T>), dim3(static_cast<unsigned>(cut * kPerTile)), dim3(256), 0, s, a);
      return hip_status(hipGetLastError(), "gated_join_kernel launch");
    }
  }
  return OW_OK;
}

template <class Ty, class Out, int MODE>
int launch_gated(const GatedArgs& a, hipStream_t s) {
  if (a.p.size == 0) return launch_gated_tile<Ty, Out, MODE, TileL>(a, s);
  if (a.p.size == 1) return launch_gated_tile<Ty, Out, MODE, TileM>(a, s);
  return launch_gated_tile<Ty, Out, MODE, TileS>(a, s);
}

template <int MODE>
int launch_gated_mode(GatedArgs& a, const GatedPlan& p, int dtype, int64_t k, float* partial, hipStream_t s) {
  a.p = p;
  a.partial = partial;
  a.k_each = static_cast<int32_t>(ceil_div(k, 64));
  const int64_t cut = p.tiles_r * p.tiles_c - p.whole;
  a.by_group = Divisor::of(8 * static_cast<uint32_t>(p.tiles_c));
  a.by_split = Divisor::of(cut > 0 ? static_cast<uint32_t>(cut) : 1u);
  a.by_each = Divisor::of(static_cast<uint32_t>(a.k_each));
  if (dtype == OW_DTYPE_BF16) return launch_gated<BF16, BF16, MODE>(a, s);
  if (dtype == OW_DTYPE_F16) return launch_gated<F16, F16, MODE>(a, s);
  return launch_gated<BF16, F32, MODE>(a, s);
}

// Tiles of k of a product over `k` values.
inline int64_t gated_k_tiles(int64_t k, int dtype) { return ceil_div(k, 64) * (dtype == OW_DTYPE_F32 ? 6 : 1); }

}  // namespace ow
