// Tiled matrix products on the matrix cores, for the linear log loss (lbt_linear_loss.hip).
//
// C[m][n] = sum_k A(m, k) B(n, k), added in 32 bits. An operand is an array of 16-bit numbers in rows, and either of its two
// directions may be the one that is contiguous:
//   k contiguous   rows are the product's m (or n), read by ds_read_b128
//   k in rows      rows are the product's k; ds_read_b64_tr_b16 turns 4 x 16 blocks on their way out of the LDS, so that
//                  no operand is ever transposed in memory
// A workgroup forms a tile of kBM x kBN, 64 values of k at a time, which go from memory into the LDS without passing
// through registers (global_load_lds, 16 bytes a lane). What lies outside an operand is read from a page of zeros, lane by
// lane, so the loop has no edges. The LDS holds 16-byte chunks in an order (an exclusive or with the row's number) in which
// the 32 rows that a fragment reads lie on all banks.
//
// A large product of 16 bits runs at 1210 to 1310 TFLOP/s, where the card's library reaches 1239 to 1304 by its size (8192 x 16384 x 4096 and
// 8192^3). The matrix cores are busy 57 to 63 % of the cycles and the clock is at 1.85 GHz then, for the library's products too: most
// likely the card's limit of power, which was not measured. Measured
// and not better: stages of 32 of k four and five deep, waves of 128 x 128, waves of raised priority.
//
// float operands are sums of three bfloat16 planes (8 + 8 + 8 significant bits, exact); of the nine products of planes the
// six that reach above 2^-24 of the result are added up, one walk over k each. (The scores, and grad_X of few rows, whose
// first operand lies in memory as floats, have a product of their own below.)
#pragma once

#include <type_traits>

#include "lbt_internal.h"

namespace lbt {

typedef __attribute__((ext_vector_type(4))) short Short4;
typedef __attribute__((ext_vector_type(8))) short Short8;
typedef __attribute__((ext_vector_type(8))) __bf16 Bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 Half8;
typedef __attribute__((ext_vector_type(16))) float Float16v;

constexpr int kProductK = 64;  // values of k in a stage of the LDS

// One operand: plane p of row r begins at base + p * plane + r * ld (elements). cols is a multiple of 8.
struct ProductOperand {
  const uint16_t* base;
  int64_t ld;
  int64_t plane;
  int32_t rows;
  int32_t cols;
};

// What the rows of a call come down to; written on the device by prepare_rows_kernel or prepare_pack_kernel.
struct RowCounts {
  int32_t rows;      // rows that count
  int32_t exponent;  // the largest exponent of a row's weight (half precision)
  int32_t reach;     // the largest exponent of a weight times a value of its row (half precision)
};

struct ProductArgs {
  ProductOperand a, b;
  int32_t k_extent;  // k ends here, or (row products over k) at the rows that count
  int32_t k_split;   // values of k of one split, a multiple of kProductK
  int32_t tiles_m, tiles_n;
  const uint16_t* zeros;  // 16 bytes of zeros
  const RowCounts* counts;
};

template <int kM, int kN, int kWaveM, int kWaveN, int kDepth>
struct ProductTile {
  static constexpr int kBM = kM, kBN = kN;              // tile of a workgroup
  static constexpr int kWM = kM / kWaveM, kWN = kN / kWaveN;  // tile of a wave
  static constexpr int kWavesM = kWaveM, kWavesN = kWaveN;
  static constexpr int kWaves = kWaveM * kWaveN, kThreads = kWaves * 64;
  static constexpr int kMT = kWM / 32, kNT = kWN / 32;  // 32 x 32 blocks of a wave
  static constexpr int kStages = kDepth;                // of the LDS
  // Steps of 16 of k whose fragments are read together: a wave of one block has too little to multiply in a step to cover a read.
  static constexpr int kGroup = kMT == 1 ? kProductK / 16 : 1;
  static constexpr int kStageA = kM * kProductK * 2, kStageB = kN * kProductK * 2;  // bytes
  static constexpr int kLds = kStages * (kStageA + kStageB);
  static constexpr int kLoads = (kM + kN) * kProductK / 8 / kThreads;               // of a lane for a stage
};

template <int kType>  // LBT_BF16 or LBT_F16
__device__ __forceinline__ Float16v mfma_32x32x16(Short8 a, Short8 b, Float16v c)
{
  if constexpr (kType == LBT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Half8, a), __builtin_bit_cast(Half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}

// 16 bytes a lane from memory into the LDS, in the order of the lanes from `lds` on. The compiler's own form of this load is waited
// for before the next read of the LDS, whichever part that reads; here the waits are those of wait_and_meet.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t lds)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds(const void* from, uint32_t lds)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}

// All but the last kLater loads of this wave have arrived, and all it has read from the LDS; then the same holds for every wave.
template <int kLater>
__device__ __forceinline__ void wait_and_meet()
{
  static_assert(kLater < 64, "the counter's range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater) : "memory");
}

// What the number of a chunk in a row of k is turned by, within the row's kTile / 8 chunks: rows that are read together lie on
// different banks, 64 bytes apart.
template <int kTile>
__device__ __forceinline__ int turned(int row)
{
  return (row & (kTile >= 128 ? 3 : 1)) << 2;
}

// One operand's way through the stages of a product: kTile of its m (or n) from `tile0` on, 64 of k at a time from `k_first`
// to `k_end`, once for each plane that is multiplied. What a stage asks of the scalar unit is an addition and a comparison:
// with small tiles that is what a stage takes.
template <bool kRowsAreK, int kTile, int kWaves>
struct StageLoader {
  static constexpr int kEach = kTile * kProductK / 8 / (kWaves * 64);  // chunks of 16 bytes of a lane
  static_assert(kEach * kWaves * 64 * 8 == kTile * kProductK, "every lane loads the same number of chunks");
  const uint16_t* at;       // first element of the next stage
  int64_t step;             // from stage to stage
  int whole;                // stages of a plane that lie inside the operand
  uint32_t offset[kEach];   // of a lane's chunks, bytes

  static __device__ __forceinline__ void place(int j, int wave, int lane, int* row, int* col)
  {
    const int q = (j * kWaves + wave) * 64 + lane;
    if constexpr (kRowsAreK) {
      constexpr int kRow = kTile / 8;  // chunks of a row
      *row = q / kRow;
      *col = ((q % kRow) ^ turned<kTile>(*row)) * 8;
    } else {
      *row = q >> 3;
      *col = ((q & 7) ^ ((*row >> 1) & 7)) * 8;
    }
  }
  __device__ __forceinline__ void begin(const ProductOperand& op, int plane, int tile0, int k_first)
  {
    at = op.base + plane * op.plane + (kRowsAreK ? static_cast<int64_t>(k_first) * op.ld + tile0 : static_cast<int64_t>(tile0) * op.ld + k_first);
  }
  __device__ __forceinline__ void init(const ProductOperand& op, int tile0, int k_first, int k_end, int wave, int lane)
  {
    const int limit = kRowsAreK ? op.rows : op.cols;  // of k
    const bool edge = tile0 + kTile > (kRowsAreK ? op.cols : op.rows);
    // (the last stage may reach past k_end: there the other operand, or this one, holds zeros)
    whole = edge ? 0 : max(0, min((k_end - k_first + kProductK - 1) / kProductK, (limit - k_first) / kProductK));
    step  = kRowsAreK ? kProductK * op.ld : kProductK;
#pragma unroll
    for (int j = 0; j < kEach; j++) {
      int row, col;
      place(j, wave, lane, &row, &col);
      offset[j] = (static_cast<uint32_t>(row) * static_cast<uint32_t>(op.ld) + col) * 2;
    }
  }
  // Asks for stage `s` of a plane. One that reaches past the operand, or that there is none of (not `live`), has zeros there.
  __device__ __forceinline__ void load(const ProductOperand& op, int tile0, int k_first, int s, bool live, const uint16_t* zeros,
                                       uint32_t lds, int wave, int lane)
  {
    if (s < whole) {
      const uint64_t bits  = reinterpret_cast<uint64_t>(at);  // (the same in all lanes, which the compiler loses sight of)
      const void* const to = reinterpret_cast<const void*>(
        static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits >> 32))) << 32 |
        static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits))));
#pragma unroll
      for (int j = 0; j < kEach; j++) load_to_lds(to, offset[j], lds + (j * kWaves + wave) * 1024);
    } else {
      const int k0   = k_first + s * kProductK;
      const int row0 = kRowsAreK ? k0 : tile0, col0 = kRowsAreK ? tile0 : k0;
#pragma unroll
      for (int j = 0; j < kEach; j++) {
        int row, col;
        place(j, wave, lane, &row, &col);
        const bool inside   = live && row0 + row < op.rows && col0 + col < op.cols;
        const uint16_t* from = at + static_cast<int64_t>(row) * op.ld + col;
        load_to_lds(inside ? from : zeros, lds + (j * kWaves + wave) * 1024);
      }
    }
    at += step;
  }
};

// Eight values of k for each of 32 values of m (or n) from `first` on: lane l has m = l % 32, k = 16 kk + 8 (l / 32) ...
template <bool kRowsAreK, int kTile>
__device__ __forceinline__ Short8 fragment(const char* lds, int first, int kk, int lane)
{
  if constexpr (kRowsAreK) {
    const int row   = kk * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2);
    const int col   = first + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    const int chunk = (col >> 3) ^ turned<kTile>(row);
    const char* at  = lds + row * (kTile * 2) + chunk * 16 + (col & 7) * 2;
    typedef __attribute__((address_space(3))) Short4* LdsPtr;
    const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)at);
    const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 4 * (kTile * 2)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int row   = first + (lane & 31);
    const int chunk = (kk * 2 + (lane >> 5)) ^ ((row >> 1) & 7);
    return *reinterpret_cast<const Short8*>(lds + row * (kProductK * 2) + chunk * 16);
  }
}

// Tile of this workgroup: workgroups go round the 8 XCDs by their number, each XCD takes a run of tiles, and a run goes
// through `kGroup` tiles of m for every tile of n, so that what an XCD has in its L2 is used by several tiles.
__device__ __forceinline__ void tile_of_block(int block, int tiles_m, int tiles_n, int* m, int* n)
{
  constexpr int kXcds = 8, kGroup = 8;
  const int tiles = tiles_m * tiles_n;
  const int share = tiles / kXcds, more = tiles % kXcds;
  const int xcd   = block % kXcds;
  const int at    = xcd * share + min(xcd, more) + block / kXcds;
  const int width = kGroup * tiles_n;
  const int group = at / width;
  const int size  = min(tiles_m - group * kGroup, kGroup);
  *m = group * kGroup + (at % width) % size;
  *n = (at % width) / size;
}

// Which planes are multiplied: the small products first.
template <int kPlanes>
struct PlanePairs;
template <>
struct PlanePairs<1> {
  static constexpr int kCount = 1;
  __device__ static int a(int) { return 0; }
  __device__ static int b(int) { return 0; }
};
template <>
struct PlanePairs<3> {
  static constexpr int kCount = 6;  // (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
  __device__ static int a(int i) { return (0x001012 >> (4 * i)) & 15; }
  __device__ static int b(int i) { return (0x010210 >> (4 * i)) & 15; }
};

// kRowsSide: which direction of the product is the call's rows
enum { kRowsN = 0, kRowsK = 1 };

// Tile `block` of split `split`, in an LDS of Tile::kLds bytes.
template <class Tile, int kType, int kPlanes, bool kAMajor, bool kBMajor, int kRowsSide, class Epilogue>
__device__ __forceinline__ void product_tile(const ProductArgs& args, const Epilogue& epilogue, int block, int split, char* lds)
{
  constexpr int kStage = Tile::kStageA + Tile::kStageB, kSteps = kProductK / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int tile_m, tile_n;
  tile_of_block(block, args.tiles_m, args.tiles_n, &tile_m, &tile_n);
  const int rows = args.counts->rows;
  int k_end      = args.k_extent;
  if (kRowsSide == kRowsN && tile_n * Tile::kBN >= rows) return;
  if (kRowsSide == kRowsK) k_end = min(k_end, rows);
  const int k_first = split * args.k_split;
  k_end             = min(k_end, k_first + args.k_split);
  const int steps   = k_end > k_first ? (k_end - k_first + kProductK - 1) / kProductK : 0;

  const int wm = wave / Tile::kWavesN, wn = wave % Tile::kWavesN;
  Float16v acc[Tile::kMT][Tile::kNT];
#pragma unroll
  for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

  const int total = steps * PlanePairs<kPlanes>::kCount;
  StageLoader<kAMajor, Tile::kBM, Tile::kWaves> load_a;
  StageLoader<kBMajor, Tile::kBN, Tile::kWaves> load_b;
  const int m0 = tile_m * Tile::kBM, n0 = tile_n * Tile::kBN;
  load_a.init(args.a, m0, k_first, k_end, wave, lane);
  load_b.init(args.b, n0, k_first, k_end, wave, lane);
  load_a.begin(args.a, PlanePairs<kPlanes>::a(0), m0, k_first);
  load_b.begin(args.b, PlanePairs<kPlanes>::b(0), n0, k_first);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  // Stages are asked for in order, the first operand's part before the second's: stage `asked` of the pair `pair` of planes.
  int asked = 0, pair = 0;
  bool live = total > 0;
  if (!live) load_a.whole = load_b.whole = 0;
  auto load = [&](int stage, auto second) {
    const uint32_t at = lds0 + stage * kStage;
    if constexpr (!decltype(second)::value) {
      load_a.load(args.a, m0, k_first, asked, live, args.zeros, at, wave, lane);
    } else {
      load_b.load(args.b, n0, k_first, asked, live, args.zeros, at + Tile::kStageA, wave, lane);
      if (++asked < steps) return;
      asked = 0;
      pair++;
      if (pair < PlanePairs<kPlanes>::kCount && steps > 0) {
        load_a.begin(args.a, PlanePairs<kPlanes>::a(pair), m0, k_first);
        load_b.begin(args.b, PlanePairs<kPlanes>::b(pair), n0, k_first);
      } else {
        live         = false;
        load_a.whole = load_b.whole = 0;
      }
    }
  };
  constexpr std::false_type kA{};
  constexpr std::true_type kB{};
  // A group of steps' fragments are read while those of the group before are multiplied.
  constexpr int kGroup = Tile::kGroup, kGroups = kSteps / kGroup;
  Short8 a[2][kGroup][Tile::kMT], b[2][kGroup][Tile::kNT];
  // The i-th part of the fragments of a step: the second operand's first, all of which the next step begins with.
  auto read = [&](const char* at, int kk, int to, int i) {
    constexpr int kAll = Tile::kMT + Tile::kNT;
#pragma unroll
    for (int p = i * kAll / Tile::kMT; p < (i + 1) * kAll / Tile::kMT; p++) {
      if (p < Tile::kNT) b[to][kk % kGroup][p] = fragment<kBMajor, Tile::kBN>(at + Tile::kStageA, wn * Tile::kWN + p * 32, kk, lane);
      else a[to][kk % kGroup][p - Tile::kNT] = fragment<kAMajor, Tile::kBM>(at, wm * Tile::kWM + (p - Tile::kNT) * 32, kk, lane);
    }
  };
  // Stages are asked for kStages ahead. The fragments of a stage's first group are read while the last one of the stage before is
  // multiplied, after all waves have met: then that stage has been read by all, and is filled again, and the next has arrived.
  // Reads and loads are dealt out between the multiplications.
#pragma unroll
  for (int s = 0; s < Tile::kStages; s++) {
    load(s, kA);
    load(s, kB);
  }
  wait_and_meet<(Tile::kStages - 1) * Tile::kLoads>();
#pragma unroll
  for (int kk = 0; kk < kGroup; kk++)
#pragma unroll
    for (int i = 0; i < Tile::kMT; i++) read(lds, kk, 0, i);
  int stage = 0;
  // `own`: which half of the fragments holds the stage's first group
  auto multiply_stage = [&](auto own) {
    const int next = stage + 1 == Tile::kStages ? 0 : stage + 1;
#pragma unroll
    for (int group = 0; group < kGroups; group++) {
      const int from  = (decltype(own)::value + group) & 1;
      const bool last = group + 1 == kGroups;
      if (last) wait_and_meet<(Tile::kStages - 2) * Tile::kLoads>();
#pragma unroll
      for (int kk = 0; kk < kGroup; kk++)
#pragma unroll
        for (int i = 0; i < Tile::kMT; i++) {
          if (last) read(lds + next * kStage, kk, 1 - from, i);
          else read(lds + stage * kStage, (group + 1) * kGroup + kk, 1 - from, i);
          if constexpr (kGroup > 1) continue;  // (all reads of a group of several steps come first)
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < Tile::kNT; j++) acc[i][j] = mfma_32x32x16<kType>(a[from][kk][i], b[from][kk][j], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
          if (last && i == 0) load(stage, kA);
          if (last && i == Tile::kMT / 2) load(stage, kB);
        }
      if constexpr (kGroup > 1) {
        if (last) {
          load(stage, kA);
          load(stage, kB);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < kGroup; kk++)
#pragma unroll
          for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
            for (int j = 0; j < Tile::kNT; j++) acc[i][j] = mfma_32x32x16<kType>(a[from][kk][i], b[from][kk][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    stage = next;
  };
  if constexpr (kGroups % 2 == 0) {
    for (int t = 0; t < total; t++) multiply_stage(std::integral_constant<int, 0>{});
  } else {
    for (int t = 0; t < total; t += 2) {
      multiply_stage(std::integral_constant<int, 0>{});
      if (t + 1 < total) multiply_stage(std::integral_constant<int, 1>{});
    }
  }
  wait_and_meet<0>();  // the LDS is free for what follows
  epilogue.template store<Tile>(acc, tile_m, tile_n, wm, wn, lane, rows, split, args.counts, lds);
}

template <class Tile, int kType, int kPlanes, bool kAMajor, bool kBMajor, int kRowsSide, class Epilogue>
__global__ void __launch_bounds__(Tile::kThreads, 2) product_kernel(const ProductArgs args, const Epilogue epilogue)
{
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  product_tile<Tile, kType, kPlanes, kAMajor, kBMajor, kRowsSide>(args, epilogue, blockIdx.x, blockIdx.y, lds);
}

// Two products that need nothing of one another in one launch: both operands' k in rows for the second, the first operand's for the
// first. What they take alone is mostly their beginning and end where both are in small tiles (64 rows of 256 floats, 1000 classes:
// 10 us, 17 as two launches).
template <class Tile, int kType, int kPlanes, class First, class Second>
__global__ void __launch_bounds__(Tile::kThreads, 2)
  two_products_kernel(const ProductArgs args, const First first, unsigned blocks, const ProductArgs more, const Second second)
{
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  if (blockIdx.x < blocks) {
    const int tiles = args.tiles_m * args.tiles_n;
    product_tile<Tile, kType, kPlanes, true, false, kRowsN>(args, first, blockIdx.x % tiles, blockIdx.x / tiles, lds);
  } else {
    const int tiles = more.tiles_m * more.tiles_n, block = blockIdx.x - blocks;
    product_tile<Tile, kType, kPlanes, true, true, kRowsK>(more, second, block % tiles, block / tiles, lds);
  }
}

// ---- float by planes: the first operand as it lies in memory ----------------------------------------
//
// C[m][n] = sum_k A(m, k) B(n, k) for an A of floats that is read once, in rows of any length of k or (kAMajor) of m, and a B laid out in planes.
// A goes into the LDS as floats and becomes three planes on its way from the registers to the matrix cores: hi is the float's upper
// half, what is left goes on exactly and is rounded, v = hi + mid + lo. The six products of a step follow one another, so a value is
// read from memory and from the LDS once where operands of planes are read up to six times, and nothing is laid out first. The eight
// values of a fragment take 44 instructions to split while its 6 products with each fragment of B take 192 cycles. Large sizes are
// bound as the products of 16 bits are (4096 rows, 30000 classes of 1000: 1.25 ms, 1200 TFLOP/s of bfloat16), few tiles by what a wave does
// between two stages: a tile of 64 is therefore two waves a SIMD, each with half of a stage's k (256 rows, 3000 classes of 4000: 75 us, 100 by
// four waves), and has two sums of a block.
template <int kM, int kN, int kWaveM, int kWaveN, int kWaveK, int kDepth>
struct FloatTile {
  static constexpr int kBM = kM, kBN = kN, kWM = kM / kWaveM, kWN = kN / kWaveN;
  static constexpr int kWavesM = kWaveM, kWavesN = kWaveN, kWavesK = kWaveK;
  static constexpr int kWaves = kWaveM * kWaveN * kWaveK, kThreads = kWaves * 64;
  static constexpr int kMT = kWM / 32, kNT = kWN / 32, kStages = kDepth;
  static constexpr int kK = 32;  // of a stage
  static constexpr int kStageA = kM * kK * 4, kRowB = 3 * kK * 2, kStage = kStageA + kN * kRowB, kLds = kStages * kStage;  // bytes
  // loads of a wave for a stage; the first kMore waves have one of B more where they do not come out even
  static constexpr int kLoadsA = kM * kK / 4 / kThreads, kPartsB = 3 * kN * kK / 8 / 64, kLoadsB = kPartsB / kWaves, kMore = kPartsB % kWaves;
  static constexpr int kEachB = kLoadsB + (kMore > 0), kLoads = kLoadsA + kLoadsB;
  static_assert(kLoadsA * 4 * kThreads == kM * kK && kPartsB * 512 == 3 * kN * kK, "a stage is whole loads");
};

struct FloatArgs {
  const float* a;        // [rows][cols]
  int32_t rows, cols;
  int32_t k_split;       // values of k of one split, a multiple of kK
  const uint16_t* b;  // [k / kK][b_rows][3][kK], padded with zeros
  int64_t b_rows;     // a multiple of the tile
  int32_t tiles_m, tiles_n;
  const uint16_t* zeros;
  const RowCounts* counts;
};

// 4 bytes a lane from memory into the LDS.
__device__ __forceinline__ void load_word_to_lds(const void* from, uint32_t lds)
{
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(from) : "memory");
}

// (infinities leave NaN in the second plane: their product with a plane that is 0 is NaN in any case)
__device__ __forceinline__ void split_eight(const float4& low, const float4& high, Short8 (&out)[3])
{
  typedef __attribute__((ext_vector_type(2))) float Float2v;
  typedef __attribute__((ext_vector_type(2))) __bf16 Bf16x2;
  const float v[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t b0 = __builtin_bit_cast(uint32_t, v[2 * i]), b1 = __builtin_bit_cast(uint32_t, v[2 * i + 1]);
    w[0][i]        = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
    const float r0 = v[2 * i] - __builtin_bit_cast(float, b0 & 0xffff0000u), r1 = v[2 * i + 1] - __builtin_bit_cast(float, b1 & 0xffff0000u);
    w[1][i]        = __builtin_bit_cast(uint32_t, __builtin_convertvector(Float2v{r0, r1}, Bf16x2));
    const float s0 = r0 - __builtin_bit_cast(float, w[1][i] << 16), s1 = r1 - __builtin_bit_cast(float, w[1][i] & 0xffff0000u);
    w[2][i]        = __builtin_bit_cast(uint32_t, __builtin_convertvector(Float2v{s0, s1}, Bf16x2));
  }
#pragma unroll
  for (int q = 0; q < 3; q++) out[q] = __builtin_bit_cast(Short8, make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]));
}

// kAMajor: A's rows are its k, its columns the product's m; a fragment's eight values are then eight reads of 4 bytes, each of 32 values
// of m beside one another, and in every second eight of k 32 values of m have changed places, which puts the lanes on all banks.
template <class Tile, bool kAMajor, class Epilogue>
__global__ void __launch_bounds__(Tile::kThreads, 2) float_product_kernel(const FloatArgs args, const Epilogue epilogue)
{
  __shared__ __attribute__((aligned(1024))) char lds[Tile::kLds];
  constexpr int kK = Tile::kK, kSteps = kK / 16 / Tile::kWavesK;  // of 16 of k, of a wave for a stage
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int tile_m, tile_n;
  tile_of_block(blockIdx.x, args.tiles_m, args.tiles_n, &tile_m, &tile_n);
  const int rows = args.counts->rows;
  if (tile_n * Tile::kBN >= rows) return;
  const int m0 = tile_m * Tile::kBM, n0 = tile_n * Tile::kBN;
  const int wk = wave / (Tile::kWavesM * Tile::kWavesN), wm = wave / Tile::kWavesN % Tile::kWavesM, wn = wave % Tile::kWavesN;
  const int k_extent = kAMajor ? args.rows : args.cols, k_first = blockIdx.y * args.k_split;
  const int steps    = (min(args.k_split, max(k_extent - k_first, 0)) + kK - 1) / kK;
  // Stages of A that are read in whole chunks: those within its rows; with k in rows, those that end, with what follows the last row of
  // the tile, within the array.
  int whole = (k_extent - k_first) / kK;
  if constexpr (kAMajor) {
    const int64_t room = static_cast<int64_t>(args.rows) * args.cols - m0 - Tile::kBM;  // for the first column of a stage's last row
    const int last     = static_cast<int>(room < 0 ? -1 : room / args.cols) - (kK - 1);  // first row of the last such stage
    whole              = min(whole, last < k_first ? 0 : (last - k_first) / kK + 1);
  }
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int a_first = min(m0, args.rows - 1), a_last = args.rows - 1 - a_first;  // (tiles may lie past the last row)
  const float* const a0 = args.a + (kAMajor ? static_cast<int64_t>(k_first) * args.cols + m0 : static_cast<int64_t>(a_first) * args.cols);
  const uint16_t* const b0 = args.b + (static_cast<int64_t>(k_first / kK) * args.b_rows + n0) * (3 * kK);
  // A: 8 chunks of 16 bytes of a row, their order turned by pairs of rows; rows past the last are the last one once more. k in rows: the
  // chunks of a row, turned by eights of rows.
  uint32_t from_a[Tile::kLoadsA], from_b[Tile::kEachB];
#pragma unroll
  for (int j = 0; j < Tile::kLoadsA; j++) {
    const int q = (j * Tile::kWaves + wave) * 64 + lane;
    constexpr int kRow = Tile::kBM / 4;  // chunks of a row of k
    const int row   = kAMajor ? q / kRow : min(q >> 3, a_last);
    const int chunk = kAMajor ? (q % kRow) ^ (((row >> 3) & 1) << 3) : (q & 7) ^ ((q >> 4) & 7);
    from_a[j]       = (static_cast<uint32_t>(row) * static_cast<uint32_t>(args.cols) + chunk * 4) * 4;
  }
  // B: 3 planes of 4 chunks of a row, turned by fours of rows
#pragma unroll
  for (int j = 0; j < Tile::kEachB; j++) {
    const int q = (j * Tile::kWaves + wave) * 64 + lane;
    from_b[j]   = (q ^ ((q / 12 >> 2) & 3)) * 16;
  }
  const bool more_loads = wave < Tile::kMore;
  auto meet = [&](auto stages) {  // wait_and_meet with the loads of so many stages on their way
    constexpr int kLater = decltype(stages)::value;
    if (Tile::kMore > 0 && more_loads) wait_and_meet<kLater * (Tile::kLoads + 1)>();
    else wait_and_meet<kLater * Tile::kLoads>();
  };
  auto uniform = [](const void* p) {
    const uint64_t bits = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const void*>(static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits >> 32))) << 32 |
                                         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bits))));
  };
  // Stage `s` into its place: kLoads of them at least, whether there is such a stage or not, as the waits count them.
  auto load = [&](int s, int place) {
    const uint32_t at = lds0 + place * Tile::kStage;
    if (s < whole) {
      const void* const a = uniform(a0 + (kAMajor ? static_cast<int64_t>(s) * kK * args.cols : s * kK));
#pragma unroll
      for (int j = 0; j < Tile::kLoadsA; j++) load_to_lds(a, from_a[j], at + (j * Tile::kWaves + wave) * 1024);
    } else if (s < steps) {  // the ends, by single floats
      for (int j = 0; j < Tile::kLoadsA * 4; j++) {
        const int q = (j * Tile::kWaves + wave) * 64 + lane;
        const float* from;
        bool inside;
        if constexpr (kAMajor) {
          const int row = s * kK + q / Tile::kBM, col = (q % Tile::kBM) ^ (((row >> 3) & 1) << 5);
          inside        = k_first + row < args.rows && m0 + col < args.cols;
          from          = a0 + static_cast<int64_t>(row) * args.cols + col;
        } else {
          const int row = q >> 5, k = s * kK + ((((q >> 2) & 7) ^ ((row >> 1) & 7)) * 4 + (q & 3));
          inside        = k < args.cols;
          from          = a0 + static_cast<int64_t>(min(row, a_last)) * args.cols + k;
        }
        load_word_to_lds(inside ? static_cast<const void*>(from) : args.zeros, at + (j * Tile::kWaves + wave) * 256);
      }
    } else {
#pragma unroll
      for (int j = 0; j < Tile::kLoadsA; j++) load_to_lds(args.zeros, at + (j * Tile::kWaves + wave) * 1024);
    }
    if (s < steps) {
      const void* const b = uniform(b0 + s * args.b_rows * (3 * kK));
#pragma unroll
      for (int j = 0; j < Tile::kEachB; j++) {
        if (j == Tile::kLoadsB && !more_loads) continue;
        load_to_lds(b, from_b[j], at + Tile::kStageA + (j * Tile::kWaves + wave) * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < Tile::kEachB; j++)
        if (j < Tile::kLoadsB || more_loads) load_to_lds(args.zeros, at + Tile::kStageA + (j * Tile::kWaves + wave) * 1024);
    }
  };
  Float16v acc[Tile::kMT][Tile::kNT];
#pragma unroll
  for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
  // a wave of one block has two sums of it, that a product does not wait for the one before
  constexpr int kSums = Tile::kMT * Tile::kNT == 1 ? 2 : 1;
  Float16v more[kSums == 2 ? 1 : Tile::kMT][kSums == 2 ? 1 : Tile::kNT];
#pragma unroll
  for (int e = 0; kSums == 2 && e < 16; e++) more[0][0][e] = 0.f;
  float4 raw[Tile::kMT][2];
  Short8 a[2][Tile::kMT][3], b[2][Tile::kNT][3];
  auto read = [&](const char* at, int step, int to) {
    const int kk = wk * kSteps + step;
#pragma unroll
    for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if constexpr (kAMajor) {
          const int m      = (wm * Tile::kWM + i * 32 + (lane & 31)) ^ ((lane >> 5) << 5);
          const float* row = reinterpret_cast<const float*>(at) + (kk * 16 + (lane >> 5) * 8 + h * 4) * Tile::kBM + m;
          raw[i][h]        = make_float4(row[0], row[Tile::kBM], row[2 * Tile::kBM], row[3 * Tile::kBM]);
        } else {
          const int row = wm * Tile::kWM + i * 32 + (lane & 31), chunk = (kk * 4 + (lane >> 5) * 2 + h) ^ ((row >> 1) & 7);
          raw[i][h]     = *reinterpret_cast<const float4*>(at + row * (kK * 4) + chunk * 16);
        }
      }
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++)
#pragma unroll
      for (int q = 0; q < 3; q++) {
        const int row = wn * Tile::kWN + j * 32 + (lane & 31), chunk = (kk * 2 + (lane >> 5)) ^ ((row >> 2) & 3);
        b[to][j][q] = *reinterpret_cast<const Short8*>(at + Tile::kStageA + row * Tile::kRowB + (q * 4 + chunk) * 16);
      }
  };
  auto multiply = [&](int from, int first, int last) {  // products first .. last - 1 of a step
    constexpr int kA[6] = {2, 1, 0, 1, 0, 0}, kB[6] = {0, 1, 2, 0, 1, 0};  // the small ones first
#pragma unroll
    for (int p = first; p < last; p++)
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
        for (int j = 0; j < Tile::kNT; j++) {
          Float16v& to = kSums == 2 && p % 2 == 0 ? more[i][j] : acc[i][j];
          to           = mfma_32x32x16<LBT_BF16>(a[from][i][kA[p]], b[from][j][kB[p]], to);
        }
  };
  // As in product_tile: what a step multiplies has been read during the one before; all waves meet before a stage's last step, when
  // that stage has been read by all and the next has arrived. The next step's planes are made between the second half of the
  // products: a wave's own instructions fill the matrix cores' time only where they stand between theirs.
#pragma unroll
  for (int s = 0; s < Tile::kStages; s++) load(s, s);
  meet(std::integral_constant<int, Tile::kStages - 1>{});
  read(lds, 0, 0);
#pragma unroll
  for (int i = 0; i < Tile::kMT; i++) split_eight(raw[i][0], raw[i][1], a[0][i]);
  int place = 0;
  auto multiply_stage = [&](int s, auto own) {  // `own`: which half of the fragments holds the stage's first step
    const int next = place + 1 == Tile::kStages ? 0 : place + 1;
#pragma unroll
    for (int kk = 0; kk < kSteps; kk++) {
      const bool last = kk + 1 == kSteps;
      const int from = (decltype(own)::value + kk) & 1, to = 1 - from;
      if (last) meet(std::integral_constant<int, Tile::kStages - 2>{});
      read(lds + (last ? next : place) * Tile::kStage, last ? 0 : kk + 1, to);
      __builtin_amdgcn_sched_barrier(0);
      if (last) load(s + Tile::kStages, place);
      __builtin_amdgcn_sched_barrier(0);
      multiply(from, 0, 3);
      __builtin_amdgcn_sched_barrier(0);
      multiply(from, 3, 6);
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++) split_eight(raw[i][0], raw[i][1], a[to][i]);
      constexpr int kHalf = 3 * Tile::kMT * Tile::kNT, kBetween = (Tile::kMT * 52 + kHalf - 1) / kHalf;
#pragma unroll
      for (int p = 0; p < kHalf; p++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, kBetween, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    place = next;
  };
  if constexpr (kSteps % 2 == 0) {
    for (int s = 0; s < steps; s++) multiply_stage(s, std::integral_constant<int, 0>{});
  } else {
    for (int s = 0; s < steps; s += 2) {
      multiply_stage(s, std::integral_constant<int, 0>{});
      if (s + 1 < steps) multiply_stage(s + 1, std::integral_constant<int, 1>{});
    }
  }
  if (kSums == 2) acc[0][0] += more[0][0];
  wait_and_meet<0>();  // the LDS is free for what follows
  if constexpr (Tile::kWavesK == 2) {
    static_assert(Tile::kMT * Tile::kNT == 1 && Tile::kThreads / 2 * 64 <= Tile::kLds / 2 && Tile::kWaves / 2 * 32 * 272 <= Tile::kLds / 2,
                  "a half's sums have room in the LDS");
    // (in its upper half: what follows begins to write in the lower one while another wave reads here)
    float4* const sums = reinterpret_cast<float4*>(lds + Tile::kLds / 2) + (wm * Tile::kWavesN + wn) * 256 + lane;
#pragma unroll
    for (int q = 0; wk == 1 && q < 4; q++) sums[q * 64] = make_float4(acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]);
    __syncthreads();
    if (wk == 1) return;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const float4 v = sums[q * 64];
      acc[0][0][4 * q] += v.x;
      acc[0][0][4 * q + 1] += v.y;
      acc[0][0][4 * q + 2] += v.z;
      acc[0][0][4 * q + 3] += v.w;
    }
  }
  epilogue.template store<Tile>(acc, tile_m, tile_n, wm, wn, lane, rows, blockIdx.y, args.counts, lds);
}

// Element e of a 32 x 32 block: its m within the block; its n is lane % 32.
__device__ __forceinline__ int block_m(int e, int lane) { return 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }

}  // namespace lbt
