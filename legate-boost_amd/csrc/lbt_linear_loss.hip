// Log loss of linear scores over many classes, without the scores in memory, and its gradient, which holds a piece of them.
//
//   s[r][c] = <X[r], weight[c]> + bias[c]      top[r] = max_c s, total[r] = sum_c exp(s - top)
//   loss[r] = log total[r] + top[r] - s[r][y[r]]
//   G[r][c] = w[r] (exp(s - top) / total - [c = y[r]])
//   grad_X = G weight,  grad_weight = G^T X,  grad_bias[c] = sum_r G[r][c]
//
// Rows whose label is no class are taken out first (prepare_rows_kernel or prepare_pack_kernel): what follows has only rows that
// count, side by side and padded with zeros, so a row that does not count costs nothing and what it holds reaches nothing.
// The scores are formed tile by tile (lbt_products.h), or for few rows straight from memory, and stay in registers: each wave leaves
// the top and the total of its share of a row, which are joined. For the gradient it also leaves u = exp(s - the share's top), where all
// classes are one piece (4 GiB of G and u): G is made from u once the totals are known, scale_kernel, instead of a second product. Where
// they are several the scores of a piece are formed a second time, GradientEpilogue. G is written in the type of the products
// and multiplied both ways. A row and class of a piece take 2 bytes in bfloat16 (6 with the gradient of a bias), 6 in half precision and 10 in
// float, 16 where G is laid out in two orders.
//
// What is rounded to fewer than 32 bits: an entry of G, to the type of the products (float: three planes, nothing lost above 2^-24 of
// it), as products of two 16-bit types are all that the matrix cores do at full rate; sums stay in float. In bfloat16 without the
// gradient of a bias u is held in 16 bits before that, 2^-11 of it beside the 2^-8 of G's own rounding. Against 64 bits the gradients
// are off 1.1 to 1.5 times as far as those of the same formulas in float, whose only such rounding is that of the result (in the norm,
// relative: 4096 rows, 32768 classes of 2048 bfloat16 0.0023 and 0.0017, 1531 rows of half precision 0.00029 and 0.00021). To hold G
// in two planes would cost two products more. Losses, sums of the bias and all results of float are as exact as those or more so.
//
// What it takes, at the card's rates of 1240 TFLOP/s for a large 16-bit product and 4.9 TB/s for a copy: 8192 rows of 4096 bfloat16 and
// 131072 classes 21.8 ms with gradients, three products at 1260 to 1310 TFLOP/s and 0.85 ms for G; 7373 rows of 2048 and 65536 classes
// 1.64 ms for the loss alone, 1210 TFLOP/s; one row of 1024 and 32768 classes 16 us, 4.2 TB/s. float is six products of bfloat16: 2048
// rows of 1024 and 16384 classes 1.14 ms with gradients, where a product in float at the card's 151 TFLOP/s would take 1.37.
//
// Half precision: G is held times 2^14 and with the weight's exponent taken out of its row (w = f 2^e, 1 <= |f| < 2), so that
// probabilities down to 2^-28 keep all their bits; grad_X gets 2^(e - 14) at its end, grad_weight multiplies rows of X times
// 2^(e - m), m such that the largest value comes to lie just below 2^15 and those of rows with small weights, 2^-29 of it, keep
// theirs. bfloat16 and float hold G as it is: their exponents reach far enough.
#include <algorithm>

#include "lbt_device.h"
#include "lbt_products.h"

namespace lbt {

namespace {

constexpr int kHalfShift = 14;
constexpr int64_t kPieceBytes  = int64_t(512) << 20;  // of packed weights at a time
constexpr int64_t kScoresBytes = int64_t(4) << 30;    // of G and of what it is made from at a time
// The same where the workspace is the least that is taken: 8192 rows, 131072 classes of 4096 bfloat16 then ask for 0.38 GiB instead of 2.25,
// and take 28.7 ms, as the scores are formed twice, instead of 21.6.
constexpr int64_t kLeastPieceBytes = int64_t(64) << 20, kLeastScoresBytes = int64_t(128) << 20;

template <int kDtype>
struct LossType;
template <>
struct LossType<LBT_BF16> {
  using Value = uint16_t;
  static constexpr int kProduct = LBT_BF16, kPlanes = 1;
};
template <>
struct LossType<LBT_F16> {
  using Value = uint16_t;
  static constexpr int kProduct = LBT_F16, kPlanes = 1;
};
template <>
struct LossType<LBT_F32> {
  using Value = float;
  static constexpr int kProduct = LBT_BF16, kPlanes = 3;
};

__device__ __forceinline__ uint16_t to_bf16(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }
__device__ __forceinline__ float from_bf16(uint16_t v) { return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16); }

// One rounding to the type of an operand's plane.
template <int kProduct>
__device__ __forceinline__ uint16_t narrow_value(float v)
{
  if constexpr (kProduct == LBT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  return to_bf16(v);
}

// A float as the sum of three bfloat16: what is left after each goes on exactly. A value that rounds up to infinity keeps
// the largest number instead; infinities and NaN are their own first plane and the others are 0.
__device__ __forceinline__ void split_planes(float v, uint16_t (&out)[3])
{
  uint16_t hi = to_bf16(v);
  if ((hi & 0x7fff) == 0x7f80 && fabsf(v) < INFINITY) hi = static_cast<uint16_t>(__builtin_bit_cast(uint32_t, v) >> 16);
  out[0]        = hi;
  const bool in = fabsf(v) < INFINITY;
  const float r = in ? v - from_bf16(hi) : 0.f;
  out[1]        = to_bf16(r);
  out[2]        = to_bf16(r - from_bf16(out[1]));
}

template <int kDtype>
__device__ __forceinline__ float load_value(const void* p, int64_t i)
{
  if constexpr (kDtype == LBT_F32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  if constexpr (kDtype == LBT_F16) return static_cast<float>(__builtin_bit_cast(_Float16, v));
  return from_bf16(v);
}

template <int kDtype>
__device__ __forceinline__ void store_value(void* p, int64_t i, float v)
{
  if constexpr (kDtype == LBT_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = narrow_value<kDtype>(v);
}

// Four values rounded to 16 bits, side by side.
template <int kType>
__device__ __forceinline__ uint2 narrow_four(const float (&v)[4])
{
  typedef __attribute__((ext_vector_type(4))) float Four;
  const Four f = {v[0], v[1], v[2], v[3]};
  if constexpr (kType == LBT_F16) {
    typedef __attribute__((ext_vector_type(4))) _Float16 Half4;
    return __builtin_bit_cast(uint2, __builtin_convertvector(f, Half4));
  } else {
    typedef __attribute__((ext_vector_type(4))) __bf16 Brain4;
    return __builtin_bit_cast(uint2, __builtin_convertvector(f, Brain4));
  }
}

// Four consecutive values of an output row of which `n` are inside. (The memory takes stores at any address: rows of an odd
// length need no others. One value at a time, grad_weight of 2519 features took twice the time of its product.)
template <int kDtype>
__device__ __forceinline__ void store_four(void* p, int64_t i, const float (&v)[4], int n)
{
  if (n >= 4) {
    if constexpr (kDtype == LBT_F32) {
      __builtin_memcpy(static_cast<float*>(p) + i, v, 16);
    } else {
      const uint2 w = narrow_four<kDtype>(v);
      __builtin_memcpy(static_cast<uint16_t*>(p) + i, &w, 8);
    }
    return;
  }
  for (int e = 0; e < 4; e++)
    if (e < n) store_value<kDtype>(p, i + e, v[e]);
}

// What is kept of each row that counts, in the order of the rows.
struct LossRows {
  int32_t* order;   // its number in the call
  int32_t* place;   // [n_rows of the call] where it went, or -1
  int32_t* label;
  float* factor;    // its weight, or (half precision) the weight's significand times 2^14
  int32_t* exponent;  // half precision: the weight's exponent
  float* picked;    // score of its label
  float* top;
  float* inverse;   // 1 / total
};

constexpr int kPrepareThreads = 1024;

// One workgroup goes through the labels, 4096 at a time: the rows that count, in order. Their weights' largest exponent is found
// on the way. It runs beside nothing, as all that follows needs it: what it takes is the latency of its loads and two meetings a turn,
// 5 us for 2048 rows, 9 for 8192.
__global__ void __launch_bounds__(kPrepareThreads)
  prepare_rows_kernel(const int64_t* __restrict__ y, const float* __restrict__ weight, int64_t n_rows, int64_t padded,
                      int n_classes, int half, LossRows out, float* __restrict__ loss, RowCounts* counts, uint16_t* zeros)
{
  constexpr int kEach = 4, kWaves = kPrepareThreads / 64;
  __shared__ int wave_sum[kEach][kWaves];
  __shared__ int largest;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x < 8) zeros[threadIdx.x] = 0;
  if (threadIdx.x == 0) largest = -1000;
  int at = 0, top_exponent = -1000;  // rows that count so far, their weights' largest exponent in this lane
  for (int64_t first = 0; first < n_rows; first += kEach * kPrepareThreads) {
    int64_t label[kEach];
    float w[kEach];
    uint64_t set[kEach];
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      const int64_t r = first + e * kPrepareThreads + threadIdx.x;
      label[e]        = r < n_rows ? y[r] : -1;
      w[e]            = weight != nullptr && r < n_rows ? weight[r] : 1.f;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      set[e] = __ballot(label[e] >= 0 && label[e] < n_classes);
      if (lane == 0) wave_sum[e][wave] = __popcll(set[e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      int before = at;
      for (int v = 0; v < kWaves; v++) {
        const int s = wave_sum[e][v];
        before += v < wave ? s : 0;
        at += s;
      }
      const int64_t r = first + e * kPrepareThreads + threadIdx.x;
      if ((set[e] >> lane) & 1) {
        const int p  = before + __popcll(set[e] & ((uint64_t(1) << lane) - 1));
        int exponent = 0;
        if (half) {
          if (w[e] != 0.f && fabsf(w[e]) < INFINITY) {
            w[e] = 2.f * frexpf(w[e], &exponent);  // 1 <= |w| < 2
            exponent -= 1;
          } else {
            exponent = w[e] == 0.f ? -1000 : 0;  // (a weight of 0 adds nothing to grad_weight)
          }
          top_exponent = max(top_exponent, exponent);
          w[e] *= 1 << kHalfShift;
        }
        out.order[p]    = static_cast<int32_t>(r);
        out.place[r]    = p;
        out.label[p]    = static_cast<int32_t>(label[e]);
        out.factor[p]   = w[e];
        out.exponent[p] = exponent;
        out.picked[p]   = -INFINITY;
      } else if (r < n_rows) {
        out.place[r] = -1;
        loss[r]      = 0.f;
      }
    }
  }
  if (half) {
    for (int s = 32; s > 0; s >>= 1) top_exponent = max(top_exponent, __shfl_xor(top_exponent, s));
    __syncthreads();  // `largest` is there
    if (lane == 0) atomicMax(&largest, top_exponent);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    counts->rows     = at;
    counts->exponent = largest > -1000 ? largest : 0;
    counts->reach    = -1000;
  }
  // (past the tiles that rows which count are in, nothing is looked at but `order`)
  for (int64_t p = at + threadIdx.x; p < padded; p += kPrepareThreads) {
    out.order[p] = -1;
    if (p >= at + 256) continue;
    out.label[p]    = -1;
    out.factor[p]   = 0.f;
    out.exponent[p] = -1000;
    out.picked[p]   = 0.f;
  }
}

// Columns col .. col + 7 of row r as they lie in an operand: zeros where r < 0 or past the row's end, a float as three planes.
template <int kDtype>
__device__ __forceinline__ void take_eight(const void* __restrict__ from, int64_t r, int col, int cols,
                                           uint16_t (&v)[LossType<kDtype>::kPlanes][8])
{
  const bool whole = r >= 0 && col + 8 <= cols;
  float f[8];
  if (whole) {  // (rows of any length: the memory takes loads at any address)
    if constexpr (kDtype == LBT_F32)
      __builtin_memcpy(f, static_cast<const float*>(from) + r * cols + col, 32);
    else
      __builtin_memcpy(v[0], static_cast<const uint16_t*>(from) + r * cols + col, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool in = r >= 0 && col + e < cols;
      if constexpr (kDtype == LBT_F32)
        f[e] = in ? static_cast<const float*>(from)[r * cols + col + e] : 0.f;
      else
        v[0][e] = in ? static_cast<const uint16_t*>(from)[r * cols + col + e] : uint16_t(0);
    }
  }
  if constexpr (kDtype == LBT_F32) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint16_t s[3];
      split_planes(f[e], s);
      v[0][e] = s[0];
      v[1][e] = s[1];
      v[2][e] = s[2];
    }
  }
}

// Where an operand's values are: plane q of row p begins at q * plane + p * row, every 32 columns are `block` further on.
struct Layout {
  int64_t plane, row, block;
  __host__ __device__ __forceinline__ int64_t at(int q, int64_t p, int col) const { return q * plane + p * row + (col >> 5) * block + (col & 31); }
};

// Rows of an array as rows of an operand: in `order` where that is given, -1 and what lies past the end as zeros, columns
// padded with zeros to `padded_cols`, floats as three planes. A thread takes 8 columns. Bound by the copy: it reads and writes
// each value once (8192 rows of 4096 bfloat16: 28 us, 4.7 TB/s). Half precision with weights: kMeasure finds counts->reach, kScale multiplies row p by 2^(exponent[p] + 14 - reach).
enum { kCopy = 0, kMeasure = 1, kScale = 2 };
constexpr int kReach = 14;
template <int kDtype>
__global__ void __launch_bounds__(256)
  pack_rows_kernel(const void* __restrict__ from, int64_t first_row, int64_t rows, int cols, const int32_t* __restrict__ order,
                   int mode, const int32_t* __restrict__ exponent, RowCounts* counts, int64_t out_rows, int padded_cols,
                   Layout layout, uint16_t* __restrict__ out)
{
  using L          = LossType<kDtype>;
  const int groups = padded_cols / 8;
  const int64_t i  = blockIdx.x * int64_t(256) + threadIdx.x;
  if (i >= out_rows * groups) return;
  const int64_t p = i / groups;
  const int col   = static_cast<int>(i % groups) * 8;
  const int64_t r = order != nullptr ? order[p] : (first_row + p < rows ? first_row + p : -1);
  uint16_t v[L::kPlanes][8];
  take_eight<kDtype>(from, r, col, cols, v);
  if constexpr (kDtype == LBT_F16) {
    if (mode == kMeasure) {
      int reach = -1000;
      if (r >= 0 && exponent[p] > -1000)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float x = load_value<kDtype>(v[0], e);
          int own       = 16;  // (infinities and NaN)
          if (fabsf(x) < INFINITY) (void)frexpf(x, &own);
          if (x != 0.f) reach = max(reach, own - 1 + exponent[p]);
        }
      for (int s = 32; s > 0; s >>= 1) reach = max(reach, __shfl_xor(reach, s));
      __shared__ int by_wave[4];
      if ((threadIdx.x & 63) == 0) by_wave[threadIdx.x >> 6] = reach;
      __syncthreads();
      // (most workgroups find a larger one there already: they need not wait their turn for the atomic)
      if (threadIdx.x == 0) {
        reach = max(max(by_wave[0], by_wave[1]), max(by_wave[2], by_wave[3]));
        if (reach > __hip_atomic_load(&counts->reach, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(&counts->reach, reach);
      }
    } else if (mode == kScale) {
      const int shift = exponent[p] + kReach - counts->reach;
#pragma unroll
      for (int e = 0; e < 8; e++)
        v[0][e] = exponent[p] <= -1000 ? uint16_t(0) : narrow_value<L::kProduct>(ldexpf(load_value<kDtype>(v[0], e), shift));
    }
  }
#pragma unroll
  for (int q = 0; q < L::kPlanes; q++)
    *reinterpret_cast<uint4*>(out + layout.at(q, p, col)) = *reinterpret_cast<const uint4*>(v[q]);
}

// prepare_rows_kernel and the laying out of X, and of the weights where they are laid out, in one launch for up to 1024 rows: a workgroup
// goes through all labels for itself and lays out up to 512 columns of 16 of the rows that count; others lay out the weights. Not for weighted rows in half
// precision, whose weights' exponents have to be known first. (1024 rows of 512 bfloat16, 10000 classes: 28.7 us in all, with one row more,
// by the kernels on their own, 31.0. 64 rows of 256 floats, 1000 classes: 4.8 us where the three launches took 9.)
constexpr int kFusedRows = 1024, kFusedEach = 16, kFusedGroups = 64;
struct FusedArgs {
  const int64_t* y;
  const float* row_weight;
  int n_rows, padded, n_classes;
  float* loss;
  RowCounts* counts;
  uint16_t* zeros;
  const void *x, *weight;
  int cols, padded_cols;
  uint16_t *x_out, *weight_out;  // (the second: null where the weights are not laid out)
  int64_t weight_rows;           // of weight_out
  uint16_t* x_blocks;            // where X goes for float_product_kernel; x_out: for the others; null: not there
  Layout blocks;
};

template <int kDtype>
__global__ void __launch_bounds__(256) prepare_pack_kernel(const FusedArgs a, const LossRows out)
{
  using L          = LossType<kDtype>;
  const int groups = a.padded_cols / 8, slices = (groups + kFusedGroups - 1) / kFusedGroups, x_blocks = a.padded / kFusedEach * slices;
  uint16_t v[L::kPlanes][8];
  if (static_cast<int>(blockIdx.x) >= x_blocks) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) - x_blocks) * 256 + threadIdx.x;
    if (i >= a.weight_rows * groups) return;
    const int64_t c = i / groups;
    const int col   = static_cast<int>(i % groups) * 8;
    take_eight<kDtype>(a.weight, c < a.n_classes ? c : -1, col, a.cols, v);
#pragma unroll
    for (int q = 0; q < L::kPlanes; q++)
      *reinterpret_cast<uint4*>(a.weight_out + (q * a.weight_rows + c) * a.padded_cols + col) = *reinterpret_cast<const uint4*>(v[q]);
    return;
  }
  constexpr int kEach = kFusedRows / 256;
  __shared__ int wave_sum[kEach][4], from[kFusedEach];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p0 = blockIdx.x / slices * kFusedEach, group0 = blockIdx.x % slices * kFusedGroups, own = min(kFusedGroups, groups - group0);
  const bool first = blockIdx.x == 0;
  if (first && threadIdx.x < 8) a.zeros[threadIdx.x] = 0;
  if (threadIdx.x < kFusedEach) from[threadIdx.x] = -1;
  int64_t label[kEach];
  uint64_t set[kEach];
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    const int r = e * 256 + threadIdx.x;
    label[e]    = r < a.n_rows ? a.y[r] : -1;
  }
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    set[e] = __ballot(label[e] >= 0 && label[e] < a.n_classes);
    if (lane == 0) wave_sum[e][wave] = __popcll(set[e]);
  }
  __syncthreads();
  int at = 0;
#pragma unroll
  for (int e = 0; e < kEach; e++) {
    int before = at;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const int s = wave_sum[e][w];
      before += w < wave ? s : 0;
      at += s;
    }
    const int r = e * 256 + threadIdx.x;
    if ((set[e] >> lane) & 1) {
      const int p = before + __popcll(set[e] & ((uint64_t(1) << lane) - 1));
      if (first) out.place[r] = p;
      if (p >= p0 && p < p0 + kFusedEach) {
        from[p - p0] = r;
        if (group0 > 0) continue;
        const float w   = a.row_weight != nullptr ? a.row_weight[r] : 1.f;
        out.order[p]    = r;
        out.label[p]    = static_cast<int32_t>(label[e]);
        out.factor[p]   = kDtype == LBT_F16 ? w * (1 << kHalfShift) : w;
        out.exponent[p] = 0;
        out.picked[p]   = -INFINITY;
      }
    } else if (first && r < a.n_rows) {
      out.place[r] = -1;
      a.loss[r]    = 0.f;
    }
  }
  if (first && threadIdx.x == 0) *a.counts = RowCounts{at, 0, -1000};
  __syncthreads();
  if (group0 == 0 && threadIdx.x < kFusedEach && p0 + static_cast<int>(threadIdx.x) >= at) {
    const int p     = p0 + threadIdx.x;
    out.order[p]    = -1;
    out.label[p]    = -1;
    out.factor[p]   = 0.f;
    out.exponent[p] = -1000;
    out.picked[p]   = 0.f;
  }
  for (int i = threadIdx.x; i < kFusedEach * own; i += 256) {
    const int p = i / own, col = (group0 + i % own) * 8;
    take_eight<kDtype>(a.x, from[p], col, a.cols, v);
#pragma unroll
    for (int q = 0; q < L::kPlanes; q++) {
      const uint4 w = *reinterpret_cast<const uint4*>(v[q]);
      if (a.x_out != nullptr) *reinterpret_cast<uint4*>(a.x_out + (static_cast<int64_t>(q) * a.padded + p0 + p) * a.padded_cols + col) = w;
      if (a.x_blocks != nullptr) *reinterpret_cast<uint4*>(a.x_blocks + a.blocks.at(q, p0 + p, col)) = w;
    }
  }
}

// ---- what the products end in -------------------------------------------------------------------

__device__ __forceinline__ float exp_of(float d, bool exact) { return exact ? expf(d) : __expf(d); }

// scores: m = classes, n = rows. Adds the bias; classes past the end count as masked. Most tiles have neither.
template <class Tile>
__device__ __forceinline__ void add_bias(Float16v (&acc)[Tile::kMT][Tile::kNT], const float* bias, int class_first, int n_classes,
                                         int lane)
{
  if (bias != nullptr) {
#pragma unroll
    for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const float b = bias[min(class_first + i * 32 + block_m(e, lane), n_classes - 1)];
#pragma unroll
        for (int j = 0; j < Tile::kNT; j++) acc[i][j][e] += b;
      }
  }
  if (class_first + Tile::kWM <= n_classes) return;
#pragma unroll
  for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const bool in = class_first + i * 32 + block_m(e, lane) < n_classes;
#pragma unroll
      for (int j = 0; j < Tile::kNT; j++) acc[i][j][e] = in ? acc[i][j][e] : -INFINITY;
    }
}

// The products end with four consecutive m of one n in a lane, and n apart from lane to lane: stored like that, a store touches 32
// rows of memory, 16 bytes each. A wave turns its part of the tile in the LDS, 32 n and up to 256 bytes of m at a time, so that
// 16 lanes store 256 bytes of a row. value(i, q, v): the four values of quad q of block i; sink(n, m, bits): 16 bytes of row n
// from value m on. The LDS is the wave's own part: no other wave is waited for. (grad_weight of 44642 classes of 3200 features, 286 MB,
// was written at 1.6 TB/s without.)
template <class Tile, int kSize, class Value, class Sink>
__device__ __forceinline__ void turn_rows(char* lds, int wave, int lane, Value value, Sink sink)
{
  constexpr int kBlocks = Tile::kMT * 32 * kSize <= 256 ? Tile::kMT : 256 / (32 * kSize);
  constexpr int kRow = kBlocks * 32 * kSize, kStride = kRow + 16, kLanes = kRow / 16, kRows = 64 / kLanes;
  static_assert(Tile::kWavesM * Tile::kWavesN * 32 * kStride <= Tile::kLds, "each wave has its part of the LDS");
  char* own = lds + wave * (32 * kStride);
#pragma unroll
  for (int group = 0; group < Tile::kMT / kBlocks; group++) {
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        float v[4];
        value(group * kBlocks + b, q, v);
        char* at = own + (lane & 31) * kStride + (b * 32 + q * 8 + 4 * (lane >> 5)) * kSize;
        if constexpr (kSize == 4) *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<uint2*>(at) = *reinterpret_cast<const uint2*>(v);  // (`value` has packed them)
      }
    meet_in_wave();
#pragma unroll
    for (int pass = 0; pass < 32 / kRows; pass++) {
      const int n = pass * kRows + lane / kLanes, c = lane % kLanes;
      sink(n, group * kBlocks * 32 + c * (16 / kSize), *reinterpret_cast<const uint4*>(own + n * kStride + c * 16));
    }
    meet_in_wave();
  }
}

// The shares of the rows' tops and totals: one of each row for the kWM classes of a wave. For scale_kernel also
// u = exp(s - the share's top), [rows][piece]: as float, or, for G in bfloat16, in 16 bits: 6 of its exponent and 10 of its significand, as
// it has no sign. That is off by at most 2^-11 where bfloat16 is by 2^-8 afterwards, down to 2^-62 of the top (half precision keeps its
// bits down to 2^-29: a row's small probabilities were off by more than its roundings). A float times 2^-64 has zeros above these 16
// bits, which then are a shift and an addition away. (3687 rows, 32768 classes of 2048 bfloat16: 83 us for G from them, where a
// second product takes 450.)
enum { kNotKept = 0, kKeptShort = 1, kKeptFloat = 2 };
constexpr float kKeptScale = 0x1p-64f;
__device__ __forceinline__ uint2 shorten_four(const float (&u)[4])
{
  uint32_t r[4];
#pragma unroll
  for (int e = 0; e < 4; e++) r[e] = (__builtin_bit_cast(uint32_t, u[e] * kKeptScale) << 3) + 0x8000u;  // rounded in the upper half
  return make_uint2(__builtin_amdgcn_perm(r[1], r[0], 0x07060302u), __builtin_amdgcn_perm(r[3], r[2], 0x07060302u));
}
// Two of them, times kKeptScale still.
__device__ __forceinline__ void widen_two(uint32_t w, float& first, float& second)
{
  first  = __builtin_bit_cast(float, (w << 13) & 0x1fffe000u);
  second = __builtin_bit_cast(float, (w >> 3) & 0x1fffe000u);
}
template <bool kExact, int kKeep>
struct LossEpilogue {
  const float* bias;
  int class_first, n_classes;  // of this launch: number of its first class; classes of the call
  int share_first;
  int64_t padded;              // rows
  LossRows rows;
  float2* partial;             // [shares][padded]: top, total
  void* kept;
  int piece;

  template <class Tile>
  __device__ __forceinline__ void store(Float16v (&acc)[Tile::kMT][Tile::kNT], int tile_m, int tile_n, int wm, int wn, int lane,
                                        int, int, const RowCounts*, char* lds) const
  {
    const int in_piece = tile_m * Tile::kBM + wm * Tile::kWM;
    const int c0       = class_first + in_piece;
    add_bias<Tile>(acc, bias, c0, n_classes, lane);
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++) {
      const int64_t row = static_cast<int64_t>(tile_n) * Tile::kBN + wn * Tile::kWN + j * 32 + (lane & 31);
      const int label   = rows.label[row] - c0;
      if (__any(label >= 0 && label < Tile::kWM)) {
        float at = 0.f;
#pragma unroll
        for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
          for (int e = 0; e < 16; e++) at = i * 32 + block_m(e, lane) == label ? acc[i][j][e] : at;
        if (label >= 0 && label < Tile::kWM && ((label >> 2) & 1) == lane >> 5) rows.picked[row] = at;
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) top = fmaxf(top, acc[i][j][e]);
      top              = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.f : top;
      float total      = 0.f;
      if constexpr (kKeep == kNotKept) {
#pragma unroll
        for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
          for (int e = 0; e < 16; e++) total += exp_of(acc[i][j][e] - from, kExact);
      } else {
        constexpr int kSize = kKeep == kKeptFloat ? 4 : 2;
        const int64_t row0  = static_cast<int64_t>(tile_n) * Tile::kBN + wn * Tile::kWN + j * 32;
        turn_rows<Tile, kSize>(
          lds, wm * Tile::kWavesN + wn, lane,
          [&](int i, int q, float(&v)[4]) {
            float u[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              u[e] = exp_of(acc[i][j][q * 4 + e] - from, kExact);
              total += u[e];
              v[e] = u[e];
            }
            if constexpr (kKeep == kKeptShort) {
              const uint2 w = shorten_four(u);
              __builtin_memcpy(v, &w, 8);
            }
          },
          [&](int n, int m, uint4 w) {
            *reinterpret_cast<uint4*>(static_cast<char*>(kept) + ((row0 + n) * piece + in_piece + m) * kSize) = w;
          });
      }
      total += __shfl_xor(total, 32);
      if (lane < 32) partial[static_cast<int64_t>(share_first + tile_m * Tile::kWavesM + wm) * padded + row] = make_float2(top, total);
    }
  }
};

template <int kCtrl, int kRows>
__device__ __forceinline__ float add_lanes(float v)
{
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, kRows, 0xf, true));
}
// Sums over lanes 0 to 31 and over 32 to 63, in the lanes' own data paths: in lanes 16 to 31 and 48 to 63.
__device__ __forceinline__ float sum_32_lanes(float v)
{
  v = add_lanes<0x128, 0xf>(v);  // row_ror:8 within 16 lanes
  v = add_lanes<0x124, 0xf>(v);
  v = add_lanes<0x122, 0xf>(v);
  v = add_lanes<0x121, 0xf>(v);
  return add_lanes<0x142, 0xa>(v);  // row_bcast:15 from the row of 16 lanes before
}

// G of a piece of the classes, [plane][rows][piece] in the products' type, and its sums over the tile's rows.
template <bool kExact, int kProduct, int kPlanes>
struct GradientEpilogue {
  const float* bias;
  int class_first, n_classes, piece;  // classes of a row of G
  LossRows rows;
  uint16_t* g;
  int64_t plane;
  float* bias_sums;  // [tiles of rows][classes], or null

  template <class Tile>
  __device__ __forceinline__ void store(Float16v (&acc)[Tile::kMT][Tile::kNT], int tile_m, int tile_n, int wm, int wn, int lane,
                                        int counted, int, const RowCounts* counts, char* lds) const
  {
    const int in_piece = tile_m * Tile::kBM + wm * Tile::kWM;
    const int c0       = class_first + in_piece;
    add_bias<Tile>(acc, bias, c0, n_classes, lane);
    float scale[Tile::kNT];  // of the sums over rows: half precision has the weights' exponents apart
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++) {
      const int64_t row   = static_cast<int64_t>(tile_n) * Tile::kBN + wn * Tile::kWN + j * 32 + (lane & 31);
      const bool in       = row < counted;
      const int label     = in ? rows.label[row] - c0 : -1;
      const float top     = in ? rows.top[row] : 0.f;
      const float inverse = in ? rows.inverse[row] : 0.f;
      const float factor  = in ? rows.factor[row] : 0.f;
      scale[j]            = 1.f;
      if (bias_sums != nullptr && kProduct == LBT_F16) scale[j] = ldexpf(1.f, in ? rows.exponent[row] - counts->exponent : 0);
      uint16_t* out = g + row * piece + in_piece + 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint16_t v[kPlanes][4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int m   = i * 32 + block_m(q * 4 + e, lane);
            const float p = exp_of(acc[i][j][q * 4 + e] - top, kExact) * inverse;
            float d       = (m == label ? p - 1.f : p) * factor;
            d             = in && c0 + m < n_classes ? d : 0.f;
            acc[i][j][q * 4 + e] = d;
            if constexpr (kPlanes == 1) {
              v[0][e] = narrow_value<kProduct>(d);
            } else {
              uint16_t s[3];
              split_planes(d, s);
              v[0][e] = s[0];
              v[1][e] = s[1];
              v[2][e] = s[2];
            }
          }
#pragma unroll
          for (int l = 0; l < kPlanes; l++)
            *reinterpret_cast<uint2*>(out + l * plane + i * 32 + q * 8) = *reinterpret_cast<const uint2*>(v[l]);
        }
    }
    if (bias_sums == nullptr) return;
    float(*share)[Tile::kBM] = reinterpret_cast<float(*)[Tile::kBM]>(lds);  // [waves over n][m]
#pragma unroll
    for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < Tile::kNT; j++) sum += acc[i][j][e] * scale[j];
        sum = sum_32_lanes(sum);
        if ((lane & 31) == 16) share[wn][wm * Tile::kWM + i * 32 + block_m(e, lane)] = sum;
      }
    __syncthreads();
    for (int m = threadIdx.x; m < Tile::kBM; m += Tile::kThreads) {
      float sum = 0.f;
      for (int w = 0; w < Tile::kWavesN; w++) sum += share[w][m];
      const int c = class_first + tile_m * Tile::kBM + m;
      if (c < n_classes) bias_sums[static_cast<int64_t>(tile_n) * n_classes + c] = sum;
    }
  }
};

// grad_X: m = features, n = rows. Adds to (or begins) the sums of this split of the classes, [split][rows][padded_cols]. The same for
// grad_weight where the rows are split or come in parts, n = classes of the piece.
struct RowsEpilogue {
  float* sums;
  int64_t split;  // values of a split
  int padded_cols;
  bool begin;
  int classes;  // n ends here; 0: at the rows that count
  bool scaled;  // the rows were multiplied by a power of two that is taken out here: each part of the rows has its own

  template <class Tile>
  __device__ __forceinline__ void store(Float16v (&acc)[Tile::kMT][Tile::kNT], int tile_m, int tile_n, int wm, int wn, int lane,
                                        int counted, int part, const RowCounts* counts, char*) const
  {
    if (scaled) {
      const int shift = counts->reach - kReach;
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
        for (int j = 0; j < Tile::kNT; j++)
#pragma unroll
          for (int e = 0; e < 16; e++) acc[i][j][e] = ldexpf(acc[i][j][e], shift);
    }
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++) {
      const int64_t row = static_cast<int64_t>(tile_n) * Tile::kBN + wn * Tile::kWN + j * 32 + (lane & 31);
      if (row >= (classes > 0 ? classes : counted)) continue;
#pragma unroll
      for (int i = 0; i < Tile::kMT; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int col = tile_m * Tile::kBM + wm * Tile::kWM + i * 32 + q * 8 + 4 * (lane >> 5);
          if (col >= padded_cols) continue;
          float4* at = reinterpret_cast<float4*>(sums + part * split + row * padded_cols + col);
          float4 v   = make_float4(acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]);
          if (!begin) {
            const float4 o = *at;
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
          }
          *at = v;
        }
    }
  }
};

// grad_weight: m = features, n = classes of the piece. Complete: written in the output's type.
template <int kDtype>
struct ClassesEpilogue {
  void* out;
  int class_first, n_classes, cols;
  bool scaled;  // the rows were multiplied by powers of two (half precision)

  template <class Tile>
  __device__ __forceinline__ void store(Float16v (&acc)[Tile::kMT][Tile::kNT], int tile_m, int tile_n, int wm, int wn, int lane,
                                        int, int, const RowCounts* counts, char* lds) const
  {
    const int shift    = (scaled ? counts->reach - kReach : 0) - kHalfShift;
    constexpr int kSize = kDtype == LBT_F32 ? 4 : 2;
    const int col0      = tile_m * Tile::kBM + wm * Tile::kWM;
#pragma unroll
    for (int j = 0; j < Tile::kNT; j++) {
      const int c0 = class_first + tile_n * Tile::kBN + wn * Tile::kWN + j * 32;
      turn_rows<Tile, kSize>(
        lds, wm * Tile::kWavesN + wn, lane,
        [&](int i, int q, float(&v)[4]) {
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] = kDtype == LBT_F16 ? ldexpf(acc[i][j][q * 4 + e], shift) : acc[i][j][q * 4 + e];
          if constexpr (kSize == 2) {
            const uint2 w = narrow_four<kDtype>(v);
            __builtin_memcpy(v, &w, 8);
          }
        },
        [&](int n, int m, uint4 w) {
          const int c = c0 + n, col = col0 + m;
          if (c >= n_classes || col >= cols) return;
          char* to = static_cast<char*>(out) + (static_cast<int64_t>(c) * cols + col) * kSize;
          if (col + 16 / kSize <= cols) {
            __builtin_memcpy(to, &w, 16);  // (rows of any length: the memory takes stores at any address)
          } else {
            uint16_t part[8];
            __builtin_memcpy(part, &w, 16);
            for (int e = 0; e < 8; e++)
              if (e * 2 < (cols - col) * kSize) reinterpret_cast<uint16_t*>(to)[e] = part[e];
          }
        });
    }
  }
};

// ---- joins ----------------------------------------------------------------------------------------

__device__ __forceinline__ float loss_of(float2 s, float picked)
{
  if (s.x == -INFINITY && s.y == 0.f) return INFINITY;  // every class is masked
  return ((s.x == -INFINITY ? 0.f : s.x) - picked) + logf(s.y);
}

constexpr int kJoinRows = 16, kJoinSlices = 64;

// Top and total of each row from its shares; its loss. 64 threads take the shares of a row between them, neighbours in a wave are
// neighbouring rows. Bound by its loads' latency: 8 us for 3687 rows of 256 shares.
__global__ void __launch_bounds__(kJoinRows * kJoinSlices)
  join_kernel(const float2* __restrict__ partial, int shares, int64_t padded, LossRows rows, const RowCounts* __restrict__ counts,
              float* __restrict__ loss)
{
  __shared__ float tops[kJoinSlices][kJoinRows], totals[kJoinSlices][kJoinRows];
  const int n       = threadIdx.x % kJoinRows, slice = threadIdx.x / kJoinRows;
  const int64_t row = blockIdx.x * int64_t(kJoinRows) + n;
  const int counted = counts->rows;
  if (blockIdx.x * int64_t(kJoinRows) >= counted) return;
  constexpr int kAhead = 8;  // shares asked for together
  float2 s[kAhead];
  auto load = [&](int first) {
#pragma unroll
    for (int e = 0; e < kAhead; e++) {
      const int t = first + e * kJoinSlices;
      s[e]        = t < shares ? partial[t * padded + row] : make_float2(-INFINITY, 0.f);
    }
  };
  float top = -INFINITY, total = 0.f;
  for (int first = slice; first < shares; first += kAhead * kJoinSlices) {
    load(first);
    float next = top;
#pragma unroll
    for (int e = 0; e < kAhead; e++) next = fmaxf(next, s[e].x);
    const float from = next == -INFINITY ? 0.f : next;
    total *= expf(top - from);
#pragma unroll
    for (int e = 0; e < kAhead; e++) total += s[e].y * expf(s[e].x - from);
    top = next;
  }
  tops[slice][n] = top;
  __syncthreads();
  float all = -INFINITY;
#pragma unroll 8
  for (int v = 0; v < kJoinSlices; v++) all = fmaxf(all, tops[v][n]);
  const float from = all == -INFINITY ? 0.f : all;
  totals[slice][n] = total * expf(top - from);
  __syncthreads();
  if (slice != 0 || row >= counted) return;
  total = 0.f;
#pragma unroll 8
  for (int v = 0; v < kJoinSlices; v++) total += totals[v][n];
  // where every class is masked there is no probability: the loss is infinite and p is 0
  rows.top[row]         = from;
  rows.inverse[row]     = all == -INFINITY && total == 0.f ? 0.f : 1.f / total;
  loss[rows.order[row]] = loss_of(make_float2(all, total), rows.picked[row]);
}

// ---- few rows -----------------------------------------------------------------------------------------
//
// A score of few rows is bound by reading the weights once. Each wave takes 16 classes, 16 bytes of a class a lane, straight from
// memory into the operand of a 16 x 16 product, with up to four blocks of 16 rows beside it (they are read over and over, from the
// L1): there is no stage in the LDS to wait for and nothing is laid out first. (One row of 1024 bfloat16, 32768 classes: 67 MB at 4.8
// TB/s. 33 rows of 1000 floats, 10007 classes: 24 us, 40 TFLOP/s of padded rows, bound by the float products and their operands' loads.) The order of k within 16 lanes' chunks is the same
// for both operands, which is all a product asks of it. float goes to the float products of the matrix cores as it is. Rows are not
// taken out: what a row that does not count holds stays in its own column.
// kShared: the four waves of a workgroup share out k instead of taking 16 classes each, where the classes would give the CUs too
// few waves to keep memory busy. More than 16 rows have two blocks of classes beside
// theirs where there are classes enough, so that the rows are read less often.

typedef __attribute__((ext_vector_type(4))) float Float4v;

constexpr int kFewThreads = 256, kFewBlock = 64;  // rows of a workgroup, at most

template <int kDtype>
struct FewStep {  // 16 bytes of a row: kValues of k
  static constexpr int kValues = kDtype == LBT_F32 ? 4 : 8;
  using Value                  = typename LossType<kDtype>::Value;
  uint4 bits;

  __device__ __forceinline__ void load(const Value* row, int k) { __builtin_memcpy(&bits, row + k, 16); }
  __device__ __forceinline__ void load_end(const Value* row, int k, int cols)
  {
    Value v[kValues];
#pragma unroll
    for (int e = 0; e < kValues; e++) v[e] = k + e < cols ? row[k + e] : Value(0);
    __builtin_memcpy(&bits, v, 16);
  }
  static __device__ __forceinline__ Float4v multiply(const FewStep& a, const FewStep& b, Float4v c)
  {
    if constexpr (kDtype == LBT_F32) {
      const Float4v x = __builtin_bit_cast(Float4v, a.bits), y = __builtin_bit_cast(Float4v, b.bits);
#pragma unroll
      for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
      return c;
    } else if constexpr (kDtype == LBT_F16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Half8, a.bits), __builtin_bit_cast(Half8, b.bits), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a.bits), __builtin_bit_cast(Bf16x8, b.bits), c, 0, 0, 0);
    }
  }
};

// For the gradient the rows are those that count, `order` names them, and u is left for scale_kernel as LossEpilogue does.
struct FewRowsArgs {
  const void *x, *weight;
  const float* bias;
  const int64_t* y;   // labels, where order is null
  int n_rows, cols, n_classes;
  int64_t share_step, row_step;  // of `partial`
  float2* partial;
  float* picked;
  const int32_t *order, *label;
  const RowCounts* counts;
  void* kept;
  int piece;
};

template <int kDtype, int kBlocks, int kClassBlocks, int kWaves, bool kShared, int kKeep>
__global__ void __launch_bounds__(kWaves * 64, 3)
  few_rows_kernel(const FewRowsArgs args)
{
  using S = FewStep<kDtype>;
  using V = typename S::Value;
  constexpr bool kExact = kDtype == LBT_F32;
  constexpr int kUnroll = kBlocks >= 3 ? 2 : 4, kStep = 4 * S::kValues;  // k of a product
  constexpr int kClasses = 16 * kClassBlocks;                            // of a wave
  const int row0 = blockIdx.y * kFewBlock, cols = args.cols, n_classes = args.n_classes;
  const int n_rows = args.order != nullptr ? args.counts->rows : args.n_rows;
  if (row0 >= n_rows) return;
  __shared__ float4 sums[kShared ? kWaves * kClassBlocks * kBlocks * 64 : 1];
  __shared__ float2 share[kWaves][kClassBlocks][16 * kBlocks];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = blockIdx.x * (kShared ? kClasses : kWaves * kClasses) + (kShared ? 0 : wave * kClasses);  // of this wave
  const V *w[kClassBlocks], *x[kBlocks];
#pragma unroll
  for (int i = 0; i < kClassBlocks; i++)
    w[i] = static_cast<const V*>(args.weight) + static_cast<int64_t>(min(c0 + i * 16 + (lane & 15), n_classes - 1)) * cols;
#pragma unroll
  for (int b = 0; b < kBlocks; b++) {
    const int r = min(row0 + b * 16 + (lane & 15), n_rows - 1);
    x[b]        = static_cast<const V*>(args.x) + static_cast<int64_t>(args.order != nullptr ? args.order[r] : r) * cols;
  }
  const int at  = (lane >> 4) * S::kValues;
  const int hop = kShared ? kWaves * kUnroll * kStep : kUnroll * kStep;  // k of a turn, from wave to wave
  Float4v acc[kClassBlocks][kBlocks];
#pragma unroll
  for (int i = 0; i < kClassBlocks; i++)
#pragma unroll
    for (int b = 0; b < kBlocks; b++) acc[i][b] = Float4v{0.f, 0.f, 0.f, 0.f};
  int k = kShared ? wave * kUnroll * kStep : 0;
  S a[kUnroll][kClassBlocks], m[kUnroll][kBlocks];
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
#pragma unroll
      for (int i = 0; i < kClassBlocks; i++) a[u][i].load(w[i], from + u * kStep + at);
#pragma unroll
      for (int b = 0; b < kBlocks; b++) m[u][b].load(x[b], from + u * kStep + at);
    }
  };
  bool whole = k + kUnroll * kStep <= cols;
  if (whole) load(k);
  while (whole) {  // the next turn is asked for before this one is multiplied
    S a1[kUnroll][kClassBlocks], m1[kUnroll][kBlocks];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
#pragma unroll
      for (int i = 0; i < kClassBlocks; i++) a1[u][i] = a[u][i];
#pragma unroll
      for (int b = 0; b < kBlocks; b++) m1[u][b] = m[u][b];
    }
    k += hop;
    whole = k + kUnroll * kStep <= cols;
    if (whole) load(k);
#pragma unroll
    for (int u = 0; u < kUnroll; u++)
#pragma unroll
      for (int i = 0; i < kClassBlocks; i++)
#pragma unroll
        for (int b = 0; b < kBlocks; b++) acc[i][b] = S::multiply(a1[u][i], m1[u][b], acc[i][b]);
  }
  for (int u = 0; u < kUnroll && k + u * kStep < cols; u++) {  // the end of the rows
    S e[kClassBlocks], f;
#pragma unroll
    for (int i = 0; i < kClassBlocks; i++) e[i].load_end(w[i], k + u * kStep + at, cols);
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {
      f.load_end(x[b], k + u * kStep + at, cols);
#pragma unroll
      for (int i = 0; i < kClassBlocks; i++) acc[i][b] = S::multiply(e[i], f, acc[i][b]);
    }
  }
  if constexpr (kShared) {
#pragma unroll
    for (int i = 0; i < kClassBlocks; i++)
#pragma unroll
      for (int b = 0; b < kBlocks; b++)
        sums[((wave * kClassBlocks + i) * kBlocks + b) * 64 + lane] = make_float4(acc[i][b][0], acc[i][b][1], acc[i][b][2], acc[i][b][3]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kClassBlocks; i++)
#pragma unroll
    for (int b = 0; b < kBlocks; b++) {  // lane: row lane % 16, classes 4 (lane / 16) ...
      if constexpr (kShared) {
        if ((i * kBlocks + b) % kWaves != wave) continue;
        Float4v t = Float4v{0.f, 0.f, 0.f, 0.f};
        for (int v = 0; v < kWaves; v++) t += __builtin_bit_cast(Float4v, sums[((v * kClassBlocks + i) * kBlocks + b) * 64 + lane]);
        acc[i][b] = t;
      }
      const int r         = row0 + b * 16 + (lane & 15);
      const int first     = c0 + i * 16 + 4 * (lane >> 4);
      const int64_t label = r >= n_rows ? -1 : args.order != nullptr ? args.label[r] : args.y[r];
      float top           = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int c  = first + e;
        acc[i][b][e] = c < n_classes ? acc[i][b][e] + (args.bias != nullptr ? args.bias[c] : 0.f) : -INFINITY;
        if (c == label && c < n_classes) args.picked[r] = acc[i][b][e];
        top = fmaxf(top, acc[i][b][e]);
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.f : top;
      float total      = 0.f, u[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        u[e] = exp_of(acc[i][b][e] - from, kExact);
        total += u[e];
      }
      if (kKeep != kNotKept && r < n_rows && first < args.piece) {
        const int64_t at = static_cast<int64_t>(r) * args.piece + first;
        if constexpr (kKeep == kKeptFloat) {
          *reinterpret_cast<float4*>(static_cast<float*>(args.kept) + at) = make_float4(u[0], u[1], u[2], u[3]);
        } else {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(args.kept) + at) = shorten_four(u);
        }
      }
      total += __shfl_xor(total, 16);
      total += __shfl_xor(total, 32);
      if constexpr (kShared) {
        if (lane < 16 && r < n_rows)
          args.partial[r * args.row_step + (blockIdx.x * kClassBlocks + i) * args.share_step] = make_float2(top, total);
      } else {
        if (lane < 16) share[wave][i][r - row0] = make_float2(top, total);
      }
    }
  if constexpr (!kShared) {
    __syncthreads();
    for (int t = threadIdx.x; t < kClassBlocks * 16 * kBlocks; t += kWaves * 64) {
      const int i = t / (16 * kBlocks), r = t % (16 * kBlocks);
      if (row0 + r >= n_rows) continue;
      float top = share[0][i][r].x;
      for (int v = 1; v < kWaves; v++) top = fmaxf(top, share[v][i][r].x);
      const float from = top == -INFINITY ? 0.f : top;
      float total      = 0.f;
      for (int v = 0; v < kWaves; v++) total += share[v][i][r].y * exp_of(share[v][i][r].x - from, kExact);
      args.partial[(row0 + r) * args.row_step + (blockIdx.x * kClassBlocks + i) * args.share_step] = make_float2(top, total);
    }
  }
}

// Top and total of a row from its shares, by a workgroup: [rows][tiles].
__device__ __forceinline__ float2 join_row(const float2* __restrict__ shares, int tiles)
{
  constexpr int kWaves = kFewThreads / 64;
  __shared__ float2 by_wave[kWaves];
  float top = -INFINITY;
  for (int t = threadIdx.x; t < tiles; t += kFewThreads) top = fmaxf(top, shares[t].x);
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
  if ((threadIdx.x & 63) == 0) by_wave[threadIdx.x >> 6].x = top;
  __syncthreads();
  for (int v = 0; v < kWaves; v++) top = fmaxf(top, by_wave[v].x);
  const float from = top == -INFINITY ? 0.f : top;
  float total      = 0.f;
  for (int t = threadIdx.x; t < tiles; t += kFewThreads) total += shares[t].y * expf(shares[t].x - from);
  for (int s = 32; s > 0; s >>= 1) total += __shfl_xor(total, s);
  if ((threadIdx.x & 63) == 0) by_wave[threadIdx.x >> 6].y = total;
  __syncthreads();
  total = 0.f;
  for (int v = 0; v < kWaves; v++) total += by_wave[v].y;
  return make_float2(top, total);
}

__global__ void __launch_bounds__(kFewThreads)
  join_few_kernel(const float2* __restrict__ partial, int tiles, const float* __restrict__ picked, const int64_t* __restrict__ y,
                  int n_classes, float* __restrict__ loss)
{
  const int r     = blockIdx.x;
  const float2 s  = join_row(partial + static_cast<int64_t>(r) * tiles, tiles);
  const int64_t l = y[r];
  if (threadIdx.x == 0) loss[r] = l >= 0 && l < n_classes ? loss_of(s, picked[r]) : 0.f;
}

// The same among the rows of a gradient, for scale_kernel.
__global__ void __launch_bounds__(kFewThreads)
  join_few_rows_kernel(const float2* __restrict__ partial, int shares, LossRows rows, const RowCounts* __restrict__ counts,
                       float* __restrict__ loss)
{
  const int r = blockIdx.x;
  if (r >= counts->rows) return;
  const float2 s = join_row(partial + static_cast<int64_t>(r) * shares, shares);
  if (threadIdx.x != 0) return;
  rows.top[r]           = s.x == -INFINITY ? 0.f : s.x;
  rows.inverse[r]       = s.x == -INFINITY && s.y == 0.f ? 0.f : 1.f / s.y;
  loss[rows.order[r]]   = loss_of(s, rows.picked[r]);
}

// G from what LossEpilogue kept, once the rows' tops and totals are known: p = u exp(top of the share - top) / total. A workgroup
// takes 16 rows and 2048 classes; bound by memory, each value is read and written once (bfloat16: in the same place; 3687 rows, 32768
// classes 83 us, 5.8 TB/s with what the last cache holds).
// The sums of G over the workgroup's rows are those of floats. Where 16 rows each would be too few workgroups they take 4; a wave
// of such a workgroup joins the shares of one of them itself (join_shares of them), which saves a launch while they are few. (64 rows,
// 1000 classes of 256 floats: 30.5 us in all, 32.7 with the launch, 42.3 by 16 rows; 4096 rows, 32768 classes of 256 bfloat16: 444 us,
// 488 by 4 rows.)
constexpr int kScaleClasses = 2048;
template <int kDtype, bool kKeptAsShort, int kRows>
__global__ void __launch_bounds__(256)
  scale_kernel(const void* kept, const float2* __restrict__ partial, int share_classes, int64_t share_step, int64_t row_step, int row_tile, LossRows rows,
               const RowCounts* __restrict__ counts, int n_classes, int piece, int64_t plane, uint16_t* g, uint16_t* g_blocks, int64_t padded, float* bias_sums,
               int join_shares, float* __restrict__ loss)
{
  using L = LossType<kDtype>;
  __shared__ float factor[kRows][kScaleClasses / 16 + 1];
  __shared__ float row_top[kRows], row_inverse[kRows];
  const int wides       = (piece + kScaleClasses - 1) / kScaleClasses;
  const int64_t block   = blockIdx.x / wides;
  const int64_t row0    = block * kRows;
  const int counted     = counts->rows;
  // (the products reach as far as their last tile of rows: up to there G is zeros)
  if (row0 >= (static_cast<int64_t>(counted) + row_tile - 1) / row_tile * row_tile) return;
  if constexpr (kRows == 4) {
    if (join_shares > 0) {
      const int lane    = threadIdx.x & 63, r = threadIdx.x >> 6;
      const int64_t row = row0 + r;
      float top = -INFINITY, total = 0.f;
      for (int t = lane; t < join_shares; t += 64) top = fmaxf(top, partial[t * share_step + row * row_step].x);
      for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
      const float from = top == -INFINITY ? 0.f : top;
      for (int t = lane; t < join_shares; t += 64) {
        const float2 s = partial[t * share_step + row * row_step];
        total += s.y * expf(s.x - from);
      }
      for (int s = 32; s > 0; s >>= 1) total += __shfl_xor(total, s);
      if (lane == 0) {
        row_top[r]     = from;
        row_inverse[r] = top == -INFINITY && total == 0.f ? 0.f : 1.f / total;
        if (blockIdx.x % wides == 0 && row < counted) loss[rows.order[row]] = loss_of(make_float2(top, total), rows.picked[row]);
      }
    }
  }
  if (join_shares == 0 && threadIdx.x < kRows) {
    row_top[threadIdx.x]     = rows.top[row0 + threadIdx.x];
    row_inverse[threadIdx.x] = rows.inverse[row0 + threadIdx.x];
  }
  __syncthreads();
  const int class0 = static_cast<int>(blockIdx.x % wides) * kScaleClasses, shares = kScaleClasses / share_classes, first = class0 / share_classes;
  for (int i = threadIdx.x; i < kRows * shares; i += 256) {
    const int64_t row = row0 + i % kRows;
    const int s       = i / kRows;
    float f           = 0.f;
    if (row < counted && class0 + s * share_classes < piece) {
      const float top = partial[(first + s) * share_step + row * row_step].x;
      // (a row that holds NaN has it in its total, not in 16 bits: the factor is NaN, where all of a share's classes are masked, too)
      const float p = top == -INFINITY ? 0.f : exp_of(top - row_top[i % kRows], kDtype == LBT_F32);
      f = p * row_inverse[i % kRows] * (kKeptAsShort ? 1.f / kKeptScale : 1.f);
    }
    factor[i % kRows][s] = f;
  }
  __syncthreads();
  const int c = class0 + static_cast<int>(threadIdx.x) * 8;
  if (c >= piece) return;
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; e++) sum[e] = 0.f;
#pragma unroll 4
  for (int r = 0; r < kRows; r++) {
    const int64_t row = row0 + r, at = row * piece + c;
    const float f   = factor[r][(c - class0) / share_classes];
    const float w   = rows.factor[row];
    const int label = rows.label[row] - c;
    float u[8];
    if constexpr (kKeptAsShort) {
      const uint4 h = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(kept) + at);
      widen_two(h.x, u[0], u[1]);
      widen_two(h.y, u[2], u[3]);
      widen_two(h.z, u[4], u[5]);
      widen_two(h.w, u[6], u[7]);
    } else {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(kept) + at);
      const float4 a = q[0], b = q[1];
      u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w; u[4] = b.x; u[5] = b.y; u[6] = b.z; u[7] = b.w;
    }
    const float scale = kDtype == LBT_F16 && bias_sums != nullptr && row < counted ? ldexpf(1.f, rows.exponent[row] - counts->exponent) : 1.f;
    uint16_t v[L::kPlanes][8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float p = u[e] * f;
      float d       = (e == label ? p - 1.f : p) * w;
      d             = row < counted ? d : 0.f;
      sum[e] += kDtype == LBT_F16 ? d * scale : d;
      if constexpr (L::kPlanes == 3) {
        uint16_t s[3];
        split_planes(d, s);
        v[0][e] = s[0];
        v[1][e] = s[1];
        v[2][e] = s[2];
      } else {
        v[0][e] = narrow_value<L::kProduct>(d);
      }
    }
#pragma unroll
    for (int l = 0; l < L::kPlanes; l++) *reinterpret_cast<uint4*>(g + l * plane + at) = *reinterpret_cast<const uint4*>(v[l]);
    if constexpr (L::kPlanes == 3)
      if (g_blocks != nullptr)
#pragma unroll
        for (int l = 0; l < 3; l++)
          *reinterpret_cast<uint4*>(g_blocks + Layout{32, 96, 96 * padded}.at(l, row, c)) = *reinterpret_cast<const uint4*>(v[l]);
  }
  if (bias_sums == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (c + e < n_classes) bias_sums[block * n_classes + c + e] = sum[e];
}

// grad_X from its sums over the splits; zeros for rows that do not count. Bound by memory: 17 us for 4096 rows of 2048, 50 MB and more.
template <int kDtype>
__global__ void __launch_bounds__(256)
  finish_rows_kernel(const float* __restrict__ sums, int splits, int64_t split, int padded_cols, int64_t n_rows, int cols,
                     LossRows rows, void* __restrict__ out)
{
  const int groups = (cols + 3) / 4;
  const int64_t i  = blockIdx.x * int64_t(256) + threadIdx.x;
  if (i >= n_rows * groups) return;
  const int64_t r = i / groups;
  const int col   = static_cast<int>(i % groups) * 4;
  const int p     = rows.place[r];
  float v[4]      = {0.f, 0.f, 0.f, 0.f};
  if (p >= 0) {
    for (int s = 0; s < splits; s++) {
      const float4 a = *reinterpret_cast<const float4*>(sums + s * split + static_cast<int64_t>(p) * padded_cols + col);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    }
    if (kDtype == LBT_F16) {
      const int e = rows.exponent[p];
      for (int q = 0; q < 4; q++) v[q] = e <= -1000 ? v[q] * 0.f : ldexpf(v[q], e - kHalfShift);
    }
  }
  store_four<kDtype>(out, r * cols + col, v, cols - col);
}

// grad_weight of a piece of the classes from its sums over the splits of the rows.
template <int kDtype>
__global__ void __launch_bounds__(256)
  finish_classes_kernel(const float* __restrict__ sums, int splits, int64_t split, int padded_cols, int64_t first, int64_t classes, int cols,
                        const RowCounts* __restrict__ counts, bool scaled, void* __restrict__ out)
{
  const int groups = (cols + 3) / 4;
  const int64_t i  = blockIdx.x * int64_t(256) + threadIdx.x;
  if (i >= classes * groups) return;
  const int64_t c = i / groups;
  const int col   = static_cast<int>(i % groups) * 4;
  float v[4]      = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s++) {
    const float4 a = *reinterpret_cast<const float4*>(sums + s * split + c * padded_cols + col);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
  }
  if (kDtype == LBT_F16)
    for (int q = 0; q < 4; q++) v[q] = ldexpf(v[q], (scaled ? counts->reach - kReach : 0) - kHalfShift);
  store_four<kDtype>(out, (first + c) * cols + col, v, cols - col);
}

// grad_bias from its sums over blocks of rows; a class's blocks are shared out among 64 threads. `add`: to that of the rows before.
__global__ void __launch_bounds__(kJoinRows * kJoinSlices)
  finish_bias_kernel(const float* __restrict__ sums, int first_class, int n_classes, int block_rows, const RowCounts* __restrict__ counts, int half,
                     bool add, float* __restrict__ out)
{
  __shared__ float share[kJoinSlices][kJoinRows];
  const int n = threadIdx.x % kJoinRows, slice = threadIdx.x / kJoinRows;
  const int c      = first_class + blockIdx.x * kJoinRows + n;
  const int blocks = (counts->rows + block_rows - 1) / block_rows;
  float sum        = 0.f;
  if (c < n_classes) {
#pragma unroll 8
    for (int t = slice; t < blocks; t += kJoinSlices) sum += sums[static_cast<int64_t>(t) * n_classes + c];
  }
  share[slice][n] = sum;
  __syncthreads();
  if (slice != 0 || c >= n_classes) return;
  sum = 0.f;
  for (int s = 0; s < kJoinSlices; s++) sum += share[s][n];
  if (half) sum = ldexpf(sum, counts->exponent - kHalfShift);
  out[c] = add ? out[c] + sum : sum;
}

__global__ void __launch_bounds__(256) clear_kernel(uint16_t* __restrict__ out, int64_t n)
{
  for (int64_t i = blockIdx.x * int64_t(256) + threadIdx.x; i < n; i += gridDim.x * int64_t(256)) out[i] = 0;
}

// ---- host -----------------------------------------------------------------------------------------

using LargeTile  = ProductTile<256, 256, 2, 4, 2>;
using MediumTile = ProductTile<128, 128, 2, 2, 2>;
using SmallTile  = ProductTile<64, 64, 2, 2, 5>;
using FloatLarge = FloatTile<128, 128, 2, 2, 1, 2>;
using FloatSmall = FloatTile<64, 64, 2, 2, 2, 4>;

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t tiles_of(int64_t v, int64_t by) { return (v + by - 1) / by; }

// How a product of m x n over `stages` stages of k is cut: tiles of 256, 128 or 64, and k into splits. A CU's time is that of its
// share of the tiles; a stage takes it 1.72 us, 0.5 and 0.2 (two workgroups at a time; 0.7 and 0.35 where it has only one, which
// then waits for memory), and a tile 8, 3 and 2 us to begin and end. Each split adds a pass over the sums. (Over forty products of
// 64 to 8192 rows the choice was mostly within a tenth of the best of all tiles and splits: 3687 x 2048 over 32768 of k 450 us in tiles
// of 256, 1026 x 1000 over 30011 128 us in tiles of 128 and splits. The times themselves are off by up to 28 %, and rows that do
// not count are priced as if they did: only the device knows how many there are.)
struct Cut {
  int tile, splits;
  double time;  // us, roughly
};
Cut cut_product(int64_t m, int64_t n, int64_t stages, int64_t most_splits)
{
  constexpr int kCus = 256;
  constexpr struct { int tile; double stage, lone, ends; } kTiles[3] = {{256, 1.72, 1.72, 8.0}, {128, 0.5, 0.7, 3.0}, {64, 0.2, 0.35, 2.0}};
  Cut best{256, 1, 1e30};
  for (const auto& t : kTiles)
    for (int splits = 1; splits <= most_splits; splits++) {
      if (splits > 1 && stages / splits < 4) break;
      const int64_t each = tiles_of(tiles_of(m, t.tile) * tiles_of(n, t.tile) * splits, kCus);
      const double time  = each * (tiles_of(stages, splits) * (each == 1 ? t.lone : t.stage) + t.ends) +
                          (splits - 1) * (1.0 + m * n * 8e-6 / 4.0);
      if (time < best.time) best = {t.tile, splits, time};
    }
  return best;
}

// Scores of few rows: the waves share the classes of a workgroup where they would be fewer than two a SIMD, and always where they
// leave u, whose shares are then 16 classes each. (One row of bfloat16: 512 features, 65000 classes 21.1 us shared, 16.3 not; 33 rows,
// 20000 classes 14.8 and 18.3.) Two blocks of classes beside more than 16 rows: 64 rows of 1024 features, 10000 classes 17.7 us, with one
// 20.0; 50000 classes 48 and 78.
constexpr int kFewRows = kFewBlock, kFewFloatRows = 4 * kFewBlock;
bool few_shared(int classes) { return classes < 32768; }
int few_class_blocks(int64_t n_rows, int classes, int dtype) { return n_rows <= 16 || classes < (dtype == LBT_F32 ? 32768 : 8192) ? 1 : 2; }
int64_t few_groups(int classes, int class_blocks, bool shared) { return tiles_of(classes, 16 * class_blocks * (shared ? 1 : 4)); }

// The same for float_product_kernel over `stages` of 32 of k: a stage takes a CU 0.5 and 1.4 us. (3000 classes of 4000 features: 256
// rows 75 us in tiles of 64, 168 in those of 128; 4096 rows 665 and 537.)
Cut cut_floats(int64_t m, int64_t n, int64_t stages, int64_t most_splits)
{
  constexpr int kCus = 256;
  constexpr struct { int tile; double stage, ends; } kTiles[2] = {{128, 1.4, 4.0}, {64, 0.5, 2.0}};
  Cut best{128, 1, 1e30};
  for (const auto& t : kTiles)
    for (int splits = 1; splits <= most_splits; splits++) {
      if (splits > 1 && stages / splits < 8) break;
      const double time = tiles_of(tiles_of(m, t.tile) * tiles_of(n, t.tile) * splits, kCus) * (tiles_of(stages, splits) * t.stage + t.ends) +
                          (splits - 1) * (1.0 + m * n * 8e-6 / 4.0);
      if (time < best.time) best = {t.tile, splits, time};
    }
  return best;
}

// Whether the scores are those of few_rows_kernel and not of tiles, whose product takes `tiles` us: its own products come at 50 TFLOP/s
// for float and 130 for 16 bits. (bfloat16, 64 rows of 1024 features: 10000 classes 18 us and 20 in tiles, 50000 classes 48 and 31.
// float, 1000 features: 33 rows 25.7 us and 32.1 in tiles over 10007 classes, 61 and 44 over 30000; 4000 features, 3000 classes: 64
// rows 42 and 72 us, 256 rows 115 and 75.)
bool few_rows(int64_t n_rows, int64_t features, int64_t classes, int dtype, double tiles)
{
  if (n_rows <= 16) return true;
  const double rate = dtype == LBT_F32 ? 4e-8 : 1.5e-8;  // us a product
  return n_rows <= (dtype == LBT_F32 ? kFewFloatRows : kFewRows) &&
         6.0 + rate * static_cast<double>(round_up(n_rows, 16)) * features * classes < 10.0 + tiles;
}
// Of the loss alone. (Weights of 16 bits in rows that are no whole chunks are laid out for tiles, at 5 TB/s.)
bool few_loss(int64_t n_rows, int64_t features, int64_t classes, int dtype)
{
  const double tiles = dtype == LBT_F32 ? cut_floats(classes, n_rows, tiles_of(features, FloatLarge::kK), 1).time
                                        : cut_product(classes, n_rows, tiles_of(features, kProductK), 1).time +
                                            (features % 8 != 0 ? 4.0 * features * classes / 5e6 : 0.0);
  return few_rows(n_rows, features, classes, dtype, tiles);
}

struct FewCall {
  float2* partial;
  float* picked;
  void carve(Arena& arena, int64_t n_rows, int classes, int dtype)
  {
    const int blocks = few_class_blocks(n_rows, classes, dtype);
    partial          = arena.take<float2>(n_rows * few_groups(classes, blocks, few_shared(classes)) * blocks);
    picked           = arena.take<float>(n_rows);
  }
};

template <int kDtype, int kKeep, int kBlocks, int kClassBlocks>
int launch_few(hipStream_t s, const FewRowsArgs& args, int64_t classes, bool shared)
{
  constexpr int kWaves = kFewThreads / 64;
  const dim3 grid(static_cast<unsigned>(few_groups(static_cast<int>(classes), kClassBlocks, shared)),
                  static_cast<unsigned>(tiles_of(args.n_rows, kFewBlock)));
  if (shared || kKeep != kNotKept)
    few_rows_kernel<kDtype, kBlocks, kClassBlocks, kWaves, true, kKeep><<<grid, kFewThreads, 0, s>>>(args);
  else
    few_rows_kernel<kDtype, kBlocks, kClassBlocks, kWaves, false, kNotKept><<<grid, kFewThreads, 0, s>>>(args);
  LBT_HIP(hipGetLastError());
  return LBT_OK;
}

template <int kDtype, int kKeep, int kBlocks>
int launch_few(hipStream_t s, const FewRowsArgs& args, int64_t classes, bool shared)
{
  if constexpr (kBlocks > 1)
    if (few_class_blocks(args.n_rows, static_cast<int>(classes), kDtype) == 2) return launch_few<kDtype, kKeep, kBlocks, 2>(s, args, classes, shared);
  return launch_few<kDtype, kKeep, kBlocks, 1>(s, args, classes, shared);
}

template <int kDtype, int kKeep>
int launch_few(hipStream_t s, const FewRowsArgs& args, int64_t classes, bool shared)
{
  if (args.n_rows <= 16) return launch_few<kDtype, kKeep, 1>(s, args, classes, shared);
  if (args.n_rows <= 32) return launch_few<kDtype, kKeep, 2>(s, args, classes, shared);
  if (args.n_rows <= 48) return launch_few<kDtype, kKeep, 3>(s, args, classes, shared);
  return launch_few<kDtype, kKeep, 4>(s, args, classes, shared);
}

template <int kDtype>
int few_log_loss(hipStream_t s, const FewCall& c, const void* X, const void* weight, const float* bias, const int64_t* y, int n_rows,
                 int features, int classes, float* loss)
{
  const bool shared = few_shared(classes);
  const int blocks  = few_class_blocks(n_rows, classes, kDtype), shares = static_cast<int>(few_groups(classes, blocks, shared)) * blocks;
  const FewRowsArgs args{X, weight, bias, y, n_rows, features, classes, 1, shares, c.partial, c.picked, nullptr, nullptr, nullptr, nullptr, 0};
  LBT_TRY((launch_few<kDtype, kNotKept>(s, args, classes, shared)));
  join_few_kernel<<<n_rows, kFewThreads, 0, s>>>(c.partial, shares, c.picked, y, classes, loss);
  LBT_HIP(hipGetLastError());
  return LBT_OK;
}

// Rows are taken in parts where they are many: what a call lays out and keeps for a row does not depend on how many there are. At most
// 131072 at a time, 2^30 values of their planes, and 2^34 rows times classes, which is 1 GiB of the rows' tops and totals: calls of up
// to 8192 rows are one part up to two million classes and 131072 features (43690 of float). (With gradients, 2,000,000 rows of 200
// floats, 8 classes: 0.8 GiB and 11.9 ms, in one part 12.6 GiB and 11.6 ms; 262144 rows of 1024 bfloat16, 32000 classes: 63.9 and 65.1 ms.)
int64_t rows_at_once(int64_t n, int f, int k, int dtype)
{
  const int64_t planes = dtype == LBT_F32 ? 3 : 1;
  int64_t most         = std::min<int64_t>({1 << 17, (int64_t(1) << 30) / (planes * round_up(f, kProductK)), (int64_t(1) << 34) / k});
  most                 = std::max<int64_t>(most / 256 * 256, 256);
  return n <= most ? n : round_up(tiles_of(n, tiles_of(n, most)), 256);
}

struct LossCall {
  int64_t n_rows;   // of this part
  bool parts;       // the call's rows are several
  int features, classes, dtype;
  bool gradient, with_bias;
  int planes;
  int64_t padded;   // rows
  int cols;         // features, padded
  bool packed;      // the weights are laid out piece by piece before they are multiplied
  int64_t piece;    // classes at a time
  int kept;         // all classes are one piece: G is made from the scores' exponentials instead of the scores once more
  int scale_rows;   // of a workgroup of scale_kernel
  bool few;         // the scores are those of few_rows_kernel
  bool floats;      // of float_product_kernel
  bool floats_back; // grad_X too: the weights are not laid out, G is, in both orders
  Cut all_scores, scores, row_product, class_product;
  LossRows rows;
  RowCounts* counts;
  uint16_t *zeros, *x, *x_blocks, *x_scaled, *weight, *g, *g_blocks;  // blocks: of float_product_kernel; x and g: of the other products
  float2* partial;
  float *row_sums, *class_sums, *bias_sums, *exps;

  LossCall(int64_t all_rows, int f, int k, int type, int grad, bool least)
    : features(f), classes(k), dtype(type), gradient(grad != 0), with_bias(grad > 1)
  {
    const int64_t scores_bytes = least ? kLeastScoresBytes : kScoresBytes, piece_bytes = least ? kLeastPieceBytes : kPieceBytes;
    const int64_t n = n_rows = rows_at_once(all_rows, f, k, type);
    parts                    = n < all_rows;
    planes = type == LBT_F32 ? 3 : 1;
    padded = round_up(n, 256);
    cols   = static_cast<int>(round_up(f, kProductK));
    // Where rows are few beside the features, laying out the weights and reading their planes up to six times costs more than G once more
    // in the other order. (1000 floats, 30000 classes: 17 rows 150 us, 271 with the weights laid out; 256 rows 372 and 458; 1024 rows 1213
    // and 1155.) Below 8 us of it the products of small gradients share a launch instead.
    floats_back = type == LBT_F32 && gradient && 10.0 * (f - n) * k / 5e6 > 8.0 && 16 * padded * round_up(k, 256) <= scores_bytes;
    packed = type == LBT_F32 ? gradient && !floats_back : f % 8 != 0;
    // a piece's G and its packed weights within their bounds; pieces of one size
    int64_t most = round_up(k, 256);
    kept                = type == LBT_BF16 && !with_bias ? kKeptShort : kKeptFloat;  // (the sums for the bias are those of floats)
    const int64_t bytes = 2 * planes + (kept == kKeptFloat ? 4 : 0);                // of an entry of G
    if (gradient) most = std::min(most, scores_bytes / (bytes * padded) / 256 * 256);
    if (packed) most = std::min(most, piece_bytes / (2 * planes * int64_t(cols)) / 256 * 256);
    most  = std::max<int64_t>(most, 256);
    piece = round_up(tiles_of(k, tiles_of(k, most)), 256);
    if (!gradient || piece < k) kept = kNotKept;
    const int64_t pairs = type == LBT_F32 ? 6 : 1;
    scores      = cut_product(std::min<int64_t>(piece, k), n, pairs * cols / kProductK, 1);
    all_scores  = type == LBT_F32 ? cut_floats(k, n, tiles_of(f, FloatLarge::kK), 1)
                  : packed        ? scores
                                  : cut_product(k, n, pairs * cols / kProductK, 1);
    few         = kept != kNotKept && few_rows(n, f, k, type, all_scores.time - 4.0);  // (X is laid out in either case)
    floats      = type == LBT_F32 && !few;
    scale_rows  = tiles_of(padded, 16) * tiles_of(piece, kScaleClasses) >= 1024 ? 16 : 4;
    row_product = floats_back ? cut_floats(f, n, piece / FloatLarge::kK, 64) : cut_product(f, n, pairs * piece / kProductK, 64);
    class_product = cut_product(f, std::min<int64_t>(piece, k), pairs * tiles_of(n, kProductK), 64);
  }

  template <typename A>
  void carve(A& arena)
  {
    counts        = arena.template take<RowCounts>(1);
    zeros         = arena.template take<uint16_t>(64);
    rows.order    = arena.template take<int32_t>(padded);
    rows.place    = arena.template take<int32_t>(padded);
    rows.label    = arena.template take<int32_t>(padded);
    rows.factor   = arena.template take<float>(padded);
    rows.exponent = arena.template take<int32_t>(padded);
    rows.picked   = arena.template take<float>(padded);
    rows.top      = arena.template take<float>(padded);
    rows.inverse  = arena.template take<float>(padded);
    x = x_blocks = nullptr;
    if (!floats || gradient) x = arena.template take<uint16_t>(planes * padded * cols);
    if (floats) x_blocks = arena.template take<uint16_t>(planes * padded * cols);
    partial       = arena.template take<float2>(std::max(few ? 2 * tiles_of(piece, 32) : 0, 2 * (tiles_of(round_up(classes, 256), all_scores.tile) + tiles_of(classes, piece))) * padded);
    weight = x_scaled = g = g_blocks = nullptr;
    row_sums = class_sums = bias_sums = exps = nullptr;
    if (packed) weight = arena.template take<uint16_t>(planes * piece * cols);
    if (!gradient) return;
    if (dtype == LBT_F16) x_scaled = arena.template take<uint16_t>(padded * cols);
    g         = arena.template take<uint16_t>(planes * padded * piece);
    if (floats_back) g_blocks = arena.template take<uint16_t>(planes * padded * piece);
    if (kept == kKeptFloat) exps = arena.template take<float>(padded * piece);
    row_sums  = arena.template take<float>(row_product.splits * padded * cols);
    // (of all classes where the rows come in parts: each part adds to them)
    if (parts) class_sums = arena.template take<float>(class_product.splits * static_cast<int64_t>(classes) * cols);
    else if (class_product.splits > 1) class_sums = arena.template take<float>(class_product.splits * piece * cols);
    if (with_bias) bias_sums = arena.template take<float>(tiles_of(padded, kept ? scale_rows : scores.tile) * classes);
  }
};

template <class Tile, class L, bool kAMajor, bool kBMajor, int kRowsSide, class Epilogue>
int launch_tiles(hipStream_t s, ProductArgs args, int64_t m, int64_t n, int splits, const Epilogue& e)
{
  args.tiles_m = static_cast<int>(tiles_of(m, Tile::kBM));
  args.tiles_n = static_cast<int>(tiles_of(n, Tile::kBN));
  const int64_t blocks = static_cast<int64_t>(args.tiles_m) * args.tiles_n;
  LBT_REQUIRE(blocks <= most_groups(Tile::kThreads), "too many tiles");
  product_kernel<Tile, L::kProduct, L::kPlanes, kAMajor, kBMajor, kRowsSide, Epilogue>
    <<<dim3(static_cast<unsigned>(blocks), splits), Tile::kThreads, 0, s>>>(args, e);
  LBT_HIP(hipGetLastError());
  return LBT_OK;
}

template <class L, bool kAMajor, bool kBMajor, int kRowsSide, class Epilogue>
int launch_product(hipStream_t s, const ProductArgs& args, int64_t m, int64_t n, Cut cut, const Epilogue& e)
{
  if (cut.tile == 256) return launch_tiles<LargeTile, L, kAMajor, kBMajor, kRowsSide>(s, args, m, n, cut.splits, e);
  if (cut.tile == 128) return launch_tiles<MediumTile, L, kAMajor, kBMajor, kRowsSide>(s, args, m, n, cut.splits, e);
  return launch_tiles<SmallTile, L, kAMajor, kBMajor, kRowsSide>(s, args, m, n, cut.splits, e);
}

template <class Tile, bool kAMajor, class Epilogue>
int launch_float_tiles(hipStream_t s, FloatArgs args, int64_t m, int64_t n, int splits, const Epilogue& e)
{
  args.tiles_m = static_cast<int>(tiles_of(m, Tile::kBM));
  args.tiles_n = static_cast<int>(tiles_of(n, Tile::kBN));
  args.k_split = static_cast<int32_t>(round_up(tiles_of(kAMajor ? args.rows : args.cols, splits), Tile::kK));
  const int64_t blocks = static_cast<int64_t>(args.tiles_m) * args.tiles_n;
  LBT_REQUIRE(blocks <= most_groups(Tile::kThreads), "too many tiles");
  float_product_kernel<Tile, kAMajor, Epilogue><<<dim3(static_cast<unsigned>(blocks), splits), Tile::kThreads, 0, s>>>(args, e);
  LBT_HIP(hipGetLastError());
  return LBT_OK;
}

template <bool kAMajor, class Epilogue>
int launch_floats(hipStream_t s, const FloatArgs& args, int64_t m, int64_t n, Cut cut, const Epilogue& e)
{
  if (cut.tile == FloatLarge::kBM) return launch_float_tiles<FloatLarge, kAMajor>(s, args, m, n, cut.splits, e);
  return launch_float_tiles<FloatSmall, kAMajor>(s, args, m, n, cut.splits, e);
}

template <int kDtype>
int launch_pack(hipStream_t s, const void* from, int64_t first_row, int64_t rows, int cols, const int32_t* order,
                int mode, const int32_t* exponent, RowCounts* counts, int64_t out_rows, int padded_cols, Layout layout, uint16_t* out)
{
  const int64_t blocks = tiles_of(out_rows * (padded_cols / 8), 256);
  LBT_REQUIRE(blocks <= most_groups(256), "too many values to lay out");
  pack_rows_kernel<kDtype><<<static_cast<unsigned>(blocks), 256, 0, s>>>(from, first_row, rows, cols, order, mode, exponent, counts,
                                                                         out_rows, padded_cols, layout, out);
  LBT_HIP(hipGetLastError());
  return LBT_OK;
}

// grad_weight of the classes first .. first + classes - 1 from their sums, as many at a time as a launch may take.
template <int kDtype>
int launch_finish_classes(hipStream_t s, const LossCall& c, const float* sums, int64_t split, int64_t first, int64_t classes, bool scaled, void* out)
{
  const int64_t groups = (c.features + 3) / 4, most = (int64_t(1) << 30) / groups;
  for (int64_t at = 0; at < classes; at += most) {
    const int64_t some = std::min(most, classes - at);
    finish_classes_kernel<kDtype><<<static_cast<unsigned>(tiles_of(some * groups, 256)), 256, 0, s>>>(
      sums + at * c.cols, c.class_product.splits, split, c.cols, first + at, some, c.features, c.counts, scaled, out);
    LBT_HIP(hipGetLastError());
  }
  return LBT_OK;
}

// Of one part of the rows; `begins` and `ends`: whether it is the first one and the last.
template <int kDtype>
int linear_log_loss(hipStream_t s, const LossCall& c, const void* X, const void* weight, const float* bias, const int64_t* y,
                    const float* sample_weight, float* loss, void* grad_X, void* grad_weight, float* grad_bias, bool begins, bool ends)
{
  using L              = LossType<kDtype>;
  constexpr bool kFine = kDtype == LBT_F32;
  constexpr bool kHalf = kDtype == LBT_F16;
  if (c.n_rows == 0) {  // no row: the gradients are zeros
    auto clear = [&](void* out, int64_t halves) {
      clear_kernel<<<static_cast<unsigned>(std::min<int64_t>(tiles_of(halves, 256), 1 << 20)), 256, 0, s>>>(static_cast<uint16_t*>(out), halves);
    };
    clear(grad_weight, int64_t(c.classes) * c.features * sizeof(typename L::Value) / 2);
    if (grad_bias != nullptr) clear(grad_bias, 2 * int64_t(c.classes));
    LBT_HIP(hipGetLastError());
    return LBT_OK;
  }
  const bool scaled = kHalf && sample_weight != nullptr;  // (without weights every exponent is 0)
  const bool fused  = c.padded <= kFusedRows && !scaled;
  const Layout x_layout{c.padded * c.cols, c.cols, 32}, x_blocks{32, 96, 96 * c.padded};
  if (fused) {
    const FusedArgs a{y,         sample_weight, static_cast<int>(c.n_rows), static_cast<int>(c.padded), c.classes, loss, c.counts, c.zeros, X, weight,
                      c.features, c.cols,        c.x,                        c.packed ? c.weight : nullptr, c.packed ? c.piece : 0, c.x_blocks, x_blocks};
    const int64_t groups = c.padded / kFusedEach * tiles_of(c.cols / 8, kFusedGroups) + tiles_of(a.weight_rows * (c.cols / 8), 256);
    LBT_REQUIRE(groups <= most_groups(256), "too many values to lay out");
    prepare_pack_kernel<kDtype><<<static_cast<unsigned>(groups), 256, 0, s>>>(a, c.rows);
    LBT_HIP(hipGetLastError());
  } else {
    prepare_rows_kernel<<<1, kPrepareThreads, 0, s>>>(y, sample_weight, c.n_rows, c.padded, c.classes, kHalf, c.rows, loss, c.counts, c.zeros);
    LBT_HIP(hipGetLastError());
    if (c.x != nullptr)
      LBT_TRY(launch_pack<kDtype>(s, X, 0, c.n_rows, c.features, c.rows.order, scaled ? kMeasure : kCopy, c.rows.exponent, c.counts, c.padded,
                                  c.cols, x_layout, c.x));
    if (c.x_blocks != nullptr)
      LBT_TRY(launch_pack<kDtype>(s, X, 0, c.n_rows, c.features, c.rows.order, kCopy, c.rows.exponent, c.counts, c.padded, c.cols, x_blocks,
                                  c.x_blocks));
  }

  // (rows that do not count are not there: x holds them side by side)
  const ProductOperand x{c.x, c.cols, c.padded * c.cols, static_cast<int32_t>(c.padded), c.cols};
  auto weights = [&](int64_t first, int64_t classes) {  // a piece, laid out by lay_out, or the caller's rows
    if (c.packed) return ProductOperand{c.weight, c.cols, c.piece * c.cols, static_cast<int32_t>(classes), c.cols};
    return ProductOperand{static_cast<const uint16_t*>(weight) + first * c.features, c.features, 0, static_cast<int32_t>(classes),
                          c.features};
  };
  auto lay_out = [&](int64_t first) {
    if (!c.packed || (!begins && c.piece >= c.classes)) return LBT_OK;  // (all of them are there from the rows before)
    return launch_pack<kDtype>(s, weight, first, c.classes, c.features, nullptr, kCopy, nullptr, c.counts, c.piece, c.cols,
                               Layout{c.piece * c.cols, c.cols, 32}, c.weight);
  };
  ProductArgs args{};
  args.zeros  = c.zeros;
  args.counts = c.counts;

  // top and total of each row; weights that are multiplied where they lie need no pieces here
  // (but launches their bound: 2^26 classes at a time where the tiles of more might be too many)
  const int64_t step = c.packed && !c.floats ? c.piece : c.kept != kNotKept ? c.classes : std::min<int64_t>(c.classes, 1 << 26);
  int64_t tiles      = 0;
  if (c.few) {
    const FewRowsArgs few{X, weight, bias, nullptr, static_cast<int>(c.n_rows), c.features, c.classes, 1, c.piece / 16, c.partial, c.rows.picked,
                          c.rows.order, c.rows.label, c.counts, c.kept == kKeptFloat ? static_cast<void*>(c.exps) : c.g,
                          static_cast<int>(c.piece)};
    if constexpr (kDtype == LBT_BF16)
      LBT_TRY((c.kept == kKeptShort ? launch_few<kDtype, kKeptShort>(s, few, c.piece, true) : launch_few<kDtype, kKeptFloat>(s, few, c.piece, true)));
    else
      LBT_TRY((launch_few<kDtype, kKeptFloat>(s, few, c.piece, true)));
  }
  for (int64_t first = 0; first < c.classes && !c.few; first += step) {
    const int64_t classes = std::min<int64_t>(step, c.classes - first);
    if (!c.floats && (first > 0 || !fused)) LBT_TRY(lay_out(first));  // (the first piece is there)
    args.a = weights(first, classes);
    args.b = x;
    args.k_extent = args.k_split = c.cols;
    const int share = 2 * static_cast<int>(tiles);  // (all tiles are two waves high)
    // (every piece in tiles of one size: they share the numbering of `partial`)
    auto scores = [&](auto kind) {
      constexpr int kKind = decltype(kind)::value;
      const int64_t m     = kKind == kNotKept ? classes : c.piece;  // (what is kept is kept for the whole piece)
      const LossEpilogue<kFine, kKind> e{bias, static_cast<int>(first), c.classes, share, c.padded, c.rows, c.partial,
                                         kKind == kKeptFloat ? static_cast<void*>(c.exps) : c.g, static_cast<int>(c.piece)};
      tiles += tiles_of(m, c.all_scores.tile);
      if constexpr (kFine) {
        const FloatArgs fa{static_cast<const float*>(weight) + first * c.features, c.classes - static_cast<int>(first), c.features, 0, c.x_blocks,
                           c.padded, 0, 0, c.zeros, c.counts};
        return launch_floats<false>(s, fa, m, c.n_rows, c.all_scores, e);
      } else {
        return launch_product<L, false, false, kRowsN>(s, args, m, c.n_rows, c.all_scores, e);
      }
    };
    if constexpr (kDtype == LBT_BF16)
      if (c.kept == kKeptShort) {
        LBT_TRY(scores(std::integral_constant<int, kKeptShort>{}));
        continue;
      }
    LBT_TRY(c.kept == kNotKept ? scores(std::integral_constant<int, kNotKept>{}) : scores(std::integral_constant<int, kKeptFloat>{}));
  }
  const int share_classes = c.few ? 16 : c.all_scores.tile / 2;
  const int shares    = c.few ? static_cast<int>(c.piece / 16) : 2 * static_cast<int>(tiles);
  const int join_here = c.kept != kNotKept && c.scale_rows == 4 && shares <= 256 ? shares : 0;  // in scale_kernel
  if (c.few && join_here == 0) {
    join_few_rows_kernel<<<static_cast<unsigned>(c.n_rows), kFewThreads, 0, s>>>(c.partial, shares, c.rows, c.counts, loss);
    LBT_HIP(hipGetLastError());
  } else if (join_here == 0) {
    join_kernel<<<static_cast<unsigned>(tiles_of(c.n_rows, kJoinRows)), kJoinRows * kJoinSlices, 0, s>>>(c.partial, shares, c.padded, c.rows,
                                                                                                       c.counts, loss);
    LBT_HIP(hipGetLastError());
  }
  if (!c.gradient) return LBT_OK;

  if (scaled)
    LBT_TRY(launch_pack<kDtype>(s, X, 0, c.n_rows, c.features, c.rows.order, kScale, c.rows.exponent, c.counts, c.padded, c.cols,
                                x_layout, c.x_scaled));
  ProductOperand x_scaled = x;
  if (scaled) x_scaled.base = c.x_scaled;
  const ProductOperand g{c.g, c.piece, c.padded * c.piece, static_cast<int32_t>(c.padded), static_cast<int32_t>(c.piece)};
  // (whether the first piece of the weights is there still, or already)
  const bool laid_out = c.few || c.floats ? fused : c.piece >= c.classes;
  for (int64_t first = 0; first < c.classes; first += c.piece) {
    const int64_t classes = std::min<int64_t>(c.piece, c.classes - first);
    if (first > 0 || !laid_out) LBT_TRY(lay_out(first));
    const ProductOperand w = weights(first, classes);
    if (c.kept != kNotKept) {
      auto scale = [&](auto narrow, auto each) {
        constexpr int kRows = decltype(each)::value;
        scale_kernel<kDtype, decltype(narrow)::value, kRows>
          <<<static_cast<unsigned>(tiles_of(c.piece, kScaleClasses) * tiles_of(c.padded, kRows)), 256, 0, s>>>(
            decltype(narrow)::value ? static_cast<const void*>(c.g) : c.exps, c.partial, share_classes, c.few ? 1 : c.padded, c.few ? shares : 1, std::max(c.row_product.tile, kProductK), c.rows, c.counts,
            c.classes, static_cast<int>(c.piece), c.padded * c.piece, c.g, c.g_blocks, c.padded, grad_bias != nullptr ? c.bias_sums : nullptr, join_here, loss);
      };
      auto scale_by = [&](auto narrow) {
        if (c.scale_rows == 16) scale(narrow, std::integral_constant<int, 16>{});
        else scale(narrow, std::integral_constant<int, 4>{});
      };
      if constexpr (kDtype == LBT_BF16) {
        if (c.kept == kKeptShort) scale_by(std::true_type{});
        else scale_by(std::false_type{});
      } else {
        scale_by(std::false_type{});
      }
      LBT_HIP(hipGetLastError());
    } else {
      args.a        = w;
      args.b        = x;
      args.k_extent = args.k_split = c.cols;
      const GradientEpilogue<kFine, L::kProduct, L::kPlanes> ge{bias, static_cast<int>(first), c.classes, static_cast<int>(c.piece),
                                                                c.rows, c.g, c.padded * c.piece,
                                                                grad_bias != nullptr ? c.bias_sums : nullptr};
      // (over the whole piece: what lies past its classes is written as zeros)
      LBT_TRY((launch_product<L, false, false, kRowsN>(s, args, c.piece, c.n_rows, c.scores, ge)));
    }
    args.a        = w;
    args.b        = g;
    args.k_extent = static_cast<int32_t>(c.piece);
    args.k_split  = static_cast<int32_t>(round_up(tiles_of(c.piece, c.row_product.splits), kProductK));
    const RowsEpilogue re{c.row_sums, c.padded * c.cols, c.cols, first == 0, 0, false};
    ProductArgs more = args;
    more.a           = x_scaled;
    more.k_extent    = static_cast<int32_t>(c.padded);
    more.k_split     = static_cast<int32_t>(round_up(tiles_of(c.padded, c.class_product.splits), kProductK));
    auto products    = [&](const auto& ce) -> int {
      if constexpr (kFine)
        if (c.floats_back) {
          const FloatArgs fa{static_cast<const float*>(weight), c.classes, c.features, 0, c.g_blocks, c.padded, 0, 0, c.zeros, c.counts};
          LBT_TRY((launch_floats<true>(s, fa, c.features, c.n_rows, c.row_product, re)));
          return launch_product<L, true, true, kRowsK>(s, more, c.features, classes, c.class_product, ce);
        }
      if (c.row_product.tile == SmallTile::kBM && c.class_product.tile == SmallTile::kBM) {
        args.tiles_m = more.tiles_m = static_cast<int>(tiles_of(c.features, SmallTile::kBM));
        args.tiles_n = static_cast<int>(tiles_of(c.n_rows, SmallTile::kBN));
        more.tiles_n = static_cast<int>(tiles_of(classes, SmallTile::kBN));
        const int64_t blocks = static_cast<int64_t>(args.tiles_m) * args.tiles_n * c.row_product.splits;
        const int64_t all    = blocks + static_cast<int64_t>(more.tiles_m) * more.tiles_n * c.class_product.splits;
        LBT_REQUIRE(all <= most_groups(SmallTile::kThreads), "too many tiles");
        two_products_kernel<SmallTile, L::kProduct, L::kPlanes>
          <<<static_cast<unsigned>(all), SmallTile::kThreads, 0, s>>>(args, re, static_cast<unsigned>(blocks), more, ce);
        LBT_HIP(hipGetLastError());
        return LBT_OK;
      }
      LBT_TRY((launch_product<L, true, false, kRowsN>(s, args, c.features, c.n_rows, c.row_product, re)));
      return launch_product<L, true, true, kRowsK>(s, more, c.features, classes, c.class_product, ce);
    };
    if (c.parts) {
      LBT_TRY(products(RowsEpilogue{c.class_sums + first * c.cols, static_cast<int64_t>(c.classes) * c.cols, c.cols, begins,
                                    static_cast<int>(classes), scaled}));
    } else if (c.class_product.splits > 1) {
      LBT_TRY(products(RowsEpilogue{c.class_sums, c.piece * c.cols, c.cols, true, static_cast<int>(classes), false}));
      LBT_TRY(launch_finish_classes<kDtype>(s, c, c.class_sums, c.piece * c.cols, first, classes, scaled, grad_weight));
    } else {
      LBT_TRY(products(ClassesEpilogue<kDtype>{grad_weight, static_cast<int>(first), c.classes, c.features, scaled}));
    }
  }
  if (c.parts && ends)
    LBT_TRY(launch_finish_classes<kDtype>(s, c, c.class_sums, static_cast<int64_t>(c.classes) * c.cols, 0, c.classes, false, grad_weight));
  const int64_t blocks = tiles_of(c.n_rows * ((c.features + 3) / 4), 256);
  LBT_REQUIRE(blocks <= most_groups(256), "too many values");
  finish_rows_kernel<kDtype><<<static_cast<unsigned>(blocks), 256, 0, s>>>(c.row_sums, c.row_product.splits, c.padded * c.cols, c.cols,
                                                                           c.n_rows, c.features, c.rows, grad_X);
  LBT_HIP(hipGetLastError());
  if (grad_bias != nullptr) {
    constexpr int kMost = 1 << 24;  // classes of a launch: 64 threads each
    for (int first = 0; first < c.classes; first += kMost) {
      finish_bias_kernel<<<static_cast<unsigned>(tiles_of(std::min(c.classes - first, kMost), kJoinRows)), kJoinRows * kJoinSlices, 0, s>>>(
        c.bias_sums, first, c.classes, c.kept ? c.scale_rows : c.scores.tile, c.counts, kHalf, !begins, grad_bias);
      LBT_HIP(hipGetLastError());
    }
  }
  return LBT_OK;
}

bool loss_shape(int64_t n_rows, int32_t n_features, int32_t n_outputs, int32_t dtype)
{
  return (dtype == LBT_F32 || dtype == LBT_BF16 || dtype == LBT_F16) && n_rows >= 0 && n_features >= 1 && n_outputs >= 1 &&
         n_rows <= (int64_t(1) << 30) && n_features <= (1 << 20) && n_outputs <= (1 << 30) - 64 &&
         n_rows * n_features < (int64_t(1) << 38) && int64_t(n_outputs) * n_features < (int64_t(1) << 38);
}

int run_loss(void* stream, const void* X, const void* weight, int32_t dtype, int64_t n_rows, int32_t n_features, int32_t n_outputs,
             const float* bias, const int64_t* y, const float* sample_weight, float* loss, void* grad_X, void* grad_weight,
             float* grad_bias, bool gradient, void* workspace, size_t workspace_bytes)
{
  LBT_REQUIRE(dtype == LBT_F32 || dtype == LBT_BF16 || dtype == LBT_F16, "unsupported dtype %d", dtype);
  LBT_REQUIRE(loss_shape(n_rows, n_features, n_outputs, dtype), "bad shape");
  LBT_REQUIRE(grad_bias == nullptr || bias != nullptr, "a gradient of the bias without a bias");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_rows == 0 && !gradient) return LBT_OK;
  LBT_REQUIRE(weight != nullptr, "null pointer");
  LBT_REQUIRE(n_rows == 0 || (X != nullptr && y != nullptr && loss != nullptr), "null pointer");
  LBT_REQUIRE(!gradient || (grad_weight != nullptr && (n_rows == 0 || grad_X != nullptr)), "null pointer");
  const uintptr_t places = reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(weight) |
                           reinterpret_cast<uintptr_t>(grad_X) | reinterpret_cast<uintptr_t>(grad_weight);
  LBT_REQUIRE((places & 15) == 0, "X, weight and their gradients must be 16-byte aligned");
  const int64_t size = dtype == LBT_F32 ? 4 : 2, rows = size * n_rows * n_features, classes = size * n_outputs * n_features;
  const MemoryRange ranges[] = {{workspace, static_cast<int64_t>(workspace_bytes)}, {loss, 4 * n_rows}, {grad_X, rows}, {grad_weight, classes},
                                {grad_bias, 4 * int64_t(n_outputs)}, {X, rows}, {weight, classes}, {bias, 4 * int64_t(n_outputs)}, {y, 8 * n_rows},
                                {sample_weight, 4 * n_rows}};
  LBT_REQUIRE(ranges_apart(ranges, 5, 10), "outputs and workspace may not overlap the inputs or one another");
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) {
    set_error("a workspace aligned to 256 bytes is needed");
    return LBT_ERR_WORKSPACE;
  }
  const int kind = !gradient ? 0 : grad_bias == nullptr ? 1 : 2;
  LossCall c(std::max<int64_t>(n_rows, 1), n_features, n_outputs, dtype, kind, false);
  const bool few = !gradient && few_loss(n_rows, n_features, n_outputs, dtype);
  FewCall f;
  Arena arena;
  arena.base = static_cast<char*>(workspace);
  arena.cap  = workspace_bytes;
  if (few) f.carve(arena, n_rows, n_outputs, dtype);
  else c.carve(arena);
  if (arena.failed && !few) {  // the least, perhaps
    LossCall smaller(std::max<int64_t>(n_rows, 1), n_features, n_outputs, dtype, kind, true);
    Arena there;
    there.base = arena.base;
    there.cap  = arena.cap;
    smaller.carve(there);
    if (!there.failed) {
      c            = smaller;
      arena.failed = false;
    }
  }
  if (arena.failed) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, arena.used);
    return LBT_ERR_WORKSPACE;
  }
  ProfScope ps(LBT_PROF_OTHER, s);
  if (few) {
    const int n = static_cast<int>(n_rows);
    if (dtype == LBT_BF16) return few_log_loss<LBT_BF16>(s, f, X, weight, bias, y, n, n_features, n_outputs, loss);
    if (dtype == LBT_F16) return few_log_loss<LBT_F16>(s, f, X, weight, bias, y, n, n_features, n_outputs, loss);
    return few_log_loss<LBT_F32>(s, f, X, weight, bias, y, n, n_features, n_outputs, loss);
  }
  const int64_t at_once = c.n_rows;
  int64_t first         = 0;
  do {
    c.n_rows              = std::min(at_once, n_rows - first);
    const int64_t value   = size * first * n_features;  // bytes before this part's rows
    const void* const x   = static_cast<const char*>(X) + value;
    void* const gx        = grad_X == nullptr ? nullptr : static_cast<char*>(grad_X) + value;
    const float* const sw = sample_weight == nullptr ? nullptr : sample_weight + first;
    const bool begins = first == 0, ends = first + at_once >= n_rows;
    switch (dtype) {
      case LBT_BF16:
        LBT_TRY(linear_log_loss<LBT_BF16>(s, c, x, weight, bias, y + first, sw, loss + first, gx, grad_weight, grad_bias, begins, ends));
        break;
      case LBT_F16:
        LBT_TRY(linear_log_loss<LBT_F16>(s, c, x, weight, bias, y + first, sw, loss + first, gx, grad_weight, grad_bias, begins, ends));
        break;
      default:
        LBT_TRY(linear_log_loss<LBT_F32>(s, c, x, weight, bias, y + first, sw, loss + first, gx, grad_weight, grad_bias, begins, ends));
    }
    first += at_once;
  } while (first < n_rows);
  return LBT_OK;
}

}  // namespace
}  // namespace lbt

extern "C" {

size_t lbt_linear_log_loss_workspace_bytes(int64_t n_rows, int32_t n_features, int32_t n_outputs, int32_t dtype, int32_t gradient)
{
  const bool least = gradient >= LBT_LEAST_WORKSPACE;
  if (least) gradient -= LBT_LEAST_WORKSPACE;
  if (!lbt::loss_shape(n_rows, n_features, n_outputs, dtype) || gradient < 0 || gradient > 2) return 0;
  lbt::LossCall c(std::max<int64_t>(n_rows, 1), n_features, n_outputs, dtype, gradient, least);
  lbt::Arena arena;
  arena.measure = true;
  if (gradient == 0 && lbt::few_loss(n_rows, n_features, n_outputs, dtype)) {
    lbt::FewCall f;
    f.carve(arena, n_rows, n_outputs, dtype);
    return std::max<size_t>(arena.used, 256);
  }
  c.carve(arena);
  return arena.used;
}

int lbt_linear_log_loss(void* stream, const void* X, const void* weight, int32_t dtype, int64_t n_rows, int32_t n_features,
                        int32_t n_outputs, const float* bias, const int64_t* y, float* loss, void* workspace,
                        size_t workspace_bytes)
{
  return lbt::run_loss(stream, X, weight, dtype, n_rows, n_features, n_outputs, bias, y, nullptr, loss, nullptr, nullptr, nullptr,
                       false, workspace, workspace_bytes);
}

int lbt_linear_log_loss_gradient(void* stream, const void* X, const void* weight, int32_t dtype, int64_t n_rows,
                                 int32_t n_features, int32_t n_outputs, const float* bias, const int64_t* y,
                                 const float* sample_weight, float* loss, void* grad_X, void* grad_weight, float* grad_bias,
                                 void* workspace, size_t workspace_bytes)
{
  return lbt::run_loss(stream, X, weight, dtype, n_rows, n_features, n_outputs, bias, y, sample_weight, loss, grad_X, grad_weight,
                       grad_bias, true, workspace, workspace_bytes);
}

}  // extern "C"
