// Rows of a table by their numbers, times a scale, and the gradient with respect to the table.
//
//   out[t] = scale * table[token[t]]                   (zeros where token[t] is no row of the table)
//   grad_table[v] = scale * sum_{t: token[t] = v} grad[t]
//
// The gradient sorts the places by their token, equal tokens by place, so that the sums have one order whatever the hardware
// does first: no atomics touch a sum. The sorted places are then cut into chunks of equal length, whatever their tokens are: a
// wave adds up the rows of a chunk for its share of the columns, in 32 bits. A run of equal tokens inside a chunk is finished
// there; of one that crosses a chunk's end each chunk leaves its part, and join_runs_kernel adds the parts in order. A token
// that takes a twentieth of all places is thus the work of many waves.
// Bound by memory: grad is read once and the table's gradient written once. 65536 places of 2048 bfloat16 into 65536 rows: 127 us for
// the sums, 537 MB at 4.2 TB/s, and 40 us for the sort and the join, which are launches and latency.
#include <algorithm>
#include <type_traits>

#include "lbt_device.h"
#include "lbt_internal.h"

namespace lbt {

namespace {

template <int kDtype>
__device__ __forceinline__ float widen(uint32_t bits)
{
  if constexpr (kDtype == LBT_F32) return __builtin_bit_cast(float, bits);
  if constexpr (kDtype == LBT_F16) return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  return __builtin_bit_cast(float, bits << 16);
}

template <int kDtype>
__device__ __forceinline__ uint32_t narrow(float v)
{
  if constexpr (kDtype == LBT_F32) return __builtin_bit_cast(uint32_t, v);
  if constexpr (kDtype == LBT_F16) return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

// v * scale as a float, whatever follows: the compiler joins a product and its rounding to half precision into one instruction
// where it can, which rounds once and not twice; the same value would then depend on how many of them a lane takes.
__device__ __forceinline__ float scaled(float v, float scale)
{
  float p = v * scale;
  asm("" : "+v"(p));
  return p;
}

// kBytes consecutive bytes of a row: its values as floats and back.
template <int kDtype, int kBytes>
struct Pack {
  static constexpr int kSize = kDtype == LBT_F32 ? 4 : 2, kValues = kBytes / kSize;
  using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>;

  static __device__ __forceinline__ void unpack(Word w, float (&v)[kValues])
  {
    if constexpr (kBytes == 16) {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < kValues; i++)
        v[i] = kSize == 4 ? widen<kDtype>(x[i % 4]) : widen<kDtype>((x[i / 2] >> (16 * (i & 1))) & 0xffffu);
    } else {
#pragma unroll
      for (int i = 0; i < kValues; i++) v[i] = kSize == 4 ? widen<kDtype>(w) : widen<kDtype>((uint32_t(w) >> (16 * i)) & 0xffffu);
    }
  }
  static __device__ __forceinline__ Word pack(const float (&v)[kValues])
  {
    if constexpr (kBytes == 16) {
      uint32_t x[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kValues; i++) {
        if constexpr (kSize == 4) x[i % 4] = narrow<kDtype>(v[i]);
        else x[i / 2] |= narrow<kDtype>(v[i]) << (16 * (i & 1));
      }
      return make_uint4(x[0], x[1], x[2], x[3]);
    } else {
      uint32_t x = 0;
#pragma unroll
      for (int i = 0; i < kValues; i++) x |= narrow<kDtype>(v[i]) << (kSize == 4 ? 0 : 16 * i);
      return static_cast<Word>(x);
    }
  }
};

// tokens as they come: 4 or 8 bytes each. What is no row of the table becomes n_rows.
__device__ __forceinline__ int token_at(const void* tokens, int bytes, int64_t t, int n_rows)
{
  const int64_t v = bytes == 8 ? static_cast<const int64_t*>(tokens)[t] : static_cast<const int32_t*>(tokens)[t];
  return v >= 0 && v < n_rows ? static_cast<int>(v) : n_rows;
}

constexpr int kRowThreads = 256, kRowWaves = kRowThreads / 64;

// A group of kLanes lanes copies a row, kEach words of a lane at a time. Bound by memory: 65536 tokens of 2048 bfloat16 74 us, 4.7 TB/s
// of what has to be read and written.
template <int kDtype, int kBytes, int kLanes>
__global__ void __launch_bounds__(kRowThreads)
  embed_rows_kernel(const void* __restrict__ table, int n_rows, int words, const void* __restrict__ tokens, int token_bytes,
                    int64_t n_tokens, float scale, void* __restrict__ out)
{
  using P             = Pack<kDtype, kBytes>;
  using Word          = typename P::Word;
  constexpr int kEach = 4;
  const int64_t t     = blockIdx.x * int64_t(kRowThreads / kLanes) + threadIdx.x / kLanes;
  if (t >= n_tokens) return;
  const int v      = token_at(tokens, token_bytes, t, n_rows);
  const Word* from = static_cast<const Word*>(table) + static_cast<int64_t>(v) * words;
  Word* to         = static_cast<Word*>(out) + t * words;
  for (int at = threadIdx.x % kLanes; at < words; at += kLanes * kEach) {
    Word w[kEach];
    if (v < n_rows) {
#pragma unroll
      for (int e = 0; e < kEach; e++)
        if (at + e * kLanes < words) w[e] = from[at + e * kLanes];
    }
#pragma unroll
    for (int e = 0; e < kEach; e++) {
      if (at + e * kLanes >= words) break;
      float x[P::kValues];
      if (v < n_rows) P::unpack(w[e], x);
#pragma unroll
      for (int i = 0; i < P::kValues; i++) x[i] = v < n_rows ? scaled(x[i], scale) : 0.f;
      to[at + e * kLanes] = P::pack(x);
    }
  }
}

// ---- places sorted by token ----------------------------------------------------------------------

struct Sorted {
  int32_t* key;    // tokens, ascending; places that name no row come last, as n_rows
  int32_t* place;  // where in `grad` each is; equal tokens in ascending order
};

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

// Few tokens: the place of each among the sorted ones is the number of those before it, counted. A workgroup counts for 64
// tokens; its waves share out the others, 64 at a time. No atomics and one launch; 8192 tokens are 128 workgroups.
__global__ void __launch_bounds__(kSortThreads)
  count_sort_kernel(const void* __restrict__ tokens, int token_bytes, int n_tokens, int n_rows, Sorted out)
{
  __shared__ int before[kSortWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int own  = blockIdx.x * 64 + lane;
  const int key  = own < n_tokens ? token_at(tokens, token_bytes, own, n_rows) : 0;
  int count      = 0;
  for (int b = wave; b * 64 < n_tokens; b += kSortWaves) {
    const int j     = b * 64 + lane;
    const int other = j < n_tokens ? token_at(tokens, token_bytes, j, n_rows) : 0x7fffffff;
    const int bound = b < static_cast<int>(blockIdx.x) ? key + 1 : key;  // equal ones count where they come first
    for (int l = 0; l < 64; l++) count += __builtin_amdgcn_readlane(other, l) < bound ? 1 : 0;
    if (b == static_cast<int>(blockIdx.x))
      for (int l = 0; l < 64; l++) count += __builtin_amdgcn_readlane(other, l) == key && l < lane ? 1 : 0;
  }
  before[wave][lane] = count;
  __syncthreads();
  if (wave != 0 || own >= n_tokens) return;
  int rank = 0;
  for (int w = 0; w < kSortWaves; w++) rank += before[w][lane];
  out.key[rank]   = key;
  out.place[rank] = own;
}

// Many tokens: by digits of up to 10 bits, least significant first; each pass counts, adds up and moves. 65536 tokens of 17 bits: two
// passes of 4 and 9 us, launches and the latency of a block's way through its entries.
constexpr int kDigits = 1024;  // at most; a block is kSortThreads * kSortEach entries

__device__ __forceinline__ int sort_key(const void* tokens, int token_bytes, const int32_t* keys, int64_t i, int n_rows)
{
  return keys != nullptr ? keys[i] : token_at(tokens, token_bytes, i, n_rows);
}

template <int kSortEach>
__global__ void __launch_bounds__(kSortThreads)
  digit_count_kernel(const void* __restrict__ tokens, int token_bytes, const int32_t* __restrict__ keys, int64_t n, int n_rows,
                     int shift, int digits, int32_t* __restrict__ counts)
{
  __shared__ int count[kDigits];
  count[threadIdx.x] = 0;
  __syncthreads();
  for (int e = 0; e < kSortEach; e++) {
    const int64_t i = blockIdx.x * int64_t(kSortThreads * kSortEach) + e * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&count[(sort_key(tokens, token_bytes, keys, i, n_rows) >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < digits) counts[static_cast<int64_t>(blockIdx.x) * digits + threadIdx.x] = count[threadIdx.x];
}

// counts [blocks][digits] become the number of entries before each: one workgroup, a thread per digit.
__global__ void __launch_bounds__(kSortThreads) digit_offsets_kernel(int digits, int blocks, int32_t* __restrict__ counts)
{
  __shared__ int wave_sum[kSortWaves];
  constexpr int kAhead = 16;  // counts asked for together
  const int d = threadIdx.x, lane = d & 63, wave = d >> 6;
  int c[kAhead], sum = 0;
  auto load = [&](int b0) {
#pragma unroll
    for (int e = 0; e < kAhead; e++) c[e] = d < digits && b0 + e < blocks ? counts[static_cast<int64_t>(b0 + e) * digits + d] : 0;
  };
  for (int b0 = 0; b0 < blocks; b0 += kAhead) {
    load(b0);
#pragma unroll
    for (int e = 0; e < kAhead; e++) sum += c[e];
  }
  int upto = sum;
  for (int s = 1; s < 64; s <<= 1) {
    const int other = __shfl_up(upto, s);
    if (lane >= s) upto += other;
  }
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < wave; w++) at += wave_sum[w];
  for (int b0 = 0; b0 < blocks; b0 += kAhead) {
    if (blocks > kAhead) load(b0);
#pragma unroll
    for (int e = 0; e < kAhead; e++) {
      if (d < digits && b0 + e < blocks) counts[static_cast<int64_t>(b0 + e) * digits + d] = at;
      at += c[e];
    }
  }
}

// Where a block's entries of each digit begin, from the counts of all blocks, by every block of the move itself: while the blocks are
// few that takes less than a launch. Thread d has digit d.
__device__ __forceinline__ int digit_offset(const int32_t* __restrict__ counts, int digits, int blocks, int block, int* wave_sum)
{
  constexpr int kAhead = 16;
  const int d = threadIdx.x, lane = d & 63, wave = d >> 6;
  int all = 0, before = 0;
  for (int b0 = 0; b0 < blocks; b0 += kAhead) {
    int c[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; e++) c[e] = d < digits && b0 + e < blocks ? counts[static_cast<int64_t>(b0 + e) * digits + d] : 0;
#pragma unroll
    for (int e = 0; e < kAhead; e++) {
      all += c[e];
      before += b0 + e < block ? c[e] : 0;
    }
  }
  int upto = all;
  for (int s = 1; s < 64; s <<= 1) {
    const int other = __shfl_up(upto, s);
    if (lane >= s) upto += other;
  }
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  int at = upto - all + before;
  for (int w = 0; w < wave; w++) at += wave_sum[w];
  return at;
}

// A wave takes 64 * kSortEach consecutive entries, 64 at a time: the lanes of equal digits find one another by ballots, the first of
// them moves the wave's count on. Ranks are then the block's offset, the waves before, and the place in the wave: stable.
template <int kSortEach>
__global__ void __launch_bounds__(kSortThreads)
  digit_move_kernel(const void* __restrict__ tokens, int token_bytes, const int32_t* __restrict__ keys,
                    const int32_t* __restrict__ places, int64_t n, int n_rows, int shift, int bits,
                    const int32_t* __restrict__ offsets, int blocks, Sorted out)
{
  __shared__ int wave_sum[kSortWaves];
  __shared__ uint16_t count[kSortWaves][kDigits];
  __shared__ int first[kDigits];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int digits = 1 << bits;
  for (int w = 0; w < kSortWaves; w++) count[w][threadIdx.x] = 0;
  if (blocks > 0) {  // `offsets` are counts still
    first[threadIdx.x] = digit_offset(offsets, digits, blocks, blockIdx.x, wave_sum);
  } else if (static_cast<int>(threadIdx.x) < digits) {
    first[threadIdx.x] = offsets[static_cast<int64_t>(blockIdx.x) * digits + threadIdx.x];
  }
  __syncthreads();
  const int64_t begin = blockIdx.x * int64_t(kSortThreads * kSortEach) + wave * (64 * kSortEach);
  int key[kSortEach], digit[kSortEach], rank[kSortEach];
  for (int e = 0; e < kSortEach; e++) {
    const int64_t i = begin + e * 64 + lane;
    const bool in   = i < n;
    key[e]          = in ? sort_key(tokens, token_bytes, keys, i, n_rows) : 0;
    digit[e]        = (key[e] >> shift) & (digits - 1);
    uint64_t same   = __ballot(in);
    for (int b = 0; b < bits; b++) {
      const uint64_t set = __ballot((digit[e] >> b) & 1);
      same &= (digit[e] >> b) & 1 ? set : ~set;
    }
    const int ahead = __popcll(same & ((uint64_t(1) << lane) - 1));
    const int so_far = in ? count[wave][digit[e]] : 0;
    rank[e]         = so_far + ahead;
    meet_in_wave();
    if (in && ahead == 0) count[wave][digit[e]] = static_cast<uint16_t>(so_far + __popcll(same));
    meet_in_wave();
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < digits) {
    int sum = 0;
    for (int w = 0; w < kSortWaves; w++) {
      const int c               = count[w][threadIdx.x];
      count[w][threadIdx.x]     = static_cast<uint16_t>(sum);
      sum += c;
    }
  }
  __syncthreads();
  for (int e = 0; e < kSortEach; e++) {
    const int64_t i = begin + e * 64 + lane;
    if (i >= n) continue;
    const int64_t to = static_cast<int64_t>(first[digit[e]]) + count[wave][digit[e]] + rank[e];
    out.key[to]      = key[e];
    out.place[to]    = places != nullptr ? places[i] : static_cast<int32_t>(i);
  }
}

// ---- sums of runs -----------------------------------------------------------------------------------

struct RunArgs {
  const void* grad;
  Sorted sorted;
  int n_tokens, n_rows;
  int words;   // of a row
  int chunk;   // sorted places of a wave, at most 64
  int slices;  // of 64 words
  float scale;
  void* out;
  int add;     // to what `out` holds
  unsigned clears;  // workgroups that clear rows without a token
  float* part; // [chunks][2][words * values]: of the run that began before the chunk, of the run that goes on after it
};

template <int kDtype, int kBytes>
__device__ __forceinline__ void write_row(const RunArgs& a, int row, int at, const float (&sum)[Pack<kDtype, kBytes>::kValues])
{
  using P    = Pack<kDtype, kBytes>;
  using Word = typename P::Word;
  Word* to   = static_cast<Word*>(a.out) + static_cast<int64_t>(row) * a.words + at;
  float x[P::kValues];
  if (a.add) {
    P::unpack(*to, x);
#pragma unroll
    for (int e = 0; e < P::kValues; e++) x[e] += scaled(sum[e], a.scale);
  } else {
#pragma unroll
    for (int e = 0; e < P::kValues; e++) x[e] = scaled(sum[e], a.scale);
  }
  *to = P::pack(x);
}

// Zeros for the rows that no token names: a workgroup looks up 64 rows in the sorted tokens and clears those that are absent.
constexpr int kClearRows = 64;
template <class Word>
__device__ __forceinline__ void clear_rows(const RunArgs& a, int64_t group)
{
  const int64_t first = group * kClearRows;
  const int64_t row   = first + (threadIdx.x & 63);
  int lo = 0, hi = a.n_tokens;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.sorted.key[mid] < row) lo = mid + 1;
    else hi = mid;
  }
  const uint64_t absent = __ballot(row < a.n_rows && !(lo < a.n_tokens && a.sorted.key[lo] == row));
  for (int r = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r < kClearRows; r += kRowWaves)
    if ((absent >> r) & 1) {
      Word* to = static_cast<Word*>(a.out) + (first + r) * a.words;
      for (int i = threadIdx.x & 63; i < a.words; i += 64) to[i] = Word{};
    }
}

template <int kDtype, int kBytes>
__global__ void __launch_bounds__(kRowThreads) sum_runs_kernel(const RunArgs a)
{
  using P    = Pack<kDtype, kBytes>;
  using Word = typename P::Word;
  // (the first workgroups clear: they are writes alone, and those that add are mostly reads)
  if (blockIdx.x < a.clears) {
    clear_rows<Word>(a, blockIdx.x);
    return;
  }
  const int lane      = threadIdx.x & 63;
  const int64_t task  = static_cast<int64_t>(blockIdx.x - a.clears) * kRowWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t chunk = task / a.slices;
  const int at        = static_cast<int>(task % a.slices) * 64 + lane;
  const int64_t p0    = chunk * a.chunk;
  if (p0 >= a.n_tokens) return;
  const int count = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.n_tokens - p0));
  // lane l has the token and place of entry l; a run ends where the next entry has another token
  const int key    = lane < count ? a.sorted.key[p0 + lane] : a.n_rows;
  const int place  = lane < count ? a.sorted.place[p0 + lane] : 0;
  const int before = p0 > 0 ? a.sorted.key[p0 - 1] : -1;
  const int after  = p0 + count < a.n_tokens ? a.sorted.key[p0 + count] : -1;
  const int below  = __shfl_down(key, 1);  // (by all lanes: what a lane reads from has to take part)
  const int next   = lane + 1 < count ? below : after;
  const uint64_t ends = __ballot(lane < count && key != next);
  const bool inside   = at < a.words;
  float sum[P::kValues];
#pragma unroll
  for (int e = 0; e < P::kValues; e++) sum[e] = 0.f;
  constexpr int kAhead = 8;  // rows asked for together
  int begin = 0;             // of the run
  for (int i = 0; i < count; i += kAhead) {
    Word w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int from = __builtin_amdgcn_readlane(place, min(i + j, count - 1));
      if (inside) w[j] = static_cast<const Word*>(a.grad)[static_cast<int64_t>(from) * a.words + at];
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (i + j >= count) break;
      float x[P::kValues];
      P::unpack(w[j], x);
#pragma unroll
      for (int e = 0; e < P::kValues; e++) sum[e] += x[e];
      const bool end = (ends >> (i + j)) & 1;
      if (!end && i + j + 1 < count) continue;
      const int row    = __builtin_amdgcn_readlane(key, i + j);
      const bool early = begin == 0 && before == row;  // began in an earlier chunk
      if (row < a.n_rows && inside) {
        if (end && !early) {
          write_row<kDtype, kBytes>(a, row, at, sum);
        } else {
          float* to = a.part + ((chunk * 2 + (early ? 0 : 1)) * a.words + at) * P::kValues;
#pragma unroll
          for (int e = 0; e < P::kValues; e++) to[e] = sum[e];
        }
      }
#pragma unroll
      for (int e = 0; e < P::kValues; e++) sum[e] = 0.f;
      begin = i + j + 1;
    }
  }
}

// Runs that cross the end of a chunk: the wave of the chunk in which one begins adds up its parts, one that reaches over 64 chunks
// and more the 16 waves of its workgroup together. (65536 places of 64 floats that are all alike: 359 us for one wave.)
constexpr int kJoinThreads = 1024, kJoinWaves = kJoinThreads / 64;
template <int kDtype, int kBytes>
__global__ void __launch_bounds__(kJoinThreads) join_runs_kernel(const RunArgs a)
{
  using P = Pack<kDtype, kBytes>;
  __shared__ int64_t heads_of[kJoinWaves];
  __shared__ float part[kJoinWaves][P::kValues][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t stride = static_cast<int64_t>(a.words) * P::kValues;
  float sum[P::kValues];
  // adds the heads begin .. end - 1 of the chunks after `chunk`
  auto add_heads = [&](int64_t chunk, int at, int64_t begin, int64_t end) {
    const float* from = a.part + (chunk + 1 + begin) * 2 * stride + static_cast<int64_t>(min(at, a.words - 1)) * P::kValues;
    constexpr int kAhead = 8;
    for (int64_t i = begin; i < end; i += kAhead, from += kAhead * 2 * stride) {
      float x[kAhead][P::kValues];
#pragma unroll
      for (int j = 0; j < kAhead; j++)
#pragma unroll
        for (int e = 0; e < P::kValues; e++) x[j][e] = from[min(static_cast<int64_t>(j), end - 1 - i) * 2 * stride + e];
#pragma unroll
      for (int j = 0; j < kAhead; j++)
#pragma unroll
        for (int e = 0; e < P::kValues; e++) sum[e] += i + j < end ? x[j][e] : 0.f;
    }
  };
  auto begin_sum = [&](int64_t chunk, int at, bool tail) {  // with the part at the tail of the chunk, where the run begins
#pragma unroll
    for (int e = 0; e < P::kValues; e++)
      sum[e] = tail && at < a.words ? a.part[(chunk * 2 + 1) * stride + static_cast<int64_t>(at) * P::kValues + e] : 0.f;
  };
  const int64_t first_task = static_cast<int64_t>(blockIdx.x) * kJoinWaves;
  const int64_t chunk = (first_task + wave) / a.slices, p0 = chunk * a.chunk, p1 = p0 + a.chunk;
  int64_t heads = 0;
  if (p1 < a.n_tokens) {
    const int row = a.sorted.key[p1 - 1];
    // (a run that began earlier is another chunk's)
    if (row < a.n_rows && a.sorted.key[p1] == row && !(p0 > 0 && a.sorted.key[p0 - 1] == row)) {
      // how many chunks begin with this token, found 64 at a time from steps of `step` chunks down to single ones
      auto in_run = [&](int64_t head) {
        const int64_t p = p1 + head * a.chunk;
        return p < a.n_tokens && a.sorted.key[min(p, static_cast<int64_t>(a.n_tokens) - 1)] == row;
      };
      auto reach = [&](int64_t from, int64_t step) {  // the lanes' first that is no longer in the run
        const uint64_t same = __ballot(in_run(from + lane * step));
        return same == ~uint64_t(0) ? 64 : __builtin_ctzll(~same);
      };
      heads = reach(0, 1);
      if (heads < 64) {
        const int at = static_cast<int>((first_task + wave) % a.slices) * 64 + lane;
        begin_sum(chunk, at, true);
        add_heads(chunk, at, 0, heads);
        if (at < a.words) write_row<kDtype, kBytes>(a, row, at, sum);
        heads = 0;
      } else {
        int64_t step = 64;
        while (step * 64 * a.chunk < a.n_tokens) step *= 64;
        heads = 0;
        for (; step > 0; step /= 64) heads += (reach(heads, step) - 1) * step;  // (head `heads` is in the run)
        heads += 1;
      }
    }
  }
  if (lane == 0) heads_of[wave] = heads;
  if (!__syncthreads_or(heads != 0)) return;
  for (int w = 0; w < kJoinWaves; w++) {
    const int64_t all = heads_of[w];
    if (all == 0) continue;
    const int64_t of = (first_task + w) / a.slices;
    const int at     = static_cast<int>((first_task + w) % a.slices) * 64 + lane;
    const int64_t share = (all + kJoinWaves - 1) / kJoinWaves;
    begin_sum(of, at, wave == 0);
    add_heads(of, at, min(wave * share, all), min((wave + 1) * share, all));
#pragma unroll
    for (int e = 0; e < P::kValues; e++) part[wave][e][lane] = sum[e];
    __syncthreads();
    if (wave == 0) {
      for (int v = 1; v < kJoinWaves; v++)
#pragma unroll
        for (int e = 0; e < P::kValues; e++) sum[e] += part[v][e][lane];
      if (at < a.words) write_row<kDtype, kBytes>(a, a.sorted.key[(of + 1) * a.chunk], at, sum);
    }
    __syncthreads();
  }
}

// ---- few places -----------------------------------------------------------------------------------------

// Few tokens need no sorting: a workgroup takes some rows of the table, lists the places that name one of them in ascending order,
// and its waves add up a row each; a long one, or one that more than 32 places name, is shared out among them afterwards. One launch.
constexpr int kDirectTokens = 2048, kDirectShared = 32, kDirectRows = 64;

template <int kDtype, int kBytes>
__global__ void __launch_bounds__(kRowThreads)
  direct_rows_kernel(const RunArgs a, const void* __restrict__ tokens, int token_bytes, int rows_each)
{
  using P    = Pack<kDtype, kBytes>;
  using Word = typename P::Word;
  __shared__ int list[kDirectTokens];  // row of the workgroup << 16 | place
  __shared__ int count[kRowWaves];
  enum { kAlone = 0, kBySlices = 1, kByPlaces = 2 };  // a row is one wave's; its slices, or the places that name it, are shared out
  __shared__ uint8_t shared[kDirectRows];
  __shared__ float part[kRowWaves][P::kValues][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = blockIdx.x * rows_each;
  int listed = 0;
  for (int base = 0; base < a.n_tokens; base += kRowThreads) {
    const int t    = base + threadIdx.x;
    const int row  = t < a.n_tokens ? token_at(tokens, token_bytes, t, a.n_rows) : a.n_rows;
    const bool in  = row < a.n_rows && row >= first && row < first + rows_each;
    const uint64_t set = __ballot(in);
    if (lane == 0) count[wave] = __popcll(set);
    __syncthreads();
    int at = listed;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) {
      at += w < wave ? count[w] : 0;
      listed += count[w];
    }
    if (in) list[at + __popcll(set & ((uint64_t(1) << lane) - 1))] = (row - first) << 16 | t;
    __syncthreads();
  }
  listed = __builtin_amdgcn_readfirstlane(listed);
  if (listed == 0) {
    if (a.add) return;
    Word* to          = static_cast<Word*>(a.out) + static_cast<int64_t>(first) * a.words;
    const int64_t all = static_cast<int64_t>(min(rows_each, a.n_rows - first)) * a.words;
    for (int64_t i = threadIdx.x; i < all; i += kRowThreads) to[i] = Word{};
    return;
  }
  // adds the rows of the places l .. l_end - 1 of the list that name row r
  auto add_up = [&](int r, int l, int l_end, int at, float(&sum)[P::kValues]) {
    constexpr int kAhead = 8;
#pragma unroll
    for (int e = 0; e < P::kValues; e++) sum[e] = 0.f;
    for (; l < l_end; l += 64) {
      const int entry = l + lane < l_end ? list[l + lane] : -1;
      uint64_t same   = __ballot(entry >> 16 == r);
      while (same != 0) {
        // (the last one again where there are no more: behind a branch the loads would be waited for one by one)
        Word w[kAhead];
        int found = 0, place = 0;
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          if (same != 0) {
            place = __builtin_amdgcn_readlane(entry, __builtin_ctzll(same)) & 0xffff;
            found++;
          }
          same &= same - 1;
          w[j] = static_cast<const Word*>(a.grad)[static_cast<int64_t>(place) * a.words + min(at, a.words - 1)];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          float x[P::kValues];
          P::unpack(w[j], x);
#pragma unroll
          for (int e = 0; e < P::kValues; e++) sum[e] += j < found ? x[e] : 0.f;
        }
      }
    }
  };
  for (int r = wave; r < rows_each && first + r < a.n_rows; r += kRowWaves) {
    int named = 0;
    for (int l = 0; l < listed; l += 64) named += __popcll(__ballot(l + lane < listed && list[min(l + lane, kDirectTokens - 1)] >> 16 == r));
    const int how = named == 0                                            ? kAlone
                    : named > kDirectShared && a.slices < kRowWaves ? kByPlaces
                    : a.slices > 1                                        ? kBySlices
                                                                          : kAlone;
    if (lane == 0) shared[r] = static_cast<uint8_t>(how);
    if (how != kAlone) continue;
    if (named == 0) {
      if (!a.add) {
        Word* to = static_cast<Word*>(a.out) + static_cast<int64_t>(first + r) * a.words;
        for (int i = lane; i < a.words; i += 64) to[i] = Word{};
      }
      continue;
    }
    float sum[P::kValues];
    add_up(r, 0, listed, lane, sum);
    if (lane < a.words) write_row<kDtype, kBytes>(a, first + r, lane, sum);
  }
  __syncthreads();
  const int share = ((listed + 63) / 64 + kRowWaves - 1) / kRowWaves * 64;
  const int begin = min(wave * share, listed), end = min(begin + share, listed);
  for (int r = 0; r < rows_each && first + r < a.n_rows; r++) {
    const int how = __builtin_amdgcn_readfirstlane(shared[r]);
    if (how == kAlone) continue;
    for (int slice = how == kBySlices ? wave : 0; slice < a.slices; slice += how == kBySlices ? kRowWaves : 1) {
      const int at = slice * 64 + lane;
      float sum[P::kValues];
      add_up(r, how == kBySlices ? 0 : begin, how == kBySlices ? listed : end, at, sum);
      if (how == kByPlaces) {
#pragma unroll
        for (int e = 0; e < P::kValues; e++) part[wave][e][lane] = sum[e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
          for (int w = 1; w < kRowWaves; w++)
#pragma unroll
            for (int e = 0; e < P::kValues; e++) sum[e] += part[w][e][lane];
        }
        __syncthreads();
      }
      if ((how == kBySlices || wave == 0) && at < a.words) write_row<kDtype, kBytes>(a, first + r, at, sum);
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------

// At most this many are sorted by counting: 3000 places of 256 bfloat16 take 20 us in all, 31 by digits; 8192 33 and 39.
constexpr int kCountSortTokens = 8192;
// Without sorting where one workgroup can add up all that is there, should it belong to one row. (2048 places of 256 bfloat16: 7 us,
// 56 if they are all alike; with one place more, sorted, 16 and 40.)
bool direct(int64_t n_tokens, int64_t row_bytes) { return n_tokens <= kDirectTokens && n_tokens * row_bytes <= (1 << 20); }

int value_bytes(int dtype) { return dtype == LBT_F32 ? 4 : 2; }

// Bytes of a row that a lane takes: 16 or 4 where rows are whole numbers of them, else one value.
int lane_bytes(int n_features, int dtype)
{
  const int64_t row = static_cast<int64_t>(n_features) * value_bytes(dtype);
  return row % 16 == 0 ? 16 : row % 4 == 0 ? 4 : 2;
}

struct EmbedCall {
  int64_t n_tokens;
  int n_features, n_rows, dtype;
  int bytes, words, slices, chunk, bits, passes, each;
  int64_t chunks, blocks;
  Sorted sorted[2];
  int32_t* counts;
  float* part;

  EmbedCall(int64_t t, int f, int rows, int type) : n_tokens(t), n_features(f), n_rows(rows), dtype(type)
  {
    bytes  = lane_bytes(f, type);
    words  = static_cast<int>(static_cast<int64_t>(f) * value_bytes(type) / bytes);
    slices = (words + 63) / 64;
    // chunks as long as they may be while there are some thousands of waves (1000000 places of 64 bfloat16: 158 us, 260 in chunks of 8;
    // 3000 places of 256: 20 us, 33 in chunks of 64)
    chunk = 64;
    while (chunk > 8 && (t / chunk) * slices < 4096) chunk /= 2;
    chunks = (t + chunk - 1) / chunk;
    // entries of a thread of the sort: one while the blocks are few, as a block is a CU's work (130000 places of 64 bfloat16: 56 us and
    // 63 with four; 200000 places 89 and 74)
    each   = t <= 131072 ? 1 : 4;
    blocks = (t + kSortThreads * each - 1) / (kSortThreads * each);
    bits   = 1;
    while ((int64_t(1) << bits) <= rows) bits++;  // keys go up to n_rows
    passes = (bits + 9) / 10;
  }

  void carve(Arena& arena)
  {
    for (int i = 0; i < 2; i++) {
      sorted[i].key   = arena.take<int32_t>(n_tokens);
      sorted[i].place = arena.take<int32_t>(n_tokens);
    }
    counts = arena.take<int32_t>(static_cast<size_t>(kDigits) * blocks);
    part   = arena.take<float>(static_cast<size_t>(chunks) * 2 * n_features);
  }
};

template <int kDtype, int kBytes>
int embed_gradient(hipStream_t s, const EmbedCall& c, const void* grad, const void* tokens, int token_bytes, float scale, bool add,
                   void* out)
{
  int at = 0;
  RunArgs a{grad,  c.sorted[0], static_cast<int>(c.n_tokens), c.n_rows, c.words, c.chunk, c.slices, scale, out, add ? 1 : 0, 0,
            c.part};
  if (direct(c.n_tokens, static_cast<int64_t>(c.words) * kBytes)) {
    int each = kDirectRows;  // rows of a workgroup: fewer where that gives too few workgroups
    while (each > 4 && c.n_rows / each < 2048) each /= 2;
    direct_rows_kernel<kDtype, kBytes><<<static_cast<unsigned>((static_cast<int64_t>(c.n_rows) + each - 1) / each), kRowThreads, 0, s>>>(
      a, tokens, token_bytes, each);
    LBT_HIP(hipGetLastError());
    return LBT_OK;
  }
  if (c.n_tokens <= kCountSortTokens) {
    count_sort_kernel<<<static_cast<unsigned>((c.n_tokens + 63) / 64), kSortThreads, 0, s>>>(
      tokens, token_bytes, static_cast<int>(c.n_tokens), c.n_rows, c.sorted[0]);
  } else {
    const int width = (c.bits + c.passes - 1) / c.passes;  // bits of a digit
    for (int p = 0; p < c.passes; p++) {
      const int shift     = p * width, bits = std::min(width, c.bits - shift);
      const int32_t* keys = p == 0 ? nullptr : c.sorted[at].key;
      const int32_t* from = p == 0 ? nullptr : c.sorted[at].place;
      const Sorted to     = c.sorted[1 - at];
      const unsigned grid = static_cast<unsigned>(c.blocks);
      auto pass = [&](auto entries) {
        constexpr int kEach = decltype(entries)::value;
        digit_count_kernel<kEach><<<grid, kSortThreads, 0, s>>>(tokens, token_bytes, keys, c.n_tokens, c.n_rows, shift, 1 << bits, c.counts);
        // each block adds up the counts for itself (500000 places: 90 us; 101 with a launch for it)
        const bool own = c.blocks <= 128;
        if (!own) digit_offsets_kernel<<<1, kSortThreads, 0, s>>>(1 << bits, static_cast<int>(c.blocks), c.counts);
        digit_move_kernel<kEach><<<grid, kSortThreads, 0, s>>>(tokens, token_bytes, keys, from, c.n_tokens, c.n_rows, shift, bits, c.counts,
                                                               own ? static_cast<int>(c.blocks) : 0, to);
      };
      if (c.each == 1) pass(std::integral_constant<int, 1>{});
      else pass(std::integral_constant<int, 4>{});
      at = 1 - at;
    }
  }
  LBT_HIP(hipGetLastError());
  a.sorted = c.sorted[at];
  if (!add) a.clears = static_cast<unsigned>((static_cast<int64_t>(c.n_rows) + kClearRows - 1) / kClearRows);
  const int64_t grid = (c.chunks * c.slices + kRowWaves - 1) / kRowWaves;
  LBT_REQUIRE(grid <= most_groups(kRowThreads), "too many elements");
  if (grid + a.clears > most_groups(kRowThreads)) {  // (only with a thousand million rows) the clears have a launch of their own
    sum_runs_kernel<kDtype, kBytes><<<a.clears, kRowThreads, 0, s>>>(a);
    LBT_HIP(hipGetLastError());
    a.clears = 0;
  }
  sum_runs_kernel<kDtype, kBytes><<<static_cast<unsigned>(grid + a.clears), kRowThreads, 0, s>>>(a);
  LBT_HIP(hipGetLastError());
  if (c.chunks > 1) {
    join_runs_kernel<kDtype, kBytes><<<static_cast<unsigned>((c.chunks * c.slices + kJoinWaves - 1) / kJoinWaves), kJoinThreads, 0, s>>>(a);
    LBT_HIP(hipGetLastError());
  }
  return LBT_OK;
}

bool embed_shape(int64_t n_tokens, int32_t n_features, int32_t n_rows, int32_t dtype)
{
  return (dtype == LBT_F32 || dtype == LBT_BF16 || dtype == LBT_F16) && n_tokens >= 0 && n_tokens <= (1 << 30) &&
         n_features >= 1 && n_features <= (1 << 24) && n_rows >= 1 && n_rows <= (1 << 30) - 64 &&
         n_tokens * n_features < (int64_t(1) << 38) && int64_t(n_rows) * n_features < (int64_t(1) << 38);
}

// Calls `f` with the type and the bytes of a lane as constants.
template <class F>
int for_type(int dtype, int bytes, const F& f)
{
  using std::integral_constant;
  if (dtype == LBT_F32)
    return bytes == 16 ? f(integral_constant<int, LBT_F32>{}, integral_constant<int, 16>{})
                       : f(integral_constant<int, LBT_F32>{}, integral_constant<int, 4>{});
  if (dtype == LBT_BF16)
    return bytes == 16  ? f(integral_constant<int, LBT_BF16>{}, integral_constant<int, 16>{})
           : bytes == 4 ? f(integral_constant<int, LBT_BF16>{}, integral_constant<int, 4>{})
                        : f(integral_constant<int, LBT_BF16>{}, integral_constant<int, 2>{});
  return bytes == 16  ? f(integral_constant<int, LBT_F16>{}, integral_constant<int, 16>{})
         : bytes == 4 ? f(integral_constant<int, LBT_F16>{}, integral_constant<int, 4>{})
                      : f(integral_constant<int, LBT_F16>{}, integral_constant<int, 2>{});
}

}  // namespace
}  // namespace lbt

extern "C" {

int lbt_embed_rows(void* stream, const void* table, int32_t dtype, int32_t n_rows, int32_t n_features, const void* tokens,
                   int32_t token_bytes, int64_t n_tokens, float scale, void* out)
{
  LBT_REQUIRE(dtype == LBT_F32 || dtype == LBT_BF16 || dtype == LBT_F16, "unsupported dtype %d", dtype);
  LBT_REQUIRE(lbt::embed_shape(n_tokens, n_features, n_rows, dtype), "bad shape");
  LBT_REQUIRE(token_bytes == 4 || token_bytes == 8, "tokens of 4 or 8 bytes, not %d", token_bytes);
  if (n_tokens == 0) return LBT_OK;
  LBT_REQUIRE(table && tokens && out, "null pointer");
  LBT_REQUIRE(((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
              "table and out must be 16-byte aligned");
  const int64_t row                = static_cast<int64_t>(n_features) * lbt::value_bytes(dtype);
  const lbt::MemoryRange ranges[] = {{out, n_tokens * row}, {table, n_rows * row}, {tokens, n_tokens * token_bytes}};
  LBT_REQUIRE(lbt::ranges_apart(ranges, 1, 3), "out may not overlap the table or the tokens");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const lbt::EmbedCall c(n_tokens, n_features, n_rows, dtype);
  lbt::ProfScope ps(LBT_PROF_OTHER, s);
  return lbt::for_type(dtype, c.bytes, [&](auto type, auto bytes) -> int {
    auto launch = [&](auto lanes) -> int {
      constexpr int kLanes = decltype(lanes)::value, kRows = lbt::kRowThreads / kLanes;
      constexpr int64_t kMost = int64_t(1) << 22;  // workgroups of a launch: 2^24 of them would be too many threads
      for (int64_t t = 0; t < n_tokens; t += kMost * kRows) {
        const int64_t some = std::min(n_tokens - t, kMost * kRows);
        lbt::embed_rows_kernel<decltype(type)::value, decltype(bytes)::value, kLanes>
          <<<static_cast<unsigned>((some + kRows - 1) / kRows), lbt::kRowThreads, 0, s>>>(
            table, n_rows, c.words, static_cast<const char*>(tokens) + t * token_bytes, token_bytes, some, scale, static_cast<char*>(out) + t * row);
        LBT_HIP(hipGetLastError());
      }
      return LBT_OK;
    };
    // a wave takes a row, or a part of one a short row; 4 words of a lane at a time (200000 rows of 32 bfloat16: 5.3 us, by whole waves 34;
    // 100000 rows of 256: 16.5 and 21)
    if (c.words > 64) LBT_TRY(launch(std::integral_constant<int, 64>{}));
    else if (c.words > 8) LBT_TRY(launch(std::integral_constant<int, 16>{}));
    else LBT_TRY(launch(std::integral_constant<int, 4>{}));
    return LBT_OK;
  });
}

size_t lbt_embed_rows_gradient_workspace_bytes(int64_t n_tokens, int32_t n_features, int32_t n_rows, int32_t dtype)
{
  if (!lbt::embed_shape(n_tokens, n_features, n_rows, dtype)) return 0;
  lbt::EmbedCall c(n_tokens, n_features, n_rows, dtype);
  lbt::Arena arena;
  arena.measure = true;
  c.carve(arena);
  return std::max<size_t>(arena.used, 256);
}

int lbt_embed_rows_gradient(void* stream, const void* grad, int32_t dtype, const void* tokens, int32_t token_bytes,
                            int64_t n_tokens, int32_t n_features, int32_t n_rows, float scale, int32_t add, void* grad_table,
                            void* workspace, size_t workspace_bytes)
{
  LBT_REQUIRE(dtype == LBT_F32 || dtype == LBT_BF16 || dtype == LBT_F16, "unsupported dtype %d", dtype);
  LBT_REQUIRE(lbt::embed_shape(n_tokens, n_features, n_rows, dtype), "bad shape");
  LBT_REQUIRE(token_bytes == 4 || token_bytes == 8, "tokens of 4 or 8 bytes, not %d", token_bytes);
  if (n_tokens == 0 && add) return LBT_OK;
  LBT_REQUIRE(grad_table && (n_tokens == 0 || (grad && tokens)), "null pointer");
  LBT_REQUIRE(((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(grad_table)) & 15) == 0,
              "grad and grad_table must be 16-byte aligned");
  const int64_t row                = static_cast<int64_t>(n_features) * lbt::value_bytes(dtype);
  const lbt::MemoryRange ranges[] = {{workspace, static_cast<int64_t>(workspace_bytes)}, {grad_table, n_rows * row}, {grad, n_tokens * row},
                                     {tokens, n_tokens * token_bytes}};
  LBT_REQUIRE(lbt::ranges_apart(ranges, 2, 4), "grad_table and workspace may not overlap the inputs or one another");
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    lbt::set_error("a workspace aligned to 16 bytes is needed");
    return LBT_ERR_WORKSPACE;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  lbt::EmbedCall c(n_tokens, n_features, n_rows, dtype);
  lbt::Arena arena;
  arena.base = static_cast<char*>(workspace);
  arena.cap  = workspace_bytes;
  c.carve(arena);
  if (arena.failed) {
    lbt::set_error("workspace of %zu bytes, %zu needed", workspace_bytes, arena.used);
    return LBT_ERR_WORKSPACE;
  }
  lbt::ProfScope ps(LBT_PROF_OTHER, s);
  return lbt::for_type(dtype, c.bytes, [&](auto type, auto bytes) {
    return lbt::embed_gradient<decltype(type)::value, decltype(bytes)::value>(s, c, grad, tokens, token_bytes, scale, add != 0,
                                                                              grad_table);
  });
}

}  // extern "C"
