/*
 * expert_kernels.hip - rows sorted by expert and back (cutt_rows.h): the stable counting sort of a router's
 * choices, the move of the tokens' rows to their experts, the weighted sum back, and the gradients of both.
 *
 * Times in the comments: MI355X, back to back in a graph, the buffers of several calls in rotation unless they say "the same buffers"; a launch
 * of an empty kernel takes about 2.2 us there, this library's copy of 512 MiB runs at 6.4 TB/s, torch's at 5.3.
 */
#include <algorithm>

#include "row_device.h"
#include "row_layer.h"

using namespace cutt;

namespace {

template <bool X>
using Is = std::integral_constant<bool, X>;
template <int X>
using Number = std::integral_constant<int, X>;

// ---------------------------------------------------------------------------
// Sort.  A stable counting sort: each workgroup places a stretch of neighbouring choices, choice a of expert e in row
//   first row of e + choices of e before the stretch + choices of e in the stretch before a.
// It needs to know how many choices each expert has in all and before the stretch.  Few choices: every workgroup counts all of them (COUNTED =
// false, one launch).  Many: a first launch counts stretch by stretch into the workspace, [stretch][experts, rounded up to 4], and a
// workgroup adds the columns up.  Whole numbers only: the order of the LDS atomics does not show.
//
// Bound by launches and latencies, not by its bytes (262144 choices are 4 MB, under 1 us): the choices, the table, the scan over the
// experts and the scattered 4-byte stores of `source` wait for each other.  512 choices 3.9 us (segments of 64
// rows; of single rows, in one workgroup, 4.6), 4096 5.4 (128 experts), 65536 8.3, 262144 11.7, 1048576
// 23.0 (256 experts, two launches); 262144 choices of 512 experts 13.6, of 1024 17.3.  Of the 11.7 (17.3) the sums over the table take 2.0 (6.7), matching
// 1.0 (1.2), the stores of `source` 1.2 (1.5).
// ---------------------------------------------------------------------------
constexpr uint32_t kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr uint32_t kCountLoads = 16;   // a workgroup's loads of the table go out at once: 262144 choices 11.7 us, of 1024 experts 17.3; 12.1 and 18.7 with 4
constexpr uint32_t kSortGroups = 256;  // at most: beyond, stretches get longer and the table does not grow
// Choices that every workgroup counts for itself.  8192 choices, 256 experts: 7.2 us so, 7.9 with the table, but 16.8 and 7.7 where all are one expert's
// and their LDS atomics follow each other.
constexpr uint32_t kCountAll = 4096;
// More workgroups for the rows that stay empty: 512 choices, 128 experts' segments in multiples of 64 rows, 5.1 us with one workgroup, 3.9 with 8.
constexpr uint32_t kRowsPerGroup = 1024, kRowGroups = 16;
// Choices that a lane places at a time: one up to the first number, two up to the second, four beyond.  More per lane are more steps in turn, fewer a
// longer table.  256 experts, us with one, two and four: 65536 choices 8.3, 8.8, 10.1; 98304 10.0, 9.4, 11.0; 262144 12.0, 11.8, 11.7 (of 1024 experts 21.9,
// 21.1, 17.3).
constexpr uint32_t kOneItem = 65536, kTwoItems = 131072;

struct SortPlan {
  uint32_t items;    // choices that a lane places at a time; a part is kSortThreads * items choices
  uint32_t stretch;  // choices per workgroup, whole parts
  uint32_t groups;
  bool counted;
  cuttHipDivisor byAlign;
};

// The expert of choice i among the `experts`, or `experts` if it is none of them.
template <typename Id>
__device__ __forceinline__ uint32_t expertOf(const cuttHipSortArgs& a, uint32_t i) {
  const uint64_t e = (uint64_t)(int64_t) static_cast<const Id*>(a.ids)[i] - (uint64_t)(int64_t)a.firstExpert;  // (wraps)
  return e < a.experts ? (uint32_t)e : a.experts;
}

template <typename Id>
__global__ __launch_bounds__(kSortThreads) void expertCountKernel(cuttHipSortArgs a, uint32_t stretch) {
  extern __shared__ uint32_t count[];  // [experts]
  const uint32_t E = a.experts;
  for (uint32_t e = threadIdx.x; e < E; e += kSortThreads) count[e] = 0;
  __syncthreads();
  const uint32_t from = blockIdx.x * stretch, to = min(from + stretch, a.n);
#pragma unroll 4
  for (uint32_t i = from + threadIdx.x; i < to; i += kSortThreads) {
    const uint32_t e = expertOf<Id>(a, i);
    if (e < E) atomicAdd(&count[e], 1u);
  }
  __syncthreads();
  const uint32_t pitch = (E + 3) / 4 * 4;
  for (uint32_t e = threadIdx.x; e < pitch; e += kSortThreads) a.workspace[(uint64_t)blockIdx.x * pitch + e] = e < E ? count[e] : 0;
}

// Lanes of the wavefront whose key is this lane's; keys have BITS bits.
template <int BITS>
__device__ __forceinline__ uint64_t sameKey(uint32_t key) {
  uint32_t low = ~0u, high = ~0u;
#pragma unroll
  for (int b = 0; b < BITS; b++) {
    const uint64_t set = __ballot((key >> b) & 1);
    const uint32_t other = (key >> b & 1) - 1;  // all ones where this lane's bit is clear
    low &= (uint32_t)set ^ other;
    high &= (uint32_t)(set >> 32) ^ other;
  }
  return (uint64_t)high << 32 | low;
}

// What the wavefront's lanes have written to LDS before is seen by its other lanes after.  LDS serves a wavefront's accesses in their order: this only
// keeps the compiler from changing it.
__device__ __forceinline__ void waveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename Id, bool COUNTED, int ITEMS, int BITS>
__global__ __launch_bounds__(kSortThreads) void expertSortKernel(cuttHipSortArgs a, SortPlan p) {
  constexpr uint32_t kSortItems = ITEMS, kSortPart = kSortThreads * ITEMS;
  const uint32_t stretch = p.stretch;
  extern __shared__ uint32_t lds[];
  const uint32_t E = a.experts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t* const next = lds;                    // [E + 1] choices before the stretch, then the row of an expert's next choice
  uint32_t* const all = next + E + 1;            // [E + 1] choices in all, then the row behind an expert's last choice
  uint32_t* const start = all + E + 1;           // [E + 1] an expert's first row
  uint32_t* const seen = start + E + 1;          // [waves][E + 1]
  __shared__ uint32_t waveSum[kSortWaves];
  const uint32_t from = blockIdx.x * stretch, to = min(from + stretch, a.n);

  // The stretch's first part, before anything is waited for.
  uint32_t expert[kSortItems];
  const auto take = [&](uint64_t part) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++) {
      const uint64_t i = part + (wave * kSortItems + j) * 64 + lane;
      expert[j] = i < to ? expertOf<Id>(a, (uint32_t)i) : E;
    }
  };
  take(from);
  for (uint32_t e = tid; e <= E; e += kSortThreads) next[e] = all[e] = 0;
  __syncthreads();
  if constexpr (COUNTED) {
    // A thread adds up four neighbouring experts over every `share`-th stretch, kCountLoads loads of 16 bytes in flight.
    const uint32_t quads = (E + 3) / 4, share = kSortThreads / quads, part = tid / quads, quad = tid - part * quads;
    uint32_t before[4] = {}, sum[4] = {};
    for (uint32_t first = part; part < share && first < gridDim.x; first += share * kCountLoads) {
      Vec<uint32_t, 4> c[kCountLoads];
#pragma unroll
      for (uint32_t u = 0; u < kCountLoads; u++)
        c[u] = *reinterpret_cast<const Vec<uint32_t, 4>*>(a.workspace + (uint64_t)min(first + u * share, gridDim.x - 1) * quads * 4 + quad * 4);
#pragma unroll
      for (uint32_t u = 0; u < kCountLoads; u++) {
        const uint32_t g = first + u * share;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          sum[x] += g < gridDim.x ? c[u][x] : 0;
          before[x] += g < blockIdx.x ? c[u][x] : 0;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 4; x++)
      if (part < share && quad * 4 + x < E) {
        atomicAdd(&next[quad * 4 + x], before[x]);
        atomicAdd(&all[quad * 4 + x], sum[x]);
      }
  } else if (gridDim.x == 1) {
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++)
      if (expert[j] < E) atomicAdd(&all[expert[j]], 1u);
  } else {
#pragma unroll 8
    for (uint32_t i = tid; i < a.n; i += kSortThreads) {
      const uint32_t e = expertOf<Id>(a, i);
      if (e < E) atomicAdd(&all[e], 1u);
      if (e < E && i < from) atomicAdd(&next[e], 1u);
    }
  }
  __syncthreads();

  // Experts' first rows: thread tid adds up experts 2 tid and 2 tid + 1 (CUTT_MAX_EXPERTS = 2 * kSortThreads).
  {
    uint32_t padded[2], sum = 0;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t e = 2 * tid + j;
      padded[j] = e < E ? divide(all[e] + a.align - 1, p.byAlign) * a.align : 0;
      sum += padded[j];
    }
    const uint32_t upTo = scanOverWave(sum, [](uint32_t x, uint32_t y) { return x + y; });
    if (lane == 63) waveSum[wave] = upTo;
    __syncthreads();
    uint32_t at = upTo - sum;
    for (uint32_t w = 0; w < wave; w++) at += waveSum[w];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t e = 2 * tid + j;
      if (e <= E) start[e] = at;
      if (e < E) {
        const uint32_t c = all[e];
        if (blockIdx.x == 0) a.counts[e] = (int32_t)c;
        all[e] = at + c;
        next[e] += at;
      }
      if (e <= E && blockIdx.x == 0) a.offsets[e] = (int32_t)at;
      at += padded[j];
    }
    if (2 * tid + 2 == E) {  // (the sum behind the last expert falls to nobody's pair when E = 2 * kSortThreads)
      start[E] = at;
      if (blockIdx.x == 0) a.offsets[E] = (int32_t)at;
    }
  }
  __syncthreads();

  // Rows without a choice: behind every expert's last one, and behind all experts.
  for (uint32_t e = blockIdx.x * kSortWaves + wave; e < E; e += gridDim.x * kSortWaves)
    for (uint64_t r = (uint64_t)all[e] + lane; r < start[e + 1] && r < a.rows; r += 64) a.source[r] = -1;
  for (uint64_t r = (uint64_t)start[E] + blockIdx.x * kSortThreads + tid; r < a.rows; r += (uint64_t)gridDim.x * kSortThreads) a.source[r] = -1;

  // The stretch, part by part.  A wavefront's choices of a part are neighbours, so that an expert's rows follow the order of the
  // wavefronts, in a wavefront that of its steps, and in a step that of the lanes.
  uint32_t* const mine = seen + wave * (E + 1);
  for (uint64_t part = from; part < to; part += kSortPart) {
    for (uint32_t e = lane; e <= E; e += 64) mine[e] = 0;
    waveFence();
    uint32_t rank[kSortItems];
    if (part != from) take(part);
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++) {
      const uint64_t same = sameKey<BITS>(expert[j]);
      const uint32_t below = __popcll(same & ((1ull << lane) - 1));
      const uint32_t before = mine[expert[j]];  // (the wavefront's lanes all read, then one lane per expert writes)
      waveFence();
      rank[j] = before + below;
      if (below == 0) mine[expert[j]] = before + __popcll(same);
      waveFence();
    }
    __syncthreads();
    for (uint32_t e = tid; e < E; e += kSortThreads) {
      uint32_t at = next[e];
#pragma unroll
      for (uint32_t w = 0; w < kSortWaves; w++) {
        const uint32_t c = seen[w * (E + 1) + e];
        seen[w * (E + 1) + e] = at;
        at += c;
      }
      next[e] = at;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++) {
      const uint64_t i = part + (wave * kSortItems + j) * 64 + lane;
      if (i >= to) continue;
      const uint32_t row = mine[expert[j]] + rank[j];
      const bool there = expert[j] < E && row < a.rows;
      a.position[i] = there ? (int32_t)row : -1;
      if (there) a.source[row] = (int32_t)i;
    }
    __syncthreads();
  }
}

SortPlan planSort(uint32_t n, uint32_t align, uint32_t rows) {
  SortPlan p;
  p.counted = n > kCountAll;
  p.items = n <= kOneItem ? 1 : n <= kTwoItems ? 2 : 4;
  const uint32_t part = kSortThreads * p.items;
  const uint64_t parts = n ? ((uint64_t)n + part - 1) / part : 1;
  const uint64_t perGroup = (parts + kSortGroups - 1) / kSortGroups;
  p.stretch = (uint32_t)(perGroup * part);
  p.groups = (uint32_t)((parts + perGroup - 1) / perGroup);
  if (!p.counted) p.groups = std::max(p.groups, std::min(rows / kRowsPerGroup, kRowGroups));  // (more, for the rows without a choice)
  p.byAlign = cuttHipMakeDivisor(align);
  return p;
}

// ---------------------------------------------------------------------------
// Rows to experts and back.  Sums of a few products per element of a row: all of it is bound by memory.  Every row is read once and written once (by the
// counters at most 2 % more HBM bytes than the algorithm's for rows on the 128-byte grid; 4 % more read off it, where two rows share a line), 16 bytes per
// lane at any alignment.  A workgroup takes a token and has a
// lane for every vector of its row, up to 1024: combine of 16 x 8 rows of 8192 bfloat16 5.7 us with 256 lanes, 4.7 with 512, 4.3 with 1024, of
// 8192 x 8 rows 217, 212, 208; dispatch of 256 x 8 rows 11.1 us with 512, 8.6 with 1024.  The gradient of combine needs more registers and takes 512 at most (16 x
// 8 rows 7.2 us, 7.6 with 1024), and so does dispatch past the caches (8192 x 8 rows 210 us, 215 with 1024).  Neighbouring tokens to the workgroups of one XCD: 208 -> 218 us for combine of 16384 x 8 rows, so the workgroups keep their order.
// ---------------------------------------------------------------------------
constexpr uint32_t kMaxRowThreads = 1024, kHalfRowThreads = 512;
constexpr uint32_t kMaxBlocks = 1u << 20;  // of tokens, and of empty rows: all lanes of a launch have to be fewer than 2^32
static_assert(2ull * kMaxBlocks * kMaxRowThreads <= CUTT_HIP_MAX_GRID_LANES, "a larger grid would be cut without an error");

// Rows without a source, which hold zeros.  Workgroup `block` of `blocks` looks at kEmptyRows rows at a time; a wavefront clears a row.  16384 x 8 rows of 512
// bfloat16, none empty: 34.1 us with 4 rows, 30.5 with 16, 31.6 with 32; 256 rows of 8320 not empty, 4096 wide: 13.1, 14.0, 15.0.
constexpr uint32_t kEmptyRows = 16;

template <typename T, int N, bool NT>
__device__ __forceinline__ void clearEmptyRows(const cuttHipExpertArgs& a, T* y, uint64_t stride, uint32_t block, uint32_t blocks) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  Pack<T, N> zero = {};
  for (uint64_t first = (uint64_t)block * kEmptyRows; first < a.rows; first += (uint64_t)blocks * kEmptyRows) {
    const uint64_t mine = first + (lane & (kEmptyRows - 1));
    uint64_t empty = __ballot(lane < kEmptyRows && mine < a.rows && a.source[mine] < 0);
    for (uint32_t n = 0; empty; n++) {
      const uint32_t r = __builtin_ctzll(empty);
      empty &= empty - 1;
      if (n % waves != wave) continue;
      T* const row = y + (first + r) * stride;
      for (uint32_t c = lane * N; c < a.width; c += 64 * N) zero.template store<NT>(row + min(c, a.width - N));
    }
  }
}

// B choices of a token from `first` on: their rows and weights.  Lane i loads choice i, so that one load brings them all; row(i) and weight(i)
// broadcast.  All lanes of the wavefront have to take part in making one and in the broadcasts, so the loops around them
// are the same for the whole wavefront: lanes beyond a row's end read its last vector again and are kept from storing.
// An absent row's number is that of a row that is there: the loads of all B can then go out back to back,
// without branches, and what an absent one brings is not used.
template <int B>
struct Choices {
  static_assert(B >= 1 && B <= 8, "a power of two of lanes holds them");
  uint32_t laneRow;
  float laneWeight;
  uint32_t there;  // bit i: choice i has a row

  __device__ __forceinline__ Choices(const cuttHipExpertArgs& a, uint32_t token, uint32_t first) {
    const uint32_t i = threadIdx.x & 7;
    const uint64_t at = (uint64_t)token * a.choices + min(first + i, a.choices - 1);
    laneRow = (uint32_t)a.position[at];
    laneWeight = 1.0f;
    if (a.weights) laneWeight = a.weights[at];
    const bool ok = i < B && first + i < a.choices && laneRow < a.rows;
    there = (uint32_t)__ballot(ok) & 0xff;
    const uint32_t some = __builtin_amdgcn_readlane(laneRow, there ? __builtin_ctz(there) : 0);
    if (!ok) laneRow = some, laneWeight = 0.0f;
  }
  __device__ __forceinline__ bool has(int i) const { return there >> i & 1; }
  __device__ __forceinline__ uint64_t row(int i) const { return (uint32_t)__builtin_amdgcn_readlane(laneRow, i); }
  __device__ __forceinline__ float weight(int i) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(laneWeight), i)); }
};

// The workgroup's wavefronts share a row's columns: wavefront w of W takes the columns w * 64 * N, (w + W) * 64 * N, ...
__device__ __forceinline__ uint32_t waveOfGroup() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// A workgroup reads a token's row once and stores it to every row that the token goes to; the last workgroups clear the empty rows.
// Rows are bytes here: any element size, any alignment.  16384 x 8 rows of 4096 bfloat16 and 8064 empty ones (1275 MB): 249 us, 216 with x left in
// the memory-side cache by whoever made it; rows that follow each other instead of the experts' order take the same time.  Row by row of y instead,
// a token's row read once per choice: 300 us.  Rows off the 128-byte grid are slower (65536 of 2002 bytes from memory 40 us, of 2048 bytes 32): two
// rows share a line; stores in windows on the grid, with a load of x per choice, make it 50 - 57, neighbouring tokens on one XCD 37, but
// aligned rows 2 - 3 % slower.
template <int N, bool NT>
__global__ __launch_bounds__(kMaxRowThreads) void dispatchKernel(cuttHipExpertArgs a, const uint8_t* x, uint64_t xStride, uint8_t* y, uint64_t yStride,
                                                                 uint32_t tokenBlocks) {
  if (blockIdx.x >= tokenBlocks) {
    clearEmptyRows<uint8_t, N, NT>(a, y, yStride, blockIdx.x - tokenBlocks, gridDim.x - tokenBlocks);
    return;
  }
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += tokenBlocks) {
    const uint8_t* const from = x + t * xStride;
    uint32_t col = waveOfGroup() * 64 * N;
    if (col >= a.width) continue;
    Pack<uint8_t, N> v;  // (asked for before the choices are waited for)
    v.load(from + min(col + lane * N, a.width - N));
    const Choices<8> begin(a, t, 0);
    for (;;) {
      const uint32_t base = col + lane * N, c = min(base, a.width - N);
      auto put = [&](const Choices<8>& ch) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (!ch.has(i)) continue;
          uint8_t* const to = y + ch.row(i) * yStride + c;
          if (base < a.width) v.template store<NT>(to);
        }
      };
      put(begin);
      for (uint32_t first = 8; first < a.choices; first += 8) put(Choices<8>(a, t, first));
      col += blockDim.x * N;
      if (col >= a.width) break;
      v.load(from + min(col + lane * N, a.width - N));
    }
  }
}

// A workgroup sums a token's rows, 16 bytes of each per lane, in 32 bits and in the order of the choices, with one rounding at the end.
// The loads of all choices are in flight together.  16384 x 8 rows of 4096 bfloat16 (1209 MB): 208 us, 5.8 TB/s; the gradient of dispatch
// of 8191 x 4 rows of 2050 floats (336 MB) 59 us.
template <typename T, int N, int B, bool NT>
__global__ __launch_bounds__(kMaxRowThreads) void combineKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, T* out, uint64_t outStride) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const Choices<B> begin(a, t, 0);
    for (uint32_t col = waveOfGroup() * 64 * N; col < a.width; col += blockDim.x * N) {
      const uint32_t base = col + lane * N, c = min(base, a.width - N);
      float sum[N] = {};
      auto add = [&](const Choices<B>& ch) __attribute__((always_inline)) {
        if (!ch.there) return;
        Pack<T, N> v[B];
#pragma unroll
        for (int i = 0; i < B; i++) v[i].template load<NT>(y + ch.row(i) * yStride + c);
#pragma unroll
        for (int i = 0; i < B; i++) {
          v[i].zeroUnless(ch.has(i));
          const float w = ch.weight(i);
#pragma unroll
          for (int e = 0; e < N; e++) sum[e] = fmaf(w, (float)v[i].get(e), sum[e]);
        }
      };
      add(begin);
      for (uint32_t first = B; first < a.choices; first += B) add(Choices<B>(a, t, first));
      Pack<T, N> o;
#pragma unroll
      for (int e = 0; e < N; e++) o.set(e, (T)sum[e]);
      if (base < a.width) o.store(out + t * outStride + c);
    }
  }
}

// Sums of B values over the wavefront: afterwards lane l holds the sum of value l / (64 / B).  Each step halves what a lane still holds.
template <int B>
__device__ __forceinline__ float sumOverWave(float (&v)[B]) {
  static_assert((B & (B - 1)) == 0, "halved step by step");
  const uint32_t lane = threadIdx.x & 63;
  uint32_t half = 32;
#pragma unroll
  for (int n = B / 2; n >= 1; n /= 2, half /= 2) {
    const bool upper = lane & half;
#pragma unroll
    for (int i = 0; i < n; i++) {
      const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor(give, half);
    }
  }
  float sum = v[0];
  for (; half >= 1; half /= 2) sum += __shfl_xor(sum, half);
  return sum;
}

// A workgroup takes a token: its gradient row is multiplied into the rows it came from, and with them.  The last workgroups clear the empty rows.
// The dot products are summed in 32 bits: a lane's columns, the lanes of a wavefront pairwise, the wavefronts in turn, always in the same order.
// 8192 x 8 rows of 4096 bfloat16 (1142 MB): 219 us, 5.2 TB/s, as much read as written; a wavefront per token, without LDS: 241 us; four choices at a
// time, for fewer registers and more wavefronts: 232.  With a tenth of the choices absent 219, the rows alone 141, the weights alone 99.  Few tokens are a chain of
// latencies (choices, rows, the sums over a wavefront and over the wavefronts): one token with 6 rows of 5120 halves 4.8 us, the rows alone 3.0, the weights alone
// 4.0; 256 such tokens 12.2, 7.2, 7.9.  Off the 128-byte grid 16384 x 8 rows of 2111 bfloat16 290 us, 4.1 TB/s.
template <typename T, int N, int B, bool ROWS, bool WEIGHTS, bool NT>
__global__ __launch_bounds__(kHalfRowThreads) void combineBackwardKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, const T* dout, uint64_t doutStride,
                                                                      T* dy, uint64_t dyStride, float* dweights, uint32_t tokenBlocks) {
  constexpr int P = B <= 1 ? 1 : B <= 2 ? 2 : B <= 4 ? 4 : 8;
  __shared__ float part[kHalfRowThreads / 64][P];
  if (ROWS && blockIdx.x >= tokenBlocks) {
    clearEmptyRows<T, N, NT>(a, dy, dyStride, blockIdx.x - tokenBlocks, gridDim.x - tokenBlocks);
    return;
  }
  const uint32_t wave = waveOfGroup(), lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += tokenBlocks)
    for (uint32_t first = 0; first < a.choices; first += B) {
      const Choices<B> ch(a, t, first);
      float dot[P] = {};
      for (uint32_t col = waveOfGroup() * 64 * N; ch.there && col < a.width; col += blockDim.x * N) {
        const uint32_t base = col + lane * N, c = min(base, a.width - N);
        Pack<T, N> g, v[B];
        g.template load<NT>(dout + t * doutStride + c);
        if (WEIGHTS)
#pragma unroll
          for (int i = 0; i < B; i++) v[i].template load<NT>(y + ch.row(i) * yStride + c);
        float grad[N];
#pragma unroll
        for (int e = 0; e < N; e++) grad[e] = (float)g.get(e);
        if (ROWS)
#pragma unroll
          for (int i = 0; i < B; i++)
            if (ch.has(i)) {
              const float w = ch.weight(i);
              T* const to = dy + ch.row(i) * dyStride + c;
              Pack<T, N> o;
#pragma unroll
              for (int e = 0; e < N; e++) o.set(e, (T)(w * grad[e]));
              if (base < a.width) o.template store<NT>(to);
            }
        if (WEIGHTS) {
          if (c != base)  // columns that the vector before it, or its row's last vector, has already counted
#pragma unroll
            for (int e = 0; e < N; e++)
              if (c + e < base) {
                grad[e] = 0;
#pragma unroll
                for (int i = 0; i < B; i++) v[i].set(e, T(0));
              }
#pragma unroll
          for (int i = 0; i < B; i++)
#pragma unroll
            for (int e = 0; e < N; e++) dot[i] = fmaf(grad[e], (float)v[i].get(e), dot[i]);
        }
      }
      if (!WEIGHTS) continue;
#pragma unroll
      for (int i = 0; i < B; i++) dot[i] = ch.has(i) ? dot[i] : 0.0f;
      const float sum = sumOverWave(dot);
      if (lane % (64 / P) == 0) part[wave][lane / (64 / P)] = sum;
      __syncthreads();
      if (threadIdx.x < B && first + threadIdx.x < a.choices) {
        float all = 0;
        for (uint32_t w = 0; w < blockDim.x / 64; w++) all += part[w][threadIdx.x];
        dweights[(uint64_t)t * a.choices + first + threadIdx.x] = all;
      }
      __syncthreads();
    }
}

constexpr uint64_t kMaxPiece = 1u << 30;  // bytes of a row that one launch of the dispatch kernel moves

uint32_t blocksFor(uint64_t n) { return (uint32_t)(n < kMaxBlocks ? n : kMaxBlocks); }
uint32_t emptyBlocks(uint32_t rows) { return blocksFor((rows + (uint64_t)kEmptyRows - 1) / kEmptyRows); }

}  // namespace

extern "C" size_t cuttHipSortWorkspace(uint32_t n, uint32_t experts) {
  const SortPlan p = planSort(n, 1, 0);
  return p.counted ? (size_t)p.groups * ((experts + 3) / 4 * 4) * 4 : 0;
}

namespace {

template <typename Id>
int sortBy(const cuttHipSortArgs* a, void* stream) {
  const SortPlan p = planSort(a->n, a->align, a->rows);
  const size_t perExpert = (size_t)(a->experts + 1) * 4, lds = (3 + kSortWaves) * perExpert;
  if (p.counted)
    if (int e = launchRows(expertCountKernel<Id>, p.groups, kSortThreads, perExpert, stream, *a, p.stretch)) return e;
  auto go = [&](auto counted, auto items) {  // (numbers up to `experts` itself, which stands for none of them)
    auto kernel = a->experts < 64 ? expertSortKernel<Id, counted, items, 6>
                                  : a->experts < 256 ? expertSortKernel<Id, counted, items, 8> : expertSortKernel<Id, counted, items, 11>;
    return launchRows(kernel, p.groups, kSortThreads, lds, stream, *a, p);
  };
  if (!p.counted) return go(Is<false>{}, Number<1>{});
  return p.items == 1 ? go(Is<true>{}, Number<1>{}) : p.items == 2 ? go(Is<true>{}, Number<2>{}) : go(Is<true>{}, Number<4>{});
}

}  // namespace

extern "C" int cuttHipExpertSort(const cuttHipSortArgs* a, void* stream) {
  return a->idBytes == 8 ? sortBy<int64_t>(a, stream) : sortBy<int32_t>(a, stream);
}

namespace {

// Lanes for rows of `width` elements, n per lane: one pass over a row if `most` lanes suffice.
uint32_t rowThreads(uint32_t width, uint32_t n, uint32_t most) {
  const uint64_t waves = ((uint64_t)width + 64 * n - 1) / (64 * n);
  return waves < most / 64 ? (uint32_t)waves * 64 : most;
}

// Rows on the 128-byte grid.  Off it, lines that two rows share have to meet in a cache: 65536 rows of 4100 bytes 69 us through the caches, 73 past them.
// So for dispatch, which only stores them; the gradient of combine, which reads as many, stores past the caches on the grid and off it: 65536 rows of 4100 bytes
// 133 us so, 144 with stores through the caches, 138 with all of it through them; 131072 of 4222 bytes 290, 298, 299.  Combine's reads of the same rows: 57 us
// past and 60 through, 129 and 123.
bool onLines(const void* p, uint64_t strideBytes) { return ((uintptr_t)p | strideBytes) % 128 == 0; }

}  // namespace

extern "C" int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t elemSize, const void* x, uint64_t xStride, void* y, uint64_t yStride, void* stream) {
  const uint64_t bytes = (uint64_t)a->width * elemSize;
  const uint32_t tokenBlocks = blocksFor(a->tokens);
  const dim3 grid(tokenBlocks + emptyBlocks(a->rows));
  // (a launch's offsets in a row have 32 bits: longer rows go piece by piece)
  for (uint64_t at = 0; at < bytes; at += kMaxPiece) {
    cuttHipExpertArgs b = *a;
    b.width = (uint32_t)(bytes - at < kMaxPiece ? bytes - at : kMaxPiece);
    const bool nt = pastCaches(a->rows, bytes) && onLines(y, yStride * elemSize);
    auto kernel = b.width < 16 ? dispatchKernel<1, false> : nt ? dispatchKernel<16, true> : dispatchKernel<16, false>;
    const uint32_t threads = rowThreads(b.width, b.width < 16 ? 1 : 16, nt ? kHalfRowThreads : kMaxRowThreads);
    if (int e = launchRows(kernel, grid, threads, 0, stream, b, (const uint8_t*)x + at, xStride * elemSize, (uint8_t*)y + at, yStride * elemSize, tokenBlocks))
      return e;
  }
  return 0;
}

namespace {

template <typename T, int N>
int combine(const cuttHipExpertArgs* a, const T* y, uint64_t yStride, T* out, uint64_t outStride, bool nt, void* stream) {
  auto go = [&](auto kernel) { return launchRows(kernel, blocksFor(a->tokens), rowThreads(a->width, N, kMaxRowThreads), 0, stream, *a, y, yStride, out, outStride); };
  if constexpr (N == 1) {
    return go(combineKernel<T, 1, 1, false>);
  } else {
    auto withChoices = [&](auto b) { return nt ? go(combineKernel<T, N, b, true>) : go(combineKernel<T, N, b, false>); };
    switch (a->choices) {
      case 1: return withChoices(Number<1>{});
      case 2: return withChoices(Number<2>{});
      case 3: return withChoices(Number<3>{});
      case 4: return withChoices(Number<4>{});
      case 5: return withChoices(Number<5>{});
      case 6: return withChoices(Number<6>{});
      case 7: return withChoices(Number<7>{});
      default: return withChoices(Number<8>{});
    }
  }
}

template <typename T>
int combineRows(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  constexpr int N = 16 / sizeof(T);
  const bool nt = pastCaches(a->rows, a->width * sizeof(T));
  if (a->width < N) return combine<T, 1>(a, (const T*)y, yStride, (T*)out, outStride, false, stream);
  return combine<T, N>(a, (const T*)y, yStride, (T*)out, outStride, nt, stream);
}

template <typename T, int N>
int combineBackward(const cuttHipExpertArgs* a, const T* y, uint64_t yStride, const T* dout, uint64_t doutStride, T* dy, uint64_t dyStride, float* dweights,
                    bool nt, void* stream) {
  const uint32_t tokenBlocks = blocksFor(a->tokens);
  auto go = [&](auto kernel) {
    return launchRows(kernel, tokenBlocks + (dy ? emptyBlocks(a->rows) : 0), rowThreads(a->width, N, kHalfRowThreads), 0, stream, *a, y, yStride, dout, doutStride, dy,
                      dyStride, dweights, tokenBlocks);
  };
  if constexpr (N == 1) {
    if (!dy) return go(combineBackwardKernel<T, 1, 1, false, true, false>);
    if (!dweights) return go(combineBackwardKernel<T, 1, 1, true, false, false>);
    return go(combineBackwardKernel<T, 1, 1, true, true, false>);
  } else {
    if (!dy) {
      auto withChoices = [&](auto b) { return nt ? go(combineBackwardKernel<T, N, b, false, true, true>) : go(combineBackwardKernel<T, N, b, false, true, false>); };
      return a->choices > 4 ? withChoices(Number<8>{}) : withChoices(Number<4>{});
    }
    if (!dweights) return nt ? go(combineBackwardKernel<T, N, 8, true, false, true>) : go(combineBackwardKernel<T, N, 8, true, false, false>);
    auto withChoices = [&](auto b) { return nt ? go(combineBackwardKernel<T, N, b, true, true, true>) : go(combineBackwardKernel<T, N, b, true, true, false>); };
    switch (a->choices) {
      case 1:
      case 2: return withChoices(Number<2>{});
      case 3:
      case 4: return withChoices(Number<4>{});
      case 5:
      case 6: return withChoices(Number<6>{});
      default: return withChoices(Number<8>{});
    }
  }
}

template <typename T>
int combineRowsBackward(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride, void* dy, uint64_t dyStride,
                        float* dweights, void* stream) {
  constexpr int N = 16 / sizeof(T);
  const bool nt = pastCaches(a->rows, a->width * sizeof(T));
  if (a->width < N) return combineBackward<T, 1>(a, (const T*)y, yStride, (const T*)dout, doutStride, (T*)dy, dyStride, dweights, false, stream);
  return combineBackward<T, N>(a, (const T*)y, yStride, (const T*)dout, doutStride, (T*)dy, dyStride, dweights, nt, stream);
}

}  // namespace

extern "C" int cuttHipCombine(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combineRows<float>(a, y, yStride, out, outStride, stream);
    case CUTT_ROW_F16: return combineRows<_Float16>(a, y, yStride, out, outStride, stream);
    default: return combineRows<__bf16>(a, y, yStride, out, outStride, stream);
  }
}

extern "C" int cuttHipCombineBackward(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride,
                                      void* dy, uint64_t dyStride, float* dweights, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combineRowsBackward<float>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    case CUTT_ROW_F16: return combineRowsBackward<_Float16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    default: return combineRowsBackward<__bf16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
  }
}
