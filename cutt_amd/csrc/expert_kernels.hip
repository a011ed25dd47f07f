/*
 * expert_kernels.hip - rows sorted by expert and back (cutt_rows.h): the stable counting sort of a router's
 * choices, the move of the tokens' rows to their experts, the weighted sum back, and the gradients of both.
 */
#include "row_device.h"
#include "row_layer.h"

using namespace cutt;

namespace {

// ---------------------------------------------------------------------------
// Sort.  A stable counting sort: each workgroup places a stretch of neighbouring choices.  It needs to know how many choices each expert has in
// all and before the stretch.  Few choices: every workgroup counts all of them (COUNTED = false, one launch).  Many: a first
// launch counts stretch by stretch into the workspace, [stretch][expert], and a workgroup adds the columns up.
// ---------------------------------------------------------------------------
constexpr uint32_t kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr uint32_t kSortItems = 4;  // choices that a lane places at a time
constexpr uint32_t kSortPart = kSortThreads * kSortItems;
constexpr uint32_t kSortGroups = 256;       // at most
constexpr uint32_t kCountAll = 16384;       // choices that every workgroup counts for itself

struct SortPlan {
  uint32_t stretch;  // choices per workgroup, a multiple of kSortPart
  uint32_t groups;
  bool counted;
};

// The expert of choice i among the `experts`, or `experts` if it is none of them.
template <typename Id>
__device__ __forceinline__ uint32_t expertOf(const cuttHipSortArgs& a, uint32_t i) {
  const uint64_t e = (uint64_t)(int64_t) static_cast<const Id*>(a.ids)[i] - (uint64_t)(int64_t)a.firstExpert;  // (wraps)
  return e < a.experts ? (uint32_t)e : a.experts;
}

template <typename Id>
__global__ __launch_bounds__(kSortThreads) void expertCountKernel(cuttHipSortArgs a, uint32_t stretch) {
  extern __shared__ uint32_t count[];  // [experts + 1]
  const uint32_t E = a.experts;
  for (uint32_t e = threadIdx.x; e <= E; e += kSortThreads) count[e] = 0;
  __syncthreads();
  const uint32_t from = blockIdx.x * stretch, to = min(from + stretch, a.n);
#pragma unroll 4
  for (uint32_t i = from + threadIdx.x; i < to; i += kSortThreads) atomicAdd(&count[expertOf<Id>(a, i)], 1u);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < E; e += kSortThreads) a.workspace[(uint64_t)blockIdx.x * E + e] = count[e];
}

// Lanes of the wavefront whose key is this lane's; keys have `bits` bits.
__device__ __forceinline__ uint64_t sameKey(uint32_t key, uint32_t bits) {
  uint64_t same = ~0ull;
  for (uint32_t b = 0; b < bits; b++) {
    const bool one = (key >> b) & 1;
    const uint64_t set = __ballot(one);
    same &= one ? set : ~set;
  }
  return same;
}

template <typename Id, bool COUNTED>
__global__ __launch_bounds__(kSortThreads) void expertSortKernel(cuttHipSortArgs a, uint32_t stretch) {
  extern __shared__ uint32_t lds[];
  const uint32_t E = a.experts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t* const next = lds;                    // [E + 1] choices before the stretch, then the row of an expert's next choice
  uint32_t* const all = next + E + 1;            // [E + 1] choices in all, then the row behind an expert's last choice
  uint32_t* const start = all + E + 1;           // [E + 1] an expert's first row
  uint32_t* const seen = start + E + 1;          // [waves][E + 1]
  __shared__ uint32_t waveSum[kSortWaves];
  const uint32_t from = blockIdx.x * stretch, to = min(from + stretch, a.n);

  if constexpr (COUNTED) {
    // The threads share the table: thread tid adds up every `share`-th stretch of expert tid % E (E <= kSortThreads), or experts
    // tid, tid + kSortThreads of all.
    for (uint32_t e = tid; e <= E; e += kSortThreads) next[e] = all[e] = 0;
    __syncthreads();
    const uint32_t share = E <= kSortThreads ? kSortThreads / E : 1, part = tid / E;
    if (part < share || share == 1)
      for (uint32_t e = share == 1 ? tid : tid - part * E; e < E; e += kSortThreads) {
        uint32_t before = 0, sum = 0;
#pragma unroll 8
        for (uint32_t g = share == 1 ? 0 : part; g < gridDim.x; g += share) {
          const uint32_t c = a.workspace[(uint64_t)g * E + e];
          sum += c;
          before += g < blockIdx.x ? c : 0;
        }
        atomicAdd(&next[e], before);
        atomicAdd(&all[e], sum);
      }
  } else {
    for (uint32_t e = tid; e <= E; e += kSortThreads) next[e] = all[e] = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = tid; i < a.n; i += kSortThreads) {
      const uint32_t e = expertOf<Id>(a, i);
      atomicAdd(&all[e], 1u);
      if (i < from) atomicAdd(&next[e], 1u);
    }
  }
  __syncthreads();

  // Experts' first rows: thread tid adds up experts 2 tid and 2 tid + 1 (CUTT_MAX_EXPERTS = 2 * kSortThreads).
  {
    uint32_t padded[2], sum = 0;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t e = 2 * tid + j;
      padded[j] = e < E ? (all[e] + a.align - 1) / a.align * a.align : 0;
      sum += padded[j];
    }
    uint32_t upTo = sum;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
      const uint32_t x = __shfl_up(upTo, d);
      if (lane >= d) upTo += x;
    }
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
  const uint32_t bits = 32 - __builtin_clz(E);
  uint32_t* const mine = seen + wave * (E + 1);
  for (uint64_t part = from; part < to; part += kSortPart) {
    for (uint32_t e = lane; e <= E; e += 64) mine[e] = 0;
    __builtin_amdgcn_wave_barrier();
    uint32_t expert[kSortItems], rank[kSortItems];
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++) {
      const uint64_t i = part + (wave * kSortItems + j) * 64 + lane;
      expert[j] = i < to ? expertOf<Id>(a, (uint32_t)i) : E;
    }
#pragma unroll
    for (uint32_t j = 0; j < kSortItems; j++) {
      const uint64_t same = sameKey(expert[j], bits);
      const uint32_t below = __popcll(same & ((1ull << lane) - 1));
      const uint32_t before = mine[expert[j]];  // (the wavefront's lanes all read, then one lane per expert writes)
      __builtin_amdgcn_wave_barrier();
      rank[j] = before + below;
      if (below == 0) mine[expert[j]] = before + __popcll(same);
      __builtin_amdgcn_wave_barrier();
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

SortPlan planSort(uint32_t n) {
  SortPlan p;
  const uint64_t parts = n ? ((uint64_t)n + kSortPart - 1) / kSortPart : 1;
  p.counted = n > kCountAll;
  const uint64_t perGroup = (parts + kSortGroups - 1) / kSortGroups;
  p.stretch = (uint32_t)(perGroup * kSortPart);
  p.groups = (uint32_t)((parts + perGroup - 1) / perGroup);
  return p;
}

// ---------------------------------------------------------------------------
// Rows to experts and back.
// ---------------------------------------------------------------------------
constexpr uint32_t kRowThreads = 256, kRowWaves = kRowThreads / 64;
constexpr uint32_t kMaxBlocks = 1u << 22;  // (workgroups x lanes have to fit 32 bits)

// Rows without a source, which hold zeros.  Workgroup `block` of `blocks` looks at kEmptyRows rows at a time; a wavefront clears a row.
constexpr uint32_t kEmptyRows = 16;

template <typename T, int N>
__device__ __forceinline__ void clearEmptyRows(const cuttHipExpertArgs& a, T* y, uint64_t stride, uint32_t block, uint32_t blocks) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  Pack<T, N> zero = {};
  for (uint64_t first = (uint64_t)block * kEmptyRows; first < a.rows; first += (uint64_t)blocks * kEmptyRows) {
    const uint64_t mine = first + (lane & (kEmptyRows - 1));
    uint64_t empty = __ballot(lane < kEmptyRows && mine < a.rows && a.source[mine] < 0);
    for (uint32_t n = 0; empty; n++) {
      const uint32_t r = __builtin_ctzll(empty);
      empty &= empty - 1;
      if (n % kRowWaves != wave) continue;
      T* const row = y + (first + r) * stride;
      for (uint32_t c = lane * N; c < a.width; c += 64 * N) zero.store(row + min(c, a.width - N));
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
  uint32_t laneRow;
  float laneWeight;
  uint32_t there;  // bit i: choice i has a row

  __device__ __forceinline__ Choices(const cuttHipExpertArgs& a, uint32_t token, uint32_t first) {
    const uint32_t i = threadIdx.x & (B - 1);
    const uint64_t at = (uint64_t)token * a.choices + min(first + i, a.choices - 1);
    laneRow = (uint32_t)a.position[at];
    laneWeight = 1.0f;
    if (a.weights) laneWeight = a.weights[at];
    const bool ok = first + i < a.choices && laneRow < a.rows;
    there = (uint32_t)__ballot(ok) & ((1u << B) - 1);
    const uint32_t some = __builtin_amdgcn_readlane(laneRow, there ? __builtin_ctz(there) : 0);
    if (!ok) laneRow = some, laneWeight = 0.0f;
  }
  __device__ __forceinline__ bool has(int i) const { return there >> i & 1; }
  __device__ __forceinline__ uint64_t row(int i) const { return (uint32_t)__builtin_amdgcn_readlane(laneRow, i); }
  __device__ __forceinline__ float weight(int i) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(laneWeight), i)); }
};

// The workgroup's wavefronts share a row's columns: wavefront w takes the columns w * 64 * N, (w + kRowWaves) * 64 * N, ...
__device__ __forceinline__ uint32_t waveOfGroup() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// A workgroup reads a token's row once and stores it to every row that the token goes to; the last workgroups clear the empty rows.
// Rows are bytes here: any element size, any alignment.
template <int N>
__global__ __launch_bounds__(kRowThreads) void dispatchKernel(cuttHipExpertArgs a, const uint8_t* x, uint64_t xStride, uint8_t* y, uint64_t yStride,
                                                              uint32_t tokenBlocks) {
  constexpr int U = N == 1 ? 1 : 2;  // vectors a lane keeps
  if (blockIdx.x >= tokenBlocks) {
    clearEmptyRows<uint8_t, N>(a, y, yStride, blockIdx.x - tokenBlocks, gridDim.x - tokenBlocks);
    return;
  }
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += tokenBlocks) {
    const uint8_t* const from = x + t * xStride;
    const Choices<8> begin(a, t, 0);
    for (uint32_t col = waveOfGroup() * 64 * N; col < a.width; col += kRowThreads * N * U) {
      Pack<uint8_t, N> v[U];
      uint32_t at[U];
      bool mine[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t base = col + u * kRowThreads * N + lane * N;
        mine[u] = base < a.width;
        at[u] = min(base, a.width - N);
        v[u].load(from + at[u]);
      }
      auto put = [&](const Choices<8>& ch) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (!ch.has(i)) continue;
          uint8_t* const to = y + ch.row(i) * yStride;
#pragma unroll
          for (int u = 0; u < U; u++)
            if (mine[u]) v[u].store(to + at[u]);
        }
      };
      put(begin);
      for (uint32_t first = 8; first < a.choices; first += 8) put(Choices<8>(a, t, first));
    }
  }
}

// A workgroup sums a token's rows, 16 bytes of each per lane.
template <typename T, int N, int B>
__global__ __launch_bounds__(kRowThreads) void combineKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, T* out, uint64_t outStride) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const Choices<B> begin(a, t, 0);
    for (uint32_t col = waveOfGroup() * 64 * N; col < a.width; col += kRowThreads * N) {
      const uint32_t base = col + lane * N, c = min(base, a.width - N);
      float sum[N] = {};
      auto add = [&](const Choices<B>& ch) __attribute__((always_inline)) {
        if (!ch.there) return;
        Pack<T, N> v[B];
#pragma unroll
        for (int i = 0; i < B; i++) v[i].load(y + ch.row(i) * yStride + c);
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
template <typename T, int N, int B, bool ROWS, bool WEIGHTS>
__global__ __launch_bounds__(kRowThreads) void combineBackwardKernel(cuttHipExpertArgs a, const T* y, uint64_t yStride, const T* dout, uint64_t doutStride,
                                                                     T* dy, uint64_t dyStride, float* dweights, uint32_t tokenBlocks) {
  __shared__ float part[kRowWaves][B];
  if (ROWS && blockIdx.x >= tokenBlocks) {
    clearEmptyRows<T, N>(a, dy, dyStride, blockIdx.x - tokenBlocks, gridDim.x - tokenBlocks);
    return;
  }
  const uint32_t wave = waveOfGroup(), lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x; t < a.tokens; t += tokenBlocks)
    for (uint32_t first = 0; first < a.choices; first += B) {
      const Choices<B> ch(a, t, first);
      float dot[B] = {};
      for (uint32_t col = waveOfGroup() * 64 * N; ch.there && col < a.width; col += kRowThreads * N) {
        const uint32_t base = col + lane * N, c = min(base, a.width - N);
        Pack<T, N> g, v[B];
        g.load(dout + t * doutStride + c);
        if (WEIGHTS)
#pragma unroll
          for (int i = 0; i < B; i++) v[i].load(y + ch.row(i) * yStride + c);
        Pack<T, N> once = g;
        if (WEIGHTS && c != base)  // columns that the vector before it, or its row's last vector, has already counted
#pragma unroll
          for (int e = 0; e < N; e++)
            if (c + e < base) {
              once.set(e, T(0));
#pragma unroll
              for (int i = 0; i < B; i++) v[i].set(e, T(0));
            }
#pragma unroll
        for (int i = 0; i < B; i++) {
          if (WEIGHTS)
#pragma unroll
            for (int e = 0; e < N; e++) dot[i] = fmaf((float)once.get(e), (float)v[i].get(e), dot[i]);
          if (ROWS && ch.has(i)) {
            const float w = ch.weight(i);
            T* const to = dy + ch.row(i) * dyStride + c;
            Pack<T, N> o;
#pragma unroll
            for (int e = 0; e < N; e++) o.set(e, (T)(w * (float)g.get(e)));
            if (base < a.width) o.store(to);
          }
        }
      }
      if (!WEIGHTS) continue;
#pragma unroll
      for (int i = 0; i < B; i++) dot[i] = ch.has(i) ? dot[i] : 0.0f;
      const float sum = sumOverWave(dot);
      if (lane % (64 / B) == 0) part[wave][lane / (64 / B)] = sum;
      __syncthreads();
      if (threadIdx.x < B && first + threadIdx.x < a.choices) {
        float all = 0;
        for (uint32_t w = 0; w < kRowWaves; w++) all += part[w][threadIdx.x];
        dweights[(uint64_t)t * a.choices + first + threadIdx.x] = all;
      }
      __syncthreads();
    }
}

constexpr uint64_t kMaxPiece = 1u << 30;

uint32_t blocksFor(uint64_t n) { return (uint32_t)(n < kMaxBlocks ? n : kMaxBlocks); }
uint32_t emptyBlocks(uint32_t rows) { return blocksFor((rows + (uint64_t)kEmptyRows - 1) / kEmptyRows); }

}  // namespace

extern "C" size_t cuttHipSortWorkspace(uint32_t n, uint32_t experts) {
  const SortPlan p = planSort(n);
  return p.counted ? (size_t)p.groups * experts * 4 : 0;
}

namespace {

template <typename Id>
int sortBy(const cuttHipSortArgs* a, void* stream) {
  const SortPlan p = planSort(a->n);
  const size_t perExpert = (size_t)(a->experts + 1) * 4, lds = (3 + kSortWaves) * perExpert;
  if (!p.counted) return launchRows(expertSortKernel<Id, false>, p.groups, kSortThreads, lds, stream, *a, p.stretch);
  if (int e = launchRows(expertCountKernel<Id>, p.groups, kSortThreads, perExpert, stream, *a, p.stretch)) return e;
  return launchRows(expertSortKernel<Id, true>, p.groups, kSortThreads, lds, stream, *a, p.stretch);
}

}  // namespace

extern "C" int cuttHipExpertSort(const cuttHipSortArgs* a, void* stream) {
  return a->idBytes == 8 ? sortBy<int64_t>(a, stream) : sortBy<int32_t>(a, stream);
}

extern "C" int cuttHipDispatch(const cuttHipExpertArgs* a, uint32_t elemSize, const void* x, uint64_t xStride, void* y, uint64_t yStride, void* stream) {
  const uint64_t bytes = (uint64_t)a->width * elemSize;
  const uint32_t tokenBlocks = blocksFor(a->tokens);
  const dim3 grid(tokenBlocks + emptyBlocks(a->rows));
  // (a launch's offsets in a row have 32 bits: longer rows go piece by piece)
  for (uint64_t at = 0; at < bytes; at += kMaxPiece) {
    cuttHipExpertArgs b = *a;
    b.width = (uint32_t)(bytes - at < kMaxPiece ? bytes - at : kMaxPiece);
    auto kernel = b.width >= 16 ? dispatchKernel<16> : dispatchKernel<1>;
    if (int e = launchRows(kernel, grid, kRowThreads, 0, stream, b, (const uint8_t*)x + at, xStride * elemSize, (uint8_t*)y + at, yStride * elemSize, tokenBlocks))
      return e;
  }
  return 0;
}

namespace {

// Calls f with the elements per vector and the choices taken at once as constants.
template <typename T, typename F>
int byShape(const cuttHipExpertArgs* a, F f) {
  constexpr int N = 16 / sizeof(T);
  if (a->width < N) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  const std::integral_constant<int, N> n;
  if (a->choices > 4) return f(n, std::integral_constant<int, 8>{});
  if (a->choices > 2) return f(n, std::integral_constant<int, 4>{});
  if (a->choices > 1) return f(n, std::integral_constant<int, 2>{});
  return f(n, std::integral_constant<int, 1>{});
}

template <typename T>
int combine(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  return byShape<T>(a, [&](auto n, auto b) {
    return launchRows(combineKernel<T, n, b>, blocksFor(a->tokens), kRowThreads, 0, stream, *a, (const T*)y, yStride, (T*)out, outStride);
  });
}

template <typename T>
int combineBackward(const cuttHipExpertArgs* a, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride, void* dy, uint64_t dyStride,
                    float* dweights, void* stream) {
  const uint32_t tokenBlocks = blocksFor(a->tokens);
  return byShape<T>(a, [&](auto n, auto b) {
    auto go = [&](auto kernel, uint32_t blocks) {
      return launchRows(kernel, tokenBlocks + blocks, kRowThreads, 0, stream, *a, (const T*)y, yStride, (const T*)dout, doutStride, (T*)dy, dyStride, dweights, tokenBlocks);
    };
    if (!dy) return go(combineBackwardKernel<T, n, b, false, true>, 0);
    if (!dweights) return go(combineBackwardKernel<T, n, b, true, false>, emptyBlocks(a->rows));
    return go(combineBackwardKernel<T, n, b, true, true>, emptyBlocks(a->rows));
  });
}

}  // namespace

extern "C" int cuttHipCombine(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, void* out, uint64_t outStride, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combine<float>(a, y, yStride, out, outStride, stream);
    case CUTT_ROW_F16: return combine<_Float16>(a, y, yStride, out, outStride, stream);
    default: return combine<__bf16>(a, y, yStride, out, outStride, stream);
  }
}

extern "C" int cuttHipCombineBackward(const cuttHipExpertArgs* a, int type, const void* y, uint64_t yStride, const void* dout, uint64_t doutStride,
                                      void* dy, uint64_t dyStride, float* dweights, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return combineBackward<float>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    case CUTT_ROW_F16: return combineBackward<_Float16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
    default: return combineBackward<__bf16>(a, y, yStride, dout, doutStride, dy, dyStride, dweights, stream);
  }
}
