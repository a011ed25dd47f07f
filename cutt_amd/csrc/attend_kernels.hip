/*
 * attend_kernels.hip - attention of new tokens' queries over keys and values in pages (cutt_products.h).
 */
#include <algorithm>

#include "product_device.h"
#include "product_layer.h"

using namespace cutt;

namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kHeads = 16;   // query heads of one key head that a workgroup takes at a time: columns of the matrix instructions
constexpr uint32_t kBlock = 64;   // tokens whose addresses a wavefront works out at a time

struct Attend {
  cuttHipAttendArgs a;
  uint32_t group, headTiles;  // query heads per key head, and workgroups that share them
  cuttHipDivisor byPage;
};

// What a query sees: tokens first .. end - 1 of request `request`; none where first == end.
struct Seen {
  uint32_t request, first, end;
  __device__ __forceinline__ Seen(const cuttHipAttendArgs& a, uint32_t query) {
    const int32_t p = a.positions[query];
    request = a.owners ? (uint32_t)a.owners[query] : query;
    const uint64_t reach = (uint64_t)a.tableWidth * a.pageSize;
    end = p < 0 || request >= a.requests ? 0 : (uint32_t)min((uint64_t)p + 1, reach);
    first = a.window && p >= 0 && (uint32_t)p >= a.window ? min((uint32_t)p - a.window + 1, end) : 0;
  }
};

// The tokens' scores and their weighted values, a tile of tokens at a time: keys times queries give the scores, heads along the instruction's columns, and each lane
// then holds the exponentials of its head's tokens just as the second product, values turned times exponentials, wants them.
template <typename T, int DP>
struct Tokens {
  static constexpr int E = kPer16<T>;
  static constexpr int TILE = sizeof(T) == 2 ? 32 : 16;  // tokens
  static constexpr int SUB = TILE / 16;                  // tiles of scores
  static constexpr int STEPS = DP / (4 * E);             // 16 bytes of each of the lane quarters
  static constexpr int VD = DP / 16;                     // a value's elements in a lane: l * VD .. for l = lane & 15
  static constexpr int VT = TILE / 4;                    // tokens whose values a lane has
};

__device__ __forceinline__ void waveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp2Of(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attendKernel(Attend p) {
  using S = Tokens<T, DP>;
  constexpr int E = S::E, TILE = S::TILE, SUB = S::SUB, STEPS = S::STEPS, VD = S::VD, VT = S::VT;
  const cuttHipAttendArgs& a = p.a;
  extern __shared__ char lds[];
  const uint32_t lane = threadIdx.x & 63, l = lane & 15, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint64_t* const offset = reinterpret_cast<uint64_t*>(lds) + wave * kBlock;  // of the block's tokens in the caches, in elements
  const uint32_t heads = p.headTiles * a.keyHeads;
  const uint32_t query = blockIdx.x / heads, part = blockIdx.x % heads, keyHead = part / p.headTiles, head0 = keyHead * p.group + part % p.headTiles * kHeads;
  const uint32_t nHeads = min(p.group - part % p.headTiles * kHeads, kHeads);
  const int width = (int)a.width;
  const Seen seen(a, query);
  const T* const kHead = static_cast<const T*>(a.k) + keyHead * a.cacheHead;
  const T* const vHead = static_cast<const T*>(a.v) + keyHead * a.cacheHead;

  Chunk<T> q[STEPS];
  {
    const T* const from = static_cast<const T*>(a.q) + query * a.qStride + (head0 + min(l, nHeads - 1)) * a.qHead;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      const int d = (s * 4 + quarter) * E;
      q[s] = loadChunk(from + d, l < nHeads ? width - d : 0);
    }
  }
  const float scale = a.scale * kLog2e;
  float top = -INFINITY, sum = 0;  // of this lane's head: the largest score so far (times log2 e), the exponentials of this quarter's tokens
  Acc acc[VD] = {};

  for (uint64_t block = seen.first + wave * kBlock; block < seen.end; block += kWaves * kBlock) {
    // Where the block's tokens are, lane by lane.
    uint64_t there;
    {
      const uint32_t t = (uint32_t)block + lane;
      const uint32_t j = t / a.pageSize;
      int32_t page = -1;
      if (t < seen.end) page = a.tables[(uint64_t)seen.request * a.tableWidth + j];
      there = __ballot((uint32_t)page < a.pages);
      if (!there) continue;
      const uint64_t at = (uint32_t)page < a.pages ? (uint64_t)(uint32_t)page * a.pageStride + (t - j * a.pageSize) * a.slotStride : 0;
      const uint32_t some = __builtin_ctzll(there);  // a token that is there stands in for one that is not, whose value counts nothing
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(at >> 32), some) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)at, some);
      offset[lane] = there >> lane & 1 ? at : other;
      waveFence();
    }
#pragma unroll 1
    for (uint32_t tile = 0; tile < kBlock && (there >> tile); tile += TILE) {
      Chunk<T> k[SUB][STEPS];
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        const T* const from = kHead + offset[tile + i * 16 + l];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          const int d = (s * 4 + quarter) * E;
          k[i][s] = loadChunk(from + d, width - d);
        }
      }
      constexpr int VC = (VD + E - 1) / E, VE = VD < E ? VD : E;  // 16-byte pieces (or one smaller) of a token's values
      AlignedVec<T, VE> v[VT][VC];
#pragma unroll
      for (int t = 0; t < VT; t++) {
        const T* const from = vHead + offset[tile + t / 4 * 16 + quarter * 4 + t % 4];
#pragma unroll
        for (int c = 0; c < VC; c++) {
          const int d = (int)l * VD + c * VE;
          v[t][c] = {};
          if (d + VE <= width) v[t][c] = __builtin_bit_cast(AlignedVec<T, VE>, *reinterpret_cast<const Vec<T, VE>*>(from + d));
          else if (d < width)
#pragma unroll
            for (int e = 0; e < VE; e++)
              if (d + e < width) v[t][c][e] = from[d + e];
          if (!(there >> (tile + t / 4 * 16 + quarter * 4 + t % 4) & 1)) v[t][c] = {};
        }
      }
      Acc score[SUB] = {};
#pragma unroll
      for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int i = 0; i < SUB; i++) score[i] = multiply(k[i][s], q[s], score[i]);
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool is = there >> (tile + i * 16 + quarter * 4 + r) & 1;
          score[i][r] = is ? score[i][r] * scale : -INFINITY;
          most = fmaxf(most, score[i][r]);
        }
      most = overQuarters(most, [](float x, float y) { return fmaxf(x, y); });
      if (__any(most > top)) {
        const float next = fmaxf(most, top), from = next == -INFINITY ? 0.0f : next;
        const float less = exp2Of(top - from);
        top = next;
        sum *= less;
#pragma unroll
        for (int j = 0; j < VD; j++) acc[j] *= less;
      }
      const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          score[i][r] = exp2Of(score[i][r] - from);
          sum += score[i][r];
        }
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int j = 0; j < VD; j++) acc[j] = multiply(v[r][j / VE][j % VE], score[0][r], acc[j]);
      } else {
        // Exponentials in two parts, what the type rounds and what it leaves, so that they count with 16 bits and more.
        Chunk<T> high, low;
#pragma unroll
        for (int t = 0; t < 8; t++) {
          high[t] = (T)score[t / 4][t % 4];
          low[t] = (T)(score[t / 4][t % 4] - (float)high[t]);
        }
#pragma unroll
        for (int j = 0; j < VD; j++) {
          Chunk<T> turned;
#pragma unroll
          for (int t = 0; t < 8; t++) turned[t] = v[t][j / VE][j % VE];
          acc[j] = multiply(turned, high, acc[j]);
          acc[j] = multiply(turned, low, acc[j]);
        }
      }
    }
    waveFence();
  }

  // The wavefronts' parts together.
  sum = overQuarters(sum, [](float x, float y) { return x + y; });
  __syncthreads();
  float* const tops = reinterpret_cast<float*>(lds);            // [waves][heads]
  float* const sums = tops + kWaves * kHeads;
  float* const parts = sums + kWaves * kHeads;                  // [waves][heads][DP + 4]
  constexpr uint32_t PITCH = DP + 4;
  if (quarter == 0) {
    tops[wave * kHeads + l] = top;
    sums[wave * kHeads + l] = sum;
  }
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; w++) all = fmaxf(all, tops[w * kHeads + l]);
  const float from = all == -INFINITY ? 0.0f : all, mine = exp2Of(top - from);
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int j = 0; j < VD; j++) parts[(wave * kHeads + l) * PITCH + (quarter * 4 + r) * VD + j] = acc[j][r] * mine;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < nHeads * a.width; i += kThreads) {
    const uint32_t h = i / a.width, d = i - h * a.width;
    float m = -INFINITY, n = 0, o = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; w++) m = fmaxf(m, tops[w * kHeads + h]);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; w++) {
      n += sums[w * kHeads + h] * exp2Of(tops[w * kHeads + h] - base);
      o += parts[(w * kHeads + h) * PITCH + d];
    }
    const bool none = n == 0 && m == -INFINITY;
    T* const to = static_cast<T*>(a.out) + query * a.outStride + (head0 + h) * a.outHead + d;
    *to = (T)(none ? 0.0f : o / n);
    if (a.logSums && d == 0) a.logSums[(uint64_t)query * a.heads + head0 + h] = none ? -INFINITY : (m + __log2f(n)) * kLn2;
  }
}

template <typename T, int DP>
int attend(const Attend& p, void* stream) {
  const size_t lds = std::max<size_t>(kWaves * kBlock * 8, (2 * kWaves * kHeads + kWaves * kHeads * (DP + 4)) * 4);
  const uint64_t blocks = (uint64_t)p.a.queries * p.a.keyHeads * p.headTiles;
  return launchRows(attendKernel<T, DP>, (uint32_t)blocks, kThreads, lds, stream, p);
}

template <typename T>
int attendWide(const Attend& p, void* stream) {
  return p.a.width <= 64 ? attend<T, 64>(p, stream) : p.a.width <= 128 ? attend<T, 128>(p, stream) : attend<T, 256>(p, stream);
}

}  // namespace

extern "C" size_t cuttHipAttendWorkspace(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }

extern "C" int cuttHipAttend(const cuttHipAttendArgs* a, int type, void* stream) {
  Attend p;
  p.a = *a;
  p.group = a->heads / a->keyHeads;
  p.headTiles = (p.group + kHeads - 1) / kHeads;
  p.byPage = cuttHipMakeDivisor(a->pageSize);
  switch (type) {
    case CUTT_ROW_F32: return attendWide<float>(p, stream);
    case CUTT_ROW_F16: return attendWide<_Float16>(p, stream);
    default: return attendWide<__bf16>(p, stream);
  }
}
