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
constexpr uint32_t kLeast = kWaves * kBlock;  // tokens of a stretch, at least
constexpr uint32_t kScan = 2048;  // queries that are cut into stretches
constexpr uint32_t kTarget = 1024;

// How the work is cut, which a launch's workgroups and the one that joins their results find out alike.
struct Attend {
  cuttHipAttendArgs a;
  uint32_t group, headTiles;  // query heads per key head, and workgroups that share them
  uint32_t stretches;         // that all tokens together are to be cut into, about; 0: each query is taken whole
  uint32_t slots;             // of partial results
  float* partial;             // [slots][heads][width]
  float2* tops;               // [slots][heads]: the largest score, and the sum of the exponentials that it was taken off
  uint2* cuts;                // [queries]: first slot and number of stretches
};

// What a query sees: tokens first .. end - 1 of request `request`; none where first == end.
struct Seen {
  uint32_t request, first, end;
  __device__ __forceinline__ Seen() {}
  __device__ __forceinline__ Seen(const cuttHipAttendArgs& a, uint32_t query) {
    const int32_t p = a.positions[query];
    request = a.owners ? (uint32_t)a.owners[query] : query;
    const uint64_t reach = (uint64_t)a.tableWidth * a.pageSize;
    end = p < 0 || request >= a.requests ? 0 : (uint32_t)min((uint64_t)p + 1, reach);
    first = a.window && p >= 0 && (uint32_t)p >= a.window ? min((uint32_t)p - a.window + 1, end) : 0;
  }
};

// A workgroup's part: the tokens of `seen`, and where the result goes.
struct Part {
  uint32_t query, slot, cut;  // cut: it is one of several
  Seen seen;
};

struct ScanLds {
  uint32_t low[kWaves], high[kWaves], counts[kWaves];
  uint32_t query, first, slot, cut, length;
};

__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return x + y; }

// Item number `item` of all queries' stretches, or false if there are fewer.  Stretches are as long as makes p.stretches of all tokens together, and a query
// that sees less is one; every workgroup scans the queries for itself.
__device__ __forceinline__ bool findPart(const Attend& p, uint32_t item, bool first, ScanLds& s, Part& part) {
  const cuttHipAttendArgs& a = p.a;
  if (!p.stretches) {
    part.query = item;
    part.cut = 0;
    part.slot = 0;
    part.seen = Seen(a, item);
    return true;
  }
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t each = (a.queries + kThreads - 1) / kThreads;  // neighbouring queries of this thread
  const uint32_t from = min(threadIdx.x * each, a.queries), to = min(from + each, a.queries);
  const auto tokensOf = [&](uint32_t query) __attribute__((always_inline)) {
    const Seen seen(a, query);
    return seen.end - seen.first;
  };
  uint32_t low = 0, high = 0;  // (sums of 2048 numbers below 2^32 in two halves)
#pragma unroll 1
  for (uint32_t i = from; i < to; i++) {
    const uint32_t n = tokensOf(i);
    low += n & 0xffff;
    high += n >> 16;
  }
  low = scanOverWave(low, plus);
  high = scanOverWave(high, plus);
  if (lane == 63) {
    s.low[wave] = low;
    s.high[wave] = high;
  }
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; w++) all += s.low[w] + ((uint64_t)s.high[w] << 16);
  const uint64_t even = ((all + p.stretches - 1) / p.stretches + kLeast - 1) / kLeast * kLeast;
  const uint32_t length = (uint32_t)min(max(even, (uint64_t)kLeast), (uint64_t)1 << 31);
  // Stretches in the lower half of a word (at most kScan + p.stretches), slots in the upper one (twice p.stretches).
  const auto countsOf = [&](uint32_t query) __attribute__((always_inline)) {
    const uint32_t tokens = tokensOf(query), n = tokens <= length ? 1 : (tokens + length - 1) / length;
    return n | (n > 1 ? n << 16 : 0);
  };
  uint32_t mine = 0;
#pragma unroll 1
  for (uint32_t i = from; i < to; i++) mine += countsOf(i);
  const uint32_t upTo = scanOverWave(mine, plus);
  if (lane == 63) s.counts[wave] = upTo;
  if (threadIdx.x == 0) s.query = a.queries;
  __syncthreads();
  uint32_t before = upTo - mine;
  for (uint32_t w = 0; w < wave; w++) before += s.counts[w];
#pragma unroll 1
  for (uint32_t i = from; i < to; i++) {
    const uint32_t counts = countsOf(i), at = before & 0xffff, n = counts & 0xffff;
    if (first) p.cuts[i] = make_uint2(before >> 16, n);
    if (item >= at && item < at + n) {
      s.query = i;
      s.first = item - at;
      s.slot = (before >> 16) + (item - at);
      s.cut = n > 1;
      s.length = length;
    }
    before += counts;
  }
  __syncthreads();
  if (s.query >= a.queries) return false;
  part.query = __builtin_amdgcn_readfirstlane(s.query);
  part.slot = __builtin_amdgcn_readfirstlane(s.slot);
  part.cut = __builtin_amdgcn_readfirstlane(s.cut);
  part.seen = Seen(a, part.query);
  const uint64_t begin = (uint64_t)part.seen.first + (uint64_t)s.first * s.length;
  part.seen.end = (uint32_t)min((uint64_t)part.seen.end, begin + s.length);
  part.seen.first = (uint32_t)min(begin, (uint64_t)part.seen.end);
  __syncthreads();
  return true;
}

// The tokens' scores and their weighted values, a tile of tokens at a time: keys times queries give the scores, heads along the instruction's columns, and each lane
// then holds the exponentials of its head's tokens just as the second product, values turned times exponentials, wants them.
template <typename T, int DP>
struct Tokens {
  static constexpr int E = kPer16<T>;
  static constexpr int TILE = sizeof(T) == 2 ? 32 : 16;  // tokens
  static constexpr int SUB = TILE / 16;                  // tiles of scores
  static constexpr int STEPS = DP / (4 * E);             // 16 bytes of each of the lane quarters
  static constexpr int VD = DP / 16;                     // a value's elements in a lane: l * VD .. for l = lane & 15
  static constexpr int VE = VD < E ? VD : E, VC = VD / VE;  // in pieces of 16 bytes, or a smaller one
  static constexpr int VT = TILE / 4;                    // tokens whose values a lane has
};

// What the wavefront's lanes have written to LDS before is seen by its other lanes after.
__device__ __forceinline__ void waveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp2Of(float x) { return __builtin_amdgcn_exp2f(x); }
// What scores are taken off from before they are exponents: their largest, unless there are only scores of -infinity.
__device__ __forceinline__ float baseOf(float top) { return top == -INFINITY ? 0.0f : top; }

// A wavefront's tokens: blocks of kBlock tokens, every kWaves-th block of the part.
struct Blocks {
  uint64_t next;       // first token of the block behind the current one
  int32_t page;        // this lane's token's page in it
  uint64_t there;      // the current block's tokens that have a page, from the current tile on
  uint32_t tile;       // first token of the current tile in the block
  uint64_t* offset;    // of the current block's tokens in the caches, in elements

  __device__ __forceinline__ void ask(const cuttHipAttendArgs& a, const Seen& seen) {
    const uint64_t t = next + (threadIdx.x & 63);
    page = -1;
    if (t < seen.end) page = a.tables[(uint64_t)seen.request * a.tableWidth + (uint32_t)t / a.pageSize];
  }
  __device__ __forceinline__ void begin(const cuttHipAttendArgs& a, const Seen& seen, uint64_t* lds) {
    offset = lds;
    next = (uint64_t)seen.first + (threadIdx.x >> 6) * kBlock;
    there = 0;
    tile = 0;
    ask(a, seen);
  }
  // On to the next tile of `tokens` that has a token with a page; false if there is none.
  __device__ __forceinline__ bool advance(const cuttHipAttendArgs& a, const Seen& seen, uint32_t tokens) {
    there = tokens < 64 ? there >> tokens : 0;
    tile += tokens;
    if (there) return true;
    const uint32_t lane = threadIdx.x & 63;
    while (next < seen.end) {
      const uint32_t t = (uint32_t)next + lane, j = t / a.pageSize;
      const int32_t mine = page;
      next += kWaves * kBlock;
      ask(a, seen);
      const bool is = (uint32_t)mine < a.pages;
      there = __ballot(is);
      if (!there) continue;
      const uint64_t at = is ? (uint64_t)(uint32_t)mine * a.pageStride + (t - j * a.pageSize) * a.slotStride : 0;
      const uint32_t some = __builtin_ctzll(there);  // a token that is there stands in for one that is not, whose value counts nothing
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(at >> 32), some) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)at, some);
      waveFence();
      offset[lane] = is ? at : other;
      waveFence();
      tile = 0;
      return true;
    }
    return false;
  }
};

template <typename T, int DP, bool FULL>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void attendKernel(Attend p, uint32_t items) {
  using S = Tokens<T, DP>;
  constexpr int E = S::E, TILE = S::TILE, SUB = S::SUB, STEPS = S::STEPS, VD = S::VD, VE = S::VE, VC = S::VC, VT = S::VT;
  const cuttHipAttendArgs& a = p.a;
  extern __shared__ char lds[];
  __shared__ ScanLds scan;
  const uint32_t lane = threadIdx.x & 63, l = lane & 15, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = p.headTiles * a.keyHeads;
  const int width = FULL ? DP : (int)a.width;
  const float scale = a.scale * kLog2e;

  for (uint64_t at = blockIdx.x; at < (uint64_t)items * heads; at += gridDim.x) {
    const uint32_t item = (uint32_t)(at / heads), share = (uint32_t)(at % heads), keyHead = share / p.headTiles;
    const uint32_t head0 = keyHead * p.group + share % p.headTiles * kHeads, nHeads = min(p.group - share % p.headTiles * kHeads, kHeads);
    Part part;
    if (!findPart(p, item, at == 0, scan, part)) return;  // (nor are there later ones)
    const T* const kHead = static_cast<const T*>(a.k) + keyHead * a.cacheHead;
    const T* const vHead = static_cast<const T*>(a.v) + keyHead * a.cacheHead;

    Blocks blocks;
    blocks.begin(a, part.seen, reinterpret_cast<uint64_t*>(lds) + wave * kBlock);
    Chunk<T> q[STEPS];
    {
      const T* const from = static_cast<const T*>(a.q) + part.query * a.qStride + (head0 + min(l, nHeads - 1)) * a.qHead;
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        const int d = (s * 4 + quarter) * E;
        q[s] = loadChunk(from + d, l < nHeads ? width - d : 0);
      }
    }
    float top = -INFINITY, sum = 0;  // of this lane's head: the largest score so far (times log2 e), the exponentials of this quarter's tokens
    Acc acc[VD] = {};

    Chunk<T> k[SUB][STEPS];
    AlignedVec<T, VE> v[VT][VC];
    const auto loadKeys = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        const T* const from = kHead + blocks.offset[blocks.tile + i * 16 + l];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          const int d = (s * 4 + quarter) * E;
          k[i][s] = loadChunk(from + d, FULL ? E : width - d);
        }
      }
    };
    const auto loadValues = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < VT; t++) {
        const T* const from = vHead + blocks.offset[blocks.tile + t / 4 * 16 + quarter * 4 + t % 4];
#pragma unroll
        for (int c = 0; c < VC; c++) {
          const int d = (int)l * VD + c * VE;
          if (FULL || d + VE <= width) {
            v[t][c] = __builtin_bit_cast(AlignedVec<T, VE>, *reinterpret_cast<const Vec<T, VE>*>(from + d));
          } else {
            v[t][c] = {};
#pragma unroll
            for (int e = 0; e < VE; e++)
              if (d + e < width) v[t][c][e] = from[d + e];
          }
        }
      }
    };

    Acc score[SUB];
    const auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < SUB; i++) score[i] = Acc(0);
#pragma unroll
      for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int i = 0; i < SUB; i++) score[i] = multiply(k[i][s], q[s], score[i]);
    };
    // The tile's part of the sums; bit i of `there`: token i of the tile is there.
    const auto addValues = [&](uint32_t there) __attribute__((always_inline)) {
      constexpr uint32_t ALL = TILE == 32 ? ~0u : (1u << (TILE & 31)) - 1;
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < SUB; i++) score[i] *= scale;
      if ((there & ALL) != ALL) {
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (!(there >> (i * 16 + quarter * 4 + r) & 1)) score[i][r] = -INFINITY;
#pragma unroll
        for (int t = 0; t < VT; t++)
          if (!(there >> (t / 4 * 16 + quarter * 4 + t % 4) & 1))
#pragma unroll
            for (int c = 0; c < VC; c++) v[t][c] = {};
      }
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) most = fmaxf(most, score[i][r]);
      most = overQuarters(most, [](float x, float y) { return fmaxf(x, y); });
      if (__any(most > top)) {
        const float next = fmaxf(most, top), less = exp2Of(top - baseOf(next));
        top = next;
        sum *= less;
#pragma unroll
        for (int j = 0; j < VD; j++) acc[j] *= less;
      }
      const float base = baseOf(top);
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          score[i][r] = exp2Of(score[i][r] - base);
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
    };

    // The next tile's keys are asked for as soon as this one's have been used, its values likewise.
    if (blocks.advance(a, part.seen, 64)) {
      loadKeys();
      loadValues();
      for (;;) {
        const uint32_t there = (uint32_t)blocks.there;
        scores();
        if (!blocks.advance(a, part.seen, TILE)) {
          addValues(there);
          break;
        }
        loadKeys();
        addValues(there);
        loadValues();
      }
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
    const float mine = exp2Of(top - baseOf(all));
    if (l < nHeads)
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < VD; j++) parts[(wave * kHeads + l) * PITCH + (quarter * 4 + r) * VD + j] = acc[j][r] * mine;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nHeads * a.width; i += kThreads) {
      const uint32_t h = i / a.width, d = i - h * a.width, head = head0 + h;
      float m = -INFINITY, n = 0, o = 0;
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) m = fmaxf(m, tops[w * kHeads + h]);
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) {
        n += sums[w * kHeads + h] * exp2Of(tops[w * kHeads + h] - baseOf(m));
        o += parts[(w * kHeads + h) * PITCH + d];
      }
      if (part.cut) {
        const uint64_t to = (uint64_t)part.slot * a.heads + head;
        p.partial[to * a.width + d] = o;
        if (d == 0) p.tops[to] = make_float2(m, n);
      } else {
        const bool none = n == 0 && m == -INFINITY;
        static_cast<T*>(a.out)[part.query * a.outStride + head * a.outHead + d] = (T)(none ? 0.0f : o / n);
        if (a.logSums && d == 0) a.logSums[(uint64_t)part.query * a.heads + head] = none ? -INFINITY : (m + __log2f(n)) * kLn2;
      }
    }
    __syncthreads();
  }
}

// The parts of the queries that were cut, joined.  A workgroup takes a query's head; its wavefronts share the parts.
template <typename T>
__global__ __launch_bounds__(kThreads) void joinKernel(Attend p) {
  const cuttHipAttendArgs& a = p.a;
  __shared__ float sums[kWaves];
  __shared__ float parts[kWaves][256];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint64_t at = blockIdx.x; at < (uint64_t)a.queries * a.heads; at += gridDim.x) {
    const uint32_t query = (uint32_t)(at / a.heads), head = (uint32_t)(at % a.heads);
    const uint2 cut = p.cuts[query];
    if (cut.y <= 1) continue;
    const float2* const tops = p.tops + (uint64_t)cut.x * a.heads + head;
    float m = -INFINITY;
    for (uint32_t i = lane; i < cut.y; i += 64) m = fmaxf(m, tops[(uint64_t)i * a.heads].x);
#pragma unroll
    for (int i = 1; i < 64; i *= 2) m = fmaxf(m, __shfl_xor(m, i));
    const float base = baseOf(m);
    float n = 0, o[4] = {};
#pragma unroll 4
    for (uint32_t i = wave; i < cut.y; i += kWaves) {
      const float2 top = tops[(uint64_t)i * a.heads];
      const float share = exp2Of(top.x - base);
      const float* const from = p.partial + ((uint64_t)(cut.x + i) * a.heads + head) * a.width;
      n += share * top.y;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t d = lane + j * 64;
        if (d < a.width) o[j] += share * from[d];
      }
    }
    if (lane == 0) sums[wave] = n;
#pragma unroll
    for (int j = 0; j < 4; j++) parts[wave][lane + j * 64] = o[j];
    __syncthreads();
    if (threadIdx.x < a.width) {
      float all = 0, sum = 0;
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) {
        sum += sums[w];
        all += parts[w][threadIdx.x];
      }
      const bool none = sum == 0 && m == -INFINITY;
      static_cast<T*>(a.out)[query * a.outStride + head * a.outHead + threadIdx.x] = (T)(none ? 0.0f : all / sum);
      if (a.logSums && threadIdx.x == 0) a.logSums[(uint64_t)query * a.heads + head] = none ? -INFINITY : (m + __log2f(sum)) * kLn2;
    }
    __syncthreads();
  }
}

constexpr uint32_t kMaxBlocks = 1u << 22;

// How sizes are cut: a query's tokens are at most `reach`.
Attend planAttend(uint32_t queries, uint32_t heads, uint32_t keyHeads, uint32_t pageSize, uint32_t tableWidth, uint32_t window) {
  Attend p = {};
  p.group = heads / keyHeads;
  p.headTiles = (p.group + kHeads - 1) / kHeads;
  uint64_t reach = (uint64_t)pageSize * tableWidth;
  if (window && window < reach) reach = window;
  if (queries <= kScan && reach > kLeast) {
    p.stretches = std::max(1u, kTarget / (p.headTiles * keyHeads));
    // A query that is cut sees more than a stretch and has less than twice its tokens' share of them.
    p.slots = (uint32_t)std::min<uint64_t>(2 * p.stretches, queries * ((reach + kLeast - 1) / kLeast));
  }
  return p;
}

template <typename T, int DP>
int attend(const Attend& p, void* stream) {
  const size_t lds = std::max<size_t>(kWaves * kBlock * 8, (2 * kWaves * kHeads + kWaves * kHeads * (DP + 4)) * 4);
  const uint32_t items = p.a.queries + p.stretches;
  const uint64_t blocks = (uint64_t)items * p.a.keyHeads * p.headTiles;
  auto kernel = p.a.width == DP ? attendKernel<T, DP, true> : attendKernel<T, DP, false>;
  if (int e = launchRows(kernel, (uint32_t)std::min<uint64_t>(blocks, kMaxBlocks), kThreads, lds, stream, p, items)) return e;
  if (!p.stretches) return 0;
  return launchRows(joinKernel<T>, (uint32_t)std::min<uint64_t>((uint64_t)p.a.queries * p.a.heads, kMaxBlocks), kThreads, 0, stream, p);
}

template <typename T>
int attendWide(const Attend& p, void* stream) {
  return p.a.width <= 64 ? attend<T, 64>(p, stream) : p.a.width <= 128 ? attend<T, 128>(p, stream) : attend<T, 256>(p, stream);
}

}  // namespace

extern "C" size_t cuttHipAttendWorkspace(uint32_t queries, uint32_t heads, uint32_t keyHeads, uint32_t width, uint32_t pageSize, uint32_t tableWidth, uint32_t window) {
  const Attend p = planAttend(queries, heads, keyHeads, pageSize, tableWidth, window);
  return p.stretches ? ((size_t)p.slots * heads * (width + 2) + 2 * (size_t)queries) * 4 : 0;
}

extern "C" int cuttHipAttend(const cuttHipAttendArgs* a, int type, void* stream) {
  Attend p = planAttend(a->queries, a->heads, a->keyHeads, a->pageSize, a->tableWidth, a->window);
  p.a = *a;
  float* const space = static_cast<float*>(a->workspace);
  p.tops = reinterpret_cast<float2*>(space);
  p.partial = space + 2 * (size_t)p.slots * a->heads;
  p.cuts = reinterpret_cast<uint2*>(p.partial + (size_t)p.slots * a->heads * a->width);
  switch (type) {
    case CUTT_ROW_F32: return attendWide<float>(p, stream);
    case CUTT_ROW_F16: return attendWide<_Float16>(p, stream);
    default: return attendWide<__bf16>(p, stream);
  }
}
