/*
 * attend_kernels.hip - attention of new tokens' queries over keys and values in pages (cutt_products.h).
 *
 * With s_t = scale q.k_t, what is wanted is sum exp(s_t) v_t / sum exp(s_t) over the tokens t that a query sees.  It is had in one pass: scores are taken off from a number `top` near
 * the largest so far, and what has been summed is scaled when that is raised.  Parts of a query's tokens, each with its `top`, are joined by the same scaling, first a workgroup's four
 * wavefronts', then, in a second launch, those of the workgroups that share the query.  All of this is in 32 bits; only the products' operands have 16 where the type has, exponentials
 * twice 16.
 *
 * Every cached element is read once, and takes two operations for each of the query heads that share it: memory bounds it, and where there is little of it the chain
 * offsets -> page -> keys -> scores -> values -> joined parts.  64 requests of up to 8192 tokens, 32 heads on 8 key heads of 128 bfloat16 (1075 MB): 177 to 197 us by where the pages lie in
 * memory, 5.5 to 6.1 TB/s, where a pure read of as much reaches 6.2 (6.9 past the caches); 256 requests of 2048 each: 338 us, 6.4 TB/s; one request of 128 tokens: 7.5 us.
 *
 * Many queries of one request are right but not fast: a workgroup has 16 columns, and every further 16 / (heads / keyHeads) queries read the keys and values again (4 requests with
 * 4096 queries for 4096 tokens each, the same heads: 3.57 ms, 0.15 PFLOP/s of what they see).
 */
#include <algorithm>
#include <cfloat>

#include "product_device.h"
#include "product_layer.h"

using namespace cutt;

namespace {

template <bool X>
using Is = std::integral_constant<bool, X>;

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kColumns = 16;  // of the matrix instructions: query heads of one key head
constexpr uint32_t kPhase = 1024;  // tokens whose addresses a workgroup works out at a time
constexpr uint32_t kScan = 2048;   // queries that are shared out evenly, at most
constexpr uint32_t kCut = 128;     // queries are cut at multiples of this many tokens: a tile for every wavefront
constexpr uint32_t kExtra = 128;   // tokens in whose time a workgroup begins a query and ends it (with 320 the 24 drafting requests take 67 us and not 62)

// How the work is shared out.  The tokens that the queries see, with kExtra more for each, lie one behind the other, and are cut into ranges of even lengths, one for each
// workgroup (of a key head's).  The cuts move to where a query begins or a little further in it, so that a range may take the end of one query's tokens, some whole
// queries and the begin of another.  Where there are many queries none looks at the others: each is a range, or a few of a length that is known before.
struct Attend {
  cuttHipAttendArgs a;
  uint32_t group, headTiles;  // query heads per key head, and workgroups that share them
  uint32_t most;              // neighbouring queries of one request that a workgroup takes together, a power of two: their heads share its columns
  uint32_t ranges;            // 0: each query has `pieces` of its own, of `length` tokens (the last one what is left)
  uint32_t pieces, length;
  float scale, scaleRest;     // of scores that are exponents of 2, and what it is off by: an error that all scores share does not average out
  float perRange;             // what length of a range, by all tokens, makes no more than `ranges`
  cuttHipDivisor byPage, byTiles, byHeads, byShares;  // divisions by pageSize, headTiles, the heads in a column tile and all workgroups of a range
  float* partial;             // [2 * ranges][most][heads][width]: of what begins within a query, and of what ends in one; or [queries][pieces][heads][width]
  float* tops;                // [2 * ranges][most][heads][2] or likewise: the largest score or near it, and the sum of the exponentials that it was taken off
  uint32_t* cuts;             // [queries][4]: first range, number of ranges, place among the queries that are taken together
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
  // What this one or another one of the same request sees.
  __device__ __forceinline__ void add(const Seen& o) {
    if (o.first == o.end) return;
    first = first == end ? o.first : min(first, o.first);
    end = max(end, o.end);
  }
};

// Whether query i is taken together with the one before it: both are of one request, and in one group of p.most queries.
__device__ __forceinline__ bool follows(const Attend& p, uint32_t i) {
  return p.a.owners && (i & (p.most - 1)) != 0 && i < p.a.queries && p.a.owners[i] == p.a.owners[i - 1];
}

// The queries that are taken together from `query` on; what they see in all.
__device__ __forceinline__ uint32_t together(const Attend& p, uint32_t query, Seen& seen) {
  uint32_t n = 1;
  seen = Seen(p.a, query);
#pragma unroll 1
  while (follows(p, query + n)) seen.add(Seen(p.a, query + n++));
  return n;
}

// Where a range begins or ends: before token `from` of those that `query` and the queries that are taken together with it see.
struct Cut {
  uint32_t query, from;
};

struct ScanLds {
  uint32_t low[kWaves], high[kWaves];
  Cut cut[2];
  Seen seen;          // what the range's first queries see, and how many they are
  uint32_t queries;   // (0: they are the ones behind those that the cut was in)
  uint64_t before;    // tokens before them
};

__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return x + y; }

// A workgroup's range of the tokens.
struct Range {
  Cut from, to;
  Seen seen;
  uint32_t queries;
  uint64_t before, length;  // length: of all ranges, before the cuts move.  (Queries that are cut by themselves: `before` is how many ranges this one has.)
};

// A cut that would come before token `at` of a query's `tokens` moves to the nearest multiple of kCut, or to the query's end (returned as ~0) if there would be little left.
__device__ __forceinline__ uint32_t moveCut(uint64_t at, uint32_t tokens) {
  const uint64_t to = (at + kCut / 2) / kCut * kCut;
  return to == 0 ? 0 : to + kCut / 2 <= tokens ? (uint32_t)to : ~0u;
}
// How many tokens of a query may lie before a cut at most, plus one, so that it stays within the query.
__device__ __forceinline__ uint64_t cutsEnd(uint32_t tokens) { return tokens < kCut / 2 ? 0 : (uint64_t)((tokens - kCut / 2) / kCut + 1) * kCut - kCut / 2; }

// Range number `index`, or false if it is empty.  Every workgroup scans the queries for itself.
__device__ __forceinline__ bool findRange(const Attend& p, uint32_t index, ScanLds& s, Range& r) {
  const cuttHipAttendArgs& a = p.a;
  if (!p.ranges) {
    const uint32_t query = index / p.pieces, piece = index - query * p.pieces;
    if (query >= a.queries || follows(p, query)) return false;
    r.queries = together(p, query, r.seen);
    const uint32_t tokens = r.seen.end - r.seen.first, begin = piece * p.length;
    if (piece && begin >= tokens) return false;
    const bool last = piece + 1 == p.pieces || tokens - begin <= p.length;
    r.from = {query, begin};
    r.to = {last ? query + r.queries : query, last ? 0 : begin + p.length};
    if (!last) r.before = min((tokens - 1) / p.length + 1, p.pieces);
    return true;
  }
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t each = (a.queries + kThreads - 1) / kThreads;  // neighbouring queries of this thread
  const uint32_t from = min(threadIdx.x * each, a.queries), to = min(from + each, a.queries);
  Seen seen;
  uint32_t low = 0, high = 0, queries = 0;  // (sums of 2048 numbers below 2^32 in two halves)
#pragma unroll 1
  for (uint32_t i = to; i-- > from;) {  // (the first one's stay in registers)
    queries = 0;
    if (follows(p, i)) continue;
    queries = together(p, i, seen);
    const uint32_t n = seen.end - seen.first + kExtra;
    low += n & 0xffff;
    high += n >> 16;
  }
  const uint32_t lowTo = scanOverWave(low, plus), highTo = scanOverWave(high, plus);
  if (lane == 63) {
    s.low[wave] = lowTo;
    s.high[wave] = highTo;
  }
  if (threadIdx.x < 2) s.cut[threadIdx.x] = {a.queries, 0};
  __syncthreads();
  uint64_t all = 0, before = (lowTo - low) + ((uint64_t)(highTo - high) << 16);
#pragma unroll
  for (uint32_t w = 0; w < kWaves; w++) {
    const uint64_t n = s.low[w] + ((uint64_t)s.high[w] << 16);
    all += n;
    if (w < wave) before += n;
  }
  r.length = max((uint64_t)((float)all * p.perRange) + 1, (uint64_t)kCut);  // (two cuts do not move to the same place within a query)
  const uint64_t begin = index * r.length, end = begin + r.length;
#pragma unroll 1
  for (uint32_t i = from; i < to; i++) {
    if (i != from) {
      if (follows(p, i)) continue;
      queries = together(p, i, seen);
    }
    if (!queries) continue;
    const uint32_t tokens = seen.end - seen.first;
    const uint64_t behind = before + tokens + kExtra;
    if (begin >= before && begin < behind) {
      const uint32_t first = moveCut(begin - before, tokens);
      const bool next = first == ~0u;
      s.cut[0] = {next ? i + queries : i, next ? 0 : first};
      s.seen = seen;
      s.queries = next ? 0 : queries;
      s.before = next ? behind : before;
    }
    if (end >= before && end < behind) {
      const uint32_t last = moveCut(end - before, tokens);
      s.cut[1] = {last == ~0u ? i + queries : i, last == ~0u ? 0 : last};
    }
    before = behind;
  }
  __syncthreads();
  const auto same = [](uint32_t x) __attribute__((always_inline)) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); };
  const auto same64 = [&](uint64_t x) __attribute__((always_inline)) { return (uint64_t)same((uint32_t)(x >> 32)) << 32 | same((uint32_t)x); };
  r.from = {same(s.cut[0].query), same(s.cut[0].from)};
  r.to = {same(s.cut[1].query), same(s.cut[1].from)};
  r.length = same64(r.length);
  if (r.from.query >= a.queries || (r.from.query == r.to.query && r.from.from == r.to.from)) return false;
  r.seen.request = same(s.seen.request);
  r.seen.first = same(s.seen.first);
  r.seen.end = same(s.seen.end);
  r.queries = same(s.queries);
  r.before = same64(s.before);
  if (!r.queries) r.queries = together(p, r.from.query, r.seen);
  return true;
}

// The tokens' scores and their weighted values, a tile of tokens at a time: keys times queries give the scores, heads along the instruction's columns, and each lane
// then holds the exponentials of its head's tokens just as the second product, values turned times exponentials, wants them.
//
// Keys and values are the instructions' A operands, 16 tokens or 16 elements, queries and exponentials their B operands: up to 16 heads that share the keys, so that few heads leave columns idle
// but no more is read, and no product waits for another wavefront.
//
// DIRECT: a wavefront's tiles go from memory to its own part of LDS, token by token, 16-byte pieces of a row exchanged so that a fragment's lanes find theirs in different banks.  Else (rows
// off the 16-byte grid) they go to registers, keys as the fragments want them and of a token's values VD neighbouring elements to each lane.  So much as is on its way to registers has to
// have its registers: with aligned rows too the 64 requests above take 229 us this way, not 194, 72 queries of 80 floats 83 and not 50.
template <typename T, int DP, bool DIRECT>
struct Tokens {
  static constexpr int E = kPer16<T>;
  static constexpr int TILE = sizeof(T) == 2 ? 32 : 16;  // tokens
  static constexpr int SUB = TILE / 16;                  // tiles of scores
  static constexpr int STEPS = DP / (4 * E);             // 16 bytes of each of the lane quarters
  static constexpr int VD = DP / 16;                     // fragments of values: 16 elements each
  static constexpr int VE = VD < E ? VD : E, VC = VD / VE;  // in pieces of 16 bytes, or a smaller one
  static constexpr int VT = TILE / 4;                    // tokens whose values a lane has
  static constexpr int PIECES = DP / E;                  // of 16 bytes per row
  static constexpr int ROWS = 64 / PIECES;               // rows that a wavefront's load brings, or (PIECES = 64) one
  static constexpr int LOADS = TILE / ROWS;
  static constexpr int NEAR = PIECES < 16 ? 16 / PIECES : 1;  // rows within 256 bytes, all banks
  static constexpr uint32_t BYTES = DIRECT ? 2 * TILE * DP * sizeof(T) : 0;  // of a wavefront's keys and values in LDS
  static __device__ __forceinline__ uint32_t keyPlace(uint32_t row, uint32_t piece) { return row * PIECES + (piece ^ (row / NEAR & (PIECES < 16 ? PIECES - 1 : 15))); }
  // (two neighbouring pieces of four rows are read at a time)
  static __device__ __forceinline__ uint32_t valuePlace(uint32_t row, uint32_t piece) {
    return row * PIECES + (sizeof(T) == 2 ? piece ^ (2 * (row / NEAR) & (PIECES < 16 ? PIECES - 1 : 15)) : piece);
  }
  // Which element of its head the i-th of fragment j is.
  static __device__ __forceinline__ uint32_t elementOf(uint32_t j, uint32_t i) {
    if (!DIRECT) return i * VD + j;
    return sizeof(T) == 2 ? j * 16 + i : j / 4 * 64 + i * 4 + j % 4;
  }
};

// What a tile holds behind a row's end: the queries' zeros must not meet just anything there.
__device__ const uint4 kZeros = {};

constexpr int kStream = 2;  // non-temporal: a step reads every cached token once.  64 requests of 4096 tokens, 8 key heads of 128 bfloat16 (1074 MB): 181 us so, 204 without

// 16 bytes from each lane's address to LDS, side by side from `to` on, which is the same for all lanes.
__device__ __forceinline__ void loadToLds(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, kStream);
}

// Loads to LDS that have left and may still be on their way: `n` at most.
template <int N>
__device__ __forceinline__ void waitForLoads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);  // vmcnt alone
  asm volatile("" ::: "memory");
}

// What stands for a weight above 0 where only infinities are wanted: so small that no sum of finite values leaves the range of 32 bits.
template <typename T>
constexpr float kSome = std::is_same_v<T, _Float16> ? 0x1p-15f : 0x1p-64f;

constexpr float kLn2 = 0.69314718055994530942f;
// Scores may exceed what they are taken off from by kSlack (times log2 e) before it is raised.  Half's exponentials are multiplied by kTimes, so that they use the type's range: they stay
// below 2^16, and of its smallest step, 2^-24, the half that is lost in both parts of an exponential is 2^-40 of the largest.
template <typename T>
constexpr float kSlack = std::is_same_v<T, _Float16> ? 0.9f : 8.0f;
template <typename T>
constexpr float kTimes = std::is_same_v<T, _Float16> ? 0x1p15f : 1.0f;
__device__ __forceinline__ float exp2Of(float x) { return __builtin_amdgcn_exp2f(x); }
// What scores are taken off from before they are exponents, unless there are only scores of -infinity.  (Finite: a score of +infinity has the exponential +infinity.)
__device__ __forceinline__ float baseOf(float top) { return top == -INFINITY ? 0.0f : fminf(top, FLT_MAX); }

struct PhaseLds {
  uint64_t offset[kPhase];      // of the phase's tokens in the caches, in elements
  uint64_t there[kPhase / 64];  // which of them have a page
};

template <typename T, int DP, bool DIRECT>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void attendKernel(Attend p, uint32_t firstRange) {
  using S = Tokens<T, DP, DIRECT>;
  constexpr int E = S::E, TILE = S::TILE, SUB = S::SUB, STEPS = S::STEPS, VD = S::VD, VE = S::VE, VC = S::VC, VT = S::VT;
  constexpr uint32_t ALL = TILE == 32 ? ~0u : (1u << (TILE & 31)) - 1;
  const cuttHipAttendArgs& a = p.a;
  extern __shared__ char lds[];
  PhaseLds& tokens = *reinterpret_cast<PhaseLds*>(lds);
  const uint32_t lane = threadIdx.x & 63, l = lane & 15, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int width = (int)a.width;
  const float scale = p.scale, scaleRest = p.scaleRest;
  // Workgroups that follow each other go to the XCDs in turn: so that none has much more to do than another, a range's heads follow each other, and the eight ranges that
  // do are turned on from eight to eight (every fourth range may be all that has work, as drafted tokens are taken together).
  const uint32_t shares = a.keyHeads * p.headTiles, at = divide(blockIdx.x, p.byShares), share = blockIdx.x - at * shares;
  const uint32_t index = firstRange + (at & ~7u) + ((at + at / 8) & 7);
  const uint32_t keyHead = divide(share, p.byTiles), headTile = share - keyHead * p.headTiles;
  const uint32_t head0 = keyHead * p.group + headTile * kColumns, nHeads = min(p.group - headTile * kColumns, kColumns);
  const T* const kHead = static_cast<const T*>(a.k) + keyHead * a.cacheHead;
  const T* const vHead = static_cast<const T*>(a.v) + keyHead * a.cacheHead;
  Range range;
  if (!findRange(p, index, *reinterpret_cast<ScanLds*>(lds), range)) return;
  for (;;) {
    // Of the range's next queries, the part of their tokens that is in it.
    const uint32_t queries = range.queries, tokensInAll = range.seen.end - range.seen.first;
    const bool ends = range.from.query != range.to.query;  // with the queries' last token
    const bool cut = range.from.from > 0 || !ends;
    const uint32_t slot = 2 * index + (range.from.from == 0);
    Seen seen = range.seen;
    if (!ends) seen.end = seen.first + range.to.from;
    seen.first += range.from.from;
    const int32_t* const table = a.tables + (uint64_t)seen.request * a.tableWidth;

    // The pages of a phase's tokens: lane i of wavefront w has token (w + j * kWaves) * 64 + i.
    constexpr uint32_t PER = kPhase / kThreads;
    int32_t page[PER];
    const auto askPages = [&](uint32_t phase) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t j = 0; j < PER; j++) {
        const uint32_t t = phase + (j * kWaves + wave) * 64 + lane;  // (below 2^32: positions are below 2^31)
        page[j] = -1;
        if (t < seen.end) page[j] = table[divide(t, p.byPage)];
      }
    };
    const auto placeTokens = [&](uint32_t phase) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t j = 0; j < PER; j++) {
        const uint32_t block = j * kWaves + wave, t = phase + block * 64 + lane;
        const bool is = (uint32_t)page[j] < a.pages;
        const uint64_t there = __ballot(is);
        const uint64_t to = is ? (uint64_t)(uint32_t)page[j] * a.pageStride + (t - divide(t, p.byPage) * a.pageSize) * a.slotStride : 0;
        const uint32_t some = there ? __builtin_ctzll(there) : 0;  // a token that is there stands in for one that is not, whose value counts nothing
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(to >> 32), some) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)to, some);
        tokens.offset[block * 64 + lane] = is ? to : other;
        if (lane == 0) tokens.there[block] = there;
      }
    };
    askPages(seen.first);

    // This lane's column: a head of one of the queries, and what that sees.
    const uint32_t place = p.most > 1 ? divide(l, p.byHeads) : 0, head = head0 + l - place * nHeads;
    const bool column = place < queries && l - place * nHeads < nHeads;
    const uint32_t query = range.from.query + (column ? place : 0);
    Seen own = range.seen;
    uint32_t from = own.first, till = own.end;  // what all columns see
    if (queries > 1) {
      own = Seen(a, query);
      from = column ? own.first : 0;
      till = column ? own.end : 0xffffffffu;
#pragma unroll
      for (int i = 1; i < 16; i *= 2) {
        from = max(from, (uint32_t)__shfl_xor(from, i));
        till = min(till, (uint32_t)__shfl_xor(till, i));
      }
      from = __builtin_amdgcn_readfirstlane(from);
      till = __builtin_amdgcn_readfirstlane(till);
    }
    if (!column) own.first = own.end = 0;
    Chunk<T> q[STEPS];
    {
      const T* const line = static_cast<const T*>(a.q) + query * a.qStride + (column ? head : head0) * a.qHead;
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        const int d = (s * 4 + quarter) * E;
        q[s] = loadChunk(line + d, column ? width - d : 0);
      }
    }
    float top, sum;  // of this lane's column: what scores are taken off from (times log2 e), the exponentials of this quarter's tokens
    Acc acc[VD];
    // An exponential's second part, 0 or below 0 as often as not, makes NaN of an infinite value.  Where the 16-bit types have got NaN, all is done again with one number in place
    // of all exponentials above 0, in both parts: what is infinite then takes the place of NaN.  (92 requests of up to 97 tokens, two queries each, 32 heads of 192 halves: 156 us; 148
    // without; 179 where the tiles at queries' ends, and all when done again, have a product of their own for such values.)
    bool again = false;
    float limit = INFINITY, times = kTimes<T>;  // (again: 0 and twice as much)

    // DIRECT: the wavefront's tiles in LDS.
    Chunk<T>* const keys = reinterpret_cast<Chunk<T>*>(lds + sizeof(PhaseLds) + wave * S::BYTES);
    Chunk<T>* const values = keys + TILE * S::PIECES;
    Chunk<T> k[DIRECT ? 1 : SUB][DIRECT ? 1 : STEPS];
    AlignedVec<T, VE> v[DIRECT ? 1 : VT][VC];
    const auto toLds = [&](const T* head, Chunk<T>* to, uint32_t tile, auto place) __attribute__((always_inline)) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);  // (lgkmcnt: what was in this place has been read)
#pragma unroll
      for (int n = 0; n < S::LOADS; n++) {
        // The lane's place in LDS is fixed; what it loads is the piece that belongs there.
        const uint32_t row = n * S::ROWS + lane / S::PIECES, at = lane % S::PIECES, piece = place(row, at) - row * S::PIECES;
        const T* const from = head + (tokens.offset[tile * TILE + row] + piece * E);
        loadToLds(piece * E < (uint32_t)width ? (const void*)from : (const void*)&kZeros, to + n * 64);
      }
      asm volatile("" ::: "memory");
    };
    const auto loadKeys = [&](uint32_t tile) __attribute__((always_inline)) {
      if constexpr (DIRECT) {
        toLds(kHead, keys, tile, S::keyPlace);
      } else {
#pragma unroll
        for (int i = 0; i < SUB; i++) {
          const T* const line = kHead + tokens.offset[tile * TILE + i * 16 + l];
#pragma unroll
          for (int s = 0; s < STEPS; s++) {
            const int d = (s * 4 + quarter) * E;
            k[i][s] = loadChunk(line + d, width - d);
          }
        }
      }
    };
    const auto loadValues = [&](uint32_t tile) __attribute__((always_inline)) {
      if constexpr (DIRECT) {
        toLds(vHead, values, tile, S::valuePlace);
      } else {
#pragma unroll
        for (int t = 0; t < VT; t++) {
          const T* const line = vHead + tokens.offset[tile * TILE + t / 4 * 16 + quarter * 4 + t % 4];
#pragma unroll
          for (int c = 0; c < VC; c++) {
            const int d = (int)l * VD + c * VE;
            if (d + VE <= width) {
              v[t][c] = __builtin_bit_cast(AlignedVec<T, VE>, *reinterpret_cast<const Vec<T, VE>*>(line + d));
            } else {
              v[t][c] = {};
#pragma unroll
              for (int e = 0; e < VE; e++)
                if (d + e < width) v[t][c][e] = line[d + e];
            }
          }
        }
      }
    };
    Acc score[SUB];
    const auto scores = [&]() __attribute__((always_inline)) {
      const auto keysOf = [&](int i, int s) __attribute__((always_inline)) -> Chunk<T> {
        if constexpr (DIRECT) return keys[S::keyPlace(i * 16 + l, s * 4 + quarter)];
        else return k[i][s];
      };
      if constexpr (sizeof(T) == 4) {
        // Four sums of a quarter of the terms each: their roundings add up to half as much, and no instruction waits for the one before it.
        Acc part[4] = {};
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
          const Chunk<T> of = keysOf(0, s);
#pragma unroll
          for (int e = 0; e < 4; e++) part[e] = multiply(of[e], q[s][e], part[e]);
        }
        score[0] = (part[0] + part[1]) + (part[2] + part[3]);
      } else {
#pragma unroll
        for (int i = 0; i < SUB; i++) score[i] = Acc(0);
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
          for (int i = 0; i < SUB; i++) score[i] = multiply(keysOf(i, s), q[s], score[i]);
      }
    };
    // Weighted values added to the sums; with a mask those of the lane's tokens t with bit t of it, for the columns that `mine` says.
    const auto addWeighted = [&](auto masked, uint32_t mask, bool mine) __attribute__((always_inline)) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < VD; j += VE) {
          Acc o[VE];
#pragma unroll
          for (int e = 0; e < VE; e++) o[e] = acc[j + e];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            AlignedVec<T, VE> line;
            if constexpr (DIRECT) line = values[S::valuePlace(quarter * 4 + r, j / 4 * 16 + l)];
            else line = v[r][j / VE];
#pragma unroll
            for (int e = 0; e < VE; e++) o[e] = multiply(!masked || mask >> r & 1 ? line[e] : 0.0f, score[0][r], o[e]);
          }
#pragma unroll
          for (int e = 0; e < VE; e++) acc[j + e] = !masked || mine ? o[e] : acc[j + e];
        }
      } else {
        // Exponentials in two parts, what the type rounds and what it leaves, so that they count with 16 bits and more.  (The matrix unit has the time: with the first
        // part alone a pass takes as long.  A third part, 24 bits of bfloat16: 64 requests of up to 8192 tokens, 8 key heads of 64, 116 -> 136 us for its registers.)
        Chunk<T> high, low;
#pragma unroll
        for (int t = 0; t < 8; t++) {
          const float e = score[t / 4][t % 4] > limit ? kSome<T> : score[t / 4][t % 4];
          high[t] = (T)(e * kTimes<T>);
          low[t] = (T)fmaf(e, times, -(float)high[t]);
        }
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
        Words keep;
        if constexpr (masked)
#pragma unroll
          for (int i = 0; i < 4; i++) keep[i] = (mask >> (2 * i) & 1 ? 0xffffu : 0u) | (mask >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < VD; j++) {
          // Values turned: of eight tokens one element of each, two tokens to a word.
          Words turned;
          if constexpr (DIRECT) {
            // Sixteen lanes load 16 elements of 4 tokens, 8 bytes each, and get one element of the four.
            typedef short Four __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) Four* Lds;
            union {
              Four four[2];
              Words whole;
            } u;
#pragma unroll
            for (int h = 0; h < 2; h++)
              u.four[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(reinterpret_cast<char*>(values + S::valuePlace(h * 16 + quarter * 4 + l / 4, j * 2 + (l & 3) / 2)) + (l & 1) * 8));
            turned = u.whole;
          } else {
            typedef uint32_t Piece __attribute__((ext_vector_type(VE / 2)));
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t even = __builtin_bit_cast(Piece, v[2 * i][j / VE])[j % VE / 2], odd = __builtin_bit_cast(Piece, v[2 * i + 1][j / VE])[j % VE / 2];
              turned[i] = __builtin_amdgcn_perm(odd, even, j % 2 ? 0x07060302 : 0x05040100);
            }
          }
          if constexpr (masked) turned &= keep;
          const Chunk<T> of = __builtin_bit_cast(Chunk<T>, turned);
          const Acc o = multiply(of, low, multiply(of, high, acc[j]));
          acc[j] = !masked || mine ? o : acc[j];
        }
      }
    };
    // A tile's part of the sums: tokens `first` on; full: all of them have a page.
    const auto addValues = [&](uint32_t tile, uint32_t first, bool full) __attribute__((always_inline)) {
      const bool whole = full && first >= from && first + TILE <= till;  // every column sees every token
      uint32_t mine = 0;  // of the lane's tokens t those that have a page
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++)  // (what the rest adds to a score of infinity must not be the other infinity)
          score[i][r] = fmaf(score[i][r], scale, __builtin_amdgcn_fmed3f(score[i][r] * scaleRest, -FLT_MAX, FLT_MAX));
      if (!whole) {
        const uint32_t there = (uint32_t)(tokens.there[tile * TILE / 64] >> (tile * TILE % 64));
#pragma unroll
        for (int t = 0; t < VT; t++) {
          const uint32_t at = t / 4 * 16 + quarter * 4 + t % 4;
          mine |= (there >> at & 1) << t;
          const bool is = (there >> at & 1) & (first + at >= own.first) & (first + at < own.end);
          score[t / 4][t % 4] = is ? score[t / 4][t % 4] : -INFINITY;
        }
      }
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) most = fmaxf(most, score[i][r]);
      if (__any(most > top + kSlack<T>)) {
        most = overQuarters(most, [](float x, float y) { return fmaxf(x, y); });
        const float next = fmaxf(most, top), less = exp2Of(top - baseOf(next));
        top = next;
        sum *= less;
#pragma unroll
        for (int j = 0; j < VD; j++) acc[j] *= again ? 1.0f : less;
      }
      const float base = baseOf(top);
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          score[i][r] = exp2Of(score[i][r] - base);
          sum += score[i][r];
        }
      if (whole) {
        addWeighted(Is<false>{}, 0, true);
      } else {
        // What a column does not see must not meet its exponential of 0, which an infinity would make NaN: one query after the other takes the values that it sees,
        // and the columns of the others stay as they were.
#pragma unroll 1
        for (uint32_t n = 0; n < queries; n++) {
          const uint32_t begin = __builtin_amdgcn_readlane(own.first, n * nHeads), end = __builtin_amdgcn_readlane(own.end, n * nHeads);
          uint32_t with = 0;
#pragma unroll
          for (int t = 0; t < VT; t++) {
            const uint32_t at = first + t / 4 * 16 + quarter * 4 + t % 4;
            with |= (uint32_t)((at >= begin) & (at < end)) << t;
          }
          addWeighted(Is<true>{}, with & mine, place == n);
        }
      }
    };

    for (;;) {
      top = -INFINITY;
      sum = 0;
#pragma unroll
      for (int j = 0; j < VD; j++) acc[j] = Acc(0);
      for (uint32_t phase = seen.first; phase < seen.end; phase += kPhase) {
        __syncthreads();
        placeTokens(phase);
        __syncthreads();
        askPages(phase + kPhase);
        // The wavefront's tiles: every kWaves-th of those that have a token.
        static_assert(kPhase / TILE <= 64, "a lane for every tile");
        uint32_t there = 0;
        if (lane < kPhase / TILE) there = (uint32_t)(tokens.there[lane * TILE / 64] >> (lane * TILE % 64)) & ALL;
        uint64_t left = __ballot(there != 0) & (0x1111111111111111ull << wave);
        const uint64_t full = __ballot(there == ALL);
        if (!left) continue;
        uint32_t tile = __builtin_ctzll(left);
        loadKeys(tile);
        loadValues(tile);
        // The next tile's keys are asked for as soon as this one's have been used, its values likewise; behind the last tile the same ones again, which nobody waits
        // for: with a condition around loads to registers the compiler, which counts the loads that it waits for, would have to wait for all.
        for (;;) {
          if constexpr (DIRECT) waitForLoads<S::LOADS>();  // (the values' loads may be under way)
          scores();
          left &= left - 1;
          const uint32_t next = left ? __builtin_ctzll(left) : tile;
          if constexpr (DIRECT) {
            if (left) {
              loadKeys(next);
              waitForLoads<S::LOADS>();
            } else {
              waitForLoads<0>();
            }
          } else {
            loadKeys(next);
          }
          addValues(tile, phase + tile * TILE, full >> tile & 1);
          if (!left) break;
          loadValues(next);
          tile = next;
        }
      }

      // The wavefronts' parts together.
      sum = overQuarters(sum, [](float x, float y) { return x + y; });
      __syncthreads();
      float* const tops = reinterpret_cast<float*>(lds);            // [waves][columns]
      float* const sums = tops + kWaves * kColumns;
      uint32_t* const odds = reinterpret_cast<uint32_t*>(sums + kWaves * kColumns);  // [waves]: whether there is NaN
      float* const parts = sums + kWaves * kColumns + kWaves;       // [waves][columns][DP + 4]
      constexpr uint32_t PITCH = DP + 4;
      if (quarter == 0) {
        tops[wave * kColumns + l] = top;
        sums[wave * kColumns + l] = sum;
      }
      if constexpr (sizeof(T) == 2) {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < VD; j++) odd |= __builtin_isunordered(acc[j][0], acc[j][1]) | __builtin_isunordered(acc[j][2], acc[j][3]);
        odd = __any(odd && column);
        if (lane == 0) odds[wave] = odd;
      }
      __syncthreads();
      uint32_t odd = 0;
      if constexpr (sizeof(T) == 2)
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) odd |= odds[w];
      float all = -INFINITY;
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) all = fmaxf(all, tops[w * kColumns + l]);
      const float mine = (again ? 1.0f : exp2Of(top - baseOf(all))) / kTimes<T>;
      if (column)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
          for (int j = 0; j < VD; j++) parts[(wave * kColumns + l) * PITCH + S::elementOf(j, quarter * 4 + r)] = acc[j][r] * mine;
      __syncthreads();
      for (uint32_t c = wave; c < queries * nHeads; c += kWaves) {
        const uint32_t n = p.most > 1 ? divide(c, p.byHeads) : 0, h = head0 + c - n * nHeads;
        float m = -INFINITY, of = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) m = fmaxf(m, tops[w * kColumns + c]);
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) of += sums[w * kColumns + c] * exp2Of(tops[w * kColumns + c] - baseOf(m));
        const bool none = of == 0 && m == -INFINITY;
        const uint64_t to = range.from.query + n;
        const uint64_t row = (p.ranges ? (uint64_t)slot * p.most + n : to * p.pieces + (index - range.from.query * p.pieces)) * a.heads + h;
        for (uint32_t d = lane; d < a.width; d += 64) {
          float o = 0;
#pragma unroll
          for (uint32_t w = 0; w < kWaves; w++) o += parts[(w * kColumns + c) * PITCH + d];
          float* const part = p.partial + (row * a.width + d);
          T* const out = static_cast<T*>(a.out) + (to * a.outStride + h * a.outHead + d);
          if (again && (fabsf(o) <= FLT_MAX || (cut ? *part == *part : *out == *out))) continue;  // (this thread has written it before)
          if (cut) *part = o;
          else *out = (T)(none ? 0.0f : o / of);
        }
        if (lane == 0) {
          if (cut) {
            p.tops[row * 2] = m;
            p.tops[row * 2 + 1] = of;
          } else if (a.logSums) a.logSums[to * a.heads + h] = none ? -INFINITY : (m + __log2f(of)) * kLn2;
        }
      }
      if (sizeof(T) == 4 || again || !__builtin_amdgcn_readfirstlane(odd)) break;
      again = true;
      limit = 0.0f;
      times = 2 * kTimes<T>;
      askPages(seen.first);
    }

    if ((p.ranges || p.pieces > 1) && range.from.from == 0 && share == 0 && threadIdx.x < queries) {
      uint32_t* const to = p.cuts + (range.from.query + threadIdx.x) * 4;
      to[0] = index;
      to[1] = ends ? 1 : !p.ranges ? (uint32_t)range.before : (uint32_t)((range.before + cutsEnd(tokensInAll) + range.length - 1) / range.length) - index;
      to[2] = threadIdx.x;
    }
    range.from = {range.from.query + queries, 0};
    if (!ends || range.from.query >= a.queries || (range.from.query == range.to.query && range.to.from == 0)) break;
    range.before += tokensInAll + kExtra;
    range.queries = together(p, range.from.query, range.seen);
    __syncthreads();  // (the next query's tokens take the place of what has been joined)
  }
}

// The parts of the queries that were cut, joined.  A workgroup takes a query's head; its wavefronts share the parts.
template <typename T>
__global__ __launch_bounds__(kThreads) void joinKernel(Attend p) {
  const cuttHipAttendArgs& a = p.a;
  __shared__ float tops[kWaves], sums[kWaves];
  __shared__ float parts[kWaves][CUTT_MAX_HEAD_WIDTH];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint64_t at = blockIdx.x; at < (uint64_t)a.queries * a.heads; at += gridDim.x) {
    const uint32_t query = (uint32_t)(at / a.heads), head = (uint32_t)(at % a.heads);
    const uint32_t* const cut = p.cuts + query * 4;
    const uint32_t first = cut[0], ranges = cut[1];
    if (ranges <= 1) continue;
    // Its first range ends in it, the others begin in it.
    const auto rowOf = [&](uint32_t i) __attribute__((always_inline)) {
      return (p.ranges ? (2 * ((uint64_t)first + i) + (i == 0)) * p.most + cut[2] : (uint64_t)query * p.pieces + i) * a.heads + head;
    };
    // A wavefront joins every kWaves-th of them, AT at a time, whose loads go out together.
    constexpr uint32_t AT = 4, PER = CUTT_MAX_HEAD_WIDTH / 64;
    float m = -INFINITY, n = 0, o[PER] = {};
    for (uint32_t i = wave; i < ranges; i += kWaves * AT) {
      float top[AT], sum[AT], part[AT][PER];
#pragma unroll
      for (uint32_t u = 0; u < AT; u++) {
        const bool is = i + u * kWaves < ranges;  // (behind the last one nothing, which its infinities must not meet)
        const uint64_t row = rowOf(is ? i + u * kWaves : ranges - 1);
        top[u] = is ? p.tops[row * 2] : -INFINITY;
        sum[u] = is ? p.tops[row * 2 + 1] : 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) part[u][j] = is && lane + j * 64 < a.width ? p.partial[row * a.width + lane + j * 64] : 0.0f;
      }
      float next = m;
#pragma unroll
      for (uint32_t u = 0; u < AT; u++) next = fmaxf(next, top[u]);
      const float less = exp2Of(m - baseOf(next));
      n *= less;
#pragma unroll
      for (uint32_t j = 0; j < PER; j++) o[j] *= less;
#pragma unroll
      for (uint32_t u = 0; u < AT; u++) {
        const float share = exp2Of(top[u] - baseOf(next));
        n += share * sum[u];
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) o[j] += share * part[u][j];
      }
      m = next;
    }
    if (lane == 0) {
      tops[wave] = m;
      sums[wave] = n;
    }
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) parts[wave][lane + j * 64] = o[j];
    __syncthreads();
    if (threadIdx.x < a.width) {
      float all = 0, sum = 0, top = -INFINITY;
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) top = fmaxf(top, tops[w]);
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) {
        const float share = exp2Of(tops[w] - baseOf(top));
        sum += share * sums[w];
        all += share * parts[w][threadIdx.x];
      }
      const bool none = sum == 0 && top == -INFINITY;
      static_cast<T*>(a.out)[query * a.outStride + head * a.outHead + threadIdx.x] = (T)(none ? 0.0f : all / sum);
      if (a.logSums && threadIdx.x == 0) a.logSums[(uint64_t)query * a.heads + head] = none ? -INFINITY : (top + __log2f(sum)) * kLn2;
    }
    __syncthreads();
  }
}

constexpr uint32_t kMaxBlocks = 1u << 22;

// Queries are cut by themselves if they are enough for all CUs even when kColumns / group of them are taken together (256 requests of 2048 tokens, 8 key heads: 338 us, with even ranges
// 360; of up to 256 tokens 48 and 53; but 24 requests of three drafted tokens, 12 heads: 104 and 50), or have so few tokens that a part of them is no less time (8 requests, 8 key heads:
// 256 tokens 9.9 and 12.9 us, 512 tokens 14.3 and 13.3).  Their pieces are long, so that what a workgroup does before and after its tokens (5 us) is little of its time (16 pieces of 1024
// tokens at least: the 338 become 370), and there are no more than kPieceBlocks workgroups, which also bounds the workspace.
constexpr uint32_t kManyBlocks = 256, kShort = 256, kPieces = 8, kLeastPiece = 2048, kPieceBlocks = 16384;

Attend planAttend(uint32_t queries, uint32_t heads, uint32_t keyHeads, uint32_t width, uint32_t pageSize, uint32_t tableWidth, uint32_t window) {
  Attend p = {};
  p.group = heads / keyHeads;
  p.headTiles = (p.group + kColumns - 1) / kColumns;
  for (p.most = 1; p.most * 2 * p.group <= kColumns;) p.most *= 2;
  p.byPage = cuttHipMakeDivisor(pageSize);
  p.byTiles = cuttHipMakeDivisor(p.headTiles);
  p.byShares = cuttHipMakeDivisor(keyHeads * p.headTiles);
  p.byHeads = cuttHipMakeDivisor(std::min(p.group, kColumns));
  const uint64_t shares = (uint64_t)keyHeads * p.headTiles, blocks = queries * shares;
  const uint64_t reach = std::min((uint64_t)tableWidth * pageSize, window ? (uint64_t)window + p.most : (uint64_t)1 << 31);
  if (queries > kScan || blocks / p.most >= kManyBlocks || reach <= kShort) {
    p.pieces = (uint32_t)std::max<uint64_t>(std::min({(uint64_t)kPieces, kPieceBlocks / std::max<uint64_t>(blocks, 1), reach / kLeastPiece}), 1);
    p.length = (uint32_t)((reach + p.pieces * kCut - 1) / (p.pieces * kCut) * kCut);
    return p;
  }
  // As many workgroups as run at a time: two to a CU, which LDS and registers allow, three of narrow heads, one of wide ones.  (Half as many: the 64 requests above 250 us, twice as many 207.)
  p.ranges = std::max(1u, (width <= 64 ? 768 : width <= 128 ? 512 : 256) / (uint32_t)shares);
  p.perRange = 1.0001f / p.ranges;
  return p;
}

// Parts of queries that the workspace has room for.
size_t rowsOf(const Attend& p, uint32_t queries) { return !queries ? 0 : p.ranges ? 2 * (size_t)p.ranges * p.most : p.pieces > 1 ? (size_t)queries * p.pieces : 0; }

template <typename T, int DP, bool DIRECT>
int attend(const Attend& p, void* stream) {
  const size_t space = sizeof(PhaseLds) + kWaves * Tokens<T, DP, DIRECT>::BYTES, join = (2 * kWaves * kColumns + kWaves + kWaves * kColumns * (DP + 4)) * 4;
  const size_t lds = std::max({space, sizeof(ScanLds), join});
  const uint32_t shares = p.a.keyHeads * p.headTiles;
  const uint32_t most = std::max(1u, (1u << 20) / shares) * 8;  // (a launch's lanes stay below 2^32)
  const uint64_t ranges = p.ranges ? p.ranges : (uint64_t)p.a.queries * p.pieces;
  for (uint64_t first = 0; first < ranges; first += most) {
    const uint32_t blocks = ((uint32_t)std::min<uint64_t>(ranges - first, most) + 7) / 8 * 8 * shares;
    if (int e = launchRows(attendKernel<T, DP, DIRECT>, blocks, kThreads, lds, stream, p, (uint32_t)first)) return e;
  }
  if (!p.ranges && p.pieces == 1) return 0;
  return launchRows(joinKernel<T>, (uint32_t)std::min<uint64_t>((uint64_t)p.a.queries * p.a.heads, kMaxBlocks), kThreads, 0, stream, p);
}

template <typename T, bool DIRECT>
int attendWide(const Attend& p, void* stream) {
  return p.a.width <= 64 ? attend<T, 64, DIRECT>(p, stream) : p.a.width <= 128 ? attend<T, 128, DIRECT>(p, stream) : attend<T, 256, DIRECT>(p, stream);
}

// (what both ways cost is said where Tokens is)
template <typename T>
int attendType(const Attend& p, void* stream) {
  const cuttHipAttendArgs& a = p.a;
  const uint64_t grid = (uintptr_t)a.k | (uintptr_t)a.v | (a.pageStride | a.slotStride | a.cacheHead | a.width) * sizeof(T);
  return grid % 16 == 0 ? attendWide<T, true>(p, stream) : attendWide<T, false>(p, stream);
}

}  // namespace

extern "C" size_t cuttHipAttendWorkspace(uint32_t queries, uint32_t heads, uint32_t keyHeads, uint32_t width, uint32_t pageSize, uint32_t tableWidth, uint32_t window) {
  const Attend p = planAttend(queries, heads, keyHeads, width, pageSize, tableWidth, window);
  const size_t rows = rowsOf(p, queries) * heads;
  return rows ? (rows * (width + 2) + 4 * (size_t)queries) * 4 : 0;
}

extern "C" int cuttHipAttend(const cuttHipAttendArgs* a, int type, void* stream) {
  Attend p = planAttend(a->queries, a->heads, a->keyHeads, a->width, a->pageSize, a->tableWidth, a->window);
  p.a = *a;
  const double scale = a->scale * 1.44269504088896340736;
  p.scale = (float)std::max(std::min(scale, (double)FLT_MAX), -(double)FLT_MAX);  // (the rest has what the largest scales exceed that by)
  p.scaleRest = (float)(scale - p.scale);
  float* const space = static_cast<float*>(a->workspace);
  const size_t rows = rowsOf(p, a->queries) * a->heads;
  p.tops = space;
  p.partial = space + 2 * rows;
  p.cuts = reinterpret_cast<uint32_t*>(p.partial + rows * a->width);
  switch (type) {
    case CUTT_ROW_F32: return attendType<float>(p, stream);
    case CUTT_ROW_F16: return attendType<_Float16>(p, stream);
    default: return attendType<__bf16>(p, stream);
  }
}
