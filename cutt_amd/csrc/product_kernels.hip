/*
 * product_kernels.hip - rows grouped by expert times their experts' weights, and the weights' gradient (cutt_products.h).
 *
 * A group's product is cut into tiles of results, one for a workgroup.  The groups' sizes are known on the GPU alone: the host launches as many workgroups as any sizes can
 * need, each finds its tile in the offsets, and those that are too many end.  No sum crosses a workgroup, so the results do not depend on timing, and an
 * expert's sums run over all its rows in 32 bits, rounded once.
 *
 * What bounds it: with few rows per group the weights, read once (512 rows of 4096 x 1536 over 128 groups, bfloat16: 242 us, 6.6 TB/s); with many the matrix
 * instructions and what feeds them (131072 rows of the same: 1640 us, 1.0 PFLOP/s; one group of 8192 rows and 8192 x 8192 weights 1.2, transposed 1.33, its gradient
 * 0.95); the gradient of few rows writes its result (64 experts of 2048 x 1536, 16 rows each: 110 us, 3.7 TB/s).
 */
#include <algorithm>

#include "product_device.h"
#include "product_layer.h"

using namespace cutt;

namespace {

// A group, the end of its rows, and the first row of one of its tiles.
struct Segment {
  uint32_t group, first, end;
  uint32_t before, tiles;  // tiles of the groups before it, and of its own
};

__device__ __forceinline__ uint32_t boundOf(const cuttHipProductArgs& a, uint32_t e) { return min((uint32_t)max(a.offsets[e], 0), a.rows); }

// The rows of tile number `tile` when every group is cut into tiles of BM rows, or false if there are fewer.  Each wavefront looks for itself, 64 groups at a
// time.  (Sums of tiles stop at 2^31 - 1: groups that share rows can have more, and what is found then is checked.)
template <int BM>
__device__ __forceinline__ bool findTile(const cuttHipProductArgs& a, uint32_t tile, Segment& s) {
  const uint32_t lane = threadIdx.x & 63;
  const auto capped = [](uint32_t x, uint32_t y) { return min(x + y, 0x7fffffffu); };
  uint32_t before = 0;
  for (uint32_t base = 0; base < a.groups; base += 64) {
    const uint32_t e = base + lane;
    uint32_t lo = 0, hi = 0;
    if (e < a.groups) {
      lo = boundOf(a, e);
      hi = max(lo, boundOf(a, e + 1));
    }
    const uint32_t n = (hi - lo + BM - 1) / BM, upTo = capped(before, scanOverWave(n, capped));
    const uint64_t found = __ballot(tile < upTo);
    if (found) {
      const uint32_t at = __builtin_ctzll(found);
      s.group = __builtin_amdgcn_readfirstlane(base + at);
      s.end = __builtin_amdgcn_readlane(hi, at);
      const uint64_t first = (uint64_t)__builtin_amdgcn_readlane(lo, at) + (uint64_t)(tile - __builtin_amdgcn_readlane(upTo - n, at)) * BM;
      s.first = __builtin_amdgcn_readfirstlane((uint32_t)first);
      s.before = __builtin_amdgcn_readlane(upTo - n, at);
      s.tiles = __builtin_amdgcn_readlane(n, at);
      return first < s.end;
    }
    before = __builtin_amdgcn_readlane(upTo, 63);
  }
  return false;
}

// ---------------------------------------------------------------------------
// Tiles.  A workgroup makes BM x BN results from 128 bytes of k's of BM rows of one operand ("M", the results' rows) and BN of the other ("N", along the
// results' rows) at a time.  An operand whose rows run along k lies in LDS row by row, one whose rows run across (ACROSS) k by k.  16-byte pieces of
// a row are exchanged (`skew`) so that the lanes of a fragment's load find them in different banks.
// ---------------------------------------------------------------------------
template <typename T, bool ACROSS, int B>
struct Tile {
  static constexpr int E = kPer16<T>, K = 128 / sizeof(T);
  static constexpr int PER = ACROSS ? B / E : 8;  // pieces per row of the tile
  static constexpr int PIECES = 8 * B;
  // Two rows lie in each 256 bytes, which are all banks.  A load of 16 bytes per lane takes 16 lanes at a time, of two quarters in part: rows 0-3 and 12-15 of one, 4-11 of the other.
  // (Counted: no conflict, where row ^ row / 8 had one cycle in three; 8192 x 8192 x 8192 transposed 828 -> 798 us.)
  static __device__ __forceinline__ uint32_t skew(uint32_t row) { return ACROSS ? 0 : row / 2 & 7; }
  static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) { return row * PER + (piece ^ skew(row)); }
};

// A workgroup's tile of M x N results, made by WAVES_M x WAVES_N wavefronts, or by PARTS that share the k's; PLACES tiles of the operands in LDS.
template <int M, int N, int WAVES_M, int WAVES_N, int PLACES, int PARTS = 1>
struct Shape {
  static constexpr int BM = M, BN = N, WM = WAVES_M, WN = WAVES_N, R = PLACES, SPLIT = PARTS, THREADS = WM * WN * SPLIT * 64;
  static_assert(SPLIT == 1 || WM * WN == 1, "one or the other");
  static constexpr uint32_t LDS = R * SPLIT * (BM + BN) * 128;
};

// An operand's part that a tile is taken from: `along` elements along k and `across` the other way.  Rows and columns of results that nobody stores are made of whatever is
// at hand: there the last line is loaded again.  A lane's 16 bytes that would reach beyond a row's end are loaded from so much further up that they end with it, and
// moved when they go to LDS; rows shorter than 16 bytes are loaded element by element.
template <typename T, bool ACROSS, int B, int THREADS, int EVERY>
struct Loader {
  using L = Tile<T, ACROSS, B>;
  static constexpr int N = (L::PIECES + THREADS - 1) / THREADS;
  static constexpr uint32_t E = L::E, ROWS = THREADS / L::PER;  // of one access of the workgroup
  static_assert(THREADS % L::PER == 0 && (!ACROSS || L::PIECES % THREADS == 0), "whole rows");
  Chunk<T> held[N];
  const T* from[ACROSS ? 1 : N];
  uint32_t turn = 0;  // bits to move
  uint64_t stride;
  uint32_t along, across;
  static __device__ __forceinline__ uint32_t row(int i) { return threadIdx.x % THREADS / L::PER + i * ROWS; }
  static __device__ __forceinline__ uint32_t column() { return threadIdx.x % L::PER * E; }
  __device__ __forceinline__ const T* at(int i) const { return ACROSS ? from[0] + i * ROWS * stride : from[i]; }
  __device__ __forceinline__ Loader(const T* base, uint64_t stride_, uint32_t along_, uint32_t across_) : stride(stride_), along(along_), across(across_) {
    if constexpr (ACROSS) {
      const uint32_t col = column() < across ? column() : 0, over = across < E ? 0 : col + E - min(col + E, across);
      from[0] = base + (row(0) * stride + col - over);
      turn = over * 8 * sizeof(T);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) from[i] = base + (min(row(i), across - 1) * stride + column());
    }
  }
  // The tile at k, which is below `along`; every EVERY-th of the tiles, one after the other.
  __device__ __forceinline__ void load(uint32_t k) {
    const auto whole = [](const T* p) __attribute__((always_inline)) { return __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const Vec<T, E>*>(p)); };
    if (along - k >= L::K && (!ACROSS || across >= E)) {
#pragma unroll
      for (int i = 0; i < N; i++) held[i] = whole(at(i));
    } else if constexpr (ACROSS) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        held[i] = {};
        if (row(i) >= along - k) continue;
        if (across >= E) held[i] = whole(at(i));
        else if (column() == 0) held[i] = loadChunk(at(i), (int)across);
      }
    } else {
      const uint32_t left = along - k > column() ? min(along - k - column(), E) : 0, over = along < E ? 0 : E - left;
      turn = over * 8 * sizeof(T) % 128;
#pragma unroll
      for (int i = 0; i < N; i++) {
        held[i] = {};
        if (along < E) held[i] = loadChunk(at(i), (int)left);
        else if (left) held[i] = whole(at(i) - over);
      }
    }
#pragma unroll
    for (int i = 0; i < (ACROSS ? 1 : N); i++) from[i] += EVERY * (ACROSS ? L::K * stride : L::K);
  }
  // What the load got.
  __device__ __forceinline__ void store(Chunk<T>* lds) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      Chunk<T> v = held[i];
      if (turn) v = __builtin_bit_cast(Chunk<T>, __builtin_bit_cast(unsigned __int128, v) >> turn);
      if (L::PIECES % THREADS == 0 || row(i) < L::PIECES / L::PER) lds[L::place(row(i), threadIdx.x % L::PER)] = v;
    }
  }
};

// Fragments of F times 16 rows (from row `first` on) for step s of the tile's two.  at(t): the instruction's operand for rows t.
// Which row of the tile a lane's row l of fragment t is: rowOf(t, l).  Across k a lane loads neighbouring rows' elements together, k by k, and turns them in its registers:
// two k's to a word, with one instruction for each.  (LDS can turn them while it reads; but the compiler, which does not know what those reads touch, then waits for all that
// is on its way to LDS.)
template <typename T, bool ACROSS, int B, int F>
struct Fragments {
  using L = Tile<T, ACROSS, B>;
  static constexpr int E = kPer16<T>, C = ACROSS ? (F < E ? F : E) : 1;  // rows that a lane has side by side
  AlignedVec<T, ACROSS ? C : E> v[ACROSS ? F / C * E : F];
  static constexpr int LOADS = ACROSS ? F / C * E : F;
  __device__ __forceinline__ void loadOne(const Chunk<T>* lds, uint32_t first, int s, int i) {
    const uint32_t l = threadIdx.x & 15, quarter = (threadIdx.x & 63) >> 4;
    if constexpr (!ACROSS) {
      v[i] = lds[L::place(first + i * 16 + l, s * 4 + quarter)];
    } else {
      const T* const line = reinterpret_cast<const T*>(lds + L::place((s * 4 + quarter) * E + i % E, 0));
      v[i] = *reinterpret_cast<const AlignedVec<T, C>*>(line + first + i / E * 16 * C + l * C);
    }
  }
  // Part i of n of the loads.
  __device__ __forceinline__ void load(const Chunk<T>* lds, uint32_t first, int s, int i = 0, int n = 1) {
#pragma unroll
    for (int j = 0; j < LOADS; j++)
      if (j * n / LOADS == i) loadOne(lds, first, s, j);
  }
  __device__ __forceinline__ Chunk<T> at(int t) const {
    if constexpr (!ACROSS) {
      return v[t];
    } else if constexpr (sizeof(T) == 4) {
      Chunk<T> c;
#pragma unroll
      for (int j = 0; j < E; j++) c[j] = v[t / C * E + j][t % C];
      return c;
    } else {
      static_assert(C >= 2, "whole words");
      typedef uint32_t Words __attribute__((ext_vector_type(4)));
      typedef uint32_t Piece __attribute__((ext_vector_type(C / 2)));
      Words c;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t even = __builtin_bit_cast(Piece, v[t / C * E + 2 * i])[t % C / 2], odd = __builtin_bit_cast(Piece, v[t / C * E + 2 * i + 1])[t % C / 2];
        c[i] = __builtin_amdgcn_perm(odd, even, t % 2 ? 0x07060302 : 0x05040100);
      }
      return __builtin_bit_cast(Chunk<T>, c);
    }
  }
  static __device__ __forceinline__ uint32_t rowOf(int t, uint32_t l) { return ACROSS ? t / C * 16 * C + l * C + t % C : t * 16 + l; }
};

// The first n of N results of a row, side by side.  ONCE: past the caches, as the weights' gradient goes: 32 groups of 2048 x 1536 (201 MB) 62 us so and 85 through them, 64 of 1000 x 520
// (66 MB) 25.2 and 27.4, 64 of 2048 x 1536 107 and 130.  (The products' results are a few lines wide: 131072 rows of 4096 elements by transposed weights 850 us through, 1023 past them.)
template <bool ONCE, typename T, int N>
__device__ __forceinline__ void storeSome(T* p, const float (&v)[N], uint32_t n) {
  Pack<T, N> o;
#pragma unroll
  for (int i = 0; i < N; i++) o.set(i, (T)v[i]);
  if (n >= N) {
    o.template store<ONCE>(p);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
      if (i < n) p[i] = o.get(i);
  }
}

// A row of results' fragments: those of M's rows b times those of N's rows a.  An instruction's result has one operand's rows along the lanes and four of the other's in each.
// Whichever a row's neighbouring results come of goes where a lane gets several side by side, and lanes beside each other go on: with N across, N's rows along the lanes.
// (The 32-bit type's four instructions for the same results wait for each other: others between them.)
template <bool NACROSS, typename T, int FN>
__device__ __forceinline__ void addProducts(const Chunk<T> (&a)[FN], const Chunk<T>& b, Acc (&acc)[FN]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[j] = NACROSS ? multiply(b[e], a[j][e], acc[j]) : multiply(a[j][e], b[e], acc[j]);
  } else {
#pragma unroll
    for (int j = 0; j < FN; j++) acc[j] = NACROSS ? multiply(b, a[j], acc[j]) : multiply(a[j], b, acc[j]);
  }
}

// A wavefront's results, rows m0 and columns n0 on of m and n, to `to`.
template <typename T, bool MACROSS, bool NACROSS, int BM, int BN, bool ONCE, int FM, int FN>
__device__ __forceinline__ void storeResults(const Acc (&acc)[FM][FN], T* to, uint64_t stride, uint32_t m0, uint32_t m, uint32_t n0, uint32_t n) {
  using N = Fragments<T, NACROSS, BN, FN>;
  const uint32_t l = threadIdx.x & 15, quarter = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < FM; i++) {
    if constexpr (NACROSS) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t row = m0 + Fragments<T, MACROSS, BM, FM>::rowOf(i, quarter * 4 + r);
        if (row >= m) continue;
#pragma unroll
        for (int j = 0; j < FN; j += N::C) {
          const uint32_t col = n0 + N::rowOf(j, l);
          float v[N::C];
#pragma unroll
          for (int x = 0; x < N::C; x++) v[x] = acc[i][j + x][r];
          if (col < n) storeSome<ONCE>(to + (row * stride + col), v, n - col);
        }
      }
    } else {
      const uint32_t row = m0 + Fragments<T, MACROSS, BM, FM>::rowOf(i, l);
      if (row >= m) continue;
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const uint32_t col = n0 + j * 16 + quarter * 4;
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        if (col < n) storeSome<ONCE>(to + (row * stride + col), v, n - col);
      }
    }
  }
}

// The sums that SPLIT wavefronts have made of the same results, each of its share of the k's, together in the first one, in the order of the wavefronts.
template <int SPLIT, int FM, int FN>
__device__ __forceinline__ void joinSums(Acc (&acc)[FM][FN], void* lds) {
  Acc* const sums = static_cast<Acc*>(lds) + (threadIdx.x & 63);
  const uint32_t wave = threadIdx.x >> 6;
  __syncthreads();
  if (wave)
#pragma unroll
    for (int i = 0; i < FM * FN; i++) sums[((wave - 1) * FM * FN + i) * 64] = acc[i / FN][i % FN];
  __syncthreads();
  if (!wave)
#pragma unroll
    for (int w = 0; w + 1 < SPLIT; w++)
#pragma unroll
      for (int i = 0; i < FM * FN; i++) acc[i / FN][i % FN] += sums[(w * FM * FN + i) * 64];
}

// One tile of results: M [m rows] times N [n rows] over `along` k's, to `to`.  SPLIT wavefronts share the k's, tile by tile, each with a part of LDS of its own.
template <typename T, bool MACROSS, bool NACROSS, typename S>
__device__ __forceinline__ void productTile(const T* from, uint64_t mStride, uint32_t m, const T* with, uint64_t nStride, uint32_t n, uint32_t along, T* to,
                                            uint64_t toStride, Chunk<T>* lds) {
  constexpr int BM = S::BM, BN = S::BN, SPLIT = S::SPLIT, THREADS = S::THREADS / SPLIT, FM = BM / S::WM / 16, FN = BN / S::WN / 16;
  constexpr uint32_t K = 128 / sizeof(T);
  const uint32_t wave = threadIdx.x >> 6, part = SPLIT > 1 ? wave : 0;
  const uint32_t m0 = SPLIT > 1 ? 0 : wave / S::WN * (BM / S::WM), n0 = SPLIT > 1 ? 0 : wave % S::WN * (BN / S::WN);
  const uint32_t rest = along - min(along, part * K);
  Chunk<T>* const ldsM = lds + part * 8 * (BM + BN);
  Chunk<T>* const ldsN = ldsM + 8 * BM;
  Loader<T, MACROSS, BM, THREADS, SPLIT> loadM(from + part * K * (MACROSS ? mStride : 1), mStride, rest, m);
  Loader<T, NACROSS, BN, THREADS, SPLIT> loadN(with + part * K * (NACROSS ? nStride : 1), nStride, rest, n);
  const auto meet = [] __attribute__((always_inline)) {
    if constexpr (SPLIT > 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wavefront's accesses to LDS are in order)
    else __syncthreads();
  };
  Acc acc[FM][FN] = {};
  if (rest) {
    loadM.load(0);
    loadN.load(0);
  }
  for (uint64_t k = 0; k < rest; k += K * SPLIT) {
    meet();
    loadM.store(ldsM);
    loadN.store(ldsN);
    meet();
    if (k + K * SPLIT < rest) {
      loadM.load((uint32_t)k + K * SPLIT);
      loadN.load((uint32_t)k + K * SPLIT);
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      Fragments<T, MACROSS, BM, FM> fm;
      Fragments<T, NACROSS, BN, FN> fn;
      fm.load(ldsM, m0, s);
      fn.load(ldsN, n0, s);
      Chunk<T> a[FN];
#pragma unroll
      for (int j = 0; j < FN; j++) a[j] = fn.at(j);
#pragma unroll
      for (int i = 0; i < FM; i++) addProducts<NACROSS, T>(a, fm.at(i), acc[i]);
    }
  }
  if constexpr (SPLIT > 1) {
    joinSums<SPLIT>(acc, lds);
    __syncthreads();  // (the next item's tiles go to the same places)
    if (wave) return;
  }
  storeResults<T, MACROSS, NACROSS, BM, BN, false>(acc, to, toStride, m0, m, n0, n);
}

// ---------------------------------------------------------------------------
// Rings of tiles.  As above, but the operands go from memory straight to LDS, to one of R places in turn, and the fragments of a half tile are read while the other half's are
// multiplied.  For operands on the 16-byte grid.  What is outside (rows behind a group's end, k's behind the last) is beyond the end that the loads' descriptor
// states, and comes as zeros without being read.
// ---------------------------------------------------------------------------
constexpr uint32_t kOutside = 0x80000000u;  // an offset beyond every descriptor's end

template <int N>
__device__ __forceinline__ void waitForLoads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);  // vmcnt alone
  asm volatile("" ::: "memory");
}
// What this wavefront reads from LDS has arrived.
__device__ __forceinline__ void waitForLds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt alone
  asm volatile("" ::: "memory");
}
// All wavefronts of the workgroup.  The operands' parts are below 2^30 bytes each, from the first to the last element.
template <typename T, bool MACROSS, bool NACROSS, typename S>
__device__ __forceinline__ void productRing(const T* from, uint32_t mStride, uint32_t m, const T* with, uint32_t nStride, uint32_t n, uint32_t along, T* to,
                                            uint64_t toStride, Chunk<T>* all) {
  constexpr int BM = S::BM, BN = S::BN, R = S::R, SPLIT = S::SPLIT, FM = BM / S::WM / 16, FN = BN / S::WN / 16;
  using LM = Tile<T, MACROSS, BM>;
  using LN = Tile<T, NACROSS, BN>;
  constexpr uint32_t WAVES = S::WM * S::WN, K = LM::K, PIECES = 8 * (BM + BN);
  constexpr uint32_t ALLM = BM / 8, ALL = (BM + BN) / 8, LOADS = (ALL + WAVES - 1) / WAVES;  // a wavefront's load: 64 pieces
  constexpr bool EVEN = ALLM % WAVES == 0 && ALL % WAVES == 0;  // (then it is known which load is of which operand)
  static_assert(R * LOADS < 64, "as the counter of loads counts");
  const uint32_t number = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t part = SPLIT > 1 ? number : 0, wave = SPLIT > 1 ? 0 : number;  // of SPLIT wavefronts each has a share of the k's, tile by tile, and a ring of its own
  const uint32_t m0 = wave / S::WN * (BM / S::WM), n0 = wave % S::WN * (BN / S::WN);
  Chunk<T>* const lds = all + part * R * PIECES;
  const auto meet = [] __attribute__((always_inline)) {
    waitForLds();
    if constexpr (SPLIT == 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // This wavefront's loads of a tile.
  __amdgpu_buffer_rsrc_t source[LOADS];
  uint32_t offset[LOADS], kOf[LOADS], step[LOADS], place[LOADS];
#pragma unroll
  for (uint32_t u = 0; u < LOADS; u++) {
    const uint32_t q = EVEN ? wave + u * WAVES : min(wave + u * WAVES, ALL - 1);  // (the last one several times if they do not come out even)
    const bool isM = EVEN ? u < ALLM / WAVES : q < ALLM;
    const uint32_t at = (isM ? q : q - ALLM) * 64 + lane, stride = isM ? mStride : nStride;
    const uint32_t rowM = at / LM::PER, rowN = at / LN::PER, row = isM ? rowM : rowN;
    const uint32_t piece = isM ? at % LM::PER ^ LM::skew(rowM) : at % LN::PER ^ LN::skew(rowN);
    const bool across = isM ? MACROSS : NACROSS;
    const uint32_t lines = across ? along : isM ? m : n, width = across ? (isM ? m : n) : along;
    source[u] = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(isM ? from : with), 0, lines ? ((lines - 1) * stride + width) * (uint32_t)sizeof(T) : 0, 0x00020000);
    const uint32_t tile = across ? K * stride * (uint32_t)sizeof(T) : 128;
    offset[u] = (row * stride + piece * LM::E) * (uint32_t)sizeof(T) + part * tile;
    kOf[u] = (across ? row : piece * LM::E) + part * K;
    step[u] = SPLIT * tile;
    place[u] = q * 64;
  }
  uint32_t asked = 0, slot = 0;  // tiles that have been asked for, and where the next one goes
  // Part i of n of the next tile's loads.
  const auto ask = [&](int i, int n) __attribute__((always_inline)) {
    Chunk<T>* const ring = lds + slot * PIECES;
#pragma unroll
    for (int u = 0; u < (int)LOADS; u++) {
      if (u * n / (int)LOADS != i) continue;
      const uint32_t o = kOf[u] + asked * (K * SPLIT) < along ? offset[u] : kOutside;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(source[u], (__attribute__((address_space(3))) void*)(ring + place[u]), 16, o, 0, 0, 0);
      offset[u] += step[u];
    }
    if (i == n - 1) {
      asked++;
      slot = slot + 1 == R ? 0 : slot + 1;
    }
  };

  Acc acc[FM][FN] = {};
  const uint32_t tiles = (along + K * SPLIT - 1 - part * K) / (K * SPLIT);
  Fragments<T, MACROSS, BM, FM> fm[2];
  Fragments<T, NACROSS, BN, FN> fn[2];
  const auto read = [&](uint32_t at, int s, int i, int n) __attribute__((always_inline)) {
    fm[s].load(lds + at * PIECES, m0, s, i, n);
    fn[s].load(lds + at * PIECES + 8 * BM, n0, s, i, n);
  };
  // A half tile's products; between them, part by part, what `other` does: there is one wavefront for a SIMD, and what it does not issue while the matrix unit works
  // is time lost.
  const auto add = [&](int s, auto other) __attribute__((always_inline)) {
    Chunk<T> a[FN];
#pragma unroll
    for (int i = 0; i < FM; i++) {
      other(i, FM);
      const Chunk<T> b = fm[s].at(i);
      if (i == 0)
#pragma unroll
        for (int j = 0; j < FN; j++) a[j] = fn[s].at(j);
      addProducts<NACROSS, T>(a, b, acc[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int r = 0; r < R; r++) ask(0, 1);
  waitForLoads<(R - 1) * LOADS>();
  meet();
  read(0, 0, 0, 1);
  uint32_t now = 0;
  for (uint32_t tile = 0; tile < tiles; tile++) {
    const uint32_t next = now + 1 == R ? 0 : now + 1;
    waitForLds();  // (before more are under way than the counter counts)
    add(0, [&](int i, int n) __attribute__((always_inline)) { read(now, 1, i, n); });
    waitForLoads<(R - 2) * LOADS>();
    meet();
    add(1, [&](int i, int n) __attribute__((always_inline)) {
      read(next, 0, i, n);
      ask(i, n);  // to where this tile was
    });
    now = next;
  }
  waitForLoads<0>();
  meet();
  if constexpr (SPLIT > 1) {
    joinSums<SPLIT>(acc, all);
    __syncthreads();  // (the next item's loads go to the same places)
    if (number) return;
  }
  storeResults<T, MACROSS, NACROSS, BM, BN, MACROSS>(acc, to, toStride, m0, m, n0, n);
}

// Items for the workgroups in groups of 2^near to an XCD, whose L2 they share.
constexpr uint32_t kNear = 4;
__device__ __forceinline__ uint64_t itemOf(uint64_t block, uint32_t near) {
  return (block >> (near + 3) << (near + 3)) + ((block & 7) << near) + (block >> 3 & ((1u << near) - 1));
}
// Which of a group's tiles x strips number `item` is: blocks of kWide strips one after the other, in a block tile by tile, so that items that follow each other share
// both operands.
constexpr uint32_t kWide = 8;
__device__ __forceinline__ void placeOf(uint32_t item, uint32_t tiles, uint32_t strips, uint32_t& tile, uint32_t& strip) {
  const uint32_t block = item / (tiles * kWide), in = item - block * tiles * kWide, wide = min(strips - block * kWide, kWide);
  tile = in / wide;
  strip = block * kWide + in - tile * wide;
}

template <typename T, bool TRANSPOSED, typename S>
__global__ __launch_bounds__(S::THREADS) void productRingKernel(cuttHipProductArgs a, uint64_t items, uint32_t near) {
  constexpr int BM = S::BM, BN = S::BN;
  extern __shared__ __attribute__((aligned(16))) char ringLds[];
  const uint32_t strips = (a.outer + BN - 1) / BN;
  for (uint64_t block = blockIdx.x; block < items; block += gridDim.x) {
    const uint64_t item = itemOf(block, near);
    Segment s;
    if (!findTile<BM>(a, (uint32_t)(item / strips), s)) continue;
    uint32_t tile, strip;
    placeOf((uint32_t)(item - (uint64_t)s.before * strips), s.tiles, strips, tile, strip);
    s.first = s.first - ((uint32_t)(item / strips) - s.before) * BM + tile * BM;
    const uint32_t col = strip * BN;
    const T* const w = static_cast<const T*>(a.w) + s.group * a.wGroup;
    productRing<T, false, !TRANSPOSED, S>(static_cast<const T*>(a.x) + s.first * a.xStride, (uint32_t)a.xStride, min(s.end - s.first, (uint32_t)BM),
                                                       TRANSPOSED ? w + col * a.wRow : w + col, (uint32_t)a.wRow, min(a.outer - col, (uint32_t)BN), a.inner,
                                                       static_cast<T*>(a.y) + (s.first * a.yStride + col), a.yStride, reinterpret_cast<Chunk<T>*>(ringLds));
  }
}

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS) void weightsRingKernel(cuttHipProductArgs a, uint64_t items, uint32_t near) {
  constexpr int BM = S::BM, BN = S::BN;
  extern __shared__ __attribute__((aligned(16))) char ringLds[];
  const uint32_t strips = (a.outer + BN - 1) / BN, tiles = (a.inner + BM - 1) / BM;
  for (uint64_t block = blockIdx.x; block < items; block += gridDim.x) {
    const uint64_t item = itemOf(block, near);
    const uint32_t group = (uint32_t)(item / ((uint64_t)tiles * strips));
    if (group >= a.groups) continue;
    uint32_t tile, strip;
    placeOf((uint32_t)(item - (uint64_t)group * tiles * strips), tiles, strips, tile, strip);
    const uint32_t row = tile * BM, col = strip * BN;
    const uint32_t first = boundOf(a, group), end = max(first, boundOf(a, group + 1));
    productRing<T, true, true, S>(static_cast<const T*>(a.x) + (first * a.xStride + row), (uint32_t)a.xStride, min(a.inner - row, (uint32_t)BM),
                                               static_cast<const T*>(a.w) + (first * a.wRow + col), (uint32_t)a.wRow, min(a.outer - col, (uint32_t)BN), end - first,
                                               static_cast<T*>(a.y) + (group * a.wGroup + row * a.yStride + col), a.yStride, reinterpret_cast<Chunk<T>*>(ringLds));
  }
}

constexpr uint32_t kMaxBlocks = 1u << 22;

template <typename T, bool TRANSPOSED, typename S>
__global__ __launch_bounds__(S::THREADS) void productKernel(cuttHipProductArgs a, uint64_t items) {
  constexpr int BM = S::BM, BN = S::BN;
  __shared__ Chunk<T> lds[S::SPLIT * 8 * (BM + BN)];
  const uint32_t strips = (uint32_t)(((uint64_t)a.outer + BN - 1) / BN);
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    Segment s;
    if (!findTile<BM>(a, (uint32_t)(item / strips), s)) return;  // (nor are there later ones)
    const uint32_t col = (uint32_t)(item % strips) * BN;
    const T* const w = static_cast<const T*>(a.w) + s.group * a.wGroup;
    productTile<T, false, !TRANSPOSED, S>(static_cast<const T*>(a.x) + s.first * a.xStride, a.xStride, min(s.end - s.first, (uint32_t)BM),
                                                       TRANSPOSED ? w + col * a.wRow : w + col, a.wRow, min(a.outer - col, (uint32_t)BN), a.inner,
                                                       static_cast<T*>(a.y) + (s.first * a.yStride + col), a.yStride, lds);
  }
}

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS) void weightsKernel(cuttHipProductArgs a, uint64_t items) {
  constexpr int BM = S::BM, BN = S::BN;
  __shared__ Chunk<T> lds[8 * (BM + BN)];
  const uint32_t strips = (uint32_t)(((uint64_t)a.outer + BN - 1) / BN), tiles = (uint32_t)(((uint64_t)a.inner + BM - 1) / BM);
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint64_t q = item / strips;
    const uint32_t group = (uint32_t)(q / tiles), row = (uint32_t)(q % tiles) * BM, col = (uint32_t)(item % strips) * BN;
    const uint32_t first = boundOf(a, group), end = max(first, boundOf(a, group + 1));
    productTile<T, true, true, S>(static_cast<const T*>(a.x) + (first * a.xStride + row), a.xStride, min(a.inner - row, (uint32_t)BM),
                                               static_cast<const T*>(a.w) + (first * a.wRow + col), a.wRow, min(a.outer - col, (uint32_t)BN), end - first,
                                               static_cast<T*>(a.y) + (group * a.wGroup + row * a.yStride + col), a.yStride, lds);
  }
}

uint32_t blocksFor(uint64_t items) { return (uint32_t)std::min<uint64_t>(items, kMaxBlocks); }
uint64_t parts(uint64_t n, uint64_t of) { return (n + of - 1) / of; }

// Whether `lines` rows of `width` elements every `stride` are on the 16-byte grid, and near enough for 32-bit offsets.  (For the weights' gradient this asks all rows, though a workgroup
// takes one group's: 16384 tokens of 8 choices, 128 experts of 4096 x 1536, rows of 2^30 bytes in bfloat16, 3010 us by weightsKernel; 16000 tokens 2085 us in rings.)
template <typename T>
bool inReach(const void* p, uint64_t group, uint64_t stride, uint64_t lines, uint64_t width) {
  return ((uintptr_t)p | group * sizeof(T) | stride * sizeof(T) | width * sizeof(T)) % 16 == 0 && stride < (1u << 30) &&
         (lines * stride + width) * sizeof(T) < (1u << 30);
}
// How many items to an XCD at a time: few enough that all XCDs have some; and what makes whole rounds of these.
uint32_t nearOf(uint64_t items) {
  uint32_t near = kNear;
  while (near && items >> near < 64) near--;
  return near;
}
uint64_t ringItems(uint64_t items) { return parts(items, 8u << nearOf(items)) * (8u << nearOf(items)); }
uint32_t ringBlocks(uint64_t items) { return (uint32_t)std::min<uint64_t>(ringItems(items), kMaxBlocks); }

// Tiles of `of` rows that suffice whatever the groups are: whole ones of all rows, and one more for every group that has a row.
uint64_t tilesOf(const cuttHipProductArgs& a, uint32_t of) { return a.rows / of + std::min(a.rows, a.groups); }

// Which shape, by what the host knows: how many rows a group has in the mean.  A larger tile reads its operands less often from the caches and feeds more products with each; a group's
// last tile is a partial one.  Measured with 64 groups of 4096 x 1536 weights, random routing, bfloat16, us (transposed weights in brackets):
//     rows per group       2          8         16         48         64         80         96        256        320        512
//     tiles of  32       123 (128)  141 (154)  162 (162)  217 (195)  242 (212)
//               64       126 (130)  139 (154)  149 (167)  169 (165)  191 (179)  216 (195)  232 (212)
//              128       152 (159)  160 (183)  165 (192)  177 (194)  180 (192)  186 (191)  191 (194)  319 (311)  388 (371)  550 (525)
//              256                                                              234 (233)  235 (235)  341 (331)  359 (356)  492 (476)
// (Up to 8 rows tiles of 32 take as long on the 16-byte grid as those of 64, and off it 175 us instead of 204.  The mean counts the rows that fill segments up, hence 80 and not 72.)
constexpr uint32_t kRows32 = 8, kRows64 = 48, kRows64Transposed = 80, kRows128 = 288;
// float, 2048 x 1536: 4 rows 132 with tiles of 16, 144 with 32; 8 rows 153 and 145; 96 rows 417 with tiles of 32, 465 with 64; 256 rows 962 and 927.
constexpr uint32_t kRows16Float = 4, kRows32Float = 128;
// Large tiles need many of them besides, or CUs have none: bfloat16, 8 groups of 512 rows, 1024 x 1024 (96 tiles of 256, 320 of 128) 32.6 us with 256, 20.7 with 128, 28.3 with 64; 8 groups of 328 rows, 320 x 448
// 18.8, 8.6 and 6.4; but 64 groups of 512 rows, 1024 x 1024 (768 of 256) 111, 117, 135.
constexpr uint64_t kFew128 = 256, kFew256 = 700;
// The weights' gradient, 64 groups of 2048 x 1536: 256 rows 222 with tiles of 128, 231 with 256; 512 rows 379 and 366; 1024 rows 627 and 614; (tiles of 128 by 4 x 1 wavefronts: 3 % less than by 2 x 2).
constexpr uint32_t kRowsWeights = 384;
// Each of its tiles goes over all of a group's rows, so that with few the longest group is all there is to wait for.  By tiles of 128 x 128, 1024 rows to a group, bfloat16, us with tiles of 64, 128, 256:
//     64 12.0, 20.0, 41.6;   256 37, 45, 95;   512 57, 50, 96;   1024 104, 67, 97;   4096 -, 234, 240;   8192 -, 433, 430
// float 64 28, 81 (with 128);   256 115, 204;   512 177, 254;   1024 341, 383;   708 tiles, groups of very unequal lengths 239, 531.  Off the 16-byte grid, bfloat16, 512: 66 with 64, 86 with 128;
// 2898: 477, 264; there 64 x 64 by 2 x 2 wavefronts where tiles are few (512 of float 200, 226 with 4 x 1), 4 x 1 where they are many (308 and 328 for 8188 rows, 60 groups, 2050 x 690).
constexpr uint64_t kFewWeights = 384, kFewWeightsUnaligned = 768, kFewWeightsFloat = 1536, kManyWeights = 6144;
// Fewer workgroups than these and the chip waits for memory: narrow tiles then, whose k's four wavefronts share.  One token of 8 experts, 4096 x 1536 (96 tiles of 128 columns): 30 -> 24 us
// (28 -> 21 transposed); 4 experts of 4096 x 1408 (44): 22.7 -> 12.9; one group of 1024 rows of 1024 x 512: 30.9 -> 7.7; 16 experts (192): 42 -> 52, so not there.
// Off the 16-byte grid, where a wavefront has one tile on its way and not a ring of them: 2047 x 1023, 8 tokens of 8 experts (512) 67 -> 57 (52 -> 44), 16 tokens in float (1024) 122 -> 160.
constexpr uint32_t kFewRows = 4;
constexpr uint64_t kFew = 176, kFewUnaligned = 768;

template <typename T, typename S>
int productInRings(const cuttHipProductArgs& a, bool transposed, void* stream) {
  const uint64_t items = tilesOf(a, S::BM) * parts(a.outer, S::BN);
  auto kernel = transposed ? productRingKernel<T, true, S> : productRingKernel<T, false, S>;
  return launchRows(kernel, ringBlocks(items), S::THREADS, S::LDS, stream, a, ringItems(items), nearOf(items));
}
template <typename T, typename S>
int productAs(const cuttHipProductArgs& a, bool transposed, bool ring, void* stream) {
  if (ring) return productInRings<T, S>(a, transposed, stream);
  const uint64_t items = tilesOf(a, S::BM) * parts(a.outer, S::BN);
  auto kernel = transposed ? productKernel<T, true, S> : productKernel<T, false, S>;
  return launchRows(kernel, blocksFor(items), S::THREADS, 0, stream, a, items);
}

template <typename T>
int product(const cuttHipProductArgs& a, bool transposed, void* stream) {
  const bool ring = inReach<T>(a.x, 0, a.xStride, 256, a.inner) && (transposed ? inReach<T>(a.w, a.wGroup, a.wRow, 256, a.inner) : inReach<T>(a.w, a.wGroup, a.wRow, a.inner, a.outer));
  const uint32_t rows = a.rows / a.groups;
  const auto items = [&](uint32_t m, uint32_t n) { return tilesOf(a, m) * parts(a.outer, n); };
  const bool few = items(32, 128) < (ring ? kFew : kFewUnaligned);
  if constexpr (sizeof(T) == 4) {
    if (few && rows <= kFewRows) return productAs<T, Shape<16, 32, 1, 1, 4, 4>>(a, transposed, ring, stream);
    if (few) return productAs<T, Shape<32, 32, 1, 1, 4, 4>>(a, transposed, ring, stream);
    if (rows <= kRows16Float) return productAs<T, Shape<16, 128, 1, 4, 4>>(a, transposed, ring, stream);
    if (rows <= kRows32Float) return productAs<T, Shape<32, 128, 1, 4, 4>>(a, transposed, ring, stream);
    return productAs<T, Shape<64, 128, 2, 2, 3>>(a, transposed, ring, stream);
  } else {
    if (few && rows <= kFewRows) return productAs<T, Shape<16, 64, 1, 1, 3, 4>>(a, transposed, ring, stream);
    if (few) return productAs<T, Shape<32, 64, 1, 1, 3, 4>>(a, transposed, ring, stream);
    if (rows <= kRows32) return productAs<T, Shape<32, 128, 1, 4, 4>>(a, transposed, ring, stream);
    if (rows <= (transposed ? kRows64Transposed : kRows64) || items(128, 128) < kFew128) return productAs<T, Shape<64, 128, 2, 2, 3>>(a, transposed, ring, stream);
    if (!ring || rows <= kRows128 || items(256, 256) < kFew256) return productAs<T, Shape<128, 128, 2, 2, 2>>(a, transposed, ring, stream);
    return productInRings<T, Shape<256, 256, 2, 2, 2>>(a, transposed, stream);
  }
}

template <typename S>
uint64_t weightsItems(const cuttHipProductArgs& a) { return parts(a.inner, S::BM) * parts(a.outer, S::BN) * a.groups; }
template <typename T, typename S>
int weightsInRings(const cuttHipProductArgs& a, void* stream) {
  const uint64_t items = weightsItems<S>(a);
  return launchRows(weightsRingKernel<T, S>, ringBlocks(items), S::THREADS, S::LDS, stream, a, ringItems(items), nearOf(items));
}
template <typename T, typename S>
int weightsAnyhow(const cuttHipProductArgs& a, void* stream) {
  return launchRows(weightsKernel<T, S>, blocksFor(weightsItems<S>(a)), S::THREADS, 0, stream, a, weightsItems<S>(a));
}

template <typename T>
int weights(const cuttHipProductArgs& a, void* stream) {
  const bool ring = inReach<T>(a.x, 0, a.xStride, a.rows, a.inner) && inReach<T>(a.w, 0, a.wRow, a.rows, a.outer);
  const uint64_t items = weightsItems<Shape<128, 128, 4, 1, 2>>(a);
  if constexpr (sizeof(T) == 4) {
    if (ring) return items < kFewWeightsFloat ? weightsInRings<T, Shape<64, 64, 4, 1, 4>>(a, stream) : weightsInRings<T, Shape<128, 128, 4, 1, 2>>(a, stream);
    return items < kFewWeightsFloat ? weightsAnyhow<T, Shape<64, 64, 2, 2, 2>>(a, stream) : weightsAnyhow<T, Shape<64, 64, 4, 1, 2>>(a, stream);
  } else {
    if (!ring) return items < kFewWeightsUnaligned ? weightsAnyhow<T, Shape<64, 64, 2, 2, 2>>(a, stream) : weightsAnyhow<T, Shape<128, 128, 4, 1, 2>>(a, stream);
    if (items < kFewWeights) return weightsInRings<T, Shape<64, 64, 2, 2, 4>>(a, stream);
    if (a.rows / a.groups <= kRowsWeights || items < kManyWeights) return weightsInRings<T, Shape<128, 128, 4, 1, 2>>(a, stream);
    return weightsInRings<T, Shape<256, 256, 2, 2, 2>>(a, stream);
  }
}

}  // namespace

extern "C" int cuttHipGroupedProduct(const cuttHipProductArgs* a, int type, int transposed, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return product<float>(*a, transposed, stream);
    case CUTT_ROW_F16: return product<_Float16>(*a, transposed, stream);
    default: return product<__bf16>(*a, transposed, stream);
  }
}

extern "C" int cuttHipGroupedWeights(const cuttHipProductArgs* a, int type, void* stream) {
  switch (type) {
    case CUTT_ROW_F32: return weights<float>(*a, stream);
    case CUTT_ROW_F16: return weights<_Float16>(*a, stream);
    default: return weights<__bf16>(*a, stream);
  }
}
