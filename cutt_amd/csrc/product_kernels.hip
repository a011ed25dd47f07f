/*
 * product_kernels.hip - rows grouped by expert times their experts' weights, and the weights' gradient (cutt_products.h).
 */
#include <algorithm>

#include "product_device.h"
#include "product_layer.h"

using namespace cutt;

namespace {

// A group's rows, and the first of the tile that a workgroup has to do.
struct Segment {
  uint32_t group, first, end;
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
      s.group = base + at;
      s.end = __builtin_amdgcn_readlane(hi, at);
      const uint64_t first = (uint64_t)__builtin_amdgcn_readlane(lo, at) + (uint64_t)(tile - __builtin_amdgcn_readlane(upTo - n, at)) * BM;
      s.first = (uint32_t)first;
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
  static __device__ __forceinline__ uint32_t skew(uint32_t row) {
    if (!ACROSS) return row & 7;
    if (sizeof(T) == 4) return 0;
    return (((row & 3) | (row >> 3 & 1) << 2) * 2) & (PER - 1);
  }
  static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) { return row * PER + (piece ^ skew(row)); }
};

// An operand's part that a tile is taken from: `along` elements along k and `across` the other way.
template <typename T, bool ACROSS, int B, int THREADS>
struct Loader {
  using L = Tile<T, ACROSS, B>;
  static constexpr int N = L::PIECES / THREADS;
  static_assert(N * THREADS == L::PIECES, "whole rounds");
  Chunk<T> held[N];
  __device__ __forceinline__ void load(const T* from, uint64_t stride, uint32_t along, uint32_t across, uint32_t k) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t p = threadIdx.x + i * THREADS, row = p / L::PER, col = p % L::PER * L::E;
      const uint32_t r = ACROSS ? k + row : row, c = ACROSS ? col : k + col;
      const uint32_t rows = ACROSS ? along : across, cols = ACROSS ? across : along;
      held[i] = loadChunk(from + (r * stride + c), r < rows && c < cols ? (int)min(cols - c, (uint32_t)L::E) : 0);
    }
  }
  __device__ __forceinline__ void store(Chunk<T>* lds) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t p = threadIdx.x + i * THREADS;
      lds[L::place(p / L::PER, p % L::PER)] = held[i];
    }
  }
};

// Fragments of F times 16 rows (from row `first` on) for step s of the tile's two.  at(t, j): the j-th instruction's operand for rows t.
// Which row of the tile a lane's row l of fragment t is: rowOf(t, l).
template <typename T, bool ACROSS, int B, int F>
struct Fragments {
  using L = Tile<T, ACROSS, B>;
  Chunk<T> v[F];
  __device__ __forceinline__ void load(const Chunk<T>* lds, uint32_t first, int s) {
    const uint32_t l = threadIdx.x & 15, quarter = (threadIdx.x & 63) >> 4;
    if constexpr (!ACROSS) {
#pragma unroll
      for (int t = 0; t < F; t++) v[t] = lds[L::place(first + t * 16 + l, s * 4 + quarter)];
    } else if constexpr (sizeof(T) == 2) {
      // Sixteen lanes load 4 k's of 16 columns, 8 bytes each, and get 4 k's of one column each.
      typedef short Four __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) Four* Lds;
#pragma unroll
      for (int t = 0; t < F; t++) {
        union {
          Four four[2];
          Chunk<T> whole;
        } u;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t k = s * 32 + quarter * 8 + h * 4 + (l >> 2), col = first + t * 16 + (l & 3) * 4;
          const char* const at = reinterpret_cast<const char*>(lds + L::place(k, col / 8)) + (col & 7) * 2;
          u.four[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at);
        }
        v[t] = u.whole;
      }
    } else {
      static_assert(F % 4 == 0, "a lane takes four neighbouring columns");
#pragma unroll
      for (int t = 0; t < F; t += 4)
#pragma unroll
        for (int j = 0; j < 4; j++) v[t + j] = lds[L::place(s * 16 + quarter * 4 + j, (first + t * 16) / 4 + l)];
    }
  }
  __device__ __forceinline__ Chunk<T> at(int t) const {
    if constexpr (ACROSS && sizeof(T) == 4) {
      Chunk<T> c;
#pragma unroll
      for (int j = 0; j < 4; j++) c[j] = v[t / 4 * 4 + j][t % 4];
      return c;
    }
    return v[t];
  }
  static __device__ __forceinline__ uint32_t rowOf(int t, uint32_t l) {
    return ACROSS && sizeof(T) == 4 ? t / 4 * 64 + l * 4 + t % 4 : t * 16 + l;
  }
};

// n results of a row, side by side.
template <typename T>
__device__ __forceinline__ void storeFour(T* p, Acc v, uint32_t n) {
  Pack<T, 4> o;
#pragma unroll
  for (int i = 0; i < 4; i++) o.set(i, (T)v[i]);
  if (n >= 4) {
    o.store(p);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (i < n) p[i] = o.get(i);
  }
}

// One tile of results: M [m rows] times N [n rows] over `along` k's, to `to`.
template <typename T, bool MACROSS, bool NACROSS, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void productTile(const T* from, uint64_t mStride, uint32_t m, const T* with, uint64_t nStride, uint32_t n, uint32_t along, T* to,
                                            uint64_t toStride, Chunk<T>* lds) {
  constexpr int THREADS = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16;
  const uint32_t wave = threadIdx.x >> 6, l = threadIdx.x & 15, quarter = (threadIdx.x & 63) >> 4;
  const uint32_t m0 = wave / WN * (BM / WM), n0 = wave % WN * (BN / WN);
  Chunk<T>* const ldsN = lds + 8 * BM;
  Loader<T, MACROSS, BM, THREADS> loadM;
  Loader<T, NACROSS, BN, THREADS> loadN;
  Acc acc[FM][FN] = {};
  if (along) {
    loadM.load(from, mStride, along, m, 0);
    loadN.load(with, nStride, along, n, 0);
  }
  constexpr uint32_t K = 128 / sizeof(T);
  for (uint64_t k = 0; k < along; k += K) {
    __syncthreads();
    loadM.store(lds);
    loadN.store(ldsN);
    __syncthreads();
    if (k + K < along) {
      loadM.load(from, mStride, along, m, (uint32_t)k + K);
      loadN.load(with, nStride, along, n, (uint32_t)k + K);
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      Fragments<T, MACROSS, BM, FM> fm;
      Fragments<T, NACROSS, BN, FN> fn;
      fm.load(lds, m0, s);
      fn.load(ldsN, n0, s);
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = multiply(fn.at(j), fm.at(i), acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const uint32_t row = m0 + Fragments<T, MACROSS, BM, FM>::rowOf(i, l);
    if (row >= m) continue;
    T* const line = to + row * toStride;
    if constexpr (NACROSS && sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < FN; j += 4)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const uint32_t col = n0 + j * 16 + (quarter * 4 + r) * 4;
          Acc v;
#pragma unroll
          for (int x = 0; x < 4; x++) v[x] = acc[i][j + x][r];
          if (col < n) storeFour(line + col, v, n - col);
        }
    } else {
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const uint32_t col = n0 + j * 16 + quarter * 4;
        if (col < n) storeFour(line + col, acc[i][j], n - col);
      }
    }
  }
}

constexpr uint32_t kMaxBlocks = 1u << 22;

template <typename T, bool TRANSPOSED, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void productKernel(cuttHipProductArgs a, uint64_t items) {
  __shared__ Chunk<T> lds[8 * (BM + BN)];
  const uint32_t strips = (uint32_t)(((uint64_t)a.outer + BN - 1) / BN);
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    Segment s;
    if (!findTile<BM>(a, (uint32_t)(item / strips), s)) return;  // (nor are there later ones)
    const uint32_t col = (uint32_t)(item % strips) * BN;
    const T* const w = static_cast<const T*>(a.w) + s.group * a.wGroup;
    productTile<T, false, !TRANSPOSED, BM, BN, WM, WN>(static_cast<const T*>(a.x) + s.first * a.xStride, a.xStride, min(s.end - s.first, (uint32_t)BM),
                                                       TRANSPOSED ? w + col * a.wRow : w + col, a.wRow, min(a.outer - col, (uint32_t)BN), a.inner,
                                                       static_cast<T*>(a.y) + (s.first * a.yStride + col), a.yStride, lds);
  }
}

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void weightsKernel(cuttHipProductArgs a, uint64_t items) {
  __shared__ Chunk<T> lds[8 * (BM + BN)];
  const uint32_t strips = (uint32_t)(((uint64_t)a.outer + BN - 1) / BN), tiles = (uint32_t)(((uint64_t)a.inner + BM - 1) / BM);
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint64_t q = item / strips;
    const uint32_t group = (uint32_t)(q / tiles), row = (uint32_t)(q % tiles) * BM, col = (uint32_t)(item % strips) * BN;
    const uint32_t first = boundOf(a, group), end = max(first, boundOf(a, group + 1));
    productTile<T, true, true, BM, BN, WM, WN>(static_cast<const T*>(a.x) + (first * a.xStride + row), a.xStride, min(a.inner - row, (uint32_t)BM),
                                               static_cast<const T*>(a.w) + (first * a.wRow + col), a.wRow, min(a.outer - col, (uint32_t)BN), end - first,
                                               static_cast<T*>(a.y) + (group * a.wGroup + row * a.yStride + col), a.yStride, lds);
  }
}

uint32_t blocksFor(uint64_t items) { return (uint32_t)std::min<uint64_t>(items, kMaxBlocks); }
uint64_t parts(uint64_t n, uint64_t of) { return (n + of - 1) / of; }

template <typename T>
int product(const cuttHipProductArgs& a, bool transposed, void* stream) {
  constexpr int BM = 128, BN = 128;
  // Tiles that suffice whatever the groups are: whole ones of all rows, and one more for every group that has a row.
  const uint64_t items = (a.rows / BM + std::min(a.rows, a.groups)) * parts(a.outer, BN);
  auto kernel = transposed ? productKernel<T, true, BM, BN, 2, 2> : productKernel<T, false, BM, BN, 2, 2>;
  return launchRows(kernel, blocksFor(items), 256, 0, stream, a, items);
}

template <typename T>
int weights(const cuttHipProductArgs& a, void* stream) {
  constexpr int BM = 128, BN = 128;
  const uint64_t items = parts(a.inner, BM) * parts(a.outer, BN) * a.groups;
  return launchRows(weightsKernel<T, BM, BN, 2, 2>, blocksFor(items), 256, 0, stream, a, items);
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
