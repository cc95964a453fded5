// Low-rank adapters of many requests beside a shared projection. Row t of a step belongs to a request
// with adapter g = row_adapter[t], or with none; the projection's output columns lie in up to four
// slices s (q, k and v of one stacked product), each with factors of its own:
//
//   h[t, s, i] = sum_k A[g, s R + i, k] x[t, k]                       i < ranks[g]
//   out[t, c] = base[t, c] + scale[g] sum_i B[g, c, i] h[t, s(c), i]
//
// Two launches, but for few rows of small rank: all slices' h, with the 24 bits of its 32-bit sums (scratch [T, S R]), then the columns. Both give a block
// tiles of 16 or 32 rows on the matrix units, whatever adapters these rows have: the products of a tile and
// one of its adapters are a block's work, the rows of others ride along unwritten. Rows of a request are
// neighbours, so a tile of a prompt's portion has one adapter, as a rule; a tile of single rows may have as
// many as rows. A step of few rows has blocks for all of them (grid.y); one of many has a block for every
// tile's first adapter, and some more that look for the tiles which have others. The rows need no order and
// the host no list of groups, so that a captured step serves whatever requests come.
//
// What bounds it: few rows, the latency of two launches that each wait for memory once (the factors
// of the step's adapters are some MB: 64 rows of three slices of 2,048 numbers and eight adapters of ranks up to 64, 15 us in a
// captured step; one row of rank 16, in one launch, 7); many rows, reading and writing x, base and out (2,055 rows of 3,584
// numbers: 34 us, 1.8 TB/s of what cannot be spared: both launches wait for rows and factors in turn). h of bfloat16 rows enters the
// second product as a sum of three bfloat16 numbers (the rounded value, what the rounding left, rounded, and what that left: 8 bits
// each, 24 together), so that none of its bits is lost and `out` alone is rounded.
//
// A tile's sums run in the same order however many rows the step has: every form cuts k among
// eight waves in the same way, and a request's numbers do not depend on its company.
//
// Where a kernel holds the projection's sums in 32 bits itself (qkv_rope.hip), it asks for what the adapters add alone, in
// 32 bits (outputs of a type of their own, without a base; rows without an adapter are not written).
#include "common.h"
#include <algorithm>
#include <type_traits>

namespace ninfer {

struct AdapterArgs {
  const void* x;         // [T, ldx]
  const void* a;         // [L, S R, K]
  const void* b;         // [L, N, R]
  const float* scale;    // [L]
  const int* ranks;      // [L]: rows of A (and columns of B) that count, clamped to [0, R]
  const int* row_adapter;   // [T]; outside [0, L): none
  const void* base;      // [T, ldb]; may be out; not read where the adapters' part is asked for alone
  void* out;             // [T, ldo]
  void* h;               // [T, S R] 32-bit numbers, or as many bfloat16 ones in each of three planes (kTerms)
  long long ldx, ldb, ldo;
  int T, K, R, S, L, N;
  int first[5];          // slice s: columns first[s] .. first[s + 1]
  int dtype;
  int single;            // the rows are of different requests each
};

constexpr int kWaves = 8;
constexpr int kExpandWaves = 4;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of a row, as the matrix units take them: a lane of quad q (lane / 16) holds numbers 8 q .. 8 q + 7 of 32
// (bfloat16) or 4 q .. 4 q + 3 of 16 (32-bit, whose products take 4 of k at a time: which ones is free as
// long as both operands agree).
template <typename T> struct Frag;
template <> struct Frag<bf16> {
  static constexpr int kLane = 8;
  bf16x8 v;
  __device__ __forceinline__ static f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  }
};
template <> struct Frag<float> {
  static constexpr int kLane = 4;
  f32x4 v;
  __device__ __forceinline__ static f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes by one load or store, which ask for addresses that are multiples of 4.
struct __attribute__((packed, aligned(4))) Sixteen { uint4 v; };
__device__ __forceinline__ uint4 load_16_bytes(const void* p) { return ((const Sixteen*)p)->v; }
__device__ __forceinline__ void store_16_bytes(void* p, uint4 v) { ((Sixteen*)p)->v = v; }

// Numbers [at, at + kLane) of a row of `n`, 0 behind its end (nothing is read there), one by one.
template <typename T>
__device__ __forceinline__ uint4 load_single(const T* row, int at, int n) {
  T e[Frag<T>::kLane];
#pragma unroll
  for (int i = 0; i < Frag<T>::kLane; ++i) e[i] = at + i < n ? row[at + i] : from_f32<T>(0.f);
  uint4 v;
  __builtin_memcpy(&v, e, 16);
  return v;
}
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* row, int at, int n) {
  Frag<T> f;
  f.v = __builtin_bit_cast(decltype(f.v), load_single(row, at, n));
  return f;
}

// The adapters of the 16 RT rows from t0 on: every wave goes through them in the order of their first rows.
template <int RT>
struct TileAdapters {
  int mine;                 // lane i < 16 RT: row t0 + i's adapter, -1 for none
  int ranks;                // lane i < L: adapter i's rank (where there are up to 64; else asked for when it is needed)
  unsigned long long left;  // rows whose adapter has not been taken yet
  __device__ __forceinline__ TileAdapters(const AdapterArgs& a, int t0) {
    const int lane = threadIdx.x & 63;
    mine = lane < 16 * RT && t0 + lane < a.T ? a.row_adapter[t0 + lane] : -1;
    ranks = a.L <= 64 && lane < a.L ? a.ranks[lane] : 0;
    if (mine >= a.L || mine < 0) mine = -1;
    left = __ballot(mine >= 0);
  }
  // The next adapter, the rows (bits) that have it, and its rank.
  __device__ __forceinline__ int next(const AdapterArgs& a, unsigned long long& rows, int& rank) {
    const int g = __builtin_amdgcn_readlane(mine, __ffsll(left) - 1);
    rows = __ballot(mine == g);
    left &= ~rows;
    rank = a.L <= 64 ? __builtin_amdgcn_readlane(ranks, g) : a.ranks[g];
    rank = min(max(rank, 0), a.R);
    return g;
  }
  // The one after `pass` others; -1: there is none.
  __device__ __forceinline__ int at(const AdapterArgs& a, int pass, unsigned long long& rows, int& rank) {
    int g = -1;
    for (int i = 0; left && i <= pass; ++i) {
      const int one = next(a, rows, rank);
      if (i == pass) g = one;
    }
    return g;
  }
};

// The `u`th of all tiles' adapters but their first ones, in the order of tiles: its tile, and which of the tile's it is (-1: there
// are fewer). By the whole block of WAVES waves: 64 tiles of 32 rows at a time, their numbers of further adapters in `counts` [64].
template <int WAVES>
__device__ int find_further(const AdapterArgs& a, int u, int* counts, int& tile) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tiles = (a.T + 31) / 32;
  for (int base = 0; base < tiles; base += 64) {
    int of[32 / WAVES];   // a wave's pairs of tiles, a row a lane
#pragma unroll
    for (int i = 0; i < 32 / WAVES; ++i) {
      const int row = (base + 2 * (w + i * WAVES)) * 32 + lane;
      of[i] = row < a.T ? a.row_adapter[row] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32 / WAVES; ++i) {
      int n0 = 0, n1 = 0;
      for (unsigned long long left = __ballot(of[i] >= 0 && of[i] < a.L); left;) {
        const unsigned long long rows = __ballot(of[i] == __builtin_amdgcn_readlane(of[i], __ffsll(left) - 1));
        n0 += (unsigned)rows != 0;
        n1 += rows >> 32 != 0;
        left &= ~rows;
      }
      if (lane < 2) counts[2 * (w + i * WAVES) + lane] = max((lane ? n1 : n0) - 1, 0);
    }
    __syncthreads();
    const int mine = counts[lane];
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    const unsigned long long hit = __ballot(upto > u);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      tile = base + l;
      return 1 + u - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
    }
    u -= __builtin_amdgcn_readlane(upto, 63);
  }
  return -1;
}

// The tile and the group of columns of block `b` of the grid's x. With `near`, blocks that run on one XCD (block id mod 8) have
// neighbouring ones, so that a request's rows find its factors in that XCD's L2. False: there is none.
__device__ __forceinline__ bool place_of(int b, bool near, int groups, int total, int& tile, int& group) {
  if (near) b = b % kXcds * ((total + kXcds - 1) / kXcds) + b / kXcds;
  tile = b / groups, group = b % groups;
  return b < total;
}

// All bits of the first `count` of 16 bytes' numbers.
template <typename T>
__device__ __forceinline__ uint4 first_numbers(int count) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int bits = (count - i * (4 / (int)sizeof(T))) * 8 * (int)sizeof(T);
    u[i] = bits >= 32 ? ~0u : bits <= 0 ? 0u : (1u << bits) - 1;
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// The 16 bytes at number `k` of a row of `n` numbers of which `rank` count: the others are 0, whatever they are.
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* row, int k, int rank, int n) {
  if (k >= rank) return make_uint4(0, 0, 0, 0);
  if (k + Frag<T>::kLane > n) return load_single(row, k, rank);
  const uint4 v = load_16_bytes(row + k), keep = first_numbers<T>(rank - k);
  return make_uint4(v.x & keep.x, v.y & keep.y, v.z & keep.z, v.w & keep.w);
}

// Between a wave's writes into its own shared memory and its lanes' reads of each other's: the memory itself keeps a wave's order.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Rows on their way to the matrix units pass through shared memory of the wave: there a lane needs 16 bytes of row `lane % 16`, and
// such loads, whose neighbouring lanes read different rows, cost the cache four times what loads of whole lines do (2,055 rows of
// 3,584 numbers, the first product: 42 us so, 18 through shared memory; the second, with h in two numbers, 26 and 17). 16 rows of 128 bytes, eight pieces each: piece c of row r lies at 8 r + (c ^ r / 2),
// so that sixteen rows' pieces of one number lie in different banks. A lane loads (and puts) piece lane % 8 of rows lane / 8 and
// lane / 8 + 8.
__device__ __forceinline__ int place8(int row, int piece) { return row * 8 + (piece ^ (row >> 1)); }
// ... and of 64 bytes, four pieces each.
__device__ __forceinline__ int place4(int row, int piece) { return row * 4 + (piece ^ (row >> 2)); }

// How rows are read: number by number; 16 bytes at a time, rows of whole steps, or with a rest behind them.
enum Rows { kSingle, kWhole, kRest };

// Products of the 16 RT rows row_of(f, 0 .. 15), f < RT, with the 16 CT that follow: this wave's part of the sums over k, the steps
// w, w + 8, .. of the block's eight waves. `lds`: memory of the block for all its rows on their way.
template <typename T, int RT, int CT, Rows ROWS, typename RowOf>
__device__ __forceinline__ void products(int K, uint4* lds, f32x4 (&acc)[RT][CT], RowOf row_of) {
  constexpr int F = RT + CT, kLane = Frag<T>::kLane, kStep = 8 * kLane;   // (a step: 128 bytes of each row, two products)
  constexpr int kDepth = RT == 1 && CT == 1 && ROWS == kWhole ? 3 : 2;    // steps on their way
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4, m = lane & 15;
  const int steps = (K + kStep - 1) / kStep;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[rt][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Frag<T> (&f)[F]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[rt][ct] = Frag<T>::mma(f[rt], f[RT + ct], acc[rt][ct]);
  };
  if constexpr (ROWS != kSingle) {
    uint4* stage = lds + w * (F * 128);
    const int r = lane >> 3, c = lane & 7, whole = K / kStep;
    const T* from[F][2];
    uint4 next[kDepth][F][2];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int i = 0; i < 2; ++i) from[f][i] = row_of(f, i * 8 + r) + c * kLane;
    auto load = [&](uint4 (&to)[F][2], int st) {
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i) to[f][i] = load_16_bytes(from[f][i] + st * kStep);
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (w + d * kWaves < whole) load(next[d], w + d * kWaves);
    for (int st0 = w; st0 < steps; st0 += kDepth * kWaves) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int st = st0 + d * kWaves;
        if (st >= steps) break;
        if (ROWS == kWhole || st < whole) {
#pragma unroll
          for (int f = 0; f < F; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) stage[f * 128 + place8(i * 8 + r, c)] = next[d][f][i];
          if (st + kDepth * kWaves < whole) load(next[d], st + kDepth * kWaves);
        } else {   // (the rest of the rows)
#pragma unroll 1
          for (int f = 0; f < F; ++f)
#pragma unroll 1
            for (int i = 0; i < 2; ++i)
              stage[f * 128 + place8(i * 8 + r, c)] = load_piece(row_of(f, i * 8 + r), st * kStep + c * kLane, K, K);
        }
        wave_fence();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          Frag<T> f[F];
#pragma unroll
          for (int i = 0; i < F; ++i) f[i].v = __builtin_bit_cast(decltype(f[i].v), stage[i * 128 + place8(m, half * 4 + quad)]);
          multiply(f);
        }
        wave_fence();
      }
    }
  } else {
    for (int st = w; st < steps; st += kWaves) {
#pragma unroll 1
      for (int k = st * kStep + quad * kLane; k < (st + 1) * kStep; k += 4 * kLane) {
        Frag<T> f[F];
#pragma unroll
        for (int i = 0; i < F; ++i) f[i] = load_frag(row_of(i, m), k, K);
        multiply(f);
      }
    }
  }
}

// The sums of the waves' parts: done(row, column, sum) for each, spread over the block's threads.
template <int RT, int CT, typename Done>
__device__ __forceinline__ void sum_parts(uint4* lds, const f32x4 (&acc)[RT][CT], Done done) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  __syncthreads();   // (the rows that lay there have been used)
  f32x4* part = (f32x4*)lds;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) part[(w * RT * CT + rt * CT + ct) * 64 + lane] = acc[rt][ct];
  __syncthreads();
  for (int o = threadIdx.x; o < RT * CT * 256; o += kWaves * 64) {
    const int f = o >> 8, l = (o >> 2) & 63;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += ((const float*)lds)[i * (RT * CT * 256) + o];
    done(f / CT * 16 + (l >> 4) * 4 + (o & 3), f % CT * 16 + (l & 15), sum);
  }
}
template <int RT, int CT> constexpr int kStageRows = kWaves * (RT + CT) * 128;   // the memory of both, in 16 bytes
template <int RT, int CT> constexpr int kStageParts = kWaves * RT * CT * 64;

template <typename T> constexpr int kTerms = sizeof(T) == 2 ? 3 : 1;   // numbers whose sum is one of h

// A number of h: 32 bits, or three bfloat16 numbers whose sum it is, `plane` apart (an infinite one is alone; what is left of numbers
// below 2^-110 may be too small for the third).
__device__ __forceinline__ void store_h(float* h, int64_t at, int64_t, float sum) { h[at] = sum; }
__device__ __forceinline__ void store_h(bf16* h, int64_t at, int64_t plane, float sum) {
  const bf16 high = from_f32<bf16>(sum);
  const float left = sum - to_f32(high), rest = __builtin_isfinite(left) ? left : 0.f;
  const bf16 mid = from_f32<bf16>(rest);
  h[at] = high;
  h[plane + at] = mid;
  h[2 * plane + at] = from_f32<bf16>(rest - to_f32(mid));
}

// h of 16 RT rows and 16 CT columns.
template <typename T, int RT, int CT, Rows ROWS>
__global__ __launch_bounds__(kWaves * 64, RT == 1 ? 4 : 2) void adapter_shrink_kernel(const AdapterArgs a, int groups, int total, int more) {
  __shared__ uint4 lds[std::max(kStageRows<RT, CT>, kStageParts<RT, CT>)];
  // `more` > 0: tiles have a block for their first adapters only, and as many more look for the further ones; else as in the other
  // kernel every gridDim.y'th.
  int further = RT > 1 ? (int)blockIdx.x - (int)(gridDim.x - more) : -1, tile_at = 0, group = 0, pass = blockIdx.y;
  if (further < 0 && !place_of(blockIdx.x, RT > 1, groups, total, tile_at, group)) return;
  const int m = threadIdx.x & 15, C = a.S * a.R;
  for (bool once = false;; once = true) {
    if (once) {
      if (RT > 1 && more && further < 0) return;
      pass += gridDim.y;
      __syncthreads();   // (the memory is the next products')
    }
    if (RT > 1 && further >= 0) {
      pass = find_further<kWaves>(a, further / groups, (int*)lds, tile_at);
      if (pass < 0) return;
      group = further % groups;
      further += more;
      __syncthreads();
    }
    const int t0 = tile_at * (16 * RT), j0 = group * (CT * 16);
    unsigned long long rows;
    int rank;
    const int g = TileAdapters<RT>(a, t0).at(a, pass, rows, rank);
    if (g < 0) return;
    bool any = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) any |= j0 + ct * 16 + m < C && (j0 + ct * 16 + m) % a.R < rank;
    if (!__ballot(any)) continue;
    f32x4 acc[RT][CT];
    products<T, RT, CT, ROWS>(a.K, lds, acc, [&](int f, int r) -> const T* {
      if (f < RT) return (const T*)a.x + (int64_t)min(t0 + f * 16 + r, a.T - 1) * a.ldx;
      return (const T*)a.a + ((int64_t)g * C + min(j0 + (f - RT) * 16 + r, C - 1)) * a.K;
    });
    sum_parts(lds, acc, [&](int row, int col, float sum) {
      const int j = j0 + col;
      if (rows >> row & 1 && j < C && j % a.R < rank) store_h((T*)a.h, (int64_t)(t0 + row) * C + j, (int64_t)a.T * C, sum);
    });
  }
}

constexpr int kRow = 68;   // floats of a row of 64 in a wave's memory: so padded that rows' columns lie in different banks

// 16 RT rows from t0 on and the `set`th 64 columns, by one wave: what the tile's `pass`th adapter adds to its rows; with `copy` the
// rows without an adapter too. h: all slices' numbers of row 0, rows `hstride` apart. False: the tile has no such adapter. With outputs
// of another type than the rows' they are the adapter's part alone.
template <typename T, int RT, bool VEC, typename O = T>
__device__ __forceinline__ bool expand_tile(const AdapterArgs& a, const T* h, int hstride, int64_t plane, int t0, int set, int sets, int pass,
                                            bool copy, uint4* stage, bool vec_out) {
  constexpr bool kAlone = !std::is_same<T, O>::value;
  constexpr int kLane = Frag<T>::kLane, kStep = 4 * kLane;   // (a step: 64 bytes of each row, one product; three for h's three numbers)
  const int lane = threadIdx.x & 63, quad = lane >> 4, m = lane & 15;
  if (set >= sets) return false;
  int s = 0;
  for (; s < a.S - 1; ++s) {
    const int here = (a.first[s + 1] - a.first[s] + 63) / 64;
    if (set < here) break;
    set -= here;
  }
  const int c0 = a.first[s] + set * 64, end = a.first[s + 1], n = min(end - c0, 64);
  const T* base = kAlone ? nullptr : (const T*)a.base + c0;
  O* out = (O*)a.out + c0;
  h += s * a.R;

  // Rows as they lie in memory: 16 bytes a lane, kCols of them side by side.
  constexpr int kEach = 16 / sizeof(O), kCols = 64 / kEach, kRows = 64 / kCols;
  const bool whole = vec_out && n == 64;
  uint4 was[RT][16 / kRows];
  auto load_base = [&](unsigned long long rows) {
    if (kAlone || !whole) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int i = 0; i < 16 / kRows; ++i) {
        const int r = rt * 16 + i * kRows + lane / kCols;
        if (rows >> r & 1) was[rt][i] = load_16_bytes(base + (t0 + r) * a.ldb + lane % kCols * kEach);
      }
  };
  auto store = [&](int rt, unsigned long long rows, float scale, const float* tile_) {   // tile_: rows of kRow floats, or null: 0
    if (whole) {
#pragma unroll
      for (int i = 0; i < 16 / kRows; ++i) {
        const int in = i * kRows + lane / kCols, r = rt * 16 + in;
        if (!(rows >> r & 1)) continue;
        O e[kEach];
        if (kAlone) {
#pragma unroll
          for (int c = 0; c < kEach; ++c) e[c] = from_f32<O>(scale * tile_[in * kRow + lane % kCols * kEach + c]);
        } else {
          __builtin_memcpy(e, &was[rt][i], 16);
          if (tile_) {
#pragma unroll
            for (int c = 0; c < kEach; ++c) e[c] = from_f32<O>(to_f32(e[c]) + scale * tile_[in * kRow + lane % kCols * kEach + c]);
          }
        }
        uint4 v;
        __builtin_memcpy(&v, e, 16);
        store_16_bytes(out + (t0 + r) * a.ldo + lane % kCols * kEach, v);
      }
    } else {
#pragma unroll 1
      for (int in = 0; in < 16; ++in) {
        const int r = rt * 16 + in;
        if (!(rows >> r & 1) || lane >= n) continue;
        if constexpr (kAlone) {
          out[(t0 + r) * a.ldo + lane] = from_f32<O>(scale * tile_[in * kRow + lane]);
        } else {
          const T v = base[(t0 + r) * a.ldb + lane];
          out[(t0 + r) * a.ldo + lane] = tile_ ? from_f32<T>(to_f32(v) + scale * tile_[in * kRow + lane]) : v;
        }
      }
    }
  };

  // (on their way before the rows' adapters are known: nearly all of them are needed)
  const unsigned long long here = (1ull << min(16 * RT, a.T - t0)) - 1;
  if (pass == 0) load_base(here);
  TileAdapters<RT> tile(a, t0);
  if (copy && (here & ~tile.left)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) store(rt, here & ~tile.left, 0.f, nullptr);
  }
  unsigned long long rows;
  int rank;
  const int g = tile.at(a, pass, rows, rank);
  if (g < 0) return false;
  const float scale = a.scale[g];
  if (pass) load_base(rows);
  auto brow = [&](int j, int r) { return (const T*)a.b + ((int64_t)g * a.N + min(c0 + j * 16 + r, end - 1)) * a.R; };
  auto hrow = [&](int rt, int r) { return h + (int64_t)min(t0 + rt * 16 + r, a.T - 1) * hstride; };
  f32x4 acc[RT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < rank; k0 += kStep) {
    if constexpr (VEC) {
      const int k = k0 + (lane & 3) * kLane, r = lane >> 2;
      auto row_of = [&](int f) { return f < 4 ? brow(f, r) : hrow((f - 4) / kTerms<T>, r) + (f - 4) % kTerms<T> * plane; };
      if (k0 + kStep <= a.R || a.R % kLane == 0) {   // (16 bytes that begin in a row end in it)
        uint4 now[4 + RT * kTerms<T>];
#pragma unroll
        for (int f = 0; f < 4 + RT * kTerms<T>; ++f) now[f] = k < rank ? load_16_bytes(row_of(f) + k) : make_uint4(0, 0, 0, 0);
        if (k0 + kStep > rank) {
          const uint4 keep = first_numbers<T>(rank - k);
#pragma unroll
          for (int f = 0; f < 4 + RT * kTerms<T>; ++f) now[f].x &= keep.x, now[f].y &= keep.y, now[f].z &= keep.z, now[f].w &= keep.w;
        }
#pragma unroll
        for (int f = 0; f < 4 + RT * kTerms<T>; ++f) stage[f * 64 + place4(r, lane & 3)] = now[f];
      } else {
#pragma unroll 1
        for (int f = 0; f < 4 + RT * kTerms<T>; ++f) stage[f * 64 + place4(r, lane & 3)] = load_piece(row_of(f), k, rank, a.R);
      }
      wave_fence();
      Frag<T> bf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bf[j].v = __builtin_bit_cast(decltype(bf[j].v), stage[j * 64 + place4(m, quad)]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < kTerms<T>; ++x) {
          Frag<T> hf;
          hf.v = __builtin_bit_cast(decltype(hf.v), stage[(4 + rt * kTerms<T> + x) * 64 + place4(m, quad)]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[rt][j] = Frag<T>::mma(bf[j], hf, acc[rt][j]);
        }
      wave_fence();
    } else {
      const int k = k0 + quad * kLane;
      Frag<T> bf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bf[j] = load_frag(brow(j, m), k, rank);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < kTerms<T>; ++x) {
          const Frag<T> hf = load_frag(hrow(rt, m) + x * plane, k, rank);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[rt][j] = Frag<T>::mma(bf[j], hf, acc[rt][j]);
        }
    }
  }
  float* floats = (float*)stage;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (RT > 1 && !(rows >> (rt * 16) & 0xffff)) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) *(f32x4*)(floats + m * kRow + j * 16 + quad * 4) = acc[rt][j];
    wave_fence();
    store(rt, rows, scale, floats);
    wave_fence();
  }
  return true;
}

template <typename T, int RT> constexpr int kStageExpand = std::max((4 + RT * kTerms<T>) * 64, 16 * kRow / 4);   // a wave's, in 16 bytes

// Four waves take neighbouring columns. `more`: as in the other kernel.
template <typename T, int RT, bool VEC, typename O = T>
__global__ __launch_bounds__(kExpandWaves * 64, RT == 1 ? 4 : 3) void adapter_expand_kernel(const AdapterArgs a, int sets, int groups, int total, int more,
                                                                           bool vec_out) {
  __shared__ uint4 lds[kExpandWaves][kStageExpand<T, RT>];
  __shared__ int counts[64];
  int further = RT > 1 && (int)blockIdx.x < more ? (int)blockIdx.x : -1, tile = 0, group = 0, pass = blockIdx.y;
  if (further < 0 && !place_of(blockIdx.x - more, RT > 1, groups, total, tile, group)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (;; pass += gridDim.y) {
    if (RT > 1 && further >= 0) {
      pass = find_further<kExpandWaves>(a, further / groups, counts, tile);
      if (pass < 0) return;
      group = further % groups;
      further += more;
    }
    const bool had = expand_tile<T, RT, VEC, O>(a, (const T*)a.h, a.S * a.R, (int64_t)a.T * a.S * a.R, tile * (16 * RT), group * kExpandWaves + wave, sets, pass,
                                                std::is_same<T, O>::value && pass == 0 && a.base != a.out, lds[wave], vec_out);
    if (further < 0 && (more || !had)) return;
  }
}

// Up to 16 rows and ranks up to kFewRank in one launch: a block makes the h that its columns (512 of a slice) need itself, into its
// own memory, in the order of the other kernels' sums. The factor A is read by every block of its slice, out of L2; what this saves
// is a launch and the wait for the first one's end. us in one and in two launches, rows of 2,048 numbers, adapters of their own: rank
// 16, 2,048 columns, one row 7.0 and 8.3; 3 x 2,048, 8 rows 10.2 and 10.9, 16 rows 13.3 and 14.2. With larger ranks every block has too
// much to read (with h in two numbers: rank 64, 3 x 2,048 columns, one row 10.4 and 9.1, 16 rows 14.1 and 11.5).
constexpr int kFewRows = 16, kFewRank = 16;

template <typename T, Rows ROWS, bool VEC, typename O = T>
__global__ __launch_bounds__(kWaves * 64, 2) void adapter_few_kernel(const AdapterArgs a, int sets, bool vec_out) {
  __shared__ uint4 lds[std::max(std::max(kStageRows<1, 1>, kStageParts<1, 1>), kWaves * kStageExpand<T, 1>)];
  __shared__ uint4 h_lds[kFewRows * kFewRank * kTerms<T> * (int)sizeof(T) / 16];
  int s = 0, first_set = 0, block = blockIdx.x, here = 0;
  for (;; ++s) {
    here = (a.first[s + 1] - a.first[s] + 63) / 64;
    const int blocks = (here + kWaves - 1) / kWaves;
    if (block < blocks) break;
    block -= blocks;
    first_set += here;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), local = block * kWaves + wave;
  const int stride = (a.R + 7) / 8 * 8;   // (pieces of 16 bytes begin at multiples of 16)
  const int64_t plane = (int64_t)kFewRows * stride;
  T* h = (T*)h_lds;
  for (int pass = blockIdx.y;; pass += gridDim.y) {
    unsigned long long rows;
    int rank;
    const int g = TileAdapters<1>(a, 0).at(a, pass, rows, rank);
    if (g >= 0 && rank > 0) {
      f32x4 acc[1][1];
      products<T, 1, 1, ROWS>(a.K, lds, acc, [&](int f, int r) -> const T* {
        if (f == 0) return (const T*)a.x + (int64_t)min(r, a.T - 1) * a.ldx;
        return (const T*)a.a + ((int64_t)g * a.S * a.R + s * a.R + min(r, a.R - 1)) * a.K;
      });
      sum_parts(lds, acc, [&](int row, int col, float sum) {
        if (col < rank) store_h(h, row * stride + col, plane, sum);
      });
      __syncthreads();
    }
    expand_tile<T, 1, VEC, O>(a, h - s * a.R, stride, plane, 0, local < here ? first_set + local : sets, sets, pass,
                           std::is_same<T, O>::value && pass == 0 && a.base != a.out, lds + wave * kStageExpand<T, 1>, vec_out);
    if (g < 0) return;
    __syncthreads();   // (both memories are the next pass's)
  }
}

// The grid of a kernel for which the tiles' first adapters are `total` blocks' work. Tiles of 32 rows: a block a CU more looks for
// further ones (fewer than that only where fewer can be there).
template <int RT>
static dim3 grid_of(const AdapterArgs& a, int total, int* more) {
  static_assert(RT == 1 || RT == 2, "find_further looks at tiles of 32 rows");
  const int most = std::min(std::min(16 * RT, a.T), a.L), cus = device_cu_count();   // adapters that a tile may have
  if (RT == 1) return dim3(total, std::max(1, std::min(most, 4 * cus / total)));
  if (most > 1) *more = (int)std::min<long long>((most - 1ll) * total, cus);
  return dim3((total + kXcds - 1) / kXcds * kXcds + *more);
}

// How a call's rows can be read and written.
template <typename T, typename O = T>
struct Forms {
  bool x, b, out;   // 16 bytes at a time: x and A, B, base and out
  bool rest;        // x and A: with a rest behind the whole steps
  int sets;         // 64 columns each, of all slices
  explicit Forms(const AdapterArgs& a) {
    auto four = [](const void* p, long long stride) { return (uintptr_t)p % 4 == 0 && stride * sizeof(T) % 4 == 0; };
    x = four(a.x, a.ldx) && four(a.a, a.K);
    rest = a.K % (8 * Frag<T>::kLane) != 0;
    b = four(a.b, a.R);
    out = std::is_same<T, O>::value ? four(a.base, a.ldb) && four(a.out, a.ldo) : (uintptr_t)a.out % 4 == 0;
    sets = 0;
    for (int s = 0; s < a.S; ++s) {
      sets += (a.first[s + 1] - a.first[s] + 63) / 64;
      out &= a.first[s] * sizeof(O) % 4 == 0;
    }
  }
};

template <typename T, int RT, int CT, typename O = T>
static void shrink(const AdapterArgs& a, const Forms<T, O>& f, hipStream_t stream) {
  const int groups = (a.S * a.R + CT * 16 - 1) / (CT * 16), total = (a.T + 16 * RT - 1) / (16 * RT) * groups;
  int more = 0;
  const dim3 grid = grid_of<RT>(a, total, &more);
  if (!f.x) adapter_shrink_kernel<T, RT, CT, kSingle><<<grid, kWaves * 64, 0, stream>>>(a, groups, total, more);
  else if (f.rest) adapter_shrink_kernel<T, RT, CT, kRest><<<grid, kWaves * 64, 0, stream>>>(a, groups, total, more);
  else adapter_shrink_kernel<T, RT, CT, kWhole><<<grid, kWaves * 64, 0, stream>>>(a, groups, total, more);
}

template <typename T, int RT, typename O = T>
static void expand(const AdapterArgs& a, const Forms<T, O>& f, hipStream_t stream) {
  const int groups = (f.sets + kExpandWaves - 1) / kExpandWaves, total = (a.T + 16 * RT - 1) / (16 * RT) * groups;
  int more = 0;
  const dim3 grid = grid_of<RT>(a, total, &more);
  if (f.b) adapter_expand_kernel<T, RT, true, O><<<grid, kExpandWaves * 64, 0, stream>>>(a, f.sets, groups, total, more, f.out);
  else adapter_expand_kernel<T, RT, false, O><<<grid, kExpandWaves * 64, 0, stream>>>(a, f.sets, groups, total, more, f.out);
}

template <typename T, typename O = T>
static void few(const AdapterArgs& a, const Forms<T, O>& f, hipStream_t stream) {
  int blocks = 0;
  for (int s = 0; s < a.S; ++s) blocks += ((a.first[s + 1] - a.first[s] + 63) / 64 + kWaves - 1) / kWaves;
  const dim3 grid(blocks, std::min(a.T, a.L));
  if (!f.x || !f.b) adapter_few_kernel<T, kSingle, false, O><<<grid, kWaves * 64, 0, stream>>>(a, f.sets, f.out);
  else if (f.rest) adapter_few_kernel<T, kRest, true, O><<<grid, kWaves * 64, 0, stream>>>(a, f.sets, f.out);
  else adapter_few_kernel<T, kWhole, true, O><<<grid, kWaves * 64, 0, stream>>>(a, f.sets, f.out);
}

// Blocks of 32 rows and 64 columns of the first product from which these are taken; blocks of 16 by 16 are many more. A portion alone is
// faster in them from some 64 on (in 32 bits 192), but single rows before it, which steps of an engine have, gain more from them below
// that than the portion alone loses. us of both products so and in blocks of 16 by 16, portions alone and with eight single rows of
// other adapters before them: bfloat16, 3 x 64 columns of 2,048, 384 rows 16.0 and 13.6, 23.4 and 25.3; 512 (48 blocks) 16.3 and 14.6, 23.9
// and 29.1; 768 19.1 and 20.3, 26.1 and 42.3; 2,048 27.5 and 34.7, 35.5 and 51.8; 3 x 16 columns, 1,024 rows (32) 18.2 and 14.9, 23.7 and
// 22.3, 2,048 (64) 24.3 and 23.6, 30.7 and 35.5; 32-bit, 3 x 64 columns, 1,024 rows (96) 48 and 37, 58 and 79, 2,048 (192) 64.9 and 64.5, 73
// and 95. Rows that each have an adapter of their own never: 512 of eight adapters in turn 100 and 63.
template <typename T> constexpr int kManyBlocks = sizeof(T) == 2 ? 48 : 192;

// The second product in tiles of 32 rows once these make three blocks for four CUs: as fast as in tiles of 16 where every tile has one
// adapter, and faster by what a tile of single rows takes that has several, whose further ones are blocks of their own here and
// one pass after the other there. us in tiles of 32 and of 16, bfloat16, 3 x 2,048 columns, rank 16, eight single rows before 256 rows of one
// request 16.0 and 21.3, 512 17.4 and 31.8, 1,024 23 and 37, without the single rows 9.9 and 10.0, 11.3 and 11.2, 14.8 and 16.9; 32-bit,
// rank 64, 256 rows 33 and 44, without 18.9 and 17.1.
static bool tiles_of_32(const AdapterArgs& a, int sets) {
  return !a.single && (a.T + 31ll) / 32 * ((sets + kExpandWaves - 1) / kExpandWaves) * 4 >= 3ll * device_cu_count();
}

template <typename T>
static void launch(const AdapterArgs& a, hipStream_t stream) {
  const Forms<T> f(a);
  const long long blocks = (a.T + 31ll) / 32 * ((a.S * a.R + 63) / 64);
  if (a.T <= kFewRows && a.R <= kFewRank) return few(a, f, stream);
  if (blocks >= kManyBlocks<T> && !a.single) shrink<T, 2, 4>(a, f, stream);
  else shrink<T, 1, 1>(a, f, stream);
  if (tiles_of_32(a, f.sets)) expand<T, 2>(a, f, stream);
  else expand<T, 1>(a, f, stream);
}

// The adapters' part alone: rows of few steps, in the tiles of 16 rows.
template <typename T, typename O>
static void launch_alone(const AdapterArgs& a, hipStream_t stream) {
  const Forms<T, O> f(a);
  if (a.T <= kFewRows && a.R <= kFewRank) return few<T, O>(a, f, stream);
  shrink<T, 1, 1, O>(a, f, stream);
  expand<T, 1, O>(a, f, stream);
}

}  // namespace ninfer

using namespace ninfer;

// Rows and ranks up to which a call needs no scratch.
extern "C" int ninfer_adapter_few_rows() { return kFewRows; }
extern "C" int ninfer_adapter_few_rank() { return kFewRank; }
extern "C" int ninfer_adapter_args_bytes() { return (int)sizeof(AdapterArgs); }
// Bytes of scratch for each of a row's S R numbers of h.
extern "C" int ninfer_adapter_h_bytes(int dtype) { return dtype == kBF16 ? kTerms<bf16> * (int)sizeof(bf16) : kTerms<float> * (int)sizeof(float); }

static int check_adapters(const AdapterArgs* args, bool alone) {
  NINFER_REQUIRE(args, "adapter_add: no arguments");
  const AdapterArgs& a = *args;
  NINFER_REQUIRE(a.T > 0 && a.K > 0 && a.R > 0 && a.L > 0, "adapter_add: T=%d K=%d R=%d L=%d must be positive", a.T, a.K, a.R, a.L);
  NINFER_REQUIRE(a.K <= 0x7fffffff - 128, "adapter_add: rows of %d numbers are too long", a.K);   // (steps are counted past the row's end)
  NINFER_REQUIRE(a.S >= 1 && a.S <= 4 && a.first[0] == 0 && a.first[a.S] == a.N, "adapter_add: %d slices of %d columns", a.S, a.N);
  for (int s = 0; s < a.S; ++s)
    NINFER_REQUIRE(a.first[s] < a.first[s + 1], "adapter_add: slice %d has no columns", s);
  NINFER_REQUIRE(a.x && a.a && a.b && a.scale && a.ranks && a.row_adapter && (a.base || alone) && a.out &&
                     (a.h || (a.T <= kFewRows && a.R <= kFewRank)), "adapter_add: a required array is null");
  NINFER_REQUIRE(a.ldx >= a.K && (alone || a.ldb >= a.N) && a.ldo >= a.N, "adapter_add: a row stride is less than the row");
  NINFER_REQUIRE(alone || a.base != a.out || a.ldb == a.ldo, "adapter_add: in place with two row strides");
  // (threads of a grid's x, in blocks of 16 rows: 512 for 16 columns of h, 64 for 64 of out)
  const long long tiles = (a.T + 15ll) / 16;
  NINFER_REQUIRE(a.S * (long long)a.R <= 0x7fffffff && tiles * ((a.S * a.R + 15ll) / 16) * 512 <= 0x7fffffffll &&
                     tiles * (a.N / 64 + 8ll) * 64 <= 0x7fffffffll, "adapter_add: %d rows are too many", a.T);
  NINFER_REQUIRE(a.dtype == kBF16 || (a.dtype == kF32 && !alone), "adapter_add: dtype %d", a.dtype);
  return 0;
}

extern "C" int ninfer_adapter_add(const AdapterArgs* args, hipStream_t stream) {
  if (const int rc = check_adapters(args, false)) return rc;
  if (args->dtype == kBF16) launch<bf16>(*args, stream);
  else launch<float>(*args, stream);
  NINFER_LAUNCH_CHECK();
  return 0;
}

// What the adapters add to bfloat16 rows alone, in 32 bits: out [T, ldo] of 32-bit numbers, of rows that have an adapter.
extern "C" int ninfer_adapter_rows(const AdapterArgs* args, hipStream_t stream) {
  if (const int rc = check_adapters(args, true)) return rc;
  launch_alone<bf16, float>(*args, stream);
  NINFER_LAUNCH_CHECK();
  return 0;
}
