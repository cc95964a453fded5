// Low-rank adapters of many requests beside a shared projection. Row t of a step belongs to a request
// with adapter g = row_adapter[t], or with none; the projection's output columns lie in up to four
// slices s (q, k and v of one stacked product), each with factors of its own:
//
//   h[t, s, i] = sum_k A[g, s R + i, k] x[t, k]                       i < ranks[g]
//   out[t, c] = base[t, c] + scale[g] sum_i B[g, c, i] h[t, s(c), i]
//
// Two launches: all slices' h, kept in 32 bits (scratch [T, S R]), then the columns. Both give a block
// tiles of 16 rows on the matrix units, whatever adapters these rows have: the block takes the tile's
// adapters one after the other, the rows of others ride along unwritten. Rows of a request are
// neighbours, so a tile of a prompt's portion has one adapter, as a rule. In a step of single rows it may
// have up to 16: these then go to blocks of their own (grid.z), side by side. The rows need no order
// and the host no list of groups, so that a captured step serves whatever requests come.
//
// What bounds it: few rows, the latency of two launches that each wait for memory once (the factors
// of the step's adapters are some MB); many rows, reading and writing x, base and out. h enters the
// second product as a sum of two bfloat16 numbers (the rounded value and what the rounding left, 16
// bits together), so that the only rounding of note is that of `out`. A lane of the second product
// holds 16 neighbouring columns of one row: which of B's rows a tile's lane takes is free, and is
// chosen so.
//
// A tile's sums run in the same order however many rows the step has: every form cuts k among
// eight waves in the same way, and a request's numbers do not depend on its company.
#include "common.h"
#include <algorithm>

namespace ninfer {

struct AdapterArgs {
  const void* x;         // [T, ldx]
  const void* a;         // [L, S R, K]
  const void* b;         // [L, N, R]
  const float* scale;    // [L]
  const int* ranks;      // [L]: rows of A (and columns of B) that count, clamped to [0, R]
  const int* row_adapter;   // [T]; outside [0, L): none
  const void* base;      // [T, ldb]; may be out
  void* out;             // [T, ldo]
  float* h;              // [T, S R]
  long long ldx, ldb, ldo;
  int T, K, R, S, L, N;
  int first[5];          // slice s: columns first[s] .. first[s + 1]
  int dtype;
};

constexpr int kShrinkWaves = 8;
constexpr int kExpandWaves = 4;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of a row, as the matrix units take them: a lane of quad q holds numbers 8 q .. 8 q + 7 of 32
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

// Numbers [at, at + kLane) of a row of `n`, 0 behind its end (nothing is read there).
template <bool VEC, typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* row, int at, int n) {
  Frag<T> f;
  if (VEC && at + Frag<T>::kLane <= n) {
    f.v = *(const decltype(f.v)*)(row + at);
  } else {
    T e[Frag<T>::kLane];
#pragma unroll
    for (int i = 0; i < Frag<T>::kLane; ++i) e[i] = at + i < n ? row[at + i] : from_f32<T>(0.f);
    __builtin_memcpy(&f.v, e, sizeof(f.v));
  }
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
};

// The work of a block: with `per` > 0 blocks that run on one XCD (block id mod 8) take neighbouring work, so that a
// request's rows find its factors in that XCD's L2; -1 behind the last.
__device__ __forceinline__ int work_of_block(int per, int total) {
  const int b = per ? blockIdx.x % kXcds * per + blockIdx.x / kXcds : blockIdx.x;
  return b < total ? b : -1;
}

// h of 16 RT rows and 16 CT columns.
template <typename T, int RT, int CT, bool VEC>
__global__ __launch_bounds__(kShrinkWaves * 64) void adapter_shrink_kernel(const AdapterArgs a, int groups, int per, int total) {
  __shared__ float part[kShrinkWaves][RT * CT][64][4];
  constexpr int kLane = Frag<T>::kLane, kStep = 4 * kLane;
  const int b = work_of_block(per, total);
  if (b < 0) return;
  const int t0 = b / groups * (16 * RT), j0 = b % groups * (CT * 16);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, quad = lane >> 4, C = a.S * a.R;
  const T* xrow[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) xrow[rt] = (const T*)a.x + (int64_t)min(t0 + rt * 16 + (lane & 15), a.T - 1) * a.ldx;
  TileAdapters<RT> tile(a, t0);
  for (int pass = 0; tile.left; ++pass) {
    unsigned long long rows;
    int rank;
    const int g = tile.next(a, rows, rank);
    if (pass % gridDim.y != blockIdx.y) continue;
    bool any = false;
    const T* arow[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int j = j0 + ct * 16 + (lane & 15);
      any |= j < C && j % a.R < rank;
      arow[ct] = (const T*)a.a + ((int64_t)g * C + min(j, C - 1)) * a.K;
    }
    if (!__ballot(any)) continue;
    f32x4 acc[RT][CT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[rt][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    // wave w takes the steps w, w + 8, ..
    int st = w;
    if constexpr (VEC) {
      const int whole = a.K / kStep;
#pragma unroll 4
      for (; st < whole; st += kShrinkWaves) {
        const int k = st * kStep + quad * kLane;
        Frag<T> xf[RT], af[CT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) xf[rt].v = *(const decltype(xf[rt].v)*)(xrow[rt] + k);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) af[ct].v = *(const decltype(af[ct].v)*)(arow[ct] + k);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[rt][ct] = Frag<T>::mma(xf[rt], af[ct], acc[rt][ct]);
      }
    }
    for (; st * kStep < a.K; st += kShrinkWaves) {
      const int k = st * kStep + quad * kLane;
      Frag<T> xf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) xf[rt] = load_frag<VEC>(xrow[rt], k, a.K);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const Frag<T> af = load_frag<VEC>(arow[ct], k, a.K);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][ct] = Frag<T>::mma(xf[rt], af, acc[rt][ct]);
      }
    }
    __syncthreads();   // (the pass before has read its sums)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) *(f32x4*)part[w][rt * CT + ct][lane] = acc[rt][ct];
    __syncthreads();
    for (int o = threadIdx.x; o < RT * CT * 256; o += kShrinkWaves * 64) {
      const int f = o >> 8, l = (o >> 2) & 63, row = f / CT * 16 + (l >> 4) * 4 + (o & 3), j = j0 + f % CT * 16 + (l & 15);
      if (!(rows >> row & 1) || j >= C || j % a.R >= rank) continue;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kShrinkWaves; ++i) sum += part[i][f][l][o & 3];
      a.h[(int64_t)(t0 + row) * C + j] = sum;
    }
  }
}

// Numbers [at, at + kLane) of a row of h as operands: their sum is the number (one operand for 32 bits).
template <bool VEC>
__device__ __forceinline__ void load_h(const float* row, int at, int n, Frag<float>& f, Frag<float>&) {
  f = load_frag<VEC>(row, at, n);
}
template <bool VEC>
__device__ __forceinline__ void load_h(const float* row, int at, int n, Frag<bf16>& high, Frag<bf16>& low) {
  float e[8];
  const Frag<float> f0 = load_frag<VEC>(row, at, n), f1 = load_frag<VEC>(row, at + 4, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = f0.v[i], e[i + 4] = f1.v[i];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    high.v[i] = (__bf16)e[i];
    const float rest = e[i] - (float)high.v[i];
    low.v[i] = (__bf16)(__builtin_isfinite(rest) ? rest : 0.f);   // (an infinite h leaves NaN)
  }
}

// Sixteen neighbouring columns of a row, the ones before `n` of them; VEC: 16 bytes at a time.
template <typename T>
__device__ __forceinline__ void load_16(const T* p, int n, bool vec, float* f) {
  constexpr int kEach = 16 / sizeof(T);
  if (vec && n >= 16) {
#pragma unroll
    for (int i = 0; i < 16; i += kEach) {
      const uint4 v = *(const uint4*)(p + i);
      T e[kEach];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int c = 0; c < kEach; ++c) f[i + c] = to_f32(e[c]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_16(T* p, int n, bool vec, const float* f) {
  constexpr int kEach = 16 / sizeof(T);
  if (vec && n >= 16) {
#pragma unroll
    for (int i = 0; i < 16; i += kEach) {
      T e[kEach];
#pragma unroll
      for (int c = 0; c < kEach; ++c) e[c] = from_f32<T>(f[i + c]);
      uint4 v;
      __builtin_memcpy(&v, e, 16);
      *(uint4*)(p + i) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
}

// 64 columns a wave, 16 RT rows.
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(kExpandWaves * 64) void adapter_expand_kernel(const AdapterArgs a, int groups, int blocks, int per, int total,
                                                                           bool vec_out) {
  constexpr int kLane = Frag<T>::kLane, kStep = 4 * kLane;
  const int b = work_of_block(per, total);
  if (b < 0) return;
  const int t0 = b / blocks * (16 * RT), lane = threadIdx.x & 63, quad = lane >> 4, m = lane & 15;
  int group = b % blocks * kExpandWaves + (threadIdx.x >> 6);
  if (group >= groups) return;
  int s = 0;
  for (; s < a.S - 1; ++s) {
    const int here = (a.first[s + 1] - a.first[s] + 63) / 64;
    if (group < here) break;
    group -= here;
  }
  const int c0 = a.first[s] + group * 64, end = a.first[s + 1];
  const int c = c0 + quad * 16, n = end - c, C = a.S * a.R;   // this lane's columns of row t0 + 16 rt + m
  TileAdapters<RT> tile(a, t0);
  if (a.base != a.out && blockIdx.y == 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int t = t0 + rt * 16 + m;
      if (t < a.T && !(tile.left >> (rt * 16 + m) & 1)) {
        float f[16];
        load_16((const T*)a.base + t * a.ldb + c, n, vec_out, f);
        store_16((T*)a.out + t * a.ldo + c, n, vec_out, f);
      }
    }
  }
  for (int pass = 0; tile.left; ++pass) {
    unsigned long long rows;
    int rank;
    const int g = tile.next(a, rows, rank);
    if (pass % gridDim.y != blockIdx.y) continue;
    const T* brow[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      brow[j] = (const T*)a.b + ((int64_t)g * a.N + min(c0 + (m >> 2) * 16 + j * 4 + (m & 3), end - 1)) * a.R;
    f32x4 acc[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < rank; k0 += kStep) {
      const int k = k0 + quad * kLane;
      Frag<T> bf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bf[j] = load_frag<VEC>(brow[j], k, rank);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (RT > 1 && !(rows >> (rt * 16) & 0xffff)) continue;
        Frag<T> high, low;
        load_h<VEC>(a.h + (int64_t)min(t0 + rt * 16 + m, a.T - 1) * C + s * a.R, k, rank, high, low);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[rt][j] = Frag<T>::mma(bf[j], high, acc[rt][j]);
          if constexpr (sizeof(T) == 2) acc[rt][j] = Frag<T>::mma(bf[j], low, acc[rt][j]);
        }
      }
    }
    const float scale = a.scale[g];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int t = t0 + rt * 16 + m;
      if (!(rows >> (rt * 16 + m) & 1)) continue;
      float f[16];
      load_16((const T*)a.base + t * a.ldb + c, n, vec_out, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[j * 4 + i] += scale * acc[rt][j][i];
      }
      store_16((T*)a.out + t * a.ldo + c, n, vec_out, f);
    }
  }
}

// Blocks side by side for the adapters that a tile of rows may have, while the tiles are few; one goes through them all where they
// are many.
static int side_by_side(const AdapterArgs& a, long long blocks, int rows) {
  const int most = std::min(std::min(rows, a.T), a.L);
  return (int)std::max(1ll, std::min<long long>(most, 4ll * device_cu_count() / blocks));
}

template <typename T, int RT, int CT>
static void shrink(const AdapterArgs& a, hipStream_t stream) {
  constexpr int kLane = Frag<T>::kLane;
  const int groups = (a.S * a.R + CT * 16 - 1) / (CT * 16), total = (a.T + 16 * RT - 1) / (16 * RT) * groups;
  const int per = RT > 1 ? (total + kXcds - 1) / kXcds : 0;
  const dim3 grid(per ? per * kXcds : total, side_by_side(a, total, 16 * RT));
  const bool vec = (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.a % 16 == 0 && a.K % kLane == 0 && a.ldx % kLane == 0;
  if (vec) adapter_shrink_kernel<T, RT, CT, true><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups, per, total);
  else adapter_shrink_kernel<T, RT, CT, false><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups, per, total);
}

template <typename T, int RT>
static void expand(const AdapterArgs& a, hipStream_t stream) {
  constexpr int kLane = Frag<T>::kLane;
  int groups = 0;
  bool vec_out = (uintptr_t)a.out % 16 == 0 && (uintptr_t)a.base % 16 == 0 && a.ldo * sizeof(T) % 16 == 0 && a.ldb * sizeof(T) % 16 == 0;
  for (int s = 0; s < a.S; ++s) {
    groups += (a.first[s + 1] - a.first[s] + 63) / 64;
    vec_out &= a.first[s] * sizeof(T) % 16 == 0;
  }
  const int blocks = (groups + kExpandWaves - 1) / kExpandWaves, total = (a.T + 16 * RT - 1) / (16 * RT) * blocks;
  const int per = RT > 1 ? (total + kXcds - 1) / kXcds : 0;
  const dim3 grid(per ? per * kXcds : total, side_by_side(a, total, 16 * RT));
  const bool vec = (uintptr_t)a.b % 16 == 0 && a.R % kLane == 0;
  if (vec) adapter_expand_kernel<T, RT, true><<<grid, kExpandWaves * 64, 0, stream>>>(a, groups, blocks, per, total, vec_out);
  else adapter_expand_kernel<T, RT, false><<<grid, kExpandWaves * 64, 0, stream>>>(a, groups, blocks, per, total, vec_out);
}

template <typename T>
static void launch(const AdapterArgs& a, hipStream_t stream) {
  if (a.T >= 512) {
    shrink<T, 2, 4>(a, stream);
    expand<T, 4>(a, stream);
  } else {
    shrink<T, 1, 1>(a, stream);
    expand<T, 1>(a, stream);
  }
}

}  // namespace ninfer

using namespace ninfer;

extern "C" int ninfer_adapter_args_bytes() { return (int)sizeof(AdapterArgs); }

extern "C" int ninfer_adapter_add(const AdapterArgs* args, hipStream_t stream) {
  NINFER_REQUIRE(args, "adapter_add: no arguments");
  const AdapterArgs& a = *args;
  NINFER_REQUIRE(a.T > 0 && a.K > 0 && a.R > 0 && a.L > 0, "adapter_add: T=%d K=%d R=%d L=%d must be positive", a.T, a.K, a.R, a.L);
  NINFER_REQUIRE(a.S >= 1 && a.S <= 4 && a.first[0] == 0 && a.first[a.S] == a.N, "adapter_add: %d slices of %d columns", a.S, a.N);
  for (int s = 0; s < a.S; ++s)
    NINFER_REQUIRE(a.first[s] < a.first[s + 1], "adapter_add: slice %d has no columns", s);
  NINFER_REQUIRE(a.x && a.a && a.b && a.scale && a.ranks && a.row_adapter && a.base && a.out && a.h, "adapter_add: a required array is null");
  NINFER_REQUIRE(a.ldx >= a.K && a.ldb >= a.N && a.ldo >= a.N, "adapter_add: a row stride is less than the row");
  NINFER_REQUIRE(a.base != a.out || a.ldb == a.ldo, "adapter_add: in place with two row strides");
  NINFER_REQUIRE((long long)a.T * a.S * a.R <= 0x7fffffff && (long long)a.T * (a.N / 64 + 8) / 16 <= 0x7fffffff,
                 "adapter_add: %d rows are too many", a.T);
  NINFER_REQUIRE(a.dtype == kF32 || a.dtype == kBF16, "adapter_add: dtype %d", a.dtype);
  if (a.dtype == kBF16) launch<bf16>(a, stream);
  else launch<float>(a, stream);
  NINFER_LAUNCH_CHECK();
  return 0;
}
