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

// The adapters of the 16 rows from t0 on: every wave goes through them in the order of their first rows.
struct TileAdapters {
  int mine;                 // lane i < 16: row t0 + i's adapter, -1 for none
  unsigned long long left;  // rows whose adapter has not been taken yet
  __device__ __forceinline__ TileAdapters(const AdapterArgs& a, int t0) {
    const int lane = threadIdx.x & 63;
    mine = lane < 16 && t0 + lane < a.T ? a.row_adapter[t0 + lane] : -1;
    if (mine >= a.L || mine < 0) mine = -1;
    left = __ballot(mine >= 0);
  }
  // The next adapter and the rows (bits) that have it.
  __device__ __forceinline__ int next(unsigned& rows) {
    const int g = __builtin_amdgcn_readlane(mine, __ffsll(left) - 1);
    rows = (unsigned)__ballot(mine == g);
    left &= ~(unsigned long long)rows;
    return g;
  }
};

template <typename T, int CT, bool VEC>
__global__ __launch_bounds__(kShrinkWaves * 64) void adapter_shrink_kernel(const AdapterArgs a, int groups) {
  __shared__ float part[kShrinkWaves][CT][64][4];
  constexpr int kLane = Frag<T>::kLane, kStep = 4 * kLane;
  const int t0 = blockIdx.x / groups * 16, j0 = blockIdx.x % groups * (CT * 16);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, quad = lane >> 4, C = a.S * a.R;
  const T* xrow = (const T*)a.x + (int64_t)min(t0 + (lane & 15), a.T - 1) * a.ldx;
  TileAdapters tile(a, t0);
  for (int pass = 0; tile.left; ++pass) {
    unsigned rows;
    const int g = tile.next(rows);
    if (pass % gridDim.y != blockIdx.y) continue;
    const int rank = min(max(a.ranks[g], 0), a.R);
    bool any = false;
    const T* arow[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int j = j0 + ct * 16 + (lane & 15);
      any |= j < C && j % a.R < rank;
      arow[ct] = (const T*)a.a + ((int64_t)g * C + min(j, C - 1)) * a.K;
    }
    if (!__ballot(any)) continue;
    f32x4 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    // wave w takes the steps w, w + 8, ..
    const int whole = VEC ? a.K / kStep : 0;
    int st = w;
    if constexpr (VEC) {
#pragma unroll 4
      for (; st < whole; st += kShrinkWaves) {
        const int k = st * kStep + quad * kLane;
        Frag<T> xf;
        xf.v = *(const decltype(xf.v)*)(xrow + k);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          Frag<T> af;
          af.v = *(const decltype(af.v)*)(arow[ct] + k);
          acc[ct] = Frag<T>::mma(xf, af, acc[ct]);
        }
      }
    }
    for (; st * kStep < a.K; st += kShrinkWaves) {
      const int k = st * kStep + quad * kLane;
      const Frag<T> xf = load_frag<VEC>(xrow, k, a.K);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[ct] = Frag<T>::mma(xf, load_frag<VEC>(arow[ct], k, a.K), acc[ct]);
    }
    __syncthreads();   // (the pass before has read its sums)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) *(f32x4*)part[w][ct][lane] = acc[ct];
    __syncthreads();
    for (int o = threadIdx.x; o < CT * 256; o += kShrinkWaves * 64) {
      const int ct = o >> 8, l = (o >> 2) & 63, row = (l >> 4) * 4 + (o & 3), j = j0 + ct * 16 + (l & 15);
      if (!(rows >> row & 1) || j >= C || j % a.R >= rank) continue;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kShrinkWaves; ++i) sum += part[i][ct][l][o & 3];
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

// Sixteen neighbouring columns of a row, the ones before `n` of them.
template <typename T>
__device__ __forceinline__ void load_16(const T* p, int n, bool vec, float* f) {
  if (vec && n >= 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_row<4>(p + 4 * i, f + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_16(T* p, int n, bool vec, const float* f) {
  if (vec && n >= 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_row<4>(p + 4 * i, f + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = from_f32<T>(f[i]);
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kExpandWaves * 64) void adapter_expand_kernel(const AdapterArgs a, int groups, int blocks, bool vec_out) {
  constexpr int kLane = Frag<T>::kLane, kStep = 4 * kLane;
  const int t0 = blockIdx.x / blocks * 16, lane = threadIdx.x & 63, quad = lane >> 4, m = lane & 15;
  int group = blockIdx.x % blocks * kExpandWaves + (threadIdx.x >> 6);
  if (group >= groups) return;
  int s = 0;
  for (; s < a.S - 1; ++s) {
    const int here = (a.first[s + 1] - a.first[s] + 63) / 64;
    if (group < here) break;
    group -= here;
  }
  const int c0 = a.first[s] + group * 64, end = a.first[s + 1];
  const int c = c0 + quad * 16, n = end - c;   // this lane's columns of row t0 + m
  const int t = min(t0 + m, a.T - 1), C = a.S * a.R;
  const T* from = (const T*)a.base + t * a.ldb + c;
  T* to = (T*)a.out + t * a.ldo + c;
  const float* hrow = a.h + (int64_t)t * C + s * a.R;
  TileAdapters tile(a, t0);
  if (a.base != a.out && blockIdx.y == 0 && t0 + m < a.T && !(tile.left >> m & 1)) {
    float f[16];
    load_16(from, n, vec_out, f);
    store_16(to, n, vec_out, f);
  }
  for (int pass = 0; tile.left; ++pass) {
    unsigned rows;
    const int g = tile.next(rows);
    if (pass % gridDim.y != blockIdx.y) continue;
    const bool mine = rows >> m & 1;
    float f[16];
    if (mine) load_16(from, n, vec_out, f);
    const int rank = min(max(a.ranks[g], 0), a.R);
    const T* brow[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      brow[j] = (const T*)a.b + ((int64_t)g * a.N + min(c0 + (m >> 2) * 16 + j * 4 + (m & 3), end - 1)) * a.R;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < rank; k0 += kStep) {
      const int k = k0 + quad * kLane;
      Frag<T> high, low;
      load_h<VEC>(hrow, k, rank, high, low);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Frag<T> bf = load_frag<VEC>(brow[j], k, rank);
        acc[j] = Frag<T>::mma(bf, high, acc[j]);
        if constexpr (sizeof(T) == 2) acc[j] = Frag<T>::mma(bf, low, acc[j]);
      }
    }
    if (!mine) continue;
    const float scale = a.scale[g];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[j * 4 + i] += scale * acc[j][i];
    }
    store_16(to, n, vec_out, f);
  }
}

template <typename T>
static void launch(const AdapterArgs& a, hipStream_t stream) {
  constexpr int kLane = Frag<T>::kLane;
  const int tiles = (a.T + 15) / 16, C = a.S * a.R, cus = device_cu_count();
  // Blocks of 64 columns share a tile of x between four products; blocks of 16 are more, where there are too few to fill the GPU.
  const bool wide = (long long)tiles * ((C + 63) / 64) >= cus;
  const int groups = wide ? (C + 63) / 64 : (C + 15) / 16;
  // A block for each adapter that a tile may have, while the tiles are few; one goes through them all where they are many.
  const int most = std::min(std::min(16, a.T), a.L);
  auto side_by_side = [&](long long blocks) { return (int)std::max(1ll, std::min<long long>(most, 8ll * cus / blocks)); };
  const bool vec = (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.a % 16 == 0 && a.K % kLane == 0 && a.ldx % kLane == 0;
  const dim3 grid(tiles * groups, side_by_side((long long)tiles * groups));
  if (wide && vec) adapter_shrink_kernel<T, 4, true><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups);
  if (wide && !vec) adapter_shrink_kernel<T, 4, false><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups);
  if (!wide && vec) adapter_shrink_kernel<T, 1, true><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups);
  if (!wide && !vec) adapter_shrink_kernel<T, 1, false><<<grid, kShrinkWaves * 64, 0, stream>>>(a, groups);
  int sets = 0;
  bool vec_out = (uintptr_t)a.out % 16 == 0 && (uintptr_t)a.base % 16 == 0 && a.ldo % 4 == 0 && a.ldb % 4 == 0;
  for (int s = 0; s < a.S; ++s) {
    sets += (a.first[s + 1] - a.first[s] + 63) / 64;
    vec_out &= a.first[s] % 4 == 0;
  }
  const int blocks = (sets + kExpandWaves - 1) / kExpandWaves;
  const dim3 egrid(tiles * blocks, side_by_side((long long)tiles * blocks));
  const bool evec = (uintptr_t)a.b % 16 == 0 && a.R % kLane == 0;
  if (evec) adapter_expand_kernel<T, true><<<egrid, kExpandWaves * 64, 0, stream>>>(a, sets, blocks, vec_out);
  else adapter_expand_kernel<T, false><<<egrid, kExpandWaves * 64, 0, stream>>>(a, sets, blocks, vec_out);
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
