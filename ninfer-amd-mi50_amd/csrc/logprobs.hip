// Log-probabilities of tokens, their places in the order of the row, and a row's first tokens with
// theirs. For a row l of V logits, m its largest,
//
//   log p(t) = (l_t - m) - log sum_i exp(l_i - m)
//   before(t) = tokens with a larger logit, or an equal one and a lower id
//
// and the best `top` tokens are those of before = 0 .. top - 1. A row in which nothing has mass (all
// -inf) has log p = -inf everywhere; tokens at +inf share the mass between them; a NaN in a row makes
// every log p of it NaN and stands behind all other tokens in the order.
//
// Two launches. The first reads the logits once, which bounds the whole: a block takes 4,096 logits of
// a row and leaves their maximum, the sum of exponentials against it, how many come before the token
// asked for, and each thread's largest key (of 16 logits). The second, a block a row, joins the parts
// in a fixed order and finds the best tokens from those keys: the top-th largest of 64 groups' maxima
// is a bound that at least `top` logits reach, and only the logits of threads whose key reaches it (about
// as many as `top`) are looked at again. A row in which very many logits are equal to the bound goes through its logits
// once per token instead. 512 rows of 151,936 tokens, no list: 53 us (5.9 TB/s with the join; the first launch alone 48); 64 rows with
// their 20 best tokens 17 (9 and 7), one row 10: the second launch's waits, and the launch itself, are most of it.
#include "sampling.h"
#include <type_traits>

namespace ninfer {

typedef float Four __attribute__((ext_vector_type(4)));

constexpr int kLpThreads = 256;
constexpr int kLpQuads = 4;   // groups of 4 logits a thread holds
constexpr int kLpPart = kLpThreads * kLpQuads * 4;
constexpr int kLpTop = 64;          // most tokens that are listed: the groups the bound is taken from
constexpr int kLpJoinThreads = 1024;
constexpr int kLpSegments = 256;    // most threads of the first launch whose logits are looked at again
constexpr int kLpMostTokens = 0x7fffffff - kLpPart;   // (a turn's and a part's tokens are counted past the row's end)
constexpr int kLpFound = 1024;      // ... and most of these logits that reach the bound

struct LogprobArgs {
  const float* logits;   // [R, ld]
  const int* tokens;     // [R], or null
  float* logprob;        // [R], or null (as tokens)
  int* before;           // [R], or null
  int* best;             // [R, top]
  float* best_logprob;   // [R, top]
  float2* sums;          // [R, parts]: maximum, sum
  int* counts;           // [R, parts]
  uint32_t* keys;        // [R, parts * kLpThreads]
  long long ld;
  int R, V, top, vec;
};

// The order of tokens: NaN behind everything.
__device__ __forceinline__ uint32_t token_key(float v) { return v != v ? 0u : ordered_key(v); }

// exp(v - m) for v <= m, as it goes into a sum; tokens at an infinite maximum count 1.
__device__ __forceinline__ float exp_above(float v, float m) { return v == m ? 1.f : __expf(v - m); }

__global__ __launch_bounds__(kLpThreads) void logprob_parts_kernel(const LogprobArgs a, int parts) {
  __shared__ float red_m[kLpThreads / 64], red_s[kLpThreads / 64];
  __shared__ int red_c[kLpThreads / 64];
  const int r = blockIdx.x / parts, part = blockIdx.x % parts, t0 = part * kLpPart, tid = threadIdx.x;
  const int n = min(kLpPart, a.V - t0), lane = tid & 63, w = tid >> 6;
  const float* row = a.logits + r * a.ld;
  const int token = a.tokens ? a.tokens[r] : -1;
  const bool asked = token >= 0 && token < a.V, whole = n == kLpPart;
  // (as many loads whatever the part, all on their way at once, and past the L2: 512 rows of 151,936 tokens 58 us through it,
  // 53 so; where the logits lie in the memory-side cache 54 and 51, 64 rows 16.2 and 15.2)
  Four v[kLpQuads];
  if (a.vec && n % 4 == 0) {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) v[u] = __builtin_nontemporal_load((const Four*)(row + t0 + min((u * kLpThreads + tid) * 4, n - 4)));
  } else {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[u][c] = row[t0 + min((u * kLpThreads + tid) * 4 + c, n - 1)];
    }
  }
  const float mine = asked ? row[token] : 0.f;
  if (!whole) {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if ((u * kLpThreads + tid) * 4 + c >= n) v[u][c] = -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < kLpQuads; ++u) m = fmaxf(fmaxf(m, fmaxf(v[u][0], v[u][1])), fmaxf(v[u][2], v[u][3]));
  // (a thread of nothing but NaN has the key of -inf, which its logits do not reach: the second launch notices)
  if (a.top) a.keys[((int64_t)r * parts + part) * kLpThreads + tid] = ordered_key(m);
  m = wave_max(m);
  if (lane == 0) red_m[w] = m;

  // What stands before the token: in parts before its own, logits as large as its own; in those behind it, larger ones.
  int count = 0;
  if (!asked) {
  } else if (mine == mine && token >= t0 + kLpPart) {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) count += v[u][c] >= mine;
    }
  } else if (mine == mine && token < t0) {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) count += v[u][c] > mine;
    }
  } else {
    const uint32_t key = token_key(mine);
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = (u * kLpThreads + tid) * 4 + c;
        const uint32_t k = token_key(v[u][c]);
        count += i < n && (k > key || (k == key && t0 + i < token));
      }
    }
  }
  __syncthreads();
  m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
  float s = 0.f;
  if (fabsf(m) < INFINITY) {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s += __expf(v[u][c] - m);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kLpQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) s += exp_above(v[u][c], m);
    }
  }
  s = wave_sum(s);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) count += __shfl_xor(count, off, 64);
  if (lane == 0) red_s[w] = s, red_c[w] = count;
  __syncthreads();
  if (tid == 0) {
    const int64_t at = (int64_t)r * parts + part;
    a.sums[at] = make_float2(m, (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]));
    a.counts[at] = (red_c[0] + red_c[1]) + (red_c[2] + red_c[3]);
  }
}

struct LpLds {
  uint32_t group[kLpJoinThreads / 64][64];
  uint32_t segment[kLpSegments];
  unsigned long long found[kLpFound];
  unsigned long long best[kLpTop], red[kLpJoinThreads / 64];
  float max, log_sum;
  uint32_t bound;
  int segments, n_found;
};

// The first key of `top` tokens of a row, one after the other: every turn the whole row.
__device__ void best_by_turns(const LogprobArgs& a, const float* row, LpLds& l) {
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    unsigned long long mine = 0;
    for (int i = threadIdx.x; i < a.V; i += kLpJoinThreads) {
      const unsigned long long k = (unsigned long long)token_key(row[i]) << 32 | ~(uint32_t)i;
      if (k < last && k > mine) mine = k;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mine = max(mine, (unsigned long long)__shfl_xor(mine, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) l.red[threadIdx.x >> 6] = mine;
    __syncthreads();
    mine = l.red[0];
    for (int i = 1; i < kLpJoinThreads / 64; ++i) mine = max(mine, l.red[i]);
    last = mine;
    if (threadIdx.x == 0) l.best[j] = mine;
  }
  __syncthreads();
}

// The logit of a key (+0 for -0; a key of NaN is asked for only in rows whose log-probabilities are all NaN).
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// Joins a row's parts; with TOP also its best tokens. Without, a block is one wave. What the second part of the work waits for,
// one load after the other, is its time (8 us for one row of 151,936 tokens): the parts are joined by the last wave while the
// others look for the bound, and keys are held from one look to the next.
template <bool TOP>
__global__ __launch_bounds__(TOP ? kLpJoinThreads : 64) void logprob_join_kernel(const LogprobArgs a, int parts) {
  __shared__ typename std::conditional<TOP, LpLds, int>::type lds;
  constexpr int kHeld = 16;   // keys a thread holds: of rows of up to 262,144 tokens all
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const float* row = a.logits + r * a.ld;
  const int64_t base = (int64_t)r * parts;
  auto log_p = [](float v, float m, float log_sum) {   // (a NaN among the logits is one in log_sum)
    return log_sum != log_sum ? log_sum : m == -INFINITY ? m : (v == m ? 0.f : v - m) - log_sum;
  };
  const int n = parts * kLpThreads;
  uint32_t held[kHeld];
  if constexpr (TOP) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int i = tid + u * kLpJoinThreads;
      held[u] = i < n ? a.keys[base * kLpThreads + i] : 0;
    }
  }
  if (tid >= (TOP ? kLpJoinThreads - 64 : 0)) {
    const int token = a.tokens ? a.tokens[r] : -1;
    const bool asked = token >= 0 && token < a.V;
    const float mine = asked ? row[token] : 0.f;
    float m = -INFINITY, s = 0.f;
    int count = 0;
    for (int p = lane; p < parts; p += 64) m = fmaxf(m, a.sums[base + p].x);
    m = wave_max(m);
    for (int p = lane; p < parts; p += 64) {
      const float2 x = a.sums[base + p];
      s += x.y * exp_above(x.x, m);
      count += a.counts[base + p];
    }
    s = wave_sum(s);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) count += __shfl_xor(count, off, 64);
    const float log_sum = logf(s);
    if (lane == 0) {
      if (a.tokens) {
        a.logprob[r] = asked ? log_p(mine, m, log_sum) : __builtin_nanf("");
        a.before[r] = asked ? count : -1;
      }
      if constexpr (TOP) lds.max = m, lds.log_sum = log_sum;
    }
  }
  if constexpr (TOP) {
    LpLds& l = lds;
    if (tid == 0) l.segments = 0, l.n_found = 0;
    const uint32_t* keys = a.keys + base * kLpThreads;
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) most = max(most, held[u]);
    for (int i = tid + kHeld * kLpJoinThreads; i < n; i += kLpJoinThreads) most = max(most, keys[i]);
    l.group[tid >> 6][lane] = most;
    __syncthreads();
    if (tid < 64) {
#pragma unroll
      for (int i = 0; i < kLpJoinThreads / 64; ++i) most = max(most, l.group[i][lane]);
      int place = 0;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const uint32_t k = __builtin_amdgcn_readlane(most, i);
        place += k > most || (k == most && i < lane);
      }
      if (place == a.top - 1) l.bound = most;
    }
    __syncthreads();
    const uint32_t bound = l.bound;
    auto list = [&](int i, uint32_t key) {
      if (key >= bound && i < n) {
        const int at = atomicAdd(&l.segments, 1);
        if (at < kLpSegments) l.segment[at] = i;
      }
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u) list(tid + u * kLpJoinThreads, held[u]);
    for (int i = tid + kHeld * kLpJoinThreads; i < n; i += kLpJoinThreads) list(i, keys[i]);
    __syncthreads();
    const int segments = l.segments;
    if (segments <= kLpSegments) {
      constexpr int kEach = kLpQuads * 4;
      for (int j = tid; j < segments * kEach; j += kLpJoinThreads) {
        const int seg = l.segment[j / kEach], x = j % kEach;
        const int i = seg / kLpThreads * kLpPart + (x / 4 * kLpThreads + seg % kLpThreads) * 4 + x % 4;
        if (i >= a.V) continue;
        const uint32_t k = token_key(row[i]);
        if (k >= bound) {
          const int at = atomicAdd(&l.n_found, 1);
          if (at < kLpFound) l.found[at] = (unsigned long long)k << 32 | ~(uint32_t)i;
        }
      }
    }
    __syncthreads();
    const int found = l.n_found;
    if (segments > kLpSegments || found > kLpFound || found < a.top) {
      best_by_turns(a, row, l);
    } else {
      for (int j = tid; j < found; j += kLpJoinThreads) {
        const unsigned long long k = l.found[j];
        int place = 0;
        for (int i = 0; i < found; ++i) place += l.found[i] > k;
        if (place < a.top) l.best[place] = k;
      }
      __syncthreads();
    }
    if (tid < a.top) {
      const unsigned long long k = l.best[tid];
      a.best[(int64_t)r * a.top + tid] = (int)~(uint32_t)k;
      a.best_logprob[(int64_t)r * a.top + tid] = log_p(logit_of((uint32_t)(k >> 32)), l.max, l.log_sum);
    }
  }
}

}  // namespace ninfer

using namespace ninfer;

extern "C" int ninfer_logprob_args_bytes() { return (int)sizeof(LogprobArgs); }
extern "C" int ninfer_logprob_most() { return kLpTop; }

// Bytes of scratch, aligned to 16: the parts' sums, counts and, with top > 0, keys.
extern "C" long long ninfer_logprob_scratch_bytes(int R, int V, int top) {
  const long long parts = ((long long)V + kLpPart - 1) / kLpPart * R;
  return parts * 8 + (parts * 4 + 15) / 16 * 16 + (top > 0 ? parts * kLpThreads * 4 : 0);
}

extern "C" int ninfer_token_logprobs(const LogprobArgs* args, void* scratch, hipStream_t stream) {
  NINFER_REQUIRE(args && scratch && (uintptr_t)scratch % 16 == 0, "token_logprobs: no arguments, or scratch not aligned");
  LogprobArgs a = *args;
  NINFER_REQUIRE(a.R > 0 && a.V > 0 && a.logits, "token_logprobs: R=%d V=%d must be positive, rows not null", a.R, a.V);
  NINFER_REQUIRE(a.V <= kLpMostTokens, "token_logprobs: rows of %d tokens are too long", a.V);
  NINFER_REQUIRE(a.ld >= a.V, "token_logprobs: row stride %lld < vocabulary %d", a.ld, a.V);
  NINFER_REQUIRE(a.top >= 0 && a.top <= kLpTop && a.top <= a.V, "token_logprobs: top %d is outside [0, min(%d, %d)]", a.top, kLpTop, a.V);
  NINFER_REQUIRE(!a.tokens || (a.logprob && a.before), "token_logprobs: tokens without a place for their numbers");
  NINFER_REQUIRE(a.top == 0 || (a.best && a.best_logprob), "token_logprobs: no place for the best tokens");
  NINFER_REQUIRE(a.tokens || a.top > 0, "token_logprobs: nothing is asked for");
  const int parts = (a.V + kLpPart - 1) / kLpPart;
  const long long blocks = (long long)parts * a.R;
  NINFER_REQUIRE(blocks <= 0xffffffffll / kLpThreads && a.R <= 0xffffffffll / kLpJoinThreads, "token_logprobs: %d rows are too many", a.R);
  a.vec = row_aligned(a.logits) && a.ld % 4 == 0;
  char* at = (char*)scratch;
  a.sums = (float2*)at;
  a.counts = (int*)(at + blocks * 8);
  a.keys = (uint32_t*)(at + blocks * 8 + (blocks * 4 + 15) / 16 * 16);
  logprob_parts_kernel<<<(unsigned)blocks, kLpThreads, 0, stream>>>(a, parts);
  NINFER_LAUNCH_CHECK();
  if (a.top > 0)
    logprob_join_kernel<true><<<a.R, kLpJoinThreads, 0, stream>>>(a, parts);
  else
    logprob_join_kernel<false><<<a.R, 64, 0, stream>>>(a, parts);
  NINFER_LAUNCH_CHECK();
  return 0;
}
