// What requests ask of their rows of logits before a token is drawn: penalties for repeated
// tokens, biases, and masks of what a grammar allows next. For a token of logit l that stands c
// times in its request's history, g of them generated, with the row's penalties p (repetition),
// f (frequency) and q (presence), a bias b, and the row's mask:
//
//   v = l > 0 ? l / p^c : l p^c     (p^c in 64 bits, so that the quotient is rounded once)
//   v = v - f g - q [g > 0] + b
//   v = -inf where the mask bars the token, whatever stands there (NaN and infinities too)
//
// One pass over the logits: what bounds it is reading and writing them. A block holds 4,096 logits
// of a row in registers and, while they are on their way, goes through the row's whole lists and
// adds up in shared memory what falls into its part. So the lists need no order, and a token may
// stand in a history more than once (whole numbers: the sums are exact in every order); of several
// biases of one token the last one of the list holds. A list is read by every block of its row, but
// out of L2. 64 rows of 151,936 tokens with 2,500 entries each take 19 us (4.3 TB/s), 256 with 6,000 87 (3.9; 72 where
// the logits lie in the memory-side cache), where a copy has 5.1 TB/s.
#include "sampling.h"

namespace ninfer {

struct AdjustArgs {
  const float* logits;      // [R, ld]
  float* out;               // [R, ldo]; may be logits
  const float *repetition, *presence, *frequency;   // [R], or null: 1, 0, 0
  const int *hist_offsets, *hist_tokens, *hist_counts, *hist_generated;   // [R + 1], [n_hist] (or null: no history)
  const int *bias_offsets, *bias_tokens;            // [R + 1], [n_bias] (or null)
  const float* bias_values;
  const uint32_t* masks;    // [n_masks, (V + 31) / 32], bit t % 32 of word t / 32: token t is allowed (or null)
  const int* mask_rows;     // [R]: the row's mask; outside [0, n_masks): none
  long long ld, ldo;
  int R, V, n_hist, n_bias, n_masks, vec;
};

typedef float Four __attribute__((ext_vector_type(4)));

constexpr int kAdjustThreads = 512;
constexpr int kAdjustQuads = 2;   // groups of 4 logits a thread holds
constexpr int kAdjustPart = kAdjustThreads * kAdjustQuads * 4;
constexpr int kAdjustLists = 8;   // entries of the history a thread has on their way at a time
constexpr int kAdjustBiases = 2;  // ... and of the biases
constexpr unsigned kMostBiases = 64;   // biases of a part that are held against one another, a lane each
constexpr unsigned kMostEntries = kAdjustPart / 2 - kMostBiases - 2;   // entries of a part: as leave room for four blocks' memory on a CU
constexpr int kFar = (int)(0xffffffffu / kAdjustPart);   // numbers of entries that a word has room for beside the token

// l / p^count, or l p^count for a logit that is not positive: the power by squaring, at most 31 turns.
__device__ __forceinline__ float penalised(float l, float p, unsigned count) {
  if (l == 0.f || fabsf(l) == INFINITY) return l;   // (p^count may be infinite, or 0)
  double power = 1., square = p;
  for (; count; count >>= 1, square *= square)
    if (count & 1) power *= square;
  return (float)(l > 0.f ? (double)l / power : (double)l * power);
}

struct AdjustLds {
  // By token of the part: first what the history's entries say of it (0: nothing), then kListed and a 32-bit float.
  unsigned long long of[kAdjustPart];
  // Entries whose token lies in the part: kAdjustPart * the entry, from the list's first on, and the token. Those of the history
  // that find no room are read where they are found.
  unsigned entry[kMostEntries], bias[kMostBiases];
  int n_entries, n_biases;

  // A thread's four neighbouring logits lie in four banks' worth of numbers side by side with its neighbours'.
  __device__ __forceinline__ unsigned long long& at(int token) { return of[(token & 3) * (kAdjustPart / 4) + (token >> 2)]; }
};
static_assert(sizeof(AdjustLds) <= 40960, "four blocks to a CU");
constexpr unsigned long long kListed = 1ull << 63;

// The tokens of a list's next entries, from e0 on a thread each; none for turns behind the list's end.
template <int N>
__device__ __forceinline__ void load_tokens(int (&t)[N], const int* tokens, int e0, int end) {
#pragma unroll
  for (int u = 0; u < N; ++u)
    if (e0 + u * kAdjustThreads < end) t[u] = tokens[min(e0 + u * kAdjustThreads + (int)threadIdx.x, end - 1)];
}

// found(entry, token of the part) for the entries [first, end) of a list whose tokens lie in the part of n logits from t0 on; `t`: the
// first ones' tokens.
template <int N, typename Found>
__device__ __forceinline__ void scan_list(int (&t)[N], const int* tokens, int first, int end, int t0, int n, Found found) {
  for (int e0 = first; e0 < end; e0 += N * kAdjustThreads) {
    if (e0 != first) load_tokens(t, tokens, e0, end);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (e0 + u * kAdjustThreads >= end) break;
      const int e = e0 + u * kAdjustThreads + (int)threadIdx.x;
      const unsigned at = (unsigned)t[u] - (unsigned)t0;   // (ids outside the vocabulary fall outside every part)
      if (e < end && at < (unsigned)n) found(e, (int)at);
    }
  }
}

// What entries say is read, and the values of their tokens are made, by as many threads as there are entries in the part: in the loop over
// the list, or over the logits that a thread holds, nearly every wave would wait for those loads, and run a power and a quotient
// in 64 bits, in every turn (256 rows of 151,936 tokens with 6,000 entries each, us: 181 so, 141 with the values alone made so). Both lists go
// through these steps together: a block's time is its waits, for memory and for its waves (these rows 100 one list after the other, 92 together).
__global__ __launch_bounds__(kAdjustThreads) void adjust_logits_kernel(const AdjustArgs a, int parts) {
  __shared__ AdjustLds l;
  constexpr int kEach = ((int)kMostEntries + kAdjustThreads - 1) / kAdjustThreads;
  const int r = blockIdx.x / parts, t0 = (blockIdx.x % parts) * kAdjustPart, tid = threadIdx.x;
  const int n = min(kAdjustPart, a.V - t0);
  const float* row = a.logits + r * a.ld + t0;
  float* to = a.out + r * a.ldo + t0;

  // (everything that says where to look next is on its way at once)
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0, m = -1;
  if (a.hist_offsets) h0 = a.hist_offsets[r], h1 = a.hist_offsets[r + 1];
  if (a.bias_offsets) b0 = a.bias_offsets[r], b1 = a.bias_offsets[r + 1];
  if (a.mask_rows) m = a.mask_rows[r];
  const float rp = a.repetition ? a.repetition[r] : 1.f;
  const float freq = a.frequency ? a.frequency[r] : 0.f, pres = a.presence ? a.presence[r] : 0.f;

  h0 = max(h0, 0), h1 = min(h1, a.n_hist), b0 = max(b0, 0), b1 = min(b1, a.n_bias);
  if (rp == 1.f && freq == 0.f && pres == 0.f) h1 = h0;
  // (the lists before the logits: a load is waited for after those that were asked for before it)
  int ht[kAdjustLists], bt[kAdjustBiases];
  if (h1 > h0) load_tokens(ht, a.hist_tokens, h0, h1);
  if (b1 > b0) load_tokens(bt, a.bias_tokens, b0, b1);
  // (as many loads whatever the part, so that the wait for the lists does not have to be one for the logits too)
  const bool fours = a.vec && n % 4 == 0;
  Four v[kAdjustQuads];
  if (fours) {
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) v[u] = *(const Four*)(row + min((u * kAdjustThreads + tid) * 4, n - 4));
  } else {
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[u][c] = row[min((u * kAdjustThreads + tid) * 4 + c, n - 1)];
    }
  }
  const bool masked = m >= 0 && m < a.n_masks;
  uint32_t words[kAdjustQuads];
  if (masked) {
    const uint32_t* mask = a.masks + (int64_t)m * ((a.V + 31) / 32);
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) words[u] = mask[(t0 + min((u * kAdjustThreads + tid) * 4, n - 1)) >> 5];
  }

  bool changed = masked || a.out != a.logits;
  if (h1 > h0 || b1 > b0) {
    struct Said { unsigned count, generated; float logit; };
    auto clear = [&] {
#pragma unroll
      for (int i = 0; i < kAdjustPart / kAdjustThreads; ++i) l.of[i * kAdjustThreads + tid] = 0;
    };
    auto read = [&](int e, int at) {
      return Said{(unsigned)max(a.hist_counts[e], 0), a.hist_generated ? (unsigned)max(a.hist_generated[e], 0) : 0u, row[at]};
    };
    // (its token's first: the others leave the value to it)
    auto note = [&](int at, const Said& s) {
      return (s.count || s.generated) && atomicAdd(&l.at(at), (unsigned long long)s.generated << 32 | s.count) == 0;
    };
    auto penalty = [&](float x, unsigned long long counts) {
      if (rp != 1.f) x = penalised(x, rp, (unsigned)counts);
      const unsigned g = (unsigned)(counts >> 32);
      return g ? x - freq * (float)g - pres : x;
    };
    clear();
    if (tid == 0) l.n_entries = l.n_biases = 0;
    __syncthreads();
    if (h1 > h0)
      scan_list(ht, a.hist_tokens, h0, h1, t0, n, [&](int e, int at) {
        const unsigned i = e - h0 < kFar ? atomicAdd(&l.n_entries, 1) : kMostEntries;
        if (i < kMostEntries) l.entry[i] = (unsigned)(e - h0) * kAdjustPart + at;
        else note(at, read(e, at));
      });
    if (b1 > b0)
      scan_list(bt, a.bias_tokens, b0, b1, t0, n, [&](int e, int at) {
        const unsigned i = e - b0 < kFar ? atomicAdd(&l.n_biases, 1) : kMostBiases;
        if (i < kMostBiases) l.bias[i] = (unsigned)(e - b0) * kAdjustPart + at;
      });
    __syncthreads();
    const int entries = min(l.n_entries, (int)kMostEntries);
    const bool all = l.n_entries <= (int)kMostEntries && h1 - h0 <= kFar;
    const bool many = l.n_biases > (int)kMostBiases || b1 - b0 > kFar;   // (biases: by the table, later)
    const int biases = many ? 0 : l.n_biases;

    unsigned mine[kEach], of_bias = 0;
    Said that[kEach];
    bool has[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      has[u] = tid + u * kAdjustThreads < entries;
      if (has[u]) {
        mine[u] = l.entry[tid + u * kAdjustThreads];
        that[u] = read(h0 + (int)(mine[u] / kAdjustPart), (int)(mine[u] % kAdjustPart));
      }
    }
    const int j = kAdjustThreads - 1 - tid;   // (the last wave, which has the fewest of the others)
    bool last = j < biases;
    float bias = 0.f, biased = 0.f;
    if (j < (int)kMostBiases && biases) {
      of_bias = l.bias[min(j, biases - 1)];
      bias = a.bias_values[b0 + (int)(of_bias / kAdjustPart)], biased = row[of_bias % kAdjustPart];
      for (int i = 0; i < biases; ++i) {
        const unsigned other = __builtin_amdgcn_readlane(of_bias, 63 - i);
        last &= other <= of_bias || (other ^ of_bias) % kAdjustPart;
      }
    }
    if (entries || !all) {
#pragma unroll
      for (int u = 0; u < kEach; ++u)
        if (has[u]) has[u] = note((int)(mine[u] % kAdjustPart), that[u]);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        if (has[u]) {
          unsigned long long& of = l.at((int)(mine[u] % kAdjustPart));
          of = kListed | __float_as_uint(penalty(that[u].logit, of));
        }
      }
      __syncthreads();
    }
    if (!all) {   // (tokens all of whose entries found no room)
      for (int at = tid; at < n; at += kAdjustThreads) {
        unsigned long long& of = l.at(at);
        if (of && !(of & kListed)) of = kListed | __float_as_uint(penalty(row[at], of));
      }
      __syncthreads();
    }
    if (biases) {
      if (last) {
        unsigned long long& of = l.at((int)(of_bias % kAdjustPart));
        of = kListed | __float_as_uint((of ? __uint_as_float((unsigned)of) : biased) + bias);
      }
      __syncthreads();
    }
    if (entries || !all || biases) {
      changed = true;
#pragma unroll
      for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const unsigned long long x = l.of[c * (kAdjustPart / 4) + u * kAdjustThreads + tid];
          if (x) v[u][c] = __uint_as_float((unsigned)x);
        }
      }
    }
    if (many) {
      changed = true;
      __syncthreads();
      clear();
      __syncthreads();
      load_tokens(bt, a.bias_tokens, b0, b1);
      scan_list(bt, a.bias_tokens, b0, b1, t0, n, [&](int e, int at) { atomicMax(&l.at(at), (unsigned long long)(e - b0) + 1); });
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const unsigned long long x = l.of[c * (kAdjustPart / 4) + u * kAdjustThreads + tid];
          if (x) v[u][c] += a.bias_values[b0 + (int)(x - 1)];
        }
      }
    }
  }
  if (!changed) return;
#pragma unroll
  for (int u = 0; u < kAdjustQuads; ++u) {
    const int i = (u * kAdjustThreads + tid) * 4;
    if (masked) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (!(words[u] >> ((t0 + i) & 28) >> c & 1)) v[u][c] = -INFINITY;
    }
    if (fours) {
      // (past the L2, where the lists and the logits looked up again are: 92 us through it, 87 so, 72 with the logits in the
      // memory-side cache; 64 rows 19.9 and 19.0)
      if (i < n) __builtin_nontemporal_store(v[u], (Four*)(to + i));
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i + c < n) to[i + c] = v[u][c];
    }
  }
}

}  // namespace ninfer

using namespace ninfer;

extern "C" int ninfer_adjust_args_bytes() { return (int)sizeof(AdjustArgs); }

extern "C" int ninfer_adjust_logits(const AdjustArgs* args, hipStream_t stream) {
  NINFER_REQUIRE(args, "adjust_logits: no arguments");
  AdjustArgs a = *args;
  NINFER_REQUIRE(a.R > 0 && a.V > 0 && a.logits && a.out, "adjust_logits: R=%d V=%d must be positive, rows not null", a.R, a.V);
  NINFER_REQUIRE(a.V <= 0x7fffffff - kAdjustPart, "adjust_logits: rows of %d tokens are too long", a.V);   // (parts are counted past the row's end)
  NINFER_REQUIRE(a.ld >= a.V && a.ldo >= a.V, "adjust_logits: row stride %lld or %lld < vocabulary %d", a.ld, a.ldo, a.V);
  NINFER_REQUIRE(a.logits != a.out || a.ld == a.ldo, "adjust_logits: in place with two row strides");
  NINFER_REQUIRE(a.n_hist >= 0 && a.n_bias >= 0 && a.n_masks >= 0, "adjust_logits: a size is negative");
  constexpr int kMost = 0x7fffffff - 2 * kAdjustLists * kAdjustThreads;   // (a turn's entries are counted past the list's end)
  NINFER_REQUIRE(a.n_hist <= kMost && a.n_bias <= kMost, "adjust_logits: lists of %d and %d entries are too many", a.n_hist, a.n_bias);
  NINFER_REQUIRE(!a.hist_offsets || a.n_hist == 0 || (a.hist_tokens && a.hist_counts), "adjust_logits: a history without tokens or counts");
  NINFER_REQUIRE(!a.bias_offsets || a.n_bias == 0 || (a.bias_tokens && a.bias_values), "adjust_logits: biases without tokens or values");
  NINFER_REQUIRE(!a.mask_rows || a.n_masks == 0 || a.masks, "adjust_logits: rows name masks that are not given");
  const int parts = (a.V + kAdjustPart - 1) / kAdjustPart;
  NINFER_REQUIRE((long long)parts * a.R <= 0xffffffffll / kAdjustThreads, "adjust_logits: %d rows are too many", a.R);
  a.vec = row_aligned(a.logits) && row_aligned(a.out) && a.ld % 4 == 0 && a.ldo % 4 == 0;
  adjust_logits_kernel<<<parts * a.R, kAdjustThreads, 0, stream>>>(a, parts);
  NINFER_LAUNCH_CHECK();
  return 0;
}
