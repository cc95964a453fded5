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
// out of L2. 64 rows of 151,936 tokens with 2,500 entries each take 22 us (3.6 TB/s), 256 with 6,000 98 (3.4): what the
// waits for the lists add to reading and writing at the 5.1 TB/s of a copy.
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

constexpr int kAdjustThreads = 512;
constexpr int kAdjustQuads = 2;   // groups of 4 logits a thread holds
constexpr int kAdjustPart = kAdjustThreads * kAdjustQuads * 4;
constexpr int kAdjustLists = 8;   // list entries a thread has on their way at a time

// l / p^count, or l p^count for a logit that is not positive: the power by squaring, at most 31 turns.
__device__ __forceinline__ float penalised(float l, float p, unsigned count) {
  if (l == 0.f || fabsf(l) == INFINITY) return l;   // (p^count may be infinite, or 0)
  double power = 1., square = p;
  for (; count; count >>= 1, square *= square)
    if (count & 1) power *= square;
  return (float)(l > 0.f ? (double)l / power : (double)l * power);
}

struct AdjustLds {
  // By token of the part: first what the list's entries say of it (0: nothing), then kListed and a 32-bit float.
  unsigned long long of[kAdjustPart];
  // Entries of the list whose token lies in the part, as many as leave room for four blocks' memory on a CU (the others are read
  // where they are found): kEntry * the entry, from the list's first on, and the token.
  unsigned entry[kAdjustPart / 2 - 2];
  int n_entries;
};
static_assert(sizeof(AdjustLds) <= 40960, "four blocks to a CU");
constexpr unsigned long long kListed = 1ull << 63;
constexpr unsigned kEntry = kAdjustPart, kMostEntries = kAdjustPart / 2 - 2;
constexpr int kEntriesEach = (kMostEntries + kAdjustThreads - 1) / kAdjustThreads;

// Where `of` has a token: a thread's four neighbouring logits in four banks' worth of numbers side by side with its neighbours'.
__device__ __forceinline__ int place_of(int token) { return (token & 3) * (kAdjustPart / 4) + (token >> 2); }

// The tokens of a list's next entries, from e0 on a thread each; none for turns behind the list's end.
__device__ __forceinline__ void load_tokens(int (&t)[kAdjustLists], const int* tokens, int e0, int end) {
#pragma unroll
  for (int u = 0; u < kAdjustLists; ++u) {
    if (e0 + u * kAdjustThreads >= end) break;
    t[u] = tokens[min(e0 + u * kAdjustThreads + (int)threadIdx.x, end - 1)];
  }
}

// One list of the row, entries [first, end), `t` the tokens of the first ones, l.of all 0. `read(entry, token)` reads what an entry
// says; `note(entry, token, that)` puts it into l.of and says whether it is its token's first; `value(what l.of has, that)`
// makes a float for the token, in the thread that had its first entry; `again(token, what l.of has)` the same for tokens all of
// whose entries found no room; `put(logit, float)` goes over the listed tokens' logits.
// What entries say is read, and the values are made, by as many threads as there are entries and tokens of the part: in the loop over
// the list, or over the logits that a thread holds, nearly every wave would wait for those loads, and run a power and a quotient
// in 64 bits, in every turn (256 rows of 151,936 tokens with 6,000 entries each, us: 181 so, 141 with the values alone made so).
template <typename Read, typename Note, typename Value, typename Again, typename Put>
__device__ __forceinline__ bool apply_list(AdjustLds& l, int (&t)[kAdjustLists], const int* tokens, int first, int end, int t0, int n,
                                           float (&v)[kAdjustQuads][4], Read read, Note note, Value value, Again again, Put put) {
  const int tid = threadIdx.x;
  for (int e0 = first; e0 < end; e0 += kAdjustLists * kAdjustThreads) {
    if (e0 != first) load_tokens(t, tokens, e0, end);
#pragma unroll
    for (int u = 0; u < kAdjustLists; ++u) {
      if (e0 + u * kAdjustThreads >= end) break;
      const int e = e0 + u * kAdjustThreads + tid;
      const unsigned at = (unsigned)t[u] - (unsigned)t0;   // (ids outside the vocabulary fall outside every part)
      if (e < end && at < (unsigned)n) {
        const unsigned i = (unsigned)(e - first) < 0xffffffffu / kEntry ? atomicAdd(&l.n_entries, 1) : kMostEntries;
        if (i < kMostEntries) l.entry[i] = (unsigned)(e - first) * kEntry + at;
        else note(e, (int)at, read(e, (int)at));
      }
    }
  }
  __syncthreads();
  const int entries = min(l.n_entries, (int)kMostEntries);
  if (l.n_entries == 0 && (unsigned)(end - first) < 0xffffffffu / kEntry) return false;
  const bool all = l.n_entries <= (int)kMostEntries && (unsigned)(end - first) < 0xffffffffu / kEntry;
  unsigned mine[kEntriesEach];
  decltype(read(0, 0)) that[kEntriesEach];
  bool has[kEntriesEach];
#pragma unroll
  for (int u = 0; u < kEntriesEach; ++u) {
    has[u] = tid + u * kAdjustThreads < entries;
    if (has[u]) {
      mine[u] = l.entry[tid + u * kAdjustThreads];
      that[u] = read(first + (int)(mine[u] / kEntry), (int)(mine[u] % kEntry));
    }
  }
#pragma unroll
  for (int u = 0; u < kEntriesEach; ++u)
    if (has[u]) has[u] = note(first + (int)(mine[u] / kEntry), (int)(mine[u] % kEntry), that[u]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kEntriesEach; ++u) {
    if (has[u]) {
      const int at = (int)(mine[u] % kEntry);
      unsigned long long& of = l.of[place_of(at)];
      of = kListed | __float_as_uint(value(of, that[u]));
    }
  }
  __syncthreads();
  if (!all) {
    for (int at = tid; at < kAdjustPart; at += kAdjustThreads) {
      unsigned long long& of = l.of[place_of(at)];
      if (of && !(of & kListed)) of = kListed | __float_as_uint(again(at, of));
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned long long x = l.of[c * (kAdjustPart / 4) + u * kAdjustThreads + tid];
      if (x) put(v[u][c], __uint_as_float((unsigned)x));
    }
  }
  return true;
}

__global__ __launch_bounds__(kAdjustThreads) void adjust_logits_kernel(const AdjustArgs a, int parts) {
  __shared__ AdjustLds l;
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
  int ht[kAdjustLists], bt[kAdjustLists];
  if (h1 > h0) load_tokens(ht, a.hist_tokens, h0, h1);
  if (b1 > b0) load_tokens(bt, a.bias_tokens, b0, b1);
  float v[kAdjustQuads][4];
#pragma unroll
  for (int u = 0; u < kAdjustQuads; ++u) {
    const int i = (u * kAdjustThreads + tid) * 4;
    if (a.vec && i + 4 <= n) {
      load_row<4>(row + i, v[u]);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[u][c] = i + c < n ? row[i + c] : 0.f;
    }
  }
  const bool masked = m >= 0 && m < a.n_masks;
  uint32_t bits[kAdjustQuads];
  if (masked) {
    const uint32_t* words = a.masks + (int64_t)m * ((a.V + 31) / 32);
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) {
      const int i = t0 + min((u * kAdjustThreads + tid) * 4, n - 1);
      bits[u] = words[i >> 5] >> (i & 28);
    }
  }

  bool changed = masked || a.out != a.logits;
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < kAdjustPart / kAdjustThreads; ++i) l.of[i * kAdjustThreads + tid] = 0;
    if (tid == 0) l.n_entries = 0;
    __syncthreads();
  };
  bool dirty = false;
  if (h1 > h0) {
    clear();
    struct Said { unsigned count, generated; float logit; };
    auto penalty = [&](float x, unsigned long long counts) {
      if (rp != 1.f) x = penalised(x, rp, (unsigned)counts);
      const unsigned g = (unsigned)(counts >> 32);
      return g ? x - freq * (float)g - pres : x;
    };
    dirty = apply_list(
        l, ht, a.hist_tokens, h0, h1, t0, n, v,
        [&](int e, int at) {
          return Said{(unsigned)max(a.hist_counts[e], 0), a.hist_generated ? (unsigned)max(a.hist_generated[e], 0) : 0u, row[at]};
        },
        [&](int, int at, const Said& s) {
          return (s.count || s.generated) && atomicAdd(&l.of[place_of(at)], (unsigned long long)s.generated << 32 | s.count) == 0;
        },
        [&](unsigned long long counts, const Said& s) { return penalty(s.logit, counts); },
        [&](int at, unsigned long long counts) { return penalty(row[at], counts); },
        [](float& logit, float x) { logit = x; });
    changed |= dirty;
  }
  if (b1 > b0) {
    if (h1 > h0) __syncthreads();   // (the list before has been put)
    if (dirty || h1 <= h0) clear();
    struct Said { int entry; float bias; };
    changed |= apply_list(
        l, bt, a.bias_tokens, b0, b1, t0, n, v,
        [&](int e, int) { return Said{e, a.bias_values[e]}; },
        [&](int e, int at, const Said&) { return atomicMax(&l.of[place_of(at)], (unsigned long long)(e - b0) + 1) == 0; },
        [&](unsigned long long last, const Said& s) {
          const int e = b0 + (int)last - 1;
          return e == s.entry ? s.bias : a.bias_values[e];
        },
        [&](int, unsigned long long last) { return a.bias_values[b0 + (int)last - 1]; },
        [](float& logit, float x) { logit += x; });
  }
  if (!changed) return;
#pragma unroll
  for (int u = 0; u < kAdjustQuads; ++u) {
    const int i = (u * kAdjustThreads + tid) * 4;
    if (masked) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (!(bits[u] >> c & 1)) v[u][c] = -INFINITY;
    }
    if (a.vec && i + 4 <= n) {
      store_row<4>(to + i, v[u]);
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
