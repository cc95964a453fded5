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
// out of L2.
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

constexpr int kAdjustThreads = 256;
constexpr int kAdjustQuads = 4;   // groups of 4 logits a thread holds
constexpr int kAdjustPart = kAdjustThreads * kAdjustQuads * 4;
constexpr int kAdjustLists = 8;   // list entries a thread has on their way at a time

// l / p^count, or l p^count for a logit that is not positive: the power by squaring, at most 31 turns.
__device__ __forceinline__ float penalised(float l, float p, unsigned count) {
  if (l == 0.f) return l;   // (p^count may be infinite)
  double power = 1., square = p;
  for (; count; count >>= 1, square *= square)
    if (count & 1) power *= square;
  return (float)(l > 0.f ? (double)l / power : (double)l * power);
}

// Calls f(entry) for the entries [first, end) whose token lies in [t0, t0 + n).
template <typename F>
__device__ __forceinline__ void for_tokens_of_part(const int* tokens, int first, int end, int t0, int n, F f) {
  for (int e0 = first + (int)threadIdx.x; e0 < end; e0 += kAdjustLists * kAdjustThreads) {
    int t[kAdjustLists];
#pragma unroll
    for (int u = 0; u < kAdjustLists; ++u) {
      const int e = e0 + u * kAdjustThreads;
      t[u] = tokens[e < end ? e : end - 1];
    }
#pragma unroll
    for (int u = 0; u < kAdjustLists; ++u) {
      const int e = e0 + u * kAdjustThreads;
      const unsigned at = (unsigned)t[u] - (unsigned)t0;   // (ids outside the vocabulary fall outside every part)
      if (e < end && at < (unsigned)n) f(e, (int)at);
    }
  }
}

__global__ __launch_bounds__(kAdjustThreads) void adjust_logits_kernel(const AdjustArgs a, int parts) {
  __shared__ unsigned long long seen[kAdjustPart];   // counts: all in the lower half, generated ones in the upper
  const int r = blockIdx.x / parts, t0 = (blockIdx.x % parts) * kAdjustPart, tid = threadIdx.x;
  const int n = min(kAdjustPart, a.V - t0);
  const float* row = a.logits + r * a.ld + t0;
  float* to = a.out + r * a.ldo + t0;

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

  const float rp = a.repetition ? a.repetition[r] : 1.f;
  const float freq = a.frequency ? a.frequency[r] : 0.f, pres = a.presence ? a.presence[r] : 0.f;
  bool changed = a.out != a.logits;
  int first = 0, end = 0;
  if (a.hist_offsets && (rp != 1.f || freq != 0.f || pres != 0.f)) {
    first = max(a.hist_offsets[r], 0);
    end = min(a.hist_offsets[r + 1], a.n_hist);
  }
  if (end > first) {
    for (int i = tid; i < kAdjustPart; i += kAdjustThreads) seen[i] = 0;
    __syncthreads();
    for_tokens_of_part(a.hist_tokens, first, end, t0, n, [&](int e, int at) {
      const unsigned c = max(a.hist_counts[e], 0), g = a.hist_generated ? max(a.hist_generated[e], 0) : 0;
      atomicAdd(&seen[at], (unsigned long long)g << 32 | c);
    });
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const unsigned long long s = seen[(u * kAdjustThreads + tid) * 4 + c];
        if (s == 0) continue;
        changed = true;
        float x = v[u][c];
        if (rp != 1.f) x = penalised(x, rp, (unsigned)s);
        const unsigned g = (unsigned)(s >> 32);
        if (g) x = x - freq * (float)g - pres;
        v[u][c] = x;
      }
    }
  }
  first = end = 0;
  if (a.bias_offsets) {
    first = max(a.bias_offsets[r], 0);
    end = min(a.bias_offsets[r + 1], a.n_bias);
  }
  if (end > first) {
    unsigned* last = (unsigned*)seen;   // 1 + the list's last entry for the token
    __syncthreads();
    for (int i = tid; i < kAdjustPart; i += kAdjustThreads) last[i] = 0;
    __syncthreads();
    for_tokens_of_part(a.bias_tokens, first, end, t0, n,
                       [&](int e, int at) { atomicMax(&last[at], (unsigned)(e - first) + 1u); });
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const unsigned at = last[(u * kAdjustThreads + tid) * 4 + c];
        if (at) {
          v[u][c] += a.bias_values[first + at - 1];
          changed = true;
        }
      }
    }
  }
  const int m = a.mask_rows ? a.mask_rows[r] : -1;
  if (m >= 0 && m < a.n_masks) {
    const uint32_t* words = a.masks + (int64_t)m * ((a.V + 31) / 32);
#pragma unroll
    for (int u = 0; u < kAdjustQuads; ++u) {
      const int i = (u * kAdjustThreads + tid) * 4;
      if (i >= n) continue;
      const uint32_t bits = words[(t0 + i) >> 5] >> ((t0 + i) & 31);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (!(bits >> c & 1)) v[u][c] = -INFINITY;
    }
    changed = true;
  }
  if (!changed) return;
#pragma unroll
  for (int u = 0; u < kAdjustQuads; ++u) {
    const int i = (u * kAdjustThreads + tid) * 4;
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
  NINFER_REQUIRE(!a.hist_offsets || a.n_hist == 0 || (a.hist_tokens && a.hist_counts), "adjust_logits: a history without tokens or counts");
  NINFER_REQUIRE(!a.bias_offsets || a.n_bias == 0 || (a.bias_tokens && a.bias_values), "adjust_logits: biases without tokens or values");
  NINFER_REQUIRE(!a.mask_rows || a.n_masks == 0 || a.masks, "adjust_logits: rows name masks that are not given");
  const int parts = (a.V + kAdjustPart - 1) / kAdjustPart;
  NINFER_REQUIRE((long long)parts * a.R <= 0x7fffffff, "adjust_logits: %d rows are too many", a.R);
  a.vec = row_aligned(a.logits) && row_aligned(a.out) && a.ld % 4 == 0 && a.ldo % 4 == 0;
  adjust_logits_kernel<<<parts * a.R, kAdjustThreads, 0, stream>>>(a, parts);
  NINFER_LAUNCH_CHECK();
  return 0;
}
