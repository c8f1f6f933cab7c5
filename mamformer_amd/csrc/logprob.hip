// Log probabilities of given tokens, with entropies and the likeliest alternatives, and the logits' gradient.
//
//   l = logits / temperature, m = max(l), S = sum exp(l - m), U = sum exp(l - m) (l - m)
//   logprob = l[target] - m - ln S,   entropy H = ln S - U / S
//   dlogits[j] = (d_lp (delta_{j, target} - p_j) - d_H p_j (ln p_j + H)) / temperature,   p_j = exp(l_j - m) / S
//
// One pass over a row with sums against a running offset m, which is a logit of the row: with d = (logit - m) k in
// powers of two, k = log2(e) / temperature,
//   S = sum 2^d, U = sum 2^d d;  a new offset m' multiplies by c = 2^((m - m') k): U <- c (U + S (m - m') k), S <- c S.
// The difference of the logits comes first, so rows of the type's lowest value stay finite at any temperature.  A thread
// moves its offset only when a logit lies 2^kSlack above it: few threads do after their first chunk, where the largest
// value itself would change in some lane of a wave at almost every chunk, and S stays small enough for ln S - U / S to
// keep its bits.  m starts at the lowest finite value, so entries of -inf weigh nothing and a row of them gives S = 0:
// such a row has logprob -inf, entropy 0 and no gradient.  The running sums are fp32.  An element costs 7 vector
// instructions and the base-2 exponential, which takes the time of 4: about 70 us of 8192 x 32000 on 256 CUs.
//
// Alternatives are ranked by (value, lowest id first) as one 64-bit key, NaN above all.  A thread's share of the row is
// bounded by its largest value and the last id of the first chunk that has it: a key at or below the share's largest, and
// in the same order as those.  Every wave finds the q-th largest of its 64 bounds by ballots, q = top / 4 rounded up; at
// least `top` keys are at or above the least of the four, and only the shares whose bound is there can hold one, so only
// those are read a second time.  (A row of fewer chunks than threads: q = top, and the largest of the four.)
//
// A row is one workgroup's, or where the rows are too few to fill the card the row is cut into spans, whose sums and
// sorted alternatives logprob_join_kernel puts together.
#include <float.h>
#include <type_traits>

#include "common.h"
#include "launch.h"
#include "rows.h"

namespace mh {

namespace {

constexpr int kNT = 256;
constexpr int kCand = 1024;                      // candidates ranked at once

constexpr float kSlack = 8.f;
constexpr float kLn2 = 0.693147180559945f;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// The forward leaves the last rows, as many as the 256 MB cache in front of the memory holds, in it for the backward, which
// takes the rows last to first; the rows before them, `left` and more from the end, go past it in both, and so does the
// gradient.  8192 x 32000 bf16, forward and backward: 259 us (232 MB so: 262, 192 MB: 272, all rows past it: 291, all through
// it: 318); 777 x 50001 fp32, whose logits fit: 91 us (gradient through it: 107, logits past it: 112).
constexpr int64_t kCacheBytes = (int64_t)256 << 20;
template <typename T>
__device__ __forceinline__ bool past_cache(int64_t left, int64_t vocab) {
  return left * vocab * (int64_t)sizeof(T) > kCacheBytes;
}

struct Soft {
  float m, s, u;
};
__device__ __forceinline__ Soft soft_none() { return {-FLT_MAX, 0.f, 0.f}; }
__device__ __forceinline__ Soft soft_move(Soft a, float m, float k) {
  const float d = fmaxf((a.m - m) * k, -200.f), c = exp2_of(d);       // 2^-200 is 0 in fp32
  return {m, a.s * c, c * (a.u + a.s * d)};
}
__device__ __forceinline__ Soft soft_join(Soft a, Soft b, float k) {
  const float m = fmaxf(a.m, b.m);
  a = soft_move(a, m, k);
  b = soft_move(b, m, k);
  return {m, a.s + b.s, a.u + b.u};
}
// Butterfly over the wave: the same sum in every lane.
__device__ __forceinline__ Soft soft_wave(Soft a, float k) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Soft o = {__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.u, off, 64)};
    a = (threadIdx.x & off) ? soft_join(o, a, k) : soft_join(a, o, k);
  }
  return a;
}
__device__ __forceinline__ float chunk_max(const float (&v)[8]) {
  float m = v[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) m = fmaxf(m, v[j]);
  return m;
}
// cm: chunk_max(v)
__device__ __forceinline__ void soft_add(Soft& a, const float (&v)[8], float cm, float k) {
  if ((cm - a.m) * k > kSlack) a = soft_move(a, cm, k);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = (v[j] - a.m) * k, e = exp2_of(d);
    a.s += e;
    a.u += e * fmaxf(d, -200.f);                 // 0 times -inf is not wanted; NaN comes through e
  }
}

// Order of the alternatives: larger value first (NaN first of all, -0 and 0 alike), then the lower id; 0 is none.
__device__ __forceinline__ uint32_t alt_order(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t alt_key(float v, uint32_t id) {
  return (uint64_t)alt_order(v) << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ float alt_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0xffffffffu ? __builtin_nanf("") : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t alt_id(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

struct AltShared {
  uint64_t cand[kCand];
  uint64_t out[kMaxAlternatives];
  uint64_t wave[kNT / 64];
  int share[kNT];
  int count, shares;
};

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, 64);
    if (o > v) v = o;
  }
  return v;
}

// The q-th largest of the lanes' keys, bit by bit from the top: its value part, and its id where values are equal.  Keys
// other than 0 differ; 0 where fewer than q are not 0.
__device__ __forceinline__ uint64_t wave_nth(uint64_t key, int q) {
  auto nth = [](uint32_t u, int n) {
    uint32_t x = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = x | 1u << bit;
      if (__popcll(__ballot(u >= t)) >= n) x = t;
    }
    return x;
  };
  const uint32_t u = (uint32_t)(key >> 32), hi = nth(u, q);
  if (hi == 0) return 0;
  const int above = __popcll(__ballot(u > hi));
  const uint64_t tie = __ballot(u == hi);
  if (above + __popcll(tie) == q) {              // all of the equal ones: the least is theirs
    uint32_t lo = u == hi ? (uint32_t)key : 0xffffffffu;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) lo = min(lo, (uint32_t)__shfl_xor((int)lo, off, 64));
    return (uint64_t)hi << 32 | lo;
  }
  return (uint64_t)hi << 32 | nth(u == hi ? (uint32_t)key : 0u, q - above);
}

// The `top` largest keys of elements [lo, hi) of a row into sh.out, largest first (0 where there are fewer); thread
// t's share are the chunks lo + 8 (t + kNT i), and `bound` its bound, 0 where it has none.
template <typename T>
__device__ void alternatives(const T* row, int64_t lo, int64_t hi, int top, uint64_t bound, AltShared& sh) {
  constexpr int kWaves = kNT / 64;
  const int t = threadIdx.x;
  const bool split = hi - lo >= 8 * kNT;         // every thread has a bound; else one wave alone stands for `top` keys
  const uint64_t mine = wave_nth(bound, split ? (top + kWaves - 1) / kWaves : top);
  if ((t & 63) == 0) sh.wave[t >> 6] = mine;
  if (t == 0) sh.count = sh.shares = 0;
  if (t < top) sh.out[t] = 0;
  __syncthreads();
  uint64_t tau = sh.wave[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const uint64_t o = sh.wave[w];
    tau = split ? (o < tau ? o : tau) : (o > tau ? o : tau);
  }
  tau = tau > 0 ? tau : 1;                       // fewer than `top` bounds: every key counts
  if (bound >= tau) sh.share[atomicAdd(&sh.shares, 1)] = t;
  __syncthreads();
  const int steps = (int)((hi - lo + 8 * kNT - 1) / (8 * kNT)), shares = sh.shares;
  auto walk = [&](auto&& f) {
    for (int i = t; i < shares * steps; i += kNT) {
      const int64_t c = lo + 8 * (int64_t)(sh.share[i % shares] + kNT * (i / shares));
      if (c >= hi) continue;
      float v[8];
      load8(row + c, (int)min(hi - c, (int64_t)8), v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < hi) f(alt_key(v[j], (uint32_t)(c + j)));
    }
  };
  walk([&](uint64_t k) {
    if (k < tau) return;
    const int n = atomicAdd(&sh.count, 1);
    if (n < kCand) sh.cand[n] = k;
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= kCand) {
    for (int i = t; i < n; i += kNT) {
      const uint64_t k = sh.cand[i];
      int r = 0;
#pragma unroll 4
      for (int q = 0; q < n; ++q) r += sh.cand[q] > k;
      if (r < top) sh.out[r] = k;
    }
  } else {                                       // many at or above the bound: one after another
    uint64_t last = ~(uint64_t)0;
    for (int r = 0; r < top; ++r) {
      uint64_t b = 0;
      walk([&](uint64_t k) {
        if (k < last && k > b) b = k;
      });
      b = wave_max(b);
      if ((t & 63) == 0) sh.wave[t >> 6] = b;
      __syncthreads();
      for (int w = 0; w < kWaves; ++w) b = sh.wave[w] > b ? sh.wave[w] : b;
      if (t == 0) sh.out[r] = b;
      last = b;
      __syncthreads();
    }
  }
  __syncthreads();
}

// The results of a row from its sums and alternatives.
template <typename T>
__device__ void finish(const LogprobParams& p, int64_t r, Soft a, const uint64_t* alts) {
  const bool none = a.s == 0.f;
  const float log2_s = none ? INFINITY : log2f(a.s);
  if (threadIdx.x == 0) {
    const float ent = none ? 0.f : (log2_s - a.u / a.s) * kLn2;
    const int64_t tgt = load_index(p.targets, p.i64, r);
    float lp = 0.f;
    if (tgt >= 0 && tgt < p.vocab && tgt != p.ignore_index)
      lp = none ? -INFINITY : ((to_f32(reinterpret_cast<const T*>(p.logits)[r * p.l_s + tgt]) - a.m) * p.k - log2_s) * kLn2;
    p.logprobs[r] = lp;
    if (p.entropy) p.entropy[r] = ent;
    p.stats[3 * r] = a.m;
    p.stats[3 * r + 1] = log2_s;
    p.stats[3 * r + 2] = ent;
  }
  for (int i = threadIdx.x; i < p.top; i += kNT) {
    p.top_ids[r * p.top + i] = alt_id(alts[i]);
    p.top_logprobs[r * p.top + i] = none ? -INFINITY : ((alt_value(alts[i]) - a.m) * p.k - log2_s) * kLn2;
  }
}

// The partial results of span i of row r in the workspace: sums, then `top` keys.
__device__ __forceinline__ Soft* span_sums(const LogprobParams& p, int64_t r, int i) {
  return reinterpret_cast<Soft*>(p.workspace) + r * p.spans + i;
}
__device__ __forceinline__ uint64_t* span_keys(const LogprobParams& p, int64_t r, int i) {
  return reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(p.workspace) + p.keys_at) + (r * p.spans + i) * p.top;
}

template <typename T, bool TOP>
__global__ __launch_bounds__(kNT) void logprob_kernel(LogprobParams p) {
  constexpr int kAhead = 2;                      // chunks a thread has on their way
  __shared__ AltShared sh;
  __shared__ Soft wsoft[kNT / 64];
  const int64_t r = grid_row();
  if (r >= p.rows) return;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.l_s;
  const int64_t lo = blockIdx.y * p.span, hi = min(p.vocab, lo + p.span);
  Soft a = soft_none();
  float best = 0.f;                              // largest value of the share and its first chunk
  int64_t best_at = -1;
  auto add = [&](const float (&v)[8], int64_t c) {
    const float cm = chunk_max(v);
    if constexpr (TOP) {
      const bool up = cm > best || best_at < 0;
      best = up ? cm : best;
      best_at = up ? c : best_at;
    }
    soft_add(a, v, cm, p.k);
  };
  auto read = [&](auto past) {
    constexpr bool NT = decltype(past)::value;
    int64_t c = lo + 8 * threadIdx.x;
    for (; c + 8 * kNT * (kAhead - 1) + 8 <= hi; c += 8 * kNT * kAhead) {
      float v[kAhead][8];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load8<NT>(row + c + 8 * kNT * i, v[i]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add(v[i], c + 8 * kNT * i);
    }
    for (; c < hi; c += 8 * kNT) {
      float v[8];
      load8<NT>(row + c, (int)min(hi - c, (int64_t)8), v, -INFINITY);
      add(v, c);
    }
  };
  if (!TOP && past_cache<T>(p.rows - r, p.vocab)) read(std::true_type{});       // alternatives are read a second time
  else read(std::false_type{});
  uint64_t bound = 0;
  if constexpr (TOP) {
    if (a.s != a.s) {                            // a NaN or an infinity in the share, which the maximum may have passed by
      uint64_t k = 0;
      for (int64_t c = lo + 8 * threadIdx.x; c < hi; c += 8 * kNT)
        for (int j = 0; j < 8 && c + j < hi; ++j) k = max(k, alt_key(to_f32(row[c + j]), (uint32_t)(c + j)));
      best = alt_value(k);
      best_at = lo + (alt_id(k) - lo) / 8 * 8;
    }
    if (best_at >= 0) bound = alt_key(best, (uint32_t)best_at + 7);
  }
  a = soft_wave(a, p.k);
  if ((threadIdx.x & 63) == 0) wsoft[threadIdx.x >> 6] = a;
  if constexpr (TOP) alternatives(row, lo, hi, p.top, bound, sh);
  else __syncthreads();
  a = wsoft[0];
  for (int w = 1; w < kNT / 64; ++w) a = soft_join(a, wsoft[w], p.k);
  if (p.spans == 1) {
    finish<T>(p, r, a, sh.out);
  } else {
    if (threadIdx.x == 0) *span_sums(p, r, blockIdx.y) = a;
    if (TOP && threadIdx.x < p.top) span_keys(p, r, blockIdx.y)[threadIdx.x] = sh.out[threadIdx.x];
  }
}

// The spans of a row: their sums in one wave, a span a lane; of their alternatives, sorted lists of `top` each, the first
// `deep` of every list bound the answer: the `lists` largest of the lists' deep-th keys stand for lists * deep >= top keys
// at or above the least of them, so only keys from there on are ranked.
template <typename T>
__global__ __launch_bounds__(kNT) void logprob_join_kernel(LogprobParams p) {
  constexpr int kAhead = 4;                      // keys a thread reads before the bound is known
  __shared__ uint64_t tau, out[kMaxAlternatives], cand[64 * kMaxAlternatives];
  __shared__ Soft total;
  __shared__ int count;
  const int64_t r = grid_row();
  if (r >= p.rows) return;
  const int t = threadIdx.x, lane = t & 63, n_keys = p.spans * p.top;
  const uint64_t* keys = span_keys(p, r, 0);
  uint64_t key[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) key[i] = t + kNT * i < n_keys ? keys[t + kNT * i] : 0;
  if (t >= 64 && t < 128) {
    const Soft a = soft_wave(lane < p.spans ? *span_sums(p, r, lane) : soft_none(), p.k);
    if (lane == 0) total = a;
  }
  if (p.top) {
    const int deep = (p.top + p.spans - 1) / p.spans, lists = (p.top + deep - 1) / deep;
    if (t < 64) {
      const uint64_t k = wave_nth(t < p.spans ? keys[t * p.top + deep - 1] : 0, lists);
      if (t == 0) { tau = k > 0 ? k : 1; count = 0; }                 // 0: spans with fewer than `deep` keys
    }
    if (t < p.top) out[t] = 0;
    __syncthreads();
    const uint64_t least = tau;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (key[i] >= least) cand[atomicAdd(&count, 1)] = key[i];
    for (int i = t + kNT * kAhead; i < n_keys; i += kNT)
      if (keys[i] >= least) cand[atomicAdd(&count, 1)] = keys[i];
    __syncthreads();
    const int n = count;
    for (int i = t; i < n; i += kNT) {
      const uint64_t k = cand[i];
      int rank = 0;
#pragma unroll 4
      for (int q = 0; q < n; ++q) rank += cand[q] > k;
      if (rank < p.top) out[rank] = k;
    }
  }
  __syncthreads();
  finish<T>(p, r, total, out);
}

// Rows last to first: what the forward read last is what the cache still holds.
template <typename T>
__global__ __launch_bounds__(kNT) void logprob_bwd_kernel(LogprobBwdParams p) {
  constexpr int kAhead = 2;
  const int64_t r = p.rows - 1 - grid_row();
  if (r < 0) return;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.l_s;
  T* out = reinterpret_cast<T*>(p.dlogits) + r * p.d_s;
  const int64_t tgt = load_index(p.targets, p.i64, r);
  const bool keep = tgt >= 0 && tgt < p.vocab && tgt != p.ignore_index;
  const float m = p.stats[3 * r], log2_s = p.stats[3 * r + 1], ent = p.stats[3 * r + 2];
  const float g = keep && p.d_logprobs ? p.d_logprobs[r] * p.inv_temp : 0.f;
  const float gh = p.d_entropy ? p.d_entropy[r] * p.inv_temp : 0.f;
  const int64_t lo = (int64_t)blockIdx.y * p.span, hi = min(p.vocab, lo + p.span);
  int64_t c = lo + 8 * threadIdx.x;
  if (log2_s == INFINITY || (g == 0.f && gh == 0.f)) {                  // nothing flows back, whatever the logits hold
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (; c < hi; c += 8 * kNT) store8(out + c, (int)min(hi - c, (int64_t)8), z);
    return;
  }
  const float g0 = g + gh * ent, g1 = gh * kLn2;
  auto grad = [&](float (&v)[8], int64_t at) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float l = (v[j] - m) * p.k - log2_s;
      v[j] = -exp2_of(l) * (g1 * fmaxf(l, -200.f) + g0);
    }
    if (tgt >= at && tgt < at + 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += at + j == tgt ? g : 0.f;
    }
  };
  auto walk = [&](auto past) {
    constexpr bool NT = decltype(past)::value;
    for (; c + 8 * kNT * (kAhead - 1) + 8 <= hi; c += 8 * kNT * kAhead) {
      float v[kAhead][8];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load8<NT>(row + c + 8 * kNT * i, v[i]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        grad(v[i], c + 8 * kNT * i);
        store8<true>(out + c + 8 * kNT * i, v[i]);
      }
    }
    for (; c < hi; c += 8 * kNT) {
      float v[8];
      const int left = (int)min(hi - c, (int64_t)8);
      load8<NT>(row + c, left, v);
      grad(v, c);
      store8<true>(out + c, left, v);
    }
  };
  if (past_cache<T>(p.rows - r, p.vocab)) walk(std::true_type{});
  else walk(std::false_type{});
}

}  // namespace

// Two workgroups a CU are wanted (777 x 50001 fp32 with its gradient, three rows a CU: 88.6 us, in two spans each 90.5; 24 x
// 128000 with 20 alternatives: 19 us at 528 and at 768 workgroups, 71 us in one kernel of a workgroup a row); a span of a
// row has more than 2048 columns, a turn of its threads, and there is one for each 4096 of the row at most.
size_t logprob_plan(LogprobParams& p) {
  const int64_t want = p.rows ? (512 + p.rows - 1) / p.rows : 1, most = (p.vocab + 4095) / 4096;
  int64_t n = want < most ? want : most;
  n = n < 64 ? n : 64;                           // the join holds a span a lane
  p.span = ((p.vocab + n - 1) / n + 7) / 8 * 8;
  p.spans = (int)((p.vocab + p.span - 1) / p.span);
  if (p.spans == 1) return 0;
  p.keys_at = ((size_t)p.rows * p.spans * sizeof(Soft) + 15) / 16 * 16;
  return p.keys_at + (size_t)p.rows * p.spans * p.top * sizeof(uint64_t);
}

template <typename T>
hipError_t run_fwd(const LogprobParams& p, hipStream_t st) {
  const dim3 g = row_grid(p.rows, p.spans);
  if (p.top) logprob_kernel<T, true><<<g, kNT, 0, st>>>(p);
  else logprob_kernel<T, false><<<g, kNT, 0, st>>>(p);
  if (p.spans > 1) logprob_join_kernel<T><<<row_grid(p.rows, 1), kNT, 0, st>>>(p);
  return hipGetLastError();
}

hipError_t launch_logprob(const LogprobParams& p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  return p.dtype == DT_F32 ? run_fwd<float>(p, st) : run_fwd<bf16>(p, st);
}

hipError_t launch_logprob_bwd(LogprobBwdParams p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  p.span = 8192;
  while ((p.vocab + p.span - 1) / p.span > 65535) p.span *= 2;
  const dim3 g = row_grid(p.rows, (unsigned)((p.vocab + p.span - 1) / p.span));
  if (p.dtype == DT_F32) logprob_bwd_kernel<float><<<g, kNT, 0, st>>>(p);
  else logprob_bwd_kernel<bf16><<<g, kNT, 0, st>>>(p);
  return hipGetLastError();
}

}  // namespace mh
