// Log probabilities of given tokens, with entropies and the likeliest alternatives, and the logits' gradient.
//
//   l = logits / temperature, m = max(l), S = sum exp(l - m), U = sum exp(l - m) (l - m)
//   logprob = l[target] - m - ln S,   entropy H = ln S - U / S
//   dlogits[j] = (d_lp (delta_{j, target} - p_j) - d_H p_j (ln p_j + H)) / temperature,   p_j = exp(l_j - m) / S
//
// One pass over a row with a running maximum: (m, S, U) move to a new maximum m' by c = exp(m - m'),
// U <- c (U + S (m - m')), S <- c S.  m starts at the lowest finite value, so entries of -inf weigh nothing and a row
// of them gives S = 0: such a row has logprob -inf, entropy 0 and no gradient.  The running sums are fp32.
//
// Alternatives are ranked by (value, lowest id first) as one 64-bit key, NaN above all.  Every thread keeps the largest
// key of its own share of the row; the top-th largest of those bounds the answer from below, and only the `top`
// threads at or above it can hold alternatives, so only their shares are read a second time.
#include <float.h>

#include "common.h"
#include "launch.h"
#include "rows.h"

namespace mh {

namespace {

constexpr int kNT = 256;
constexpr int kCand = 1024;                      // candidates ranked at once

// exp: of fp32 logits the accurate one, of bf16 logits (8 bits of value) the hardware's base-2 exponential
__device__ __forceinline__ float exp_of(float x, float) { return expf(x); }
__device__ __forceinline__ float exp_of(float x, bf16) { return __expf(x); }

struct Soft {
  float m, s, u;
};
__device__ __forceinline__ Soft soft_none() { return {-FLT_MAX, 0.f, 0.f}; }
__device__ __forceinline__ Soft soft_move(Soft a, float m) {
  const float d = fmaxf(a.m - m, -200.f), c = expf(d);                // exp(-200) is 0 in fp32
  return {m, a.s * c, c * (a.u + a.s * d)};
}
__device__ __forceinline__ Soft soft_join(Soft a, Soft b) {
  const float m = fmaxf(a.m, b.m);
  a = soft_move(a, m);
  b = soft_move(b, m);
  return {m, a.s + b.s, a.u + b.u};
}

// Order of the alternatives: larger value first (NaN first of all, -0 and 0 alike), then the lower id; 0 is none.
__device__ __forceinline__ uint64_t alt_key(float v, uint32_t id) {
  uint32_t u = __float_as_uint(v + 0.f);
  u = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ float alt_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0xffffffffu ? __builtin_nanf("") : __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t alt_id(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

struct AltShared {
  uint64_t best[kNT];
  uint64_t cand[kCand];
  uint64_t out[kMaxAlternatives];
  uint64_t tau;
  uint64_t wave[kNT / 64];
  int share[kMaxAlternatives];
  int count;
};

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, 64);
    if (o > v) v = o;
  }
  return v;
}

// The `top` largest keys of elements [lo, hi) of a row into sh.out, largest first (0 where there are fewer); thread
// t's share are the chunks lo + 8 (t + kNT i), and `best` its largest key.
template <typename T>
__device__ void alternatives(const T* row, int64_t lo, int64_t hi, int top, uint64_t best, AltShared& sh) {
  const int t = threadIdx.x;
  sh.best[t] = best;
  if (t == 0) sh.count = 0;
  if (t < top) sh.out[t] = 0;
  __syncthreads();
  int rank = 0;
  for (int i = 0; i < kNT; ++i) rank += sh.best[i] > best || (sh.best[i] == best && i < t);
  if (rank < top) sh.share[rank] = t;
  if (rank == top - 1) sh.tau = best > 0 ? best : 1;                  // fewer shares than `top`: all they hold
  __syncthreads();
  const uint64_t tau = sh.tau;
  const int steps = (int)((hi - lo + 8 * kNT - 1) / (8 * kNT));
  auto walk = [&](auto&& f) {
    for (int i = t; i < top * steps; i += kNT) {
      const int64_t c = lo + 8 * (int64_t)(sh.share[i / steps] + kNT * (i % steps));
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
      for (int w = 0; w < kNT / 64; ++w) b = sh.wave[w] > b ? sh.wave[w] : b;
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
  const float ln_s = none ? INFINITY : logf(a.s);
  if (threadIdx.x == 0) {
    const float ent = none ? 0.f : ln_s - a.u / a.s;
    const int64_t tgt = load_index(p.targets, p.i64, r);
    float lp = 0.f;
    if (tgt >= 0 && tgt < p.vocab && tgt != p.ignore_index)
      lp = none ? -INFINITY : to_f32(reinterpret_cast<const T*>(p.logits)[r * p.l_s + tgt]) * p.inv_temp - a.m - ln_s;
    p.logprobs[r] = lp;
    if (p.entropy) p.entropy[r] = ent;
    p.stats[3 * r] = a.m;
    p.stats[3 * r + 1] = ln_s;
    p.stats[3 * r + 2] = ent;
  }
  for (int i = threadIdx.x; i < p.top; i += kNT) {
    p.top_ids[r * p.top + i] = alt_id(alts[i]);
    p.top_logprobs[r * p.top + i] = none ? -INFINITY : alt_value(alts[i]) * p.inv_temp - a.m - ln_s;
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(kNT) void logprob_kernel(LogprobParams p) {
  __shared__ AltShared sh;
  __shared__ Soft wsoft[kNT / 64];
  const int64_t r = blockIdx.x;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.l_s;
  const int64_t lo = 0, hi = p.vocab;
  Soft a = soft_none();
  uint64_t best = 0;
  for (int64_t c = lo + 8 * threadIdx.x; c < hi; c += 8 * kNT) {
    float v[8];
    load8(row + c, (int)min(hi - c, (int64_t)8), v, -INFINITY);
    if constexpr (TOP) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint64_t k = c + j < hi ? alt_key(v[j], (uint32_t)(c + j)) : 0;
        best = k > best ? k : best;
      }
    }
    float cm = a.m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] *= p.inv_temp;
      cm = fmaxf(cm, v[j]);
    }
    if (cm > a.m) a = soft_move(a, cm);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[j] - a.m, e = exp_of(d, T());
      a.s += e;
      a.u += e * fmaxf(d, -200.f);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Soft o = {__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.u, off, 64)};
    a = soft_join(a, o);
  }
  if ((threadIdx.x & 63) == 0) wsoft[threadIdx.x >> 6] = a;
  if constexpr (TOP) alternatives(row, lo, hi, p.top, best, sh);
  else __syncthreads();
  a = wsoft[0];
  for (int w = 1; w < kNT / 64; ++w) a = soft_join(a, wsoft[w]);
  finish<T>(p, r, a, sh.out);
}

template <typename T>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogprobBwdParams p) {
  const int64_t r = blockIdx.x;
  const T* row = reinterpret_cast<const T*>(p.logits) + r * p.l_s;
  T* out = reinterpret_cast<T*>(p.dlogits) + r * p.d_s;
  const int64_t tgt = load_index(p.targets, p.i64, r);
  const bool keep = tgt >= 0 && tgt < p.vocab && tgt != p.ignore_index;
  const float m = p.stats[3 * r], ln_s = p.stats[3 * r + 1], ent = p.stats[3 * r + 2];
  const float g = keep && p.d_logprobs ? p.d_logprobs[r] * p.inv_temp : 0.f;
  const float gh = p.d_entropy ? p.d_entropy[r] * p.inv_temp : 0.f;
  const bool none = ln_s == INFINITY || (g == 0.f && gh == 0.f);      // nothing flows back, whatever the logits hold
  const int64_t lo = (int64_t)blockIdx.y * p.span, hi = min(p.vocab, lo + p.span);
  for (int64_t c = lo + 8 * threadIdx.x; c < hi; c += 8 * 256) {
    const int left = (int)min(hi - c, (int64_t)8);
    float v[8];
    if (none) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    } else {
      load8(row + c, left, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lnp = v[j] * p.inv_temp - m - ln_s, pr = exp_of(lnp, T());
        v[j] = (c + j == tgt ? g : 0.f) - pr * (g + gh * (fmaxf(lnp, -200.f) + ent));
      }
    }
    store8(out + c, left, v);
  }
}

}  // namespace

size_t logprob_workspace_bytes(const LogprobParams&) { return 0; }

hipError_t launch_logprob(const LogprobParams& p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  const unsigned g = (unsigned)p.rows;
  if (p.dtype == DT_F32) {
    if (p.top) logprob_kernel<float, true><<<g, kNT, 0, st>>>(p);
    else logprob_kernel<float, false><<<g, kNT, 0, st>>>(p);
  } else {
    if (p.top) logprob_kernel<bf16, true><<<g, kNT, 0, st>>>(p);
    else logprob_kernel<bf16, false><<<g, kNT, 0, st>>>(p);
  }
  return hipGetLastError();
}

hipError_t launch_logprob_bwd(LogprobBwdParams p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  p.span = 8192;
  while ((p.vocab + p.span - 1) / p.span > 65535) p.span *= 2;
  const dim3 g((unsigned)p.rows, (unsigned)((p.vocab + p.span - 1) / p.span));
  if (p.dtype == DT_F32) logprob_bwd_kernel<float><<<g, 256, 0, st>>>(p);
  else logprob_bwd_kernel<bf16><<<g, 256, 0, st>>>(p);
  return hipGetLastError();
}

}  // namespace mh
