// Token table: scaled lookup, and its gradient by sorted tokens.
//
//   out[t] = scale W[ids[t]]  (zeros for an id outside [0, vocab));
//   dW[v] = scale sum of dy[t] over the tokens t with ids[t] = v != padding_idx, in the order of t.
//
// The gradient sorts (id, t) by id with a stable radix sort of 9 bits a pass (two passes up to 2^18 rows), so that the
// sum of a row runs in the order of its tokens and gives the same bits at every call; no floating-point atomics.  The
// sorted tokens are cut into pieces of equal length whatever their ids, so a word that fills a tenth of the batch is
// summed by many workgroups.  A run of one id that lies within a piece is written to dW at once; a run that crosses a
// border leaves fp32 partial rows, which embed_join_kernel adds in order.  Dropped tokens (padding, ids out of range)
// sort behind the last row.
#include "common.h"
#include "launch.h"
#include "rows.h"

namespace mh {

namespace {

constexpr int kBits = 9, kDigits = 1 << kBits;   // a pass: 512 counters, two a thread

template <typename T>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedParams p) {
  const int64_t per = (p.dim + 7) / 8, total = p.tokens * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per;
    const int c = (int)(i - t * per) * 8;
    const int64_t id = load_index(p.ids, p.i64, t);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (id >= 0 && id < p.vocab) {
      load8(reinterpret_cast<const T*>(p.weight) + id * p.w_s + c, p.dim - c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= p.scale;
    }
    store8(reinterpret_cast<T*>(p.out) + t * p.out_s + c, p.dim - c, v);
  }
}

// The sort key of token t: its row, or vocab where it has none.
__device__ __forceinline__ uint32_t token_key(const EmbedBwdParams& p, int64_t t) {
  const int64_t id = load_index(p.ids, p.i64, t);
  return id >= 0 && id < p.vocab && id != p.padding_idx ? (uint32_t)id : (uint32_t)p.vocab;
}

// Counts of the first pass's digits in this workgroup's tile; clears the later passes' counts.
__global__ __launch_bounds__(256) void embed_count_kernel(EmbedBwdParams p) {
  __shared__ uint32_t cnt[kDigits];
  cnt[threadIdx.x] = cnt[threadIdx.x + 256] = 0;
  for (int q = 1; q < p.passes; ++q) {
    uint32_t* h = p.hist + ((int64_t)q * p.tiles + blockIdx.x) * kDigits;
    h[threadIdx.x] = h[threadIdx.x + 256] = 0;
  }
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * p.tile, hi = min(p.tokens, lo + p.tile);
  for (int64_t t = lo + threadIdx.x; t < hi; t += 256) atomicAdd(&cnt[token_key(p, t) & (kDigits - 1)], 1u);
  __syncthreads();
  uint32_t* h = p.hist + (int64_t)blockIdx.x * kDigits;
  h[threadIdx.x] = cnt[threadIdx.x];
  h[threadIdx.x + 256] = cnt[threadIdx.x + 256];
}

// One stable pass.  Each wave owns a quarter of the tile and walks it 64 tokens at a time: a token's place is its
// digit's start (all smaller digits, then the digit's tokens of earlier tiles, earlier waves and earlier steps) plus
// the number of lanes before it with the same digit (ballots over the digit's bits).
__global__ __launch_bounds__(256) void embed_sort_kernel(EmbedBwdParams p, int pass) {
  __shared__ uint32_t at[4][kDigits];
  __shared__ uint32_t wsum[4];
  const int lane = lane_id(), wave = wave_id(), shift = pass * kBits;
  const uint32_t* key_in = p.keys[pass & 1];
  const uint32_t* tok_in = p.order[pass & 1];
  uint32_t* key_out = p.keys[(pass & 1) ^ 1];
  uint32_t* tok_out = p.order[(pass & 1) ^ 1];
  for (int i = threadIdx.x; i < 4 * kDigits; i += 256) at[0][i] = 0;
  __syncthreads();
  const int64_t quarter = p.tile / 4, lo = (int64_t)blockIdx.x * p.tile + wave * quarter;
  const int64_t hi = min(p.tokens, lo + quarter);
  for (int64_t t = lo + lane; t < hi; t += 64) {
    const uint32_t k = pass ? key_in[t] : token_key(p, t);
    atomicAdd(&at[wave][(k >> shift) & (kDigits - 1)], 1u);
  }
  // digits 2 x, 2 x + 1 of thread x: their counts in earlier tiles and in all
  const uint32_t* hist = p.hist + (int64_t)pass * p.tiles * kDigits;
  uint32_t before[2] = {0, 0}, total[2] = {0, 0};
  for (int b = 0; b < p.tiles; ++b) {
    const uint2 n = reinterpret_cast<const uint2*>(hist + (int64_t)b * kDigits)[threadIdx.x];
    if (b < (int)blockIdx.x) { before[0] += n.x; before[1] += n.y; }
    total[0] += n.x;
    total[1] += n.y;
  }
  uint32_t incl = total[0] + total[1];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)incl, off, 64);
    if (lane >= off) incl += o;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();                               // also: every wave's counts are in `at`
  uint32_t base = incl - total[0] - total[1];
  for (int w = 0; w < wave; ++w) base += wsum[w];
  uint32_t start[2] = {base + before[0], base + total[0] + before[1]};
#pragma unroll
  for (int d = 0; d < 2; ++d)
    for (int w = 0; w < 4; ++w) {
      const uint32_t n = at[w][2 * threadIdx.x + d];
      at[w][2 * threadIdx.x + d] = start[d];
      start[d] += n;
    }
  __syncthreads();
  uint32_t* next = pass + 1 < p.passes ? p.hist + (int64_t)(pass + 1) * p.tiles * kDigits : nullptr;
  volatile uint32_t* mine = at[wave];
  for (int64_t t0 = lo; t0 < hi; t0 += 64) {
    const int64_t t = t0 + lane;
    const bool live = t < hi;
    uint32_t k = 0, tok = 0;
    if (live) {
      k = pass ? key_in[t] : token_key(p, t);
      tok = pass ? tok_in[t] : (uint32_t)t;
    }
    const uint32_t d = (k >> shift) & (kDigits - 1);
    uint64_t same = __ballot(live);
#pragma unroll
    for (int bit = 0; bit < kBits; ++bit) {
      const bool on = (d >> bit) & 1;
      const uint64_t b = __ballot(on);
      same &= on ? b : ~b;
    }
    const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
    if (live) {
      const uint32_t first = mine[d], pos = first + rank;
      __builtin_amdgcn_wave_barrier();           // every lane has read its digit's place before the first lane moves it
      if (rank == 0) mine[d] = first + (uint32_t)__popcll(same);
      key_out[pos] = k;
      tok_out[pos] = tok;
      if (next) atomicAdd(&next[(int64_t)(pos / (uint32_t)p.tile) * kDigits + ((k >> (shift + kBits)) & (kDigits - 1))], 1u);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename TW>
__global__ __launch_bounds__(256) void embed_clear_kernel(EmbedBwdParams p) {
  const int64_t per = (p.dim + 7) / 8, total = p.vocab * per;
  const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t v = i / per;
    const int c = (int)(i - v * per) * 8;
    store8(reinterpret_cast<TW*>(p.dweight) + v * p.dim + c, p.dim - c, z);
  }
}

// A piece of the sorted tokens and up to 2048 columns of it, 8 a thread.
template <typename T, typename TW>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedBwdParams p) {
  const int lane = threadIdx.x % p.cthreads;
  const int64_t piece = (int64_t)blockIdx.x * (256 / p.cthreads) + threadIdx.x / p.cthreads;
  const int c = 8 * (blockIdx.y * p.cthreads + lane), left = p.dim - c;
  if (piece >= p.pieces || left <= 0) return;
  const uint32_t* keys = p.keys[p.passes & 1];
  const uint32_t* order = p.order[p.passes & 1];
  const int64_t lo = piece * p.piece, hi = min(p.tokens, lo + p.piece);
  const T* dy = reinterpret_cast<const T*>(p.dy) + c;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  uint32_t cur = keys[lo];
  bool cont = lo > 0 && keys[lo - 1] == cur;     // the run began in an earlier piece
  auto flush = [&](bool goes_on) {
    if (cont || goes_on) {
      store8(p.part + (2 * piece + (cont ? 0 : 1)) * (int64_t)p.dim + c, left, acc);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store8(reinterpret_cast<TW*>(p.dweight) + (int64_t)cur * p.dim + c, left, acc);
    }
  };
  for (int64_t i = lo; i < hi; ++i) {
    const uint32_t k = keys[i];
    if (k != cur) {
      flush(false);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      cur = k;
      cont = false;
    }
    if (k >= (uint32_t)p.vocab) return;          // only dropped tokens follow
    float v[8];
    load8(dy + (int64_t)order[i] * p.dy_s, left, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  flush(hi < p.tokens && keys[hi] == cur);
}

// The run that begins in this piece and goes beyond it, if there is one: its partial rows in order.
template <typename TW>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedBwdParams p) {
  const uint32_t* keys = p.keys[p.passes & 1];
  const int64_t piece = blockIdx.x, lo = piece * p.piece, hi = lo + p.piece;
  if (hi >= p.tokens) return;
  const uint32_t cur = keys[hi - 1];
  if (cur >= (uint32_t)p.vocab || keys[hi] != cur) return;
  if (keys[lo] == cur && lo > 0 && keys[lo - 1] == cur) return;       // an earlier piece's
  const int c = 8 * (blockIdx.y * 256 + threadIdx.x), left = p.dim - c;
  if (left <= 0) return;
  float acc[8], v[8];
  load8(p.part + (2 * piece + 1) * (int64_t)p.dim + c, left, acc);
  for (int64_t q = piece + 1; q < p.pieces && keys[q * p.piece] == cur; ++q) {
    load8(p.part + 2 * q * (int64_t)p.dim + c, left, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
  store8(reinterpret_cast<TW*>(p.dweight) + (int64_t)cur * p.dim + c, left, acc);
}

unsigned chunk_blocks(int64_t total) {
  const int64_t b = (total + 255) / 256;
  return (unsigned)(b < 8192 ? b : 8192);
}

template <typename T, typename TW>
hipError_t run_bwd(const EmbedBwdParams& p, hipStream_t st) {
  embed_clear_kernel<TW><<<chunk_blocks(p.vocab * ((p.dim + 7) / 8)), 256, 0, st>>>(p);
  if (p.tokens == 0) return hipGetLastError();
  embed_count_kernel<<<p.tiles, 256, 0, st>>>(p);
  for (int pass = 0; pass < p.passes; ++pass) embed_sort_kernel<<<p.tiles, 256, 0, st>>>(p, pass);
  const int groups = 256 / p.cthreads;
  const unsigned slabs = (unsigned)((p.dim + 8 * p.cthreads - 1) / (8 * p.cthreads));
  embed_sum_kernel<T, TW><<<dim3((unsigned)((p.pieces + groups - 1) / groups), slabs), 256, 0, st>>>(p);
  if (p.pieces > 1)
    embed_join_kernel<TW><<<dim3((unsigned)p.pieces, (unsigned)((p.dim + 2047) / 2048)), 256, 0, st>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st) {
  const int64_t total = p.tokens * ((p.dim + 7) / 8);
  if (total == 0) return hipSuccess;
  if (p.dtype == DT_F32) embed_fwd_kernel<float><<<chunk_blocks(total), 256, 0, st>>>(p);
  else embed_fwd_kernel<bf16><<<chunk_blocks(total), 256, 0, st>>>(p);
  return hipGetLastError();
}

size_t embed_bwd_plan(EmbedBwdParams& p, void* workspace) {
  p.passes = 1;
  while (p.passes < 4 && (p.vocab >> (kBits * p.passes)) > 0) ++p.passes;     // keys 0 .. vocab
  p.tile = 1024;
  while ((p.tokens + p.tile - 1) / p.tile > 128) p.tile *= 2;
  p.tiles = (int)((p.tokens + p.tile - 1) / p.tile);
  p.piece = 8;
  while (p.piece < 256 && p.tokens / p.piece > 1024) p.piece *= 2;
  p.pieces = (p.tokens + p.piece - 1) / p.piece;
  p.cthreads = 8;
  while (p.cthreads < 256 && 8 * p.cthreads < p.dim) p.cthreads *= 2;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    void* q = workspace ? reinterpret_cast<char*>(workspace) + off : nullptr;
    off += (bytes + 15) & ~(size_t)15;
    return q;
  };
  for (int i = 0; i < 2; ++i) {
    p.keys[i] = reinterpret_cast<uint32_t*>(take((size_t)p.tokens * 4));
    p.order[i] = reinterpret_cast<uint32_t*>(take((size_t)p.tokens * 4));
  }
  p.hist = reinterpret_cast<uint32_t*>(take((size_t)p.passes * p.tiles * kDigits * 4));
  p.part = reinterpret_cast<float*>(take((size_t)2 * p.pieces * p.dim * 4));
  return off;
}

hipError_t launch_embed_bwd(const EmbedBwdParams& p, hipStream_t st) {
  if (p.dtype == DT_F32) return p.dw_f32 ? run_bwd<float, float>(p, st) : run_bwd<float, bf16>(p, st);
  return p.dw_f32 ? run_bwd<bf16, float>(p, st) : run_bwd<bf16, bf16>(p, st);
}

}  // namespace mh
