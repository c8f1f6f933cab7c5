// Token table: scaled lookup, and its gradient, of many tokens by sorting them.
//
//   out[t] = scale W[ids[t]]  (zeros for an id outside [0, vocab));
//   dW[v] = scale sum of dy[t] over the tokens t with ids[t] = v != padding_idx, in the order of t.
//
// The gradient of up to 2048 tokens is one launch that compares every token's id with all others (embed_few_kernel: 1927
// tokens, 10777 x 1000 fp32: 17 us, sorted 24).  Otherwise it sorts (id, t) by id with a stable radix sort of 9 bits a
// pass (two passes up to 2^18 rows), so that the
// sum of a row runs in the order of its tokens and gives the same bits at every call; no floating-point atomics.  Most of
// what has to be moved is the table's zeros: the sort's launches carry them in workgroups of their own, a share a pass, so
// that a pass (a chain of dependent steps on few CUs) costs no time of its own where the table is large.  The
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
constexpr int kSortThreads = 1024;               // 64 tokens a wave of the smallest tile
constexpr int kClearThreads = 256;               // of these, the ones that clear beside a sort
// Up to here, in a table of up to kFewRows, nothing is sorted.  us, compared and sorted, for ids whose frequencies fall as the
// inverse of the rank, for even ones and for one id alone: 32000 x 1024 bf16, 16 tokens 13 and 18, 14 and 19, 14 and 20;
// 1000 tokens 16 and 21, 16 and 21, 22 and 25; 2000 tokens 21 and 22, 18 and 22, 39 and 32; 3000 tokens (with kFew = 4096) 28
// and 24, 21 and 24, 65 and 40.  1000 x 1024, 1000 tokens 13 and 18, 6 and 17, 21 and 22; 2000 tokens 17 and 21, 8 and 19,
// 37 and 30; 3000 tokens 22 and 22, 14 and 21, 54 and 38.  32000 x 2048, 2000 tokens 36 and 33, 31 and 32, 48 and 40.
constexpr int kFew = 2048;
constexpr int kFewRows = 1 << 18;
// up to here a pass counts all tokens by itself (32000 x 1024 bf16: 4096 tokens 28 us, counted for 40; 16000: both 49;
// 30000: 76 and 68)
constexpr int64_t kDirect = 16384;

// cthreads threads (a power of two) take 8 columns each of kRows tokens, whose loads are all on their way at once.
template <typename T>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedParams p) {
  constexpr int kRows = 2;
  const int lane = threadIdx.x & (p.cthreads - 1), groups = 256 / p.cthreads;
  const int c = 8 * (blockIdx.y * p.cthreads + lane), left = p.dim - c;
  const int64_t t0 = grid_row() * groups * kRows + threadIdx.x / p.cthreads;
  if (left <= 0) return;
  int64_t id[kRows];
  Raw8<T> v[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t t = t0 + i * groups;
    id[i] = t < p.tokens ? load_index(p.ids, p.i64, t) : -1;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    v[i].clear();
    if (id[i] >= 0 && id[i] < p.vocab) load_raw(v[i], reinterpret_cast<const T*>(p.weight) + id[i] * p.w_s + c, left);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t t = t0 + i * groups;
    if (t >= p.tokens) return;
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[i].get(j) * p.scale;
    store8(reinterpret_cast<T*>(p.out) + t * p.out_s + c, left, o);
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

// Zeros for share `pass` of the table's `passes` equal shares, by workgroup b of n, past the caches (the whole gradient of 8192
// tokens, 131 MB of table: 45 us, through them 48) and by a quarter of the threads: 2 x 256 a CU that move along the table
// together write faster than 2 x 1024 (200 MB alone: 33 us, 39; the gradient of the 8192 tokens: 43 us, 45).
__device__ void clear_share(const EmbedBwdParams& p, int pass, int64_t b, int64_t n) {
  typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
  const int64_t bytes = p.vocab * p.dim * (p.dw_f32 ? 4 : 2), share = (bytes / p.passes + 15) / 16 * 16;
  const int64_t lo = pass * share, hi = pass + 1 == p.passes ? bytes : min(bytes, lo + share);
  char* base = reinterpret_cast<char*>(p.dweight);
  const u32x4_any z = {0u, 0u, 0u, 0u};
  if (threadIdx.x >= kClearThreads) return;
  int64_t at = lo + 16 * (b * kClearThreads + threadIdx.x);
  for (; at + 16 <= hi; at += 16 * kClearThreads * n) __builtin_nontemporal_store(z, reinterpret_cast<u32x4_any*>(base + at));
  for (; at < hi; at += 2) *reinterpret_cast<uint16_t*>(base + at) = 0;         // the last thread's tail, if any
}
__global__ __launch_bounds__(kSortThreads) void embed_clear_kernel(EmbedBwdParams p) {
  for (int pass = 0; pass < p.passes; ++pass) clear_share(p, pass, blockIdx.x, gridDim.x);
}

// The lanes with this lane's digit (`same`), and how many of them come before it.
__device__ __forceinline__ int digit_rank(uint32_t d, bool live, int lane, uint64_t& same) {
  same = __ballot(live);
#pragma unroll
  for (int bit = 0; bit < kBits; ++bit) {
    const bool on = (d >> bit) & 1;
    const uint64_t b = __ballot(on);
    same &= on ? b : ~b;
  }
  return __popcll(same & (((uint64_t)1 << lane) - 1));
}

// One stable pass.  Each of a workgroup's 16 waves owns a share of the tile and walks it 64 tokens at a time: a token's
// place is its digit's start (all smaller digits, then the digit's tokens of earlier tiles, earlier waves and earlier
// steps) plus the number of lanes before it with the same digit (ballots over the digit's bits).  The digits of the other
// tiles are counted here from their keys where there are few (DIRECT: no launch and no atomics in memory for it; the
// keys of 16384 tokens are 64 KB), or come from `hist`.  Workgroups beyond the tiles clear their share of the table.
template <bool DIRECT>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedBwdParams p, int pass) {
  constexpr int kWaves = kSortThreads / 64;
  constexpr int kAhead = 4;                      // steps whose loads are on their way together
  __shared__ uint32_t at[kWaves][kDigits];
  __shared__ uint32_t early[DIRECT ? kDigits : 1], late[DIRECT ? kDigits : 1];
  __shared__ uint32_t wsum[kDigits / 64];
  if ((int)blockIdx.x >= p.tiles) return clear_share(p, pass, blockIdx.x - p.tiles, gridDim.x - p.tiles);
  const int lane = lane_id(), wave = wave_id(), shift = pass * kBits;
  const uint32_t* key_in = p.keys[pass & 1];
  const uint32_t* tok_in = p.order[pass & 1];
  uint32_t* key_out = p.keys[(pass & 1) ^ 1];
  uint32_t* tok_out = p.order[(pass & 1) ^ 1];
  for (int i = threadIdx.x; i < kWaves * kDigits; i += kSortThreads) at[0][i] = 0;
  if (DIRECT && threadIdx.x < kDigits) early[threadIdx.x] = late[threadIdx.x] = 0;
  __syncthreads();
  const int64_t part = p.tile / kWaves, first = (int64_t)blockIdx.x * p.tile, lo = first + wave * part;
  const int64_t hi = min(p.tokens, lo + part);
  auto digit = [&](int64_t t) {
    return ((pass ? key_in[t] : token_key(p, t)) >> shift) & (kDigits - 1);
  };
  // digit x of thread x: its counts in earlier tiles and in all
  uint32_t before = 0, total = 0;
  if (DIRECT) {
    const int bits = __builtin_ctzll(part);
    for (int64_t t0 = threadIdx.x; t0 < p.tokens; t0 += kSortThreads * kAhead) {
      uint32_t d[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) d[i] = t0 + kSortThreads * i < p.tokens ? digit(t0 + kSortThreads * i) : 0;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int64_t t = t0 + kSortThreads * i;
        if (t >= p.tokens) break;
        uint32_t* n = t < first ? early : t >= first + p.tile ? late : at[(t - first) >> bits];
        atomicAdd(&n[d[i]], 1u);
      }
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      before = early[threadIdx.x];
      total = before + late[threadIdx.x];
      for (int w = 0; w < kWaves; ++w) total += at[w][threadIdx.x];
    }
  } else {
    for (int64_t t0 = lo + lane; t0 < hi; t0 += 64 * kAhead) {
      uint32_t d[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) d[i] = t0 + 64 * i < hi ? digit(t0 + 64 * i) : 0;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (t0 + 64 * i < hi) atomicAdd(&at[wave][d[i]], 1u);
    }
    if (threadIdx.x < kDigits) {
      const uint32_t* hist = p.hist + (int64_t)pass * p.tiles * kDigits + threadIdx.x;
#pragma unroll 8
      for (int b = 0; b < p.tiles; ++b) {
        const uint32_t n = hist[b * kDigits];
        before += b < (int)blockIdx.x ? n : 0;
        total += n;
      }
    }
  }
  uint32_t incl = total;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)incl, off, 64);
    if (lane >= off) incl += o;
  }
  if (lane == 63 && wave < kDigits / 64) wsum[wave] = incl;
  __syncthreads();                               // also: every wave's counts are in `at`
  if (threadIdx.x < kDigits) {
    uint32_t start = incl - total + before;
    for (int w = 0; w < wave; ++w) start += wsum[w];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t n = at[w][threadIdx.x];
      at[w][threadIdx.x] = start;
      start += n;
    }
  }
  __syncthreads();
  uint32_t* next = !DIRECT && pass + 1 < p.passes ? p.hist + (int64_t)(pass + 1) * p.tiles * kDigits : nullptr;
  volatile uint32_t* mine = at[wave];
  for (int64_t t0 = lo; t0 < hi; t0 += 64 * kAhead) {
    uint32_t key[kAhead], tok[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t t = t0 + 64 * i + lane;
      key[i] = tok[i] = 0;
      if (t < hi) {
        key[i] = pass ? key_in[t] : token_key(p, t);
        tok[i] = pass ? tok_in[t] : (uint32_t)t;
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t0 + 64 * i >= hi) break;
      const bool live = t0 + 64 * i + lane < hi;
      const uint32_t k = key[i], d = (k >> shift) & (kDigits - 1);
      uint64_t same;
      const int rank = digit_rank(d, live, lane, same);
      if (live) {
        const uint32_t place = mine[d], pos = place + rank;
        __builtin_amdgcn_wave_barrier();         // every lane has read its digit's place before the first lane moves it
        if (rank == 0) mine[d] = place + (uint32_t)__popcll(same);
        key_out[pos] = k;
        tok_out[pos] = tok[i];
        if (next) atomicAdd(&next[(int64_t)(pos / (uint32_t)p.tile) * kDigits + ((k >> (shift + kBits)) & (kDigits - 1))], 1u);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// Zeros for the rows whose bit is not set, by workgroup b of n: 16 bytes a thread along the table whatever its rows' length,
// so that stores stay whole and in line; the pieces at the ends of rows that have a token go by elements.
template <typename TW>
__device__ void clear_absent(const EmbedBwdParams& p, const uint32_t* bits, int64_t b, int64_t n) {
  typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
  const u32x4_any z = {0u, 0u, 0u, 0u};
  // rows and bytes of a row in 32 bits (2^18 each at most): the arithmetic of a piece is what a store has to hide
  const int row_bytes = p.dim * (int)sizeof(TW);
  const int64_t bytes = p.vocab * row_bytes, step = 16 * kSortThreads * n, at = 16 * (b * kSortThreads + threadIdx.x);
  const int rows = (int)(step / row_bytes), rest = (int)(step % row_bytes);
  int row = (int)(at / row_bytes), in = (int)(at % row_bytes);        // the piece begins at byte `in` of `row`
  char* q = reinterpret_cast<char*>(p.dweight) + at;
  const char* end = reinterpret_cast<char*>(p.dweight) + bytes;
  auto has = [&](int v) { return bits[v >> 5] >> (v & 31) & 1; };
  for (; q < end; q += step) {
    const bool whole = q + 16 <= end, mine = has(row);
    if (whole && (in + 16 <= row_bytes || (row_bytes >= 16 && mine == has(row + 1)))) {
      if (!mine) __builtin_nontemporal_store(z, reinterpret_cast<u32x4_any*>(q));
    } else {
      int v = row, e = in;
      for (int o = 0; o < 16 && q + o < end; o += sizeof(TW), e += sizeof(TW)) {
        if (e >= row_bytes) { e -= row_bytes; ++v; }
        if (!has(v)) *reinterpret_cast<TW*>(q + o) = from_f32<TW>(0.f);
      }
    }
    row += rows;
    in += rest;
    if (in >= row_bytes) { in -= row_bytes; ++row; }
  }
}

// Few tokens: one launch without a sort.  The first workgroups take 16 tokens each, a wave a token and up to 512 columns of
// it: the wave compares the token's row with all tokens' (in LDS), and the one occurrence that is to answer for the row
// sums its tokens in their order.  Which occurrence that is goes by the row, so that a few frequent rows, all of which
// show up among the first tokens, are not one workgroup's.  A row with more than kList tokens is summed by the whole
// workgroup, an equal share of its tokens a wave, the shares joined in order.  The other workgroups write the zeros of the
// rows that have no token, which a bit for each row in LDS tells.
template <typename T, typename TW>
__global__ __launch_bounds__(kSortThreads) void embed_few_kernel(EmbedBwdParams p, int sums) {
  constexpr int kWaves = kSortThreads / 64, kList = 32, kAhead = 8;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  struct Sum {
    u32x4 keys[kFew / 4];
    uint16_t list[kWaves][kList], run[kFew];
    uint32_t longs[kWaves];
    float park[kWaves][8][64];
    int n_longs, found;
  };
  __shared__ union {
    Sum s;
    uint32_t bits[kFewRows / 32];
  } sh;
  const int n = (int)p.tokens, lane = lane_id(), wave = wave_id();
  if ((int)blockIdx.x >= sums) {
    const int words = (int)((p.vocab + 31) / 32);
    for (int i = threadIdx.x; i < words; i += kSortThreads) sh.bits[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < n; t += kSortThreads) {
      const uint32_t k = token_key(p, t);
      if (k < (uint32_t)p.vocab) atomicOr(&sh.bits[k / 32], 1u << (k % 32));
    }
    __syncthreads();
    clear_absent<TW>(p, sh.bits, blockIdx.x - sums, gridDim.x - sums);
    return;
  }
  const int slabs = (p.dim + 511) / 512, slab = blockIdx.x % slabs, t = blockIdx.x / slabs * kWaves + wave;
  const int c = 512 * slab + 8 * lane, left = p.dim - c;
  const T* dy = reinterpret_cast<const T*>(p.dy) + c;
  const int n256 = (n + 255) / 256 * 256;
  uint32_t* keys = reinterpret_cast<uint32_t*>(sh.s.keys);
  for (int i = threadIdx.x; i < n256; i += kSortThreads) keys[i] = i < n ? token_key(p, i) : 0xffffffffu;
  if (threadIdx.x == 0) sh.s.n_longs = 0;
  __syncthreads();
  // the tokens of row `key` in order into list (as many as it holds); their number, and how many come before token t.  Four
  // tokens a lane at a time, most of which are other rows'.
  auto find = [&](uint32_t key, uint16_t* list, int room, int& before) {
    int found = 0;
    before = 0;
#pragma unroll 2
    for (int q = 0; q < n256; q += 256) {
      const u32x4 k = sh.s.keys[q / 4 + lane];
      const bool hit[4] = {k[0] == key, k[1] == key, k[2] == key, k[3] == key};
      if (!__ballot(hit[0] | hit[1] | hit[2] | hit[3])) continue;
      const uint64_t lower = ((uint64_t)1 << lane) - 1;
      int at = found;
#pragma unroll
      for (int j = 0; j < 4; ++j) at += __popcll(__ballot(hit[j]) & lower);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int token = q + 4 * lane + j;
        before += __popcll(__ballot(hit[j] && token < t));
        found += __popcll(__ballot(hit[j]));
        if (hit[j]) {
          if (at < room) list[at] = (uint16_t)token;
          ++at;
        }
      }
    }
    return found;
  };
  // dy of tokens list[from .. to) added up in order
  auto sum = [&](const uint16_t* list, int from, int to, float (&acc)[8]) {
    for (int i0 = from; i0 < to; i0 += kAhead) {
      Raw8<T> v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < to && left > 0) load_raw(v[i], dy + (int64_t)list[i0 + i] * p.dy_s, left);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < to && left > 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += v[i].get(j);
        }
    }
  };
  auto put = [&](uint32_t key, float (&acc)[8]) {
    if (left <= 0) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
    store8(reinterpret_cast<TW*>(p.dweight) + (int64_t)key * p.dim + c, left, acc);
  };
  const uint32_t key = t < n ? keys[t] : (uint32_t)p.vocab;
  if (key < (uint32_t)p.vocab) {
    int before;
    const int found = find(key, sh.s.list[wave], kList, before);
    if ((uint32_t)before == key % (uint32_t)found) {
      if (found <= kList) {
        __builtin_amdgcn_wave_barrier();
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        sum(sh.s.list[wave], 0, found, acc);
        put(key, acc);
      } else if (lane == 0) {
        sh.s.longs[atomicAdd(&sh.s.n_longs, 1)] = key;
      }
    }
  }
  __syncthreads();
  const int longs = sh.s.n_longs;
  for (int r = 0; r < longs; ++r) {
    const uint32_t k = sh.s.longs[r];
    int before;
    if (wave == 0) {
      const int found = find(k, sh.s.run, kFew, before);
      if (lane == 0) sh.s.found = found;
    }
    __syncthreads();
    const int found = sh.s.found, per = (found + kWaves - 1) / kWaves, from = wave * per;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    sum(sh.s.run, from, min(found, from + per), acc);
#pragma unroll
    for (int j = 0; j < 8; ++j) sh.s.park[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kWaves; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += sh.s.park[w][j][lane];
      put(k, acc);
    }
    __syncthreads();
  }
}

// A piece of the sorted tokens and up to 2048 columns of it, 8 a thread; the rows of 8 tokens are on their way at once.
template <typename T, typename TW>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedBwdParams p) {
  constexpr int kAhead = 8;                      // pieces are multiples of it
  const int lane = threadIdx.x & (p.cthreads - 1);
  const int64_t piece = (int64_t)blockIdx.x * (256 / p.cthreads) + threadIdx.x / p.cthreads;
  const int c = 8 * (blockIdx.y * p.cthreads + lane), left = p.dim - c;
  if (piece >= p.pieces || left <= 0) return;
  const uint32_t* keys = p.keys[p.passes & 1];
  const uint32_t* order = p.order[p.passes & 1];
  const int64_t lo = piece * p.piece, hi = min(p.tokens, lo + p.piece);
  const T* dy = reinterpret_cast<const T*>(p.dy) + c;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const uint32_t prev = lo > 0 ? keys[lo - 1] : 0xffffffffu, after = hi < p.tokens ? keys[hi] : 0xffffffffu;
  uint32_t cur = keys[lo];
  bool cont = prev == cur;                       // the run began in an earlier piece
  auto flush = [&](bool goes_on) {
    if (cont || goes_on) {
      store8(p.part + (2 * piece + (cont ? 0 : 1)) * (int64_t)p.dim + c, left, acc);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store8(reinterpret_cast<TW*>(p.dweight) + (int64_t)cur * p.dim + c, left, acc);
    }
  };
  for (int64_t i0 = lo; i0 < hi; i0 += kAhead) {
    uint32_t k[kAhead], tok[kAhead];
    Raw8<T> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      k[i] = i0 + i < hi ? keys[i0 + i] : 0xffffffffu;
      tok[i] = i0 + i < hi ? order[i0 + i] : 0u;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (k[i] < (uint32_t)p.vocab) load_raw(v[i], dy + (int64_t)tok[i] * p.dy_s, left);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= hi) break;
      if (k[i] != cur) {
        flush(false);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
        cur = k[i];
        cont = false;
      }
      if (k[i] >= (uint32_t)p.vocab) return;     // only dropped tokens follow
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += v[i].get(j);
    }
  }
  flush(after == cur);
}

// The runs that begin in this workgroup's pieces and go beyond their piece: cthreads threads, a wave (WAVE) at most, of 8 columns each,
// the partial rows in equal shares to the workgroup's groups of threads, the shares joined in order.
template <typename TW, bool WAVE>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedBwdParams p) {
  __shared__ float park[8][256];
  const uint32_t* keys = p.keys[p.passes & 1];
  const int jt = WAVE ? 64 : p.cthreads, groups = 256 / jt, group = WAVE ? wave_id() : threadIdx.x / jt;
  const int c = 8 * (blockIdx.y * jt + (threadIdx.x & (jt - 1))), left = p.dim - c;
  const int64_t end = min(p.pieces, (int64_t)(blockIdx.x + 1) * p.join);
  for (int64_t piece = (int64_t)blockIdx.x * p.join; piece < end; ++piece) {
    const int64_t lo = piece * p.piece, hi = lo + p.piece;
    if (hi >= p.tokens) return;
    const uint32_t cur = keys[hi - 1], after = keys[hi], first = keys[lo], prev = lo > 0 ? keys[lo - 1] : 0xffffffffu;
    if (cur >= (uint32_t)p.vocab) return;
    if (after != cur || (first == cur && prev == cur)) continue;      // ends here, or is an earlier piece's
    int n = 1;                                   // the pieces that begin in the run follow this one
    for (int64_t q = piece + 1;; q += 64) {
      const bool in = q + lane_id() < p.pieces && keys[(q + lane_id()) * p.piece] == cur;
      const uint64_t out = ~__ballot(in);
      n += out ? __builtin_ctzll(out) : 64;
      if (out) break;
    }
    const int per = (n + groups - 1) / groups, from = group * per, to = min(n, from + per);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (left > 0) {
#pragma unroll 4
      for (int i = from; i < to; ++i) {
        float v[8];
        load8(p.part + (2 * (piece + i) + (i ? 0 : 1)) * (int64_t)p.dim + c, left, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) park[j][threadIdx.x] = acc[j];
    __syncthreads();
    if (group == 0 && left > 0) {
      const int used = (n + per - 1) / per;
      for (int w = 1; w < used; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += park[j][w * jt + threadIdx.x];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= p.scale;
      store8(reinterpret_cast<TW*>(p.dweight) + (int64_t)cur * p.dim + c, left, acc);
    }
    __syncthreads();
  }
}

// Workgroups that clear: 64 KB each, `most` at most.  Beside the sort two a CU.  Beside the sums of few tokens 2048, which
// follow the sums' as those end (1999 tokens, 49999 x 1001 fp32: 43 us, with 512 at most 52; with 32 KB each and 4096 at
// most 51, each having the rows' bits to set first).
unsigned clear_blocks(int64_t bytes, int64_t most) {
  const int64_t b = (bytes + 65535) / 65536;
  return (unsigned)(b < most ? b : most);
}

bool few_tokens(const EmbedBwdParams& p) {
  return p.tokens <= kFew && p.vocab <= kFewRows && p.dim <= (1 << 16);
}

template <typename T, typename TW>
hipError_t run_bwd(const EmbedBwdParams& p, hipStream_t st) {
  const int64_t bytes = p.vocab * p.dim * (int64_t)sizeof(TW);
  if (p.tokens == 0) {
    embed_clear_kernel<<<clear_blocks(bytes, 512), kSortThreads, 0, st>>>(p);
    return hipGetLastError();
  }
  const unsigned grid = p.tiles + clear_blocks(bytes / p.passes + 16, 512);
  if (few_tokens(p)) {
    const int sums = (int)((p.tokens + 15) / 16) * ((p.dim + 511) / 512);
    embed_few_kernel<T, TW><<<sums + clear_blocks(bytes, 2048), kSortThreads, 0, st>>>(p, sums);
    return hipGetLastError();
  }
  const bool direct = p.tokens <= kDirect;
  if (!direct) embed_count_kernel<<<p.tiles, 256, 0, st>>>(p);
  for (int pass = 0; pass < p.passes; ++pass) {
    if (direct) embed_sort_kernel<true><<<grid, kSortThreads, 0, st>>>(p, pass);
    else embed_sort_kernel<false><<<grid, kSortThreads, 0, st>>>(p, pass);
  }
  const int groups = 256 / p.cthreads, jt = p.cthreads < 64 ? p.cthreads : 64;
  const unsigned slabs = (unsigned)((p.dim + 8 * p.cthreads - 1) / (8 * p.cthreads));
  embed_sum_kernel<T, TW><<<dim3((unsigned)((p.pieces + groups - 1) / groups), slabs), 256, 0, st>>>(p);
  if (p.pieces > 1) {
    const dim3 g((unsigned)((p.pieces + p.join - 1) / p.join), (unsigned)((p.dim + 8 * jt - 1) / (8 * jt)));
    if (jt == 64) embed_join_kernel<TW, true><<<g, 256, 0, st>>>(p);
    else embed_join_kernel<TW, false><<<g, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_embed_fwd(EmbedParams p, hipStream_t st) {
  if (p.tokens == 0) return hipSuccess;
  p.cthreads = row_threads(p.dim);
  const int64_t rows = 2 * (256 / p.cthreads);
  const dim3 g = row_grid((p.tokens + rows - 1) / rows, (unsigned)((p.dim + 8 * p.cthreads - 1) / (8 * p.cthreads)));
  if (p.dtype == DT_F32) embed_fwd_kernel<float><<<g, 256, 0, st>>>(p);
  else embed_fwd_kernel<bf16><<<g, 256, 0, st>>>(p);
  return hipGetLastError();
}

size_t embed_bwd_plan(EmbedBwdParams& p, void* workspace) {
  p.passes = 1;
  while (p.passes < 4 && (p.vocab >> (kBits * p.passes)) > 0) ++p.passes;     // keys 0 .. vocab
  p.tile = 1024;
  while ((p.tokens + p.tile - 1) / p.tile > 128) p.tile *= 2;
  p.tiles = (int)((p.tokens + p.tile - 1) / p.tile);
  p.cthreads = row_threads(p.dim);
  // the shortest pieces (their rows' loads go out together) that make no more than 8 workgroups a CU of the sums
  p.piece = 8;
  while (p.piece < 256 && p.tokens / p.piece * p.cthreads > (int64_t)2048 * 256) p.piece *= 2;
  p.pieces = (p.tokens + p.piece - 1) / p.piece;
  p.join = (p.pieces + 2047) / 2048;
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
  if (few_tokens(p)) return off;                 // which use none of it; 16 bytes a token are asked for at every size
  p.hist = reinterpret_cast<uint32_t*>(take((size_t)p.passes * p.tiles * kDigits * 4));
  p.part = reinterpret_cast<float*>(take((size_t)2 * p.pieces * p.dim * 4));
  return off;
}

hipError_t launch_embed_bwd(const EmbedBwdParams& p, hipStream_t st) {
  if (p.dtype == DT_F32) return p.dw_f32 ? run_bwd<float, float>(p, st) : run_bwd<float, bf16>(p, st);
  return p.dw_f32 ? run_bwd<bf16, float>(p, st) : run_bwd<bf16, bf16>(p, st);
}

}  // namespace mh
