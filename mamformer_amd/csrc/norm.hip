// Layer norm of a residual stream, its backward with the parameters' gradients, and activations in 8 bits.
//
//   h = x + residual (rounded to the stream's type, which is what the next layer adds to; without a residual h = x)
//   mu = mean(h), r = 1 / sqrt(mean((h - mu)^2) + eps), y = (h - mu) r w + b
// and, with c = (h - mu) r and g = dy w,
//   dx = r (g - mean(g) - c mean(g c)) + d_h,   dw = sum over rows of dy c,   db = sum over rows of dy.
//
// A row lives in the registers of a group of threads (8 channels a thread and step), so every tensor is read and
// written once and the variance is that of the centred values.  Groups: as many lanes of a wave as the row has chunks,
// from 8 (heads of 64 channels) to a wave, which needs no barrier; beyond, a workgroup of 128 to 1024 threads.  Sums are
// fp32.  Bound by memory: 32768 x 4096 bf16 with 8-bit rows moves 1.2 GB forward in 199 us and 0.94 GB backward in 154.
#include <type_traits>

#include "common.h"
#include "launch.h"
#include "rows.h"

namespace mh {

namespace {

// Sums of two values over the threads of a row's group: in the wave, or over the workgroup through LDS (two buffers by
// turns, one barrier a sum).
template <int TPR>
struct RowSum {
  __device__ __forceinline__ explicit RowSum(float2*) {}
  __device__ __forceinline__ float2 operator()(float a, float b) { return {group_sum<TPR>(a), group_sum<TPR>(b)}; }
};
template <int NT>
struct BlockSum {
  float2* buf;                                   // (2, NT / 64)
  int turn = 0;
  __device__ __forceinline__ explicit BlockSum(float2* b) : buf(b) {}
  __device__ __forceinline__ float2 operator()(float a, float b) {
    const float2 v = {group_sum<64>(a), group_sum<64>(b)};
    float2* at = buf + turn * (NT / 64);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    lds_barrier();                               // leaves the loads of the next row in flight
    float2 s = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      s.x += at[w].x;
      s.y += at[w].y;
    }
    return s;
  }
};
template <> struct RowSum<128> : BlockSum<128> { using BlockSum<128>::BlockSum; };
template <> struct RowSum<256> : BlockSum<256> { using BlockSum<256>::BlockSum; };
template <> struct RowSum<512> : BlockSum<512> { using BlockSum<512>::BlockSum; };
template <> struct RowSum<1024> : BlockSum<1024> { using BlockSum<1024>::BlockSum; };

// Channels in all from which a group takes two rows: 2048 workgroups of 256 threads, 2 chunks of 8 a thread.
constexpr int64_t kTwoRows = (int64_t)2048 * 256 * 2 * 8;

// s / n by the reciprocal and one correction (n up to 16384, inv_n = 1 / n rounded): the quotient to its last bit or the one
// beside it, in 3 instructions instead of a division's 10.
__device__ __forceinline__ float mean_of(float s, float n, float inv_n) {
  const float q = s * inv_n;
  return fmaf(fmaf(-q, n, s), inv_n, q);
}
// 1 / sqrt(v) from the hardware's estimate and a Newton step; values that the step could leave the range with, zero and
// the subnormal ones among them, by the two exact operations.
__device__ __forceinline__ float inv_sqrt(float v) {
  if (!(v > 1e-30f && v < 1e30f)) return 1.f / sqrtf(v);
  const float r = __builtin_amdgcn_rsqf(v);
  return fmaf(0.5f * r, fmaf(-v * r, r, 1.f), r);
}

template <int TPR> constexpr int kThreads = TPR <= 64 ? 256 : TPR;

// ROWS rows a group, one after another with their loads all on their way at the start; the parameters are read once, with
// the rows where a thread holds one chunk of them and after the sums where it holds more.
template <typename T, int TPR, int NV, int ROWS, bool NT>
__global__ __launch_bounds__(kThreads<TPR>) void norm_fwd_kernel(NormParams p) {
  constexpr int G = kThreads<TPR> / TPR;
  __shared__ float2 sums[2 * 16];
  const int lane = threadIdx.x % TPR;
  const int64_t row0 = grid_row() * (G * ROWS) + threadIdx.x / TPR;
  if (row0 >= p.rows) return;                    // whole groups, and whole workgroups where a group is one
  RowSum<TPR> sum(sums);
  Raw8<T> x[ROWS][NV], res[ROWS][NV];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t row = row0 + k * G;
    if (k > 0 && row >= p.rows) break;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + lane);
      load_raw<NT>(x[k][i], reinterpret_cast<const T*>(p.x) + row * p.x_s + c, p.dim - c);
      if (p.residual) load_raw<NT>(res[k][i], reinterpret_cast<const T*>(p.residual) + row * p.res_s + c, p.dim - c);
    }
  }
  float w[8], b[8];
  auto params = [&](int c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { w[j] = 1.f; b[j] = 0.f; }
    if (p.weight && c < p.dim) load_par8(p.weight, p.w_f32, c, p.dim, w);
    if (p.bias && c < p.dim) load_par8(p.bias, p.w_f32, c, p.dim, b);
  };
  if constexpr (NV == 1) params(8 * lane);
  const float n = (float)p.dim, inv_n = 1.f / n;
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t row = row0 + k * G;
    if (k > 0 && row >= p.rows) return;
    float v[NV][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = x[k][i].get(j);
      if (p.residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = to_f32(from_f32<T>(v[i][j] + res[k][i].get(j)));   // the stream's own rounding
        store8<NT>(reinterpret_cast<T*>(p.h) + row * p.h_s + c, p.dim - c, v[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
    const float mu = mean_of(sum(s, 0.f).x, n, inv_n);
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = 8 * (i * TPR + lane) + j < p.dim ? v[i][j] - mu : 0.f;
        s2 += d * d;
      }
    const float r = inv_sqrt(mean_of(sum(s2, 0.f).x, n, inv_n) + p.eps);
    if (p.stats && lane == 0) {
      p.stats[2 * row] = mu;
      p.stats[2 * row + 1] = r;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + lane);
      if (p.codes) {
        const uint32_t e = pack_exponent(v[i]);
        if (c < p.code_s) {
          *reinterpret_cast<uint64_t*>(p.codes + row * p.code_s + c) = pack_codes(v[i], e);
          if ((lane & 7) == 0) p.exps[(row * p.code_s + c) / kPackGroup] = (uint8_t)e;
        }
      }
      if (c >= p.dim) continue;
      if constexpr (NV > 1) params(c);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = (v[i][j] - mu) * r * w[j] + b[j];
      store8<NT>(reinterpret_cast<T*>(p.y) + row * p.y_s + c, p.dim - c, o);
    }
  }
}

// What a thread holds of a row that it will normalise again: the stream's chunks, or their codes and steps.
template <typename T, bool PACKED, bool NT> struct RowChunk;
template <typename T, bool NT> struct RowChunk<T, false, NT> {
  Raw8<T> h, dy;
  __device__ __forceinline__ void load(const NormBwdParams& p, int64_t row, int c) {
    load_raw<NT>(h, reinterpret_cast<const T*>(p.h) + row * p.h_s + c, p.dim - c);
    load_raw<NT>(dy, reinterpret_cast<const T*>(p.dy) + row * p.dy_s + c, p.dim - c);
  }
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ float centred(int j, float mu, float r) const { return (h.get(j) - mu) * r; }
};
template <typename T, bool NT> struct RowChunk<T, true, NT> {
  Raw8<T> dy;
  uint64_t code;
  uint32_t byte;
  float step;
  __device__ __forceinline__ void load(const NormBwdParams& p, int64_t row, int c) {
    const int64_t at = row * p.code_s + c;
    code = 0;
    byte = 0;
    if (c < p.dim) {
      code = *reinterpret_cast<const uint64_t*>(p.codes + at);
      byte = p.exps[at / kPackGroup];
    }
    load_raw<NT>(dy, reinterpret_cast<const T*>(p.dy) + row * p.dy_s + c, p.dim - c);
  }
  __device__ __forceinline__ void begin() { step = pack_step(byte); }
  __device__ __forceinline__ float centred(int j, float mu, float r) const { return (pack_code(code, j) * step - mu) * r; }
};

// A workgroup walks rows blockIdx, + gridDim, ..., the next row's chunks on their way while it works on one; both the sums
// and dx are formed from the chunks as loaded.  The sums for dw and db stay in registers until its end and go to its own
// row of the partials, which norm_params_kernel adds in order: the same bits at every call.
template <typename T, int TPR, int NV, bool PACKED, bool NT>
__global__ __launch_bounds__(kThreads<TPR>) void norm_bwd_kernel(NormBwdParams p) {
  constexpr int G = kThreads<TPR> / TPR;         // rows at a time
  constexpr int W = TPR * NV * 8;                // channels of a group
  static_assert(G == 1 || NV == 1, "one chunk a thread where a workgroup has several rows");
  // Two chunks a thread, 1024 threads of 128 registers: the sums for dw and db wait in LDS (every thread's own, read and
  // written once a row).  The weight stays in registers: read again with every row it would wait for the next row's chunks.
  // Of bf16 rows that fits (8192 x 12000: 142 us with the join, 590 MB, at a copy's rate 95; from 8 bits 122); of fp32 rows
  // 80 bytes a lane go to scratch memory, 20 from 8 bits (4096 x 12000: 159 us, 590 MB; 108).
  constexpr bool kKeep = NV == 1;
  __shared__ float2 sums[2 * 16];
  __shared__ float park[G > 1 ? G * W : 1];
  __shared__ f32x4 wait[kKeep ? 1 : 4 * NV * TPR];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  RowSum<TPR> sum(sums);
  const float n = (float)p.dim, inv_n = 1.f / n;
  float w[NV][8], dw[8], db[8];
  auto swap_in = [&](int i) {                    // chunk i's sums from LDS
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw[j] = wait[(4 * i + j / 4) * TPR + threadIdx.x][j & 3];
      db[j] = wait[(4 * i + 2 + j / 4) * TPR + threadIdx.x][j & 3];
    }
  };
  auto swap_out = [&](int i) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      wait[(4 * i + q) * TPR + threadIdx.x] = f32x4{dw[4 * q], dw[4 * q + 1], dw[4 * q + 2], dw[4 * q + 3]};
      wait[(4 * i + 2 + q) * TPR + threadIdx.x] = f32x4{db[4 * q], db[4 * q + 1], db[4 * q + 2], db[4 * q + 3]};
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (i * TPR + lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[i][j] = 1.f;
    if (p.weight && c < p.dim) load_par8(p.weight, p.w_f32, c, p.dim, w[i]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = db[j] = 0.f;
  if constexpr (!kKeep) {
#pragma unroll
    for (int i = 0; i < NV; ++i) swap_out(i);
  }
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + group;
  RowChunk<T, PACKED, NT> cur[NV], next[NV];
  float2 st = {0.f, 0.f}, st_next = {0.f, 0.f};
  auto fetch = [&](int64_t at, float2& s, RowChunk<T, PACKED, NT>* chunk) {
    s = {p.stats[2 * at], p.stats[2 * at + 1]};
#pragma unroll
    for (int i = 0; i < NV; ++i) chunk[i].load(p, at, 8 * (i * TPR + lane));
  };
  if (row < p.rows) fetch(row, st, cur);
  for (; row < p.rows; row += step) {
    Raw8<T> dh[NV];
    if (p.d_h) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + lane);
        load_raw<NT>(dh[i], reinterpret_cast<const T*>(p.d_h) + row * p.dh_s + c, p.dim - c);
      }
    }
    if (row + step < p.rows) fetch(row + step, st_next, next);
    const float mu = st.x, r = st.y;
    float sg = 0.f, sgc = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      cur[i].begin();
      if constexpr (!kKeep) swap_in(i);
#pragma unroll
      for (int j = 0; j < 8; ++j) {              // beyond the row dy is 0, which keeps those channels out of the sums
        const float d = cur[i].dy.get(j), c = cur[i].centred(j, mu, r), g = d * w[i][j];
        db[j] += d;
        dw[j] += d * c;
        sg += g;
        sgc += g * c;
      }
      if constexpr (!kKeep) swap_out(i);
    }
    const float2 s = sum(sg, sgc);
    const float mg = mean_of(s.x, n, inv_n), mgc = mean_of(s.y, n, inv_n);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (i * TPR + lane);
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = r * (cur[i].dy.get(j) * w[i][j] - mg - cur[i].centred(j, mu, r) * mgc);
      if (p.d_h) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += dh[i].get(j);
      }
      store8<NT>(reinterpret_cast<T*>(p.dx) + row * p.dx_s + c, p.dim - c, o);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) cur[i] = next[i];
    st = st_next;
  }
  if (!p.dweight && !p.dbias) return;
  // the groups' sums, first to last, into this workgroup's rows of the partials (dw at 0, db at 1), or where it is the only
  // one to where they belong
  for (int which = 0; which < 2; ++which) {
    void* par = which ? p.dbias : p.dweight;
    float* dst = gridDim.x > 1 ? p.part + ((int64_t)which * gridDim.x + blockIdx.x) * p.dim : nullptr;
    if (!par) continue;
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) park[group * W + 8 * lane + j] = which ? db[j] : dw[j];
      __syncthreads();
      for (int c = threadIdx.x; c < p.dim; c += kThreads<TPR>) {
        float t = 0.f;
        for (int k = 0; k < G; ++k) t += park[k * W + c];
        if (dst) dst[c] = t;
        else if (p.w_f32) reinterpret_cast<float*>(par)[c] = t;
        else reinterpret_cast<bf16*>(par)[c] = (bf16)t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (i * TPR + lane);
        if constexpr (!kKeep) swap_in(i);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = which ? db[j] : dw[j];
        if (dst) store8(dst + c, p.dim - c, v);
        else if (p.w_f32) store8(reinterpret_cast<float*>(par) + c, p.dim - c, v);
        else store8(reinterpret_cast<bf16*>(par) + c, p.dim - c, v);
      }
    }
  }
}

// dw / db from the partials: 64 columns a workgroup, 16 threads of 4 columns for each of 64 runs of partial rows, whose
// sums are joined in order.  Few columns make few workgroups, so the rows are what is spread over the threads (512
// partials of 2048 channels: 4.5 us; with one wave for a quarter of the rows: 32 us).
__global__ __launch_bounds__(1024) void norm_params_kernel(const float* part, int nb, int dim, void* dw, void* db,
                                                           int f32) {
  __shared__ f32x4 park[64][17];
  const int which = blockIdx.y, run = threadIdx.x >> 4, c = blockIdx.x * 64 + 4 * (threadIdx.x & 15);
  void* dst = which ? db : dw;
  if (!dst) return;
  const float* src = part + (int64_t)which * nb * dim;
  const int per = (nb + 63) / 64, lo = run * per, hi = min(nb, lo + per);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (c + 4 <= dim) {
#pragma unroll 8
    for (int b = lo; b < hi; ++b) s += *reinterpret_cast<const f32x4_any*>(src + (int64_t)b * dim + c);
  } else {
    for (int b = lo; b < hi; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += c + j < dim ? src[(int64_t)b * dim + c + j] : 0.f;
  }
  park[run][threadIdx.x & 15] = s;
  __syncthreads();
  const int col = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x < 64 && col < dim) {
    float t = 0.f;
#pragma unroll 8
    for (int k = 0; k < 64; ++k) t += park[k][threadIdx.x >> 2][threadIdx.x & 3];
    if (f32) reinterpret_cast<float*>(dst)[col] = t;
    else reinterpret_cast<bf16*>(dst)[col] = (bf16)t;
  }
}

// cthreads threads hold a row (or 2048 channels of it), a chunk of 8 channels each and 8 threads a group; kPackRows rows a
// thread, whose loads are all on their way at once.
constexpr int kPackRows = 2;

template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(PackParams p) {
  const int groups = 256 / p.cthreads;
  const int c = 8 * (blockIdx.y * p.cthreads + (threadIdx.x & (p.cthreads - 1)));
  const int64_t row0 = grid_row() * groups * kPackRows + threadIdx.x / p.cthreads;
  Raw8<T> x[kPackRows];
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int64_t row = row0 + i * groups;
    x[i].clear();
    if (row < p.rows && c < p.dim) load_raw(x[i], reinterpret_cast<const T*>(p.x) + row * p.x_s + c, p.dim - c);
  }
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int64_t row = row0 + i * groups;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[i].get(j);
    const uint32_t e = pack_exponent(v);
    if (row >= p.rows || c >= p.code_s) continue;
    *reinterpret_cast<uint64_t*>(p.codes + row * p.code_s + c) = pack_codes(v, e);
    if ((threadIdx.x & 7) == 0) p.exps[(row * p.code_s + c) / kPackGroup] = (uint8_t)e;
  }
}
template <typename T>
__global__ __launch_bounds__(256) void unpack_kernel(PackParams p) {
  const int groups = 256 / p.cthreads;
  const int c = 8 * (blockIdx.y * p.cthreads + (threadIdx.x & (p.cthreads - 1)));
  const int64_t row0 = grid_row() * groups * kPackRows + threadIdx.x / p.cthreads;
  if (c >= p.dim) return;
  uint64_t code[kPackRows];
  uint32_t byte[kPackRows];
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int64_t row = row0 + i * groups, at = row * p.code_s + c;
    code[i] = byte[i] = 0;
    if (row < p.rows) {
      code[i] = *reinterpret_cast<const uint64_t*>(p.codes + at);
      byte[i] = p.exps[at / kPackGroup];
    }
  }
#pragma unroll
  for (int i = 0; i < kPackRows; ++i) {
    const int64_t row = row0 + i * groups;
    if (row >= p.rows) return;
    const float step = pack_step(byte[i]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = pack_code(code[i], j) * step;
    store8(reinterpret_cast<T*>(p.out) + row * p.x_s + c, p.dim - c, v);
  }
}

// Calls f with (TPR, NV, ROWS) of the group that holds a row of dim channels.  Rows of up to 512 channels, one chunk a
// thread, go two to a group where that leaves 8 workgroups a CU (131072 x 128 bf16: 13.0 us, 13.8 by one; 60000 x 512:
// 24.0 and 26.0).  Rows of up to 2048 go to a workgroup each where there are up to four a CU of them (256 x 2048: 4.8
// us, a wave each 5.4; 1024 x 2048: 5.1 and 5.6), and to a wave each beyond (2048 x 1000: 4.4 us, a workgroup each 5.2;
// 4096 x 1000: 5.8 and 8.0).
template <int TPR, int NV, int ROWS = 1> struct Group {};
template <typename F>
auto with_fwd_group(int64_t rows, int dim, F&& f) {
  const bool many = rows * dim >= kTwoRows;
  if (dim <= 64) return many ? f(Group<8, 1, 2>{}) : f(Group<8, 1>{});
  if (dim <= 128) return many ? f(Group<16, 1, 2>{}) : f(Group<16, 1>{});
  if (dim <= 256) return many ? f(Group<32, 1, 2>{}) : f(Group<32, 1>{});
  if (dim <= 512) return many ? f(Group<64, 1, 2>{}) : f(Group<64, 1>{});
  if (rows <= 1024 && dim <= 2048) return f(Group<256, 1>{});
  if (dim <= 1024) return f(Group<64, 2>{});
  if (dim <= 2048) return f(Group<64, 4>{});
  if (dim <= 4096) return f(Group<256, 2>{});
  if (dim <= 8192) return f(Group<512, 2>{});
  return f(Group<1024, 2>{});
}
// The backward's sums take two registers a channel more: one chunk a thread as far as a workgroup goes, which leaves
// registers for more waves and the next row (with the join, 32768 x 4096 from 8-bit rows: 512 threads with one chunk 153 us,
// 256 with two 165; from bf16 rows 187 and 182; 4001 x 8192 fp32: 1024 with one 91, 512 with two 96).
template <typename F>
auto with_bwd_group(int dim, F&& f) {
  if (dim <= 64) return f(Group<8, 1>{});
  if (dim <= 128) return f(Group<16, 1>{});
  if (dim <= 256) return f(Group<32, 1>{});
  if (dim <= 512) return f(Group<64, 1>{});
  if (dim <= 1024) return f(Group<128, 1>{});
  if (dim <= 2048) return f(Group<256, 1>{});
  if (dim <= 4096) return f(Group<512, 1>{});
  if (dim <= 8192) return f(Group<1024, 1>{});
  return f(Group<1024, 2>{});
}

// Calls whose tensors together are larger than the cache in front of the memory read and write them past it (32768 x 4096
// bf16 with 8-bit rows: backward, 0.9 GB, 152 us, through it 179; forward, 1.2 GB, after a backward 195 and 206); smaller
// ones leave there what the next call will read (8192 x 2048, backward on what the forward left: 25 us, past it 31).
bool past_cache(int64_t rows, int dim, int tensors, size_t es) {
  return rows * dim * tensors * (int64_t)es > (int64_t)256 << 20;
}

template <typename T, int TPR, int NV, int ROWS>
hipError_t run_fwd(const NormParams& p, hipStream_t st, Group<TPR, NV, ROWS>) {
  constexpr int R = kThreads<TPR> / TPR * ROWS;
  const dim3 g = row_grid((p.rows + R - 1) / R, 1);
  if (past_cache(p.rows, p.dim, p.residual ? 4 : 2, sizeof(T)))
    norm_fwd_kernel<T, TPR, NV, ROWS, true><<<g, kThreads<TPR>, 0, st>>>(p);
  else
    norm_fwd_kernel<T, TPR, NV, ROWS, false><<<g, kThreads<TPR>, 0, st>>>(p);
  return hipGetLastError();
}

// Every workgroup leaves a row of partials each for dw and db, written and read again, so there are fewer workgroups than
// would hide more latency: two a CU, one of 1024 threads (8192 x 2048: 25 us with 512 workgroups and 4.0 for the partials'
// sums, 24.6 and 5.0 with 1024), four of the short rows, whose partials are small (131072 x 128: 18.1 with 1024, 19.8 with
// 512).  Of 128 threads, for 513 to 1024 channels, eight: many rows need them (with the join, 32768 x 1024 bf16: 48 us,
// with 512 in all 80; 100001 x 1000: 146 and 395), few rows pay for the partials (8192 x 1024: 22.5 both, fp32 28 and 25;
// 2048 x 1024, a row a workgroup: 20 and 11).
template <int TPR, int NV>
int bwd_blocks(int64_t rows, Group<TPR, NV>) {
  constexpr int G = kThreads<TPR> / TPR;
  const int64_t need = (rows + G - 1) / G, cap = TPR == 1024 ? 256 : TPR < 128 ? 1024 : TPR == 128 ? 2048 : 512;
  return (int)(need < cap ? need : cap);
}

template <typename T, int TPR, int NV>
hipError_t run_bwd(const NormBwdParams& p, hipStream_t st, Group<TPR, NV> gr) {
  const int nb = bwd_blocks(p.rows, gr);
  const bool past = past_cache(p.rows, p.dim, p.d_h ? 4 : 3, sizeof(T));
  auto go = [&](auto packed, auto nt) {
    norm_bwd_kernel<T, TPR, NV, decltype(packed)::value, decltype(nt)::value><<<nb, kThreads<TPR>, 0, st>>>(p);
  };
  if (p.codes) past ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else past ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
  if (p.part && nb > 1)
    norm_params_kernel<<<dim3((p.dim + 63) / 64, 2), 1024, 0, st>>>(p.part, nb, p.dim, p.dweight, p.dbias, p.w_f32);
  return hipGetLastError();
}

__global__ __launch_bounds__(256) void zero_params_kernel(void* dw, void* db, int dim, int f32) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  void* dst = blockIdx.y ? db : dw;
  if (!dst || c >= dim) return;
  if (f32) reinterpret_cast<float*>(dst)[c] = 0.f;
  else reinterpret_cast<bf16*>(dst)[c] = (bf16)0.f;
}

}  // namespace

hipError_t launch_norm_fwd(const NormParams& p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  return with_fwd_group(p.rows, p.dim, [&](auto g) {
    return p.dtype == DT_F32 ? run_fwd<float>(p, st, g) : run_fwd<bf16>(p, st, g);
  });
}

size_t norm_bwd_workspace_bytes(int64_t rows, int dim) {
  if (rows == 0) return 0;
  return (size_t)with_bwd_group(dim, [&](auto g) { return bwd_blocks(rows, g); }) * dim * 2 * sizeof(float);
}

hipError_t launch_norm_bwd(const NormBwdParams& p, hipStream_t st) {
  if (p.rows == 0) {
    if (p.dweight || p.dbias)
      zero_params_kernel<<<dim3((p.dim + 255) / 256, 2), 256, 0, st>>>(p.dweight, p.dbias, p.dim, p.w_f32);
    return hipGetLastError();
  }
  return with_bwd_group(p.dim, [&](auto g) {
    return p.dtype == DT_F32 ? run_bwd<float>(p, st, g) : run_bwd<bf16>(p, st, g);
  });
}

hipError_t launch_pack(PackParams p, bool back, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  p.cthreads = row_threads(p.code_s);
  const int64_t rows = kPackRows * (256 / p.cthreads);
  const dim3 g = row_grid((p.rows + rows - 1) / rows, (unsigned)((p.code_s + 8 * p.cthreads - 1) / (8 * p.cthreads)));
  if (p.dtype == DT_F32) {
    if (back) unpack_kernel<float><<<g, 256, 0, st>>>(p);
    else pack_kernel<float><<<g, 256, 0, st>>>(p);
  } else {
    if (back) unpack_kernel<bf16><<<g, 256, 0, st>>>(p);
    else pack_kernel<bf16><<<g, 256, 0, st>>>(p);
  }
  return hipGetLastError();
}

}  // namespace mh
