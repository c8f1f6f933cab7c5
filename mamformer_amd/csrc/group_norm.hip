// Group norm, channels last: x (batch, space, channels), mean and variance of each (batch, group) over the space and the
// group's channels, z = (x - mean) / sqrt(var + eps) * weight + bias, y = z or silu(z).  Backward, with dz = dy act'(z),
// gw = dz weight and xh the normalised x: dx = (gw - mean(gw) - xh mean(gw xh)) / sqrt(var + eps), dweight = sum dz xh,
// dbias = sum dz.  Bound by the tensors' bytes.
//
// Two ways.  One position in the space (a token's heads): the lanes of a group hold its channels, one reading of x, the
// variance that of the centred values.  Otherwise the sums of a (batch, group) come from many workgroups: a pass for the
// sums, then a pass that reads x again (from the caches where it fits).  There the sums are those of x - x0 and its square in
// fp64, x0 the group's first value: the mean's distance from x0 is at most sqrt(n) deviations of n values, so that the
// variance, sum / n less its square, loses a factor n of fp64's 2^-53 at most, however far the values are from zero.
// Either way values are centred by the mean in two parts, as its rounding to fp32 may be many deviations.
// Channels are taken 8 at a time within a group, so that a chunk never belongs to two groups.
//
// Measured (bf16, silu): 8192 tokens of 16 groups of 128 channels, one reading: 18 us for 67 MB (3.7 TB/s), backward 29 for
// 101 MB and 4 for the parameters' sums; 8 x 4096 x 512 in 32 groups: 10 for the sums, 17 for the rest.  Where a workgroup
// has few rows, its first loads, its reduction and its stores follow each other: a copy of these sizes takes 10.
#include <cfloat>
#include <type_traits>

#include "launch.h"
#include "rows.h"

namespace mh {
namespace {

constexpr int kRowsMax = 512;                    // channels of a group that one wave holds

template <int N> __device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (N == 1) return v;
  else if constexpr (N == 2) return v + dppf<0xB1>(v);
  else if constexpr (N == 4) return sum_quad(v);
  else return group_sum<N>(v);
}

// z to y; and the factor of dy in dz
__device__ __forceinline__ float act(bool silu, float z) { return silu ? silu_f(z) : z; }
__device__ __forceinline__ float act_slope(bool silu, float z) {
  if (!silu) return 1.f;
  const float s = sigmoid_f(z);
  return s * (1.f + z * (1.f - s));
}

// 1 / sqrt(var + eps); squares that left fp32's range make a NaN, as an infinite deviation would turn values to the bias.
__device__ __forceinline__ float deviation(float var, float eps) {
  return var <= FLT_MAX ? 1.f / sqrtf(fmaxf(var, 0.f) + eps) : __builtin_nanf("");
}

struct Affine {
  float w[8], b[8];
  __device__ __forceinline__ Affine(const GroupNormParams& p, int c, int end) {      // channels c .. of a group ending at `end`
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = 1.f;
      b[j] = 0.f;
    }
    if (p.weight) load_par8(p.weight, p.w_f32, c, end, w);
    if (p.bias) load_par8(p.bias, p.w_f32, c, end, b);
  }
};

// Chunks of rows r, r + step .. (beyond `last` that row again), all under way before the first is used; `full`: no chunk is
// cut by its group's end.
template <int U, typename T>
__device__ __forceinline__ void load_rows(const T* src, int64_t stride, int64_t r, int64_t step, int64_t last, bool full, int left, Raw8<T> (&x)[U]) {
  if (full) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(src + min(r + u * step, last) * stride);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) load_raw(x[u], src + min(r + u * step, last) * stride, left);
  }
}
template <typename T> constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;

// A value that is loaded before others and waited for where it is taken, behind their loads.
template <typename T>
struct Ahead {
  uint32_t bits;
  __device__ __forceinline__ explicit Ahead(const T* p) {
    if constexpr (sizeof(T) == 4) bits = *reinterpret_cast<const uint32_t*>(p);
    else bits = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ double get() const {
    uint32_t b = bits;
    asm volatile("" : "+v"(b));
    return (double)__uint_as_float(sizeof(T) == 4 ? b : b << 16);
  }
};

// ------------------------------------------------------------------ one position
// A workgroup takes 256 / TG groups (or all, and several batch entries at once) and walks the batch with them, so that the
// parameters stay in registers.  The variance is that of values centred by the rounded mean, which is mended by what is left.
template <typename T, int TG>
__global__ __launch_bounds__(256) void group_rows_kernel(GroupNormParams p, int gb, int side) {
  constexpr int U = kAhead<T>;
  const int cg = p.channels / p.groups, c8 = threadIdx.x % TG * 8, left = cg - c8, slot = threadIdx.x / TG;
  const int g = blockIdx.y * gb + slot % gb, sub = slot / gb;
  if (sub >= side || g >= p.groups) return;      // no barrier follows; lanes of a group go together
  const bool full = cg % 8 == 0;
  const int c = g * cg + (left > 0 ? c8 : 0);
  const float inv = 1.f / (float)cg;
  const Affine a(p, c, (g + 1) * cg);
  const int64_t step = (int64_t)gridDim.x * side;
  for (int64_t n0 = (int64_t)blockIdx.x * side + sub; n0 < p.batch; n0 += U * step) {
    Raw8<T> raw[U];
    load_rows(reinterpret_cast<const T*>(p.x) + c, p.x_sb, n0, step, p.batch - 1, full, left, raw);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * step;
      if (n >= p.batch) break;
      float x[8], s = 0.f, q = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = j < left ? raw[u].get(j) : 0.f;
        s += x[j];
      }
      const float mean = lanes_sum<TG>(s) * inv;
      s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = j < left ? x[j] - mean : 0.f;
        s += x[j];
        q += x[j] * x[j];
      }
      const float rest = lanes_sum<TG>(s) * inv;
      const float var = lanes_sum<TG>(q) * inv - rest * rest;
      const float rstd = deviation(var, p.eps);
      if (left > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = act(p.silu, (x[j] - rest) * (rstd * a.w[j]) + a.b[j]);
        store8(reinterpret_cast<T*>(p.y) + n * p.y_sb + c, left, x);
      }
      if (p.stats && c8 == 0) {
        p.stats[2 * (n * p.groups + g)] = mean + rest;
        p.stats[2 * (n * p.groups + g) + 1] = rstd;
      }
    }
  }
}

// The same walk, a thread adding its channels' gradients in registers; `part` (rows, channels, 2) gets a row for each that
// walked.
template <typename T, int TG>
__global__ __launch_bounds__(256) void group_rows_bwd_kernel(GroupNormBwdParams q, int gb, int side) {
  constexpr int U = kAhead<T>;
  const GroupNormParams& p = q.f;
  const int cg = p.channels / p.groups, c8 = threadIdx.x % TG * 8, left = cg - c8, slot = threadIdx.x / TG;
  const int g = blockIdx.y * gb + slot % gb, sub = slot / gb;
  if (sub >= side || g >= p.groups) return;      // no barrier follows; lanes of a group go together
  const bool full = cg % 8 == 0;
  const int c = g * cg + (left > 0 ? c8 : 0);
  const float inv = 1.f / (float)cg;
  const Affine a(p, c, (g + 1) * cg);
  float A[8] = {}, B[8] = {};
  const int64_t step = (int64_t)gridDim.x * side;
  for (int64_t n0 = (int64_t)blockIdx.x * side + sub; n0 < p.batch; n0 += U * step) {
    Raw8<T> rx[U], rd[U];
    float mean[U], rstd[U];
    load_rows(reinterpret_cast<const T*>(p.x) + c, p.x_sb, n0, step, p.batch - 1, full, left, rx);
    load_rows(reinterpret_cast<const T*>(q.dy) + c, q.dy_sb, n0, step, p.batch - 1, full, left, rd);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* st = p.stats + 2 * (min(n0 + u * step, p.batch - 1) * p.groups + g);
      mean[u] = st[0];
      rstd[u] = st[1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * step;
      if (n >= p.batch) break;
      float x[8], d[8], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = j < left ? (rx[u].get(j) - mean[u]) * rstd[u] : 0.f;
        const float dz = j < left ? rd[u].get(j) * act_slope(p.silu, x[j] * a.w[j] + a.b[j]) : 0.f;
        A[j] += dz;
        B[j] += dz * x[j];
        d[j] = dz * a.w[j];
        s1 += d[j];
        s2 += d[j] * x[j];
      }
      s1 = lanes_sum<TG>(s1) * inv;
      s2 = lanes_sum<TG>(s2) * inv;
      if (left > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = rstd[u] * (d[j] - s1 - x[j] * s2);
        store8(reinterpret_cast<T*>(q.dx) + n * q.dx_sb + c, left, x);
      }
    }
  }
  if (q.part && left > 0) {
    float* to = q.part + (((int64_t)blockIdx.x * side + sub) * p.channels + c) * 2;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) *reinterpret_cast<f32x2*>(to + 2 * j) = f32x2{A[j], B[j]};
  }
}

// dbias and dweight: sums over the rows of part (rows, channels, 2), 16 lanes of rows a channel, in a fixed order.
__global__ __launch_bounds__(256) void group_params_kernel(const float* part, int64_t rows, int channels, void* dweight, void* dbias,
                                                           int f32) {
  __shared__ float sa[16][17], sb[16][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float a = 0.f, b = 0.f;
  if (c < channels)
    for (int64_t r = rl; r < rows; r += 16 * 8) {
      f32x2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const f32x2*>(part + (min(r + 16 * u, rows - 1) * channels + c) * 2);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        a += r + 16 * u < rows ? v[u][0] : 0.f;
        b += r + 16 * u < rows ? v[u][1] : 0.f;
      }
    }
  sa[rl][cl] = a;
  sb[rl][cl] = b;
  __syncthreads();
  if (rl == 0 && c < channels) {
    for (int i = 1; i < 16; ++i) {
      a += sa[i][cl];
      b += sb[i][cl];
    }
    if (dbias) {
      if (f32) reinterpret_cast<float*>(dbias)[c] = a;
      else reinterpret_cast<bf16*>(dbias)[c] = (bf16)a;
    }
    if (dweight) {
      if (f32) reinterpret_cast<float*>(dweight)[c] = b;
      else reinterpret_cast<bf16*>(dweight)[c] = (bf16)b;
    }
  }
}

// ------------------------------------------------------------------ many positions
// A workgroup's part of (batch, space, groups): gb groups of cpg chunks, `side` positions at once, `rows` positions.
struct Split {
  int cg, cpg, gb, ub, side, cblocks, splits;
  int64_t rows, units;
  __host__ explicit Split(const GroupNormParams& p) {
    cg = p.channels / p.groups;
    cpg = (cg + 7) / 8;
    gb = cpg >= 256 ? 1 : 256 / cpg < p.groups ? 256 / cpg : p.groups;
    ub = gb * cpg;
    side = ub <= 256 ? 256 / ub : 1;
    cblocks = (p.groups + gb - 1) / gb;
    // enough workgroups for the card, each with at least 4 passes over its positions
    int64_t want = 1024 / (p.batch * cblocks) + 1, most = (p.space + 4 * side - 1) / (4 * side);
    splits = (int)(want < most ? want : most);
    rows = (p.space + splits - 1) / splits;
    splits = (int)((p.space + rows - 1) / rows);
    units = p.batch * splits * cblocks;
  }
  __device__ __forceinline__ void at(int64_t u, int64_t& n, int& s, int& cb) const {
    cb = (int)(u % cblocks);
    const int64_t v = u / cblocks;
    s = (int)(v % splits);
    n = v / splits;
  }
};

template <typename T>
__global__ __launch_bounds__(256) void group_sums_kernel(GroupNormParams p, Split sp) {
  constexpr int U = kAhead<T>;
  __shared__ double sa[256], sb[256];
  const int tid = threadIdx.x, u0 = sp.ub <= 256 ? tid % sp.ub : tid, sub = sp.ub <= 256 ? tid / sp.ub : 0;
  for (int64_t unit = blockIdx.x; unit < sp.units; unit += gridDim.x) {
    int64_t n;
    int s, cb;
    sp.at(unit, n, s, cb);
    const int64_t r0 = s * sp.rows, r1 = min(p.space, r0 + sp.rows);
    double a = 0., b = 0.;
    for (int u = u0; u < sp.ub && sub < sp.side; u += 256) {
      const int g = cb * sp.gb + u / sp.cpg, c8 = u % sp.cpg * 8;
      if (g >= p.groups) break;
      const T* src = reinterpret_cast<const T*>(p.x) + n * p.x_sb + g * sp.cg + c8;
      const Ahead<T> first(src - c8);
      const bool full = sp.cg % 8 == 0;
      const int left = sp.cg - c8;
      for (int64_t r = r0 + sub; r < r1; r += U * sp.side) {
        Raw8<T> raw[U];
        load_rows(src, p.x_ss, r, sp.side, p.space - 1, full, left, raw);
        const double x0 = first.get();
#pragma unroll
        for (int v = 0; v < U; ++v) {
          if (r + v * sp.side >= r1) break;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const double x = full || j < left ? (double)raw[v].get(j) - x0 : 0.;
            a += x;
            b = __builtin_fma(x, x, b);
          }
        }
      }
    }
    __syncthreads();
    sa[tid] = a;
    sb[tid] = b;
    __syncthreads();
    if (tid < sp.gb && cb * sp.gb + tid < p.groups) {
      const int per = sp.cpg < 256 ? sp.cpg : 256;
      a = b = 0.;
      for (int i = 0; i < sp.side; ++i)
        for (int j = 0; j < per; ++j) {
          a += sa[i * sp.ub + tid * sp.cpg + j];
          b += sb[i * sp.ub + tid * sp.cpg + j];
        }
      double* to = p.part + ((n * sp.splits + s) * p.groups + cb * sp.gb + tid) * 2;
      to[0] = a;
      to[1] = b;
    }
  }
}

// Four workgroups a CU, as Split asks for: 17 us with 128 registers (8 x 4096 x 512), 19.4 with the 132 it would take.
// What the mean's rounding left goes to the bias, for a thread once: (x - mean) is exact where that counts, an fma adds the rest.
template <typename T>
__global__ __launch_bounds__(256, 4) void group_apply_kernel(GroupNormParams p, Split sp) {
  constexpr int U = kAhead<T>;
  __shared__ float sm[256], sl[256], sr[256];    // the mean and what its rounding left, 1 / deviation
  __shared__ double sa[256], sb[256];
  const int tid = threadIdx.x, u0 = sp.ub <= 256 ? tid % sp.ub : tid, sub = sp.ub <= 256 ? tid / sp.ub : 0;
  for (int64_t unit = blockIdx.x; unit < sp.units; unit += gridDim.x) {
    int64_t n;
    int s, cb;
    sp.at(unit, n, s, cb);
    const int64_t r0 = s * sp.rows, r1 = min(p.space, r0 + sp.rows);
    const bool full = sp.cg % 8 == 0;
    Raw8<T> raw[U];
    auto load = [&](int u, int64_t r) {
      const int g = min(cb * sp.gb + u / sp.cpg, p.groups - 1), c8 = u % sp.cpg * 8;
      load_rows(reinterpret_cast<const T*>(p.x) + n * p.x_sb + g * sp.cg + c8, p.x_ss, r, sp.side, p.space - 1, full, sp.cg - c8, raw);
    };
    if (u0 < sp.ub && sub < sp.side) load(u0, r0 + sub);               // under way while the sums are joined
    const bool mine = tid < sp.gb && cb * sp.gb + tid < p.groups;      // a group a thread
    const Ahead<T> first(reinterpret_cast<const T*>(p.x) + n * p.x_sb + min(cb * sp.gb + tid, p.groups - 1) * sp.cg);
    __syncthreads();
    const int shares = 256 / sp.gb;              // the splits' sums, by all threads
    if (tid < sp.gb * shares) {
      const int g = min(cb * sp.gb + tid % sp.gb, p.groups - 1);
      double a = 0., b = 0.;
      for (int i = tid / sp.gb; i < sp.splits; i += 8 * shares) {
        double2 t[8];
#pragma unroll
        for (int v = 0; v < 8; ++v)
          t[v] = *reinterpret_cast<const double2*>(p.part + ((n * sp.splits + min(i + v * shares, sp.splits - 1)) * p.groups + g) * 2);
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          a += i + v * shares < sp.splits ? t[v].x : 0.;
          b += i + v * shares < sp.splits ? t[v].y : 0.;
        }
      }
      sa[tid] = a;
      sb[tid] = b;
    }
    __syncthreads();
    if (mine) {
      const int g = cb * sp.gb + tid;
      double a = sa[tid], b = sb[tid];
      for (int i = 1; i < shares; ++i) {
        a += sa[i * sp.gb + tid];
        b += sb[i * sp.gb + tid];
      }
      const double count = (double)p.space * sp.cg, off = a / count, mean = first.get() + off, var = b / count - off * off;
      sm[tid] = (float)mean;
      sl[tid] = (float)(mean - sm[tid]);
      sr[tid] = deviation((float)var, p.eps);
      if (p.stats && s == 0) {
        p.stats[2 * (n * p.groups + g)] = sm[tid];
        p.stats[2 * (n * p.groups + g) + 1] = sr[tid];
      }
    }
    __syncthreads();
    for (int u = u0; u < sp.ub && sub < sp.side; u += 256) {
      const int g = cb * sp.gb + u / sp.cpg, c8 = u % sp.cpg * 8, left = sp.cg - c8;
      if (g >= p.groups) break;
      const int c = g * sp.cg + c8;
      Affine a(p, c, (g + 1) * sp.cg);
      const float mean = sm[u / sp.cpg], rest = sl[u / sp.cpg], rstd = sr[u / sp.cpg];
      float rw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rw[j] = rstd * a.w[j];
        a.b[j] = __builtin_fmaf(-rest, rw[j], a.b[j]);
      }
      T* dst = reinterpret_cast<T*>(p.y) + n * p.y_sb + c;
      if (u != u0) load(u, r0 + sub);
      for (int64_t r = r0 + sub; r < r1; r += U * sp.side) {
        Raw8<T> now[U];
#pragma unroll
        for (int v = 0; v < U; ++v) now[v] = raw[v];
        if (r + U * sp.side < r1) load(u, r + U * sp.side);
#pragma unroll
        for (int v = 0; v < U; ++v) {
          if (r + v * sp.side >= r1) break;
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = act(p.silu, __builtin_fmaf(now[v].get(j) - mean, rw[j], a.b[j]));
          store8(dst + (r + v * sp.side) * p.y_ss, left, x);
        }
      }
    }
  }
}

// Sums of dz and dz xh for every channel of a workgroup's positions: part (batch, splits, channels, 2).
template <typename T>
__global__ __launch_bounds__(256) void group_bwd_sums_kernel(GroupNormBwdParams q, Split sp) {
  constexpr int U = kAhead<T>;
  __shared__ float sa[256][17];
  const GroupNormParams& p = q.f;
  const int tid = threadIdx.x, u0 = sp.ub <= 256 ? tid % sp.ub : tid, sub = sp.ub <= 256 ? tid / sp.ub : 0;
  for (int64_t unit = blockIdx.x; unit < sp.units; unit += gridDim.x) {
    int64_t n;
    int s, cb;
    sp.at(unit, n, s, cb);
    const int64_t r0 = s * sp.rows, r1 = min(p.space, r0 + sp.rows);
    for (int base = 0; base < sp.ub; base += 256) {
      const int u = base + u0, g = cb * sp.gb + u / sp.cpg, c8 = u % sp.cpg * 8, left = sp.cg - c8;
      const bool on = u < sp.ub && sub < sp.side && g < p.groups;
      const int c = g * sp.cg + c8;
      float A[8] = {}, B[8] = {};
      if (on) {
        const Affine a(p, c, (g + 1) * sp.cg);
        const float mean = p.stats[2 * (n * p.groups + g)], rstd = p.stats[2 * (n * p.groups + g) + 1];
        const T* xs = reinterpret_cast<const T*>(p.x) + n * p.x_sb + c;
        const T* ds = reinterpret_cast<const T*>(q.dy) + n * q.dy_sb + c;
        for (int64_t r = r0 + sub; r < r1; r += U * sp.side) {
          Raw8<T> rx[U], rd[U];
          load_rows(xs, p.x_ss, r, sp.side, p.space - 1, sp.cg % 8 == 0, left, rx);
          load_rows(ds, q.dy_ss, r, sp.side, p.space - 1, sp.cg % 8 == 0, left, rd);
#pragma unroll
          for (int v = 0; v < U; ++v) {
            if (r + v * sp.side >= r1) break;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float x = (rx[v].get(j) - mean) * rstd;
              const float dz = j < left ? rd[v].get(j) * act_slope(p.silu, x * a.w[j] + a.b[j]) : 0.f;
              A[j] += dz;
              B[j] += dz * x;
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sa[tid][j] = A[j];
        sa[tid][8 + j] = B[j];
      }
      __syncthreads();
      if (on && sub == 0) {
        float* to = q.part + ((n * sp.splits + s) * p.channels + c) * 2;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          for (int i = 1; i < sp.side; ++i) {
            A[j] += sa[tid + i * sp.ub][j];
            B[j] += sa[tid + i * sp.ub][8 + j];
          }
          if (j < left) {
            to[2 * j] = A[j];
            to[2 * j + 1] = B[j];
          }
        }
      }
    }
  }
}

// The splits joined: `whole` (batch, channels, 2), and mean(gw), mean(gw xh) of each (batch, group) into `means`.  A
// workgroup for each (batch, group), its waves a fourth of the splits each.
__global__ __launch_bounds__(256) void group_bwd_join_kernel(GroupNormBwdParams q, Split sp, float* whole, float* means) {
  __shared__ f32x2 sv[4][64];
  const GroupNormParams& p = q.f;
  const int lane = threadIdx.x & 63, w = wave_id();
  for (int64_t it = blockIdx.x; it < p.batch * p.groups; it += gridDim.x) {
    const int64_t n = it / p.groups;
    const int g = (int)(it % p.groups);
    float s1 = 0.f, s2 = 0.f;
    for (int i0 = 0; i0 < sp.cg; i0 += 64) {
      const int i = i0 + lane, c = g * sp.cg + min(i, sp.cg - 1);
      f32x2 v = {};
      for (int s = w; s < sp.splits; s += 4 * 8) {
        f32x2 t[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) t[u] = *reinterpret_cast<const f32x2*>(q.part + ((n * sp.splits + min(s + 4 * u, sp.splits - 1)) * p.channels + c) * 2);
#pragma unroll
        for (int u = 0; u < 8; ++u) v += s + 4 * u < sp.splits ? t[u] : f32x2{};
      }
      __syncthreads();
      sv[w][lane] = v;
      __syncthreads();
      if (w == 0 && i < sp.cg) {
        v = (sv[0][lane] + sv[1][lane]) + (sv[2][lane] + sv[3][lane]);
        *reinterpret_cast<f32x2*>(whole + (n * p.channels + c) * 2) = v;
        const float wt = !p.weight ? 1.f : p.w_f32 ? reinterpret_cast<const float*>(p.weight)[c] : to_f32(reinterpret_cast<const bf16*>(p.weight)[c]);
        s1 += wt * v[0];
        s2 += wt * v[1];
      }
    }
    if (w != 0) continue;
    s1 = group_sum<64>(s1);
    s2 = group_sum<64>(s2);
    if (lane == 0) {
      const float count = (float)p.space * (float)sp.cg;
      means[2 * it] = s1 / count;
      means[2 * it + 1] = s2 / count;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void group_bwd_apply_kernel(GroupNormBwdParams q, Split sp, const float* means) {
  constexpr int U = kAhead<T>;
  const GroupNormParams& p = q.f;
  const int tid = threadIdx.x, u0 = sp.ub <= 256 ? tid % sp.ub : tid, sub = sp.ub <= 256 ? tid / sp.ub : 0;
  if (sub >= sp.side) return;
  for (int64_t unit = blockIdx.x; unit < sp.units; unit += gridDim.x) {
    int64_t n;
    int s, cb;
    sp.at(unit, n, s, cb);
    const int64_t r0 = s * sp.rows, r1 = min(p.space, r0 + sp.rows);
    for (int u = u0; u < sp.ub; u += 256) {
      const int g = cb * sp.gb + u / sp.cpg, c8 = u % sp.cpg * 8, left = sp.cg - c8;
      if (g >= p.groups) break;
      const int c = g * sp.cg + c8;
      const int64_t ng = n * p.groups + g;
      const Affine a(p, c, (g + 1) * sp.cg);
      const float mean = p.stats[2 * ng], rstd = p.stats[2 * ng + 1], m1 = means[2 * ng], m2 = means[2 * ng + 1];
      const T* xs = reinterpret_cast<const T*>(p.x) + n * p.x_sb + c;
      const T* ds = reinterpret_cast<const T*>(q.dy) + n * q.dy_sb + c;
      T* out = reinterpret_cast<T*>(q.dx) + n * q.dx_sb + c;
      for (int64_t r = r0 + sub; r < r1; r += U * sp.side) {
        Raw8<T> rx[U], rd[U];
        load_rows(xs, p.x_ss, r, sp.side, p.space - 1, sp.cg % 8 == 0, left, rx);
        load_rows(ds, q.dy_ss, r, sp.side, p.space - 1, sp.cg % 8 == 0, left, rd);
#pragma unroll
        for (int v = 0; v < U; ++v) {
          if (r + v * sp.side >= r1) break;
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[j] = (rx[v].get(j) - mean) * rstd;
            const float gw = rd[v].get(j) * act_slope(p.silu, x[j] * a.w[j] + a.b[j]) * a.w[j];
            x[j] = rstd * (gw - m1 - x[j] * m2);
          }
          store8(out + (r + v * sp.side) * q.dx_ss, left, x);
        }
      }
    }
  }
}

bool by_rows(const GroupNormParams& p) { return p.space == 1 && p.channels / p.groups <= kRowsMax; }

int rows_lanes(const GroupNormParams& p) {
  int n = 1;
  while (8 * n < p.channels / p.groups) n *= 2;
  return n;
}

struct RowsGrid {
  int gb, side, x, y;
  RowsGrid(const GroupNormParams& p, int workgroups) {
    const int slots = 256 / rows_lanes(p);
    gb = slots < p.groups ? slots : p.groups;
    side = slots / gb;
    y = (p.groups + gb - 1) / gb;
    const int64_t most = (p.batch + side - 1) / side;
    const int64_t want = workgroups / y + 1;
    x = (int)(want < most ? want : most);
  }
};

unsigned grid_of(int64_t n) { return (unsigned)(n < (1 << 20) ? n : 1 << 20); }

template <typename F>
hipError_t with_lanes(int n, F f) {
  switch (n) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    case 16: f(std::integral_constant<int, 16>()); break;
    case 32: f(std::integral_constant<int, 32>()); break;
    default: f(std::integral_constant<int, 64>()); break;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t fwd(const GroupNormParams& p, hipStream_t st) {
  if (by_rows(p)) {
    const RowsGrid rg(p, 2048);
    return with_lanes(rows_lanes(p), [&](auto n) { group_rows_kernel<T, decltype(n)::value><<<dim3(rg.x, rg.y), 256, 0, st>>>(p, rg.gb, rg.side); });
  }
  const Split sp(p);
  group_sums_kernel<T><<<grid_of(sp.units), 256, 0, st>>>(p, sp);
  group_apply_kernel<T><<<grid_of(sp.units), 256, 0, st>>>(p, sp);
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const GroupNormBwdParams& q, hipStream_t st) {
  const GroupNormParams& p = q.f;
  const bool params = q.dweight || q.dbias;
  const float* rows = q.part;
  int64_t nrows = p.batch;
  if (by_rows(p)) {
    const RowsGrid rg(p, 512);
    GroupNormBwdParams r = q;
    if (!params) r.part = nullptr;
    const hipError_t e = with_lanes(rows_lanes(p), [&](auto n) {
      group_rows_bwd_kernel<T, decltype(n)::value><<<dim3(rg.x, rg.y), 256, 0, st>>>(r, rg.gb, rg.side);
    });
    if (e != hipSuccess) return e;
    nrows = (int64_t)rg.x * rg.side;
  } else {
    const Split sp(p);
    float* whole = q.part + p.batch * sp.splits * p.channels * 2;
    float* means = whole + p.batch * p.channels * 2;
    group_bwd_sums_kernel<T><<<grid_of(sp.units), 256, 0, st>>>(q, sp);
    group_bwd_join_kernel<<<grid_of(p.batch * p.groups), 256, 0, st>>>(q, sp, whole, means);
    group_bwd_apply_kernel<T><<<grid_of(sp.units), 256, 0, st>>>(q, sp, means);
    rows = whole;
  }
  if (params)
    group_params_kernel<<<(p.channels + 15) / 16, 256, 0, st>>>(rows, nrows, p.channels, q.dweight, q.dbias, p.w_f32);
  return hipGetLastError();
}

// No rows: the parameters' gradients are cleared.
__global__ void group_clear_kernel(void* dweight, void* dbias, int channels, int f32) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= channels) return;
  if (dweight) {
    if (f32) reinterpret_cast<float*>(dweight)[c] = 0.f;
    else reinterpret_cast<bf16*>(dweight)[c] = (bf16)0.f;
  }
  if (dbias) {
    if (f32) reinterpret_cast<float*>(dbias)[c] = 0.f;
    else reinterpret_cast<bf16*>(dbias)[c] = (bf16)0.f;
  }
}

}  // namespace

size_t group_norm_workspace_bytes(const GroupNormParams& p) {
  if (by_rows(p) || p.batch == 0 || p.space == 0) return 0;
  return (size_t)p.batch * Split(p).splits * p.groups * 2 * sizeof(double);
}

hipError_t launch_group_norm(const GroupNormParams& p, hipStream_t st) {
  if (p.batch == 0 || p.space == 0) return hipSuccess;
  return p.dtype == DT_F32 ? fwd<float>(p, st) : fwd<bf16>(p, st);
}

size_t group_norm_bwd_workspace_bytes(const GroupNormParams& p) {
  if (p.batch == 0 || p.space == 0) return 0;
  if (by_rows(p)) {
    const RowsGrid rg(p, 512);
    return (size_t)rg.x * rg.side * p.channels * 2 * sizeof(float);
  }
  return ((size_t)p.batch * (Split(p).splits + 1) * p.channels + (size_t)p.batch * p.groups) * 2 * sizeof(float);
}

hipError_t launch_group_norm_bwd(const GroupNormBwdParams& q, hipStream_t st) {
  const GroupNormParams& p = q.f;
  if (p.batch == 0 || p.space == 0) {
    if (!q.dweight && !q.dbias) return hipSuccess;
    group_clear_kernel<<<(p.channels + 255) / 256, 256, 0, st>>>(q.dweight, q.dbias, p.channels, p.w_f32);
    return hipGetLastError();
  }
  return p.dtype == DT_F32 ? bwd<float>(q, st) : bwd<bf16>(q, st);
}

}  // namespace mh
