// Rows of channels as 8-element chunks, for the operators that walk (rows, dim) tensors of any width and row stride.
// A chunk is one 16-byte (bf16) or two 16-byte (fp32) accesses that need the alignment of an element only (gfx950
// takes unaligned vector accesses to global memory), so odd widths and strides run the same code as even ones; the
// last chunk of a row whose width is no multiple of 8 goes element by element.
#pragma once

#include "common.h"

namespace mh {

typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// NT: past the caches, for tensors larger than those that are read or written once (512 MiB read: 7.0 TB/s against 6.2,
// copied: 6.2 against 5.6).
template <bool NT> __device__ __forceinline__ bf16x8 get_vec(const bf16* p) {
  const bf16x8_any* q = reinterpret_cast<const bf16x8_any*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool NT> __device__ __forceinline__ f32x4 get_vec(const float* p) {
  const f32x4_any* q = reinterpret_cast<const f32x4_any*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool NT> __device__ __forceinline__ void put_vec(bf16* p, bf16x8 v) {
  bf16x8_any* q = reinterpret_cast<bf16x8_any*>(p);
  if constexpr (NT) __builtin_nontemporal_store(v, q);
  else *q = v;
}
template <bool NT> __device__ __forceinline__ void put_vec(float* p, f32x4 v) {
  f32x4_any* q = reinterpret_cast<f32x4_any*>(p);
  if constexpr (NT) __builtin_nontemporal_store(v, q);
  else *q = v;
}

// A chunk as it was loaded, so that what is fetched ahead holds no more registers than its bytes.
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  bf16x8 v;
  template <bool NT = false> __device__ __forceinline__ void load(const bf16* p) {
    v = get_vec<NT>(p);
  }
  __device__ __forceinline__ void set(int j, bf16 x) { v[j] = x; }
  __device__ __forceinline__ void clear() { v = bf16x8{}; }
  __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
};
template <> struct Raw8<float> {
  f32x4 a, b;
  template <bool NT = false> __device__ __forceinline__ void load(const float* p) {
    a = get_vec<NT>(p);
    b = get_vec<NT>(p + 4);
  }
  __device__ __forceinline__ void set(int j, float x) {
    if (j < 4) a[j] = x;
    else b[j & 3] = x;
  }
  __device__ __forceinline__ void clear() { a = b = f32x4{}; }
  __device__ __forceinline__ float get(int j) const { return j < 4 ? a[j] : b[j & 3]; }
};
// left: elements from p to the end of the row; those beyond it read as 0.
template <bool NT = false, typename T>
__device__ __forceinline__ void load_raw(Raw8<T>& r, const T* p, int left) {
  if (left >= 8) {
    r.template load<NT>(p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.set(j, j < left ? p[j] : from_f32<T>(0.f));
  }
}

template <bool NT = false, typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  Raw8<T> r;
  r.template load<NT>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = r.get(j);
}
// Elements beyond `left` read as `pad`.
template <bool NT = false, typename T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8], float pad = 0.f) {
  if (left >= 8) {
    load8<NT>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? to_f32(p[j]) : pad;
  }
}

template <bool NT = false>
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
  bf16x8 b;
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = (bf16)v[j];
  put_vec<NT>(p, b);
}
template <bool NT = false>
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  put_vec<NT>(p, f32x4{v[0], v[1], v[2], v[3]});
  put_vec<NT>(p + 4, f32x4{v[4], v[5], v[6], v[7]});
}
template <bool NT = false, typename T>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if (left >= 8) {
    store8<NT>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = from_f32<T>(v[j]);
  }
}

// A parameter chunk in fp32 or bf16 (`f32` is uniform); element c of a vector of `dim`.
__device__ __forceinline__ void load_par8(const void* p, bool f32, int c, int dim, float (&v)[8]) {
  if (f32) load8(reinterpret_cast<const float*>(p) + c, dim - c, v);
  else load8(reinterpret_cast<const bf16*>(p) + c, dim - c, v);
}

// Index i of a vector of 32- or 64-bit indices.
__device__ __forceinline__ int64_t load_index(const void* p, bool i64, int64_t i) {
  return i64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// One workgroup for each of `n` things along a grid of at most 2^20 by z (a grid's threads along x have to stay below
// 2^32); grid_row() is the workgroup's own, which may lie behind the last one.
constexpr int64_t kGridRows = (int64_t)1 << 20;
inline dim3 row_grid(int64_t n, unsigned y) {
  const int64_t x = n < kGridRows ? n : kGridRows;
  return dim3((unsigned)x, y, (unsigned)((n + x - 1) / x));
}
// Threads of 256 for a row, a power of two from 8 to 256, of 8 columns each.
inline int row_threads(int dim) {
  int n = 8;
  while (n < 256 && 8 * n < dim) n *= 2;
  return n;
}
__device__ __forceinline__ int64_t grid_row() { return (int64_t)blockIdx.z * kGridRows + blockIdx.x; }

// Sum over aligned groups of N = 8, 16, 32 or 64 lanes, the same in every lane of the group: quad permutes and mirrors on
// the DPP crossbar, then row and half swaps -- no LDS permutes.
template <int N>
__device__ __forceinline__ float group_sum(float v) {
  v = sum_quad(v);
  v += dppf<0x141>(v);                           // row_half_mirror: the other quad of 8
  if constexpr (N >= 16) v += dppf<0x140>(v);    // row_mirror: the other 8 of 16
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (N >= 64) v = sum_halves(v);
  return v;
}

// ---------------------------------------------------------------- activations in 8 bits
// A group of 64 channels (8 lanes of one chunk each) shares an exponent e, the least with max|x| <= 127 2^e; a code
// is x 2^-e rounded to nearest even, |code| <= 127, and stands for code 2^e: 8 significant bits at most, so a bf16 or
// fp32 holds it exactly.  A power of two costs up to one bit of the 8 against a scale of max/127 but makes every step
// exact.  The exponent is kept as a byte e + 132; e is at least -132, where all codes of a group below 2^-126 end.
// 255 marks a group that holds an infinity or a NaN: all of it reads back as NaN, so that a diverged step is not hidden.
constexpr int kPackGroup = 64;
constexpr int kPackBias = 132;
constexpr int kPackNan = 255;

__device__ __forceinline__ uint32_t pack_exponent(const float (&x)[8]) {
  uint32_t u = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) u = max(u, __float_as_uint(x[j]) & 0x7fffffffu);
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, false));      // the 8 lanes' maximum as in
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, false));      // group_sum
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x141, 0xf, 0xf, false));
  if (u >= 0x7f800000u) return kPackNan;
  // max = f 2^k, 1 <= f < 2: 127 2^(k - 6) is enough up to f = 127/64 (mantissa 0x7e0000)
  const int k = max((int)(u >> 23), 1) - 127;
  return (uint32_t)(k - 6 + ((u & 0x7fffffu) > 0x7e0000u && u >= 0x00800000u) + kPackBias);
}
// |x 2^-e| is below 128, so adding 1.5 2^23 rounds it to a whole number, ties to even, in the sum's low bits.
__device__ __forceinline__ uint64_t pack_codes(const float (&x)[8], uint32_t byte) {
  if (byte == kPackNan) return 0;
  const int e = (int)byte - kPackBias;
  uint32_t q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = __float_as_uint(__builtin_amdgcn_ldexpf(x[j], -e) + 12582912.f);
  auto bytes = [&](int j) {
    const uint32_t lo = __builtin_amdgcn_perm(q[j + 1], q[j], 0x0c0c0400), hi = __builtin_amdgcn_perm(q[j + 3], q[j + 2], 0x0c0c0400);
    return lo | hi << 16;
  };
  return (uint64_t)bytes(4) << 32 | bytes(0);
}
// What a code of 1 stands for (2^e, exact; NaN for the byte of a group that holds one).
__device__ __forceinline__ float pack_step(uint32_t byte) {
  return byte == kPackNan ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(1.f, (int)byte - kPackBias);
}
__device__ __forceinline__ float pack_code(uint64_t c, int j) { return (float)(int8_t)(uint8_t)(c >> (8 * j)); }

}  // namespace mh
