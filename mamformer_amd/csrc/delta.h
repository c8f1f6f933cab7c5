// Pieces shared by the gated delta rule's kernels (gfx950): fp16 operands in two parts, their LDS tiles and fragments,
// and the workspace's layout.
//
// Arithmetic.  The state, its gradient and the gates' gradients leave in fp32, and products of operands rounded once to
// bf16 or fp16 are too coarse for them (2^-9, 2^-12), while the fp32 matrix instructions run at 1/16 of the 16-bit rate.
// A matrix x is therefore held as (hi + lo) s: a power of two s that brings its largest magnitude into [2^12, 2^13), hi
// the fp16 nearest x / s and lo the fp16 nearest what is left.  That is x to 2^-22 of itself down to 2^-16 of the largest
// value, and to 2^-38 of the largest value below it.  A product is hi hi + hi lo + lo hi in fp32 accumulators (lo lo
// would add 2^-22); a bf16 matrix is exact in hi alone within 2^-18 of its largest value, which saves a product.
// The power of two is what fp16's range costs: bf16 parts would need none but take three of them, six products, for the
// same result.
//
// Fragments are those of the 16x16x32 fp16 instruction: lane l holds row (A) or column (B) l % 16 and, with g = l / 16,
// the k-values KS(g, j) = 4 g + j (j < 4), 16 + 4 g + j - 4 (j >= 4).  The accumulator of a 16x16 tile holds rows
// 4 g + r of column l % 16, so that two tiles below each other are a B operand as they stand: a wave keeps 16 columns of
// the state through all of its products without moving a value to another lane.
#pragma once

#include <type_traits>

#include "launch.h"
#include "rows.h"
#include "tiles.h"

namespace mh {

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

constexpr int DC = 64;                           // tokens of a piece

__device__ __forceinline__ f32x4 mma_h(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// DC rows of W fp16 (64 or 128), 16-byte chunks XOR-swizzled by row so that both accesses below meet every LDS bank once:
// 16 rows of 16 bytes (row_frag16's half wave) and 8 rows of 32 bytes (col_frag16's).
template <int W>
struct HTile {
  static constexpr int ELEMS = DC * W;
  __host__ __device__ static constexpr int swz(int r) {
    return W == 128 ? ((r & 7) << 1) | ((r >> 3) & 1) : (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  }
  __host__ __device__ static constexpr int at(int r, int c) { return r * W + (((c >> 3) ^ swz(r)) << 3) + (c & 7); }
};

// Operand with k along the rows' columns: row r0 + l % 16, k0 + KS(g, j).
template <int W>
__device__ __forceinline__ f16x8 row_frag16(const f16* t, int r0, int k0, int lane) {
  const int r = r0 + (lane & 15), k = k0 + 4 * (lane >> 4);
  const f16x4 a = *reinterpret_cast<const f16x4*>(t + HTile<W>::at(r, k));
  const f16x4 b = *reinterpret_cast<const f16x4*>(t + HTile<W>::at(r, k + 16));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Operand with k down the rows: rows k0 + KS(g, j) of column c0 + l % 16, by two transposing reads (each 16 lanes name 4
// elements of each of 4 rows, lane i receives the i-th of the 16 columns).
template <int W>
__device__ __forceinline__ f16x8 col_frag16(const f16* t, int c0, int k0, int lane) {
  const int i = lane & 15, r = k0 + 4 * (lane >> 4) + (i >> 2), c = c0 + 4 * (i & 3);
  const i16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(t + HTile<W>::at(r, c)));
  const i16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(t + HTile<W>::at(r + 16, c)));
  return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int CTRL> __device__ __forceinline__ float max_dpp(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)));
}
// The largest of a value over the lanes of a column (l % 16), and over the wave, in every lane.
__device__ __forceinline__ float col_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row16_max(float v) {
  return max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(v))));
}
__device__ __forceinline__ float wave_max(float v) { return col_max(row16_max(v)); }

// The power of two s (`inv`) with amax / s in [2^12, 2^13), and 1 / s (`mult`).  A maximum below 2^-114 is taken as that;
// an infinity stays one in every part, so that it reaches the results.
struct Scale {
  float mult, inv;
  __device__ __forceinline__ explicit Scale(float amax) {
    const int e = max((int)(__float_as_uint(amax) >> 23) & 0xff, 13);
    mult = __uint_as_float((uint32_t)(266 - e) << 23);
    inv = __uint_as_float((uint32_t)(e - 12) << 23);
  }
};
__device__ __forceinline__ f16 part_hi(float x, float mult) { return (f16)(x * mult); }
__device__ __forceinline__ f16 part_lo(float x, float mult, f16 hi) { return (f16)__builtin_fmaf(x, mult, -(float)hi); }

// B operand of k-step c from accumulator tiles 2 c and 2 c + 1 (rows 32 c .. 32 c + 31), on a scale of the lane's column.
// `zero` is a 0 that the compiler does not see through: x mult + 0 rounded to fp16 is one instruction, the product alone
// one and a half.
template <int PLANES, int N>
__device__ __forceinline__ void parts_of(const f32x4 (&t)[N], float mult, f16x8 (&hi)[N / 2], f16x8 (&lo)[N / 2]) {
  float zero = 0.f;
  asm volatile("" : "+v"(zero));
#pragma unroll
  for (int c = 0; c < N / 2; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = t[2 * c + (j >> 2)][j & 3];
      hi[c][j] = (f16)__builtin_fmaf(x, mult, zero);
      if constexpr (PLANES == 2) lo[c][j] = part_lo(x, mult, hi[c][j]);
    }
}
template <int N>
__device__ __forceinline__ float abs_max(const f32x4 (&t)[N], float m = 0.f) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(t[i][r]));
  return m;
}

// A gate's logarithm as the kernels take it: e^-200 is 0 in fp32 as e^-inf is, and sums of it stay finite.
__device__ __forceinline__ float gate_log(float g) { return g < -200.f ? -200.f : g; }

// Inclusive sums over the wave's 64 lanes in fp64 (differences of sums keep fp32's precision however far the sums went), by
// the row shifts and broadcasts of wave_incl_scan_dpp on both halves of a value.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan64(double v) {
  v = add_dpp64<0x111, 0xf>(v);
  v = add_dpp64<0x112, 0xf>(v);
  v = add_dpp64<0x114, 0xf>(v);
  v = add_dpp64<0x118, 0xf>(v);
  v = add_dpp64<0x142, 0xa>(v);
  return add_dpp64<0x143, 0xc>(v);
}
__device__ __forceinline__ double last_lane64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// e^x for x log2 e in fp64 (sums of gates are kept so): v_exp_f32, 1 ulp, of its nearest fp32.
constexpr double kLog2e64 = 1.4426950408889634;
__device__ __forceinline__ float exp_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

// ------------------------------------------------------------------ workspace
// Operands are kept as the instructions take them, a fragment of 64 lanes x 8 values (1 KB) after the other, so that they
// are read by 16 bytes a lane without conflicts, and the scans need no transposing reads.
//   For each (batch, key head, piece), NP parts of each: Q by rows (i KS + s: rows 16 i .., k-step s), K by rows, K by
//     columns (2 n + s: channels 16 n .., tokens 32 s ..), and for the backward Q by columns.
//   For each (batch, value head, piece): T by rows in two parts (its 6 fragments that are not zero), P by rows in two parts,
//     then for the backward T and P by columns in two parts each.
//   `vec` for the same: e^{G_t}, beta_t e^{G_end - G_t}, then e^{G_end} and the scales of T, P, K and Q.
//   For the backward, for each (batch, value head, piece, 16 columns of v): the entering state and delta, two parts each,
//     in the order in which waves hold them as operands ([part][k-step]), and the scales of their columns in either half
//     of the rows ([half][which][column]).  In a room of their own (DeltaScratch), as only the backward writes them: the
//     state's gradient behind the piece and y in the same way, and the scales of dO's columns behind theirs.
constexpr int FR = 512;                          // halfs of a fragment
template <int DKP> constexpr int kKFrags = DKP / 8;                    // of K or Q, rows or columns
constexpr int kTFrags = 6;
__device__ __forceinline__ constexpr int t_frag(int i, int s) { return s ? 2 + i : i; }      // by rows: i >= 2 s
__device__ __forceinline__ constexpr int tt_frag(int i, int s) { return 2 * s + i; }         // by columns: i < 2 + 2 s
__device__ __forceinline__ f16x8 frag(const f16* t, int f, int lane) { return *reinterpret_cast<const f16x8*>(t + f * FR + lane * 8); }
__device__ __forceinline__ void put_frag(f16* t, int f, int lane, f16x8 v) { *reinterpret_cast<f16x8*>(t + f * FR + lane * 8) = v; }

constexpr int kVecFloats = 256;
enum { VEC_W = 64, VEC_GAMMA = 128, VEC_ST, VEC_SP, VEC_SK, VEC_SQ };
constexpr int kScales = 64, kGradScales = 80;    // floats
template <int DKP> constexpr int keep_halfs() { return 2 * 16 * DKP + 2 * 16 * DC; }
template <int DKP> constexpr int kTokens = 2 * 16 * DKP;               // where delta and y begin, behind the states
// k-steps s0 .. s0 + N - 1 of ALL.
template <int ALL, int N>
__device__ __forceinline__ void keep_parts(f16* to, int s0, const f16x8 (&hi)[N], const f16x8 (&lo)[N], int lane) {
#pragma unroll
  for (int s = 0; s < N; ++s) {
    put_frag(to, s0 + s, lane, hi[s]);
    put_frag(to, ALL + s0 + s, lane, lo[s]);
  }
}

int delta_segments(const DeltaParams& p);        // how many a sequence is scanned in
constexpr int64_t kCUs = 256;                    // a workgroup of a scan fills one
// bf16: pairs of waves in workgroups of their own where every one of them has a CU to itself.
inline bool delta_one_pair(const DeltaParams& p, int segs) { return (int64_t)p.batch * p.heads * segs * ((p.dv + 15) / 16) <= kCUs; }
// A scan's workgroup: pairs, and for bf16 a wave that fetches and one for each 32 columns of v.
template <int PAIRS> constexpr int kIoWaves = PAIRS == 4 ? 2 : 1;
template <int PAIRS> constexpr int kIoCols = PAIRS == 1 ? 16 : 32;
template <typename T, int PAIRS> constexpr int kDeltaThreads = 64 * (2 * PAIRS + (sizeof(T) == 4 ? 0 : 1 + kIoWaves<PAIRS>));

struct DeltaLayout {
  size_t kq, tp, vec, keep, scales, total;       // byte offsets
  size_t kq_unit, tp_unit;                       // bytes of a piece
  size_t seg_states, seg_trans;                  // of segments, each (batch, head, segment)
  int segs, per;                                 // segments, pieces of one
  __host__ DeltaLayout(const DeltaParams& p, bool backward) {
    const size_t np = p.dtype == DT_F32 ? 2 : 1, dkp = p.dk <= 64 ? 64 : 128;
    const size_t kpieces = (size_t)p.batch * p.kheads * p.pieces, pieces = (size_t)p.batch * p.heads * p.pieces;
    const size_t blocks = backward ? pieces * ((p.dv + 15) / 16) : 0;
    kq_unit = (backward ? 4 : 3) * np * (dkp / 8) * FR * 2;
    tp_unit = (backward ? 8 : 4) * kTFrags * FR * 2;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t was = at; at += (bytes + 1023) / 1024 * 1024; return was; };
    kq = take(kpieces * kq_unit);
    tp = take(pieces * tp_unit);
    vec = take(pieces * kVecFloats * 4);
    keep = take(blocks * (dkp == 64 ? keep_halfs<64>() : keep_halfs<128>()) * 2);
    scales = take(blocks * kScales * 4);
    segs = delta_segments(p);
    per = (p.pieces + segs - 1) / segs;
    const size_t units = segs > 1 ? (size_t)p.batch * p.heads * segs : 0;
    seg_states = take(units * p.dk * p.dv * 4);
    seg_trans = take(units * dkp * dkp * 4);
    total = at;
  }
};
struct DeltaScratch {
  size_t keep, scales, total;
  __host__ explicit DeltaScratch(const DeltaParams& p) {
    const size_t blocks = (size_t)p.batch * p.heads * p.pieces * ((p.dv + 15) / 16);
    keep = 0;
    scales = (blocks * (p.dk <= 64 ? keep_halfs<64>() : keep_halfs<128>()) * 2 + 1023) / 1024 * 1024;
    total = scales + (blocks * kGradScales * 4 + 1023) / 1024 * 1024;
  }
};

// N fragments by LDS DMA, wave w of NW taking N / NW in a row.
typedef __attribute__((address_space(3))) f16 lds_f16_t;
template <int N, int NW>
__device__ __forceinline__ void fetch_share(lds_f16_t* to, const char* from, int w, int lane) {
  static_assert(N % NW == 0, "equal shares");
  const char* src = from + w * (N / NW) * 1024;
  lds_f16_t* dst = to + w * (N / NW) * FR;
  uint32_t off = 16u * lane;
  asm volatile("" : "+v"(off));                  // 32 bits beside a scalar base, not a 64-bit address held for the loop
#pragma unroll
  for (int i = 0; i < N / NW; ++i)
    __builtin_amdgcn_global_load_lds((glb_void_t*)(src + i * 1024 + off), (lds_void_t*)(dst + i * FR), 16, 0, 0);
}

// Lines of a later piece's fragments, read so that the L2 holds them when the waves that fetch ask: `wg` of `nwg` workgroups
// that want the same takes its share of A + B + 1 KB in blocks of 8 KB, a line a lane.  With a pair a workgroup, eight of
// which share 128 columns, that took the scan from 201 to 175 us (b 2, H 16, L 4096); with two pairs, whose share is twice as
// large and whose fetching waves are as busy, it cost 5 of 86 (b 4, H 16, L 2048), so that those go without.
struct Warm {
  static constexpr int N = 5;
  uint32_t x[N];
  template <int A, int B>
  __device__ __forceinline__ void load(const char* a, const char* b, const char* c, int wg, int nwg, int lane) {
    constexpr int NA = (A + 7) / 8, NB = (B + 7) / 8;
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = wg + nwg * i;
      x[i] = 0;
      if (j >= NA + NB + 1) continue;
      const char* from = j < NA ? a + j * 8192 : j < NA + NB ? b + (j - NA) * 8192 : c;
      const int lines = j < NA ? 8 * A - 64 * j : j < NA + NB ? 8 * B - 64 * (j - NA) : 8;
      x[i] = *reinterpret_cast<const uint32_t*>(from + 128u * min(lane, lines - 1));
    }
  }
  __device__ __forceinline__ void done() const {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" ::"v"(x[i]));
  }
};

// 32 rows of 16 columns in the accumulators' order: v[i] is row 16 (i / 4) + 4 g + i % 4 of column l % 16.  `at` is the
// first row at the first column; rows beyond `len` read the last one, or row 0 (their gates are zero), columns beyond the
// last one as 0.  A row's address is the wave's, one offset the lane's.
template <typename T>
__device__ __forceinline__ void load_rows8(const T* at, int64_t stride, int len, bool cv, bool all_cv, int l16, int g4, T (&v)[8]) {
  int c = cv ? l16 : 0;
  asm volatile("" : "+v"(c), "+v"(g4));          // addresses formed here, not held for the loop
  if (len >= 32) {
    const int64_t off = 4 * g4 * stride + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (at + (16 * (i >> 2) + (i & 3)) * stride)[off];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at[(int64_t)min(16 * (i >> 2) + 4 * g4 + (i & 3), len - 1) * stride + c];
  }
  if (!all_cv)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = cv ? v[i] : from_f32<T>(0.f);
}
template <typename T>
__device__ __forceinline__ void store_rows8(T* at, int64_t stride, int len, bool cv, int l16, int g4, const float (&v)[8]) {
  if (!cv) return;
  asm volatile("" : "+v"(l16), "+v"(g4));
  if (len >= 32) {
    const int64_t off = 4 * g4 * stride + l16;
#pragma unroll
    for (int i = 0; i < 8; ++i) (at + (16 * (i >> 2) + (i & 3)) * stride)[off] = from_f32<T>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 16 * (i >> 2) + 4 * g4 + (i & 3);
      if (r < len) at[(int64_t)r * stride + l16] = from_f32<T>(v[i]);
    }
  }
}

// 32 columns of a piece's rows by a wave that does nothing else, a token a lane, to and from LDS by columns
// ([column][token]), where the waves that compute read and write 4 tokens of a column at once.
constexpr int IO_PITCH = 68;                     // 34 banks a column: 16 columns of 8 bytes meet every bank once
template <int COLS> struct IoRows {
  bf16x8 v[COLS / 8];
  // `at`: column 0 of the lane's token, of which `left` columns exist; FULL: all of them, then without a branch, so that a
  // load stays under way until to_lds of the piece after next
  template <bool FULL>
  __device__ __forceinline__ void load(const bf16* at, int left) {
#pragma unroll
    for (int i = 0; i < COLS / 8; ++i) {
      Raw8<bf16> r;
      if constexpr (!FULL) r.clear();
      if (FULL || left > 8 * i) load_raw(r, at + 8 * i, FULL ? 8 : left - 8 * i);
      v[i] = r.v;
    }
  }
  template <bool FULL>
  __device__ __forceinline__ void store(bf16* at, bool row, int left) const {
    if (!row) return;
#pragma unroll
    for (int i = 0; i < COLS / 8; ++i) {
      if (FULL || left >= 8 * i + 8) put_vec<false>(at + 8 * i, v[i]);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (8 * i + j < left) at[8 * i + j] = v[i][j];
    }
  }
  __device__ __forceinline__ void to_lds(bf16* t, int lane) const {
#pragma unroll
    for (int c = 0; c < COLS; ++c) t[c * IO_PITCH + lane] = v[c / 8][c % 8];
  }
  __device__ __forceinline__ void zero_unless(bool row) {
#pragma unroll
    for (int i = 0; i < COLS / 8; ++i) v[i] = row ? v[i] : bf16x8{};
  }
  __device__ __forceinline__ void from_lds(const bf16* t, int lane) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) v[c / 8][c % 8] = t[c * IO_PITCH + lane];
  }
};

// Workgroup n of heads x blocks, with the blocks of a head on one XCD (workgroups go to the 8 XCDs in turn): they share the
// head's tiles through its L2.  False beyond the last head.
__device__ __forceinline__ bool head_block(int n, int heads, int blocks, int& head, int& block) {
  const int y = n >> 3;
  head = (y / blocks) * 8 + (n & 7);
  block = y % blocks;
  return head < heads;
}
inline unsigned head_block_grid(int heads, int blocks) { return (unsigned)((heads + 7) / 8 * 8 * blocks); }

}  // namespace mh
