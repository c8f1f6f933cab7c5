// Rotary positions: channel pairs (x0, x1) turned by the angle position * inv_freq[i], (x0 c - x1 s, x1 c + x0 s) * scale,
// the pairs being channels (i, n + i) or (2 i, 2 i + 1) of the first 2 n; the rest pass.  The turn by the negative angle is
// its gradient (and its inverse where scale is 1).
//
// Bound by the rows' bytes.  Angles: position * inv_freq / (2 pi) in fp64, three roundings of the whole angle (less than
// 2^-24 radians up to angles of 2^27), of which the fraction of a turn is left; then the sine and cosine of that many turns
// in fp32.  A thread computes those of its 8 pairs once, while its first heads' channels are under way, and runs through its share of the heads of queries and
// keys with them, four heads' loads at once (one at a time: 23.8 us).  b 2, 16 + 8 heads of 128, L 4096 in bf16: 21 us for
// 101 MB, 4.8 TB/s, of which the angles take about 3 before the first store.
#include "launch.h"
#include "rows.h"

namespace mh {
namespace {

constexpr int U = 4;                             // heads whose loads are under way at once

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, int chunks, int shares, int per) {
  const int64_t id = grid_row() * 256 + threadIdx.x;
  const int64_t units = (int64_t)p.batch * p.seqlen * chunks;
  const int share = blockIdx.y;
  if (id >= units) return;
  const int c = (int)(id % chunks);
  const int64_t tok = id / chunks;
  const int l = (int)(tok % p.seqlen), b = (int)(tok / p.seqlen);
  // chunks of 8 pairs first, then chunks of 8 channels that pass
  const int turning = (p.pairs + 7) / 8;
  const bool turn = c < turning;
  const int n = turn ? min(8, p.pairs - 8 * c) : 0;
  const int ch = turn ? (INTER ? 16 * c : 8 * c) : 2 * p.pairs + 8 * (c - turning);
  const int left0 = turn ? (INTER ? 2 * n : n) : p.dim - ch, off1 = turn ? (INTER ? 8 : p.pairs) : 0;
  const int left1 = turn ? (INTER ? 2 * n - 8 : n) : left0;            // a chunk that passes is read twice, written once
  const bool full = p.pairs % 8 == 0 && (p.dim - 2 * p.pairs) % 8 == 0;
  const int total = p.q_heads + p.k_heads, h0 = share * per, h1 = min(total, h0 + per);
  Raw8<T> a[U], e[U];
  auto load = [&](int h) {                       // of U heads
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hu = h + u;
      if (hu >= h1) break;
      const bool isq = hu < p.q_heads;
      const RotaryTensor& x = isq ? p.q : p.k;
      const T* in = reinterpret_cast<const T*>(x.in) + (isq ? hu : hu - p.q_heads) * x.in_s.h + b * x.in_s.b + l * x.in_s.l + ch;
      if (full) {
        a[u].load(in);
        e[u].load(in + off1);
      } else {
        load_raw(a[u], in, left0);
        load_raw(e[u], in + off1, left1);
      }
    }
  };
  load(h0);
  float cs[8], sn[8];
  if (turn) {
    const double pos = (double)((p.positions ? load_index(p.positions, p.i64, b * p.pos_sb + l) : (int64_t)l) + p.offset);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 8 * c + min(j, n - 1);
      const double f = p.freq64 ? reinterpret_cast<const double*>(p.inv_freq)[i] : (double)reinterpret_cast<const float*>(p.inv_freq)[i];
      const double r = pos * (f * 0.15915494309189535);
      float s, co;
      sincospif((float)(2.0 * (r - rint(r))), &s, &co);
      cs[j] = co * p.scale;
      sn[j] = (p.inverse ? -s : s) * p.scale;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j] = sn[j] = 0.f;
  }
  for (int h = h0; h < h1; h += U) {
    if (h != h0) load(h);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u >= h1) break;
      const bool isq = h + u < p.q_heads;
      const RotaryTensor& x = isq ? p.q : p.k;
      T* out = reinterpret_cast<T*>(x.out) + (isq ? h + u : h + u - p.q_heads) * x.out_s.h + b * x.out_s.b + l * x.out_s.l + ch;
      float y0[8], y1[8];
      if (INTER) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p0 = a[u].get(2 * j), p1 = a[u].get(2 * j + 1), r0 = e[u].get(2 * j), r1 = e[u].get(2 * j + 1);
          y0[2 * j] = p0 * cs[j] - p1 * sn[j];
          y0[2 * j + 1] = p1 * cs[j] + p0 * sn[j];
          y1[2 * j] = r0 * cs[4 + j] - r1 * sn[4 + j];
          y1[2 * j + 1] = r1 * cs[4 + j] + r0 * sn[4 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x0 = a[u].get(j), x1 = e[u].get(j);
          y0[j] = x0 * cs[j] - x1 * sn[j];
          y1[j] = x1 * cs[j] + x0 * sn[j];
        }
      }
      if (!turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y0[j] = a[u].get(j);
      }
      store8(out, left0, y0);
      if (turn && left1 > 0) store8(out + off1, left1, y1);
    }
  }
}

template <typename T>
hipError_t run(const RotaryParams& p, hipStream_t st) {
  const int chunks = (p.pairs + 7) / 8 + (p.dim - 2 * p.pairs + 7) / 8, total = p.q_heads + p.k_heads;
  const int64_t blocks = ((int64_t)p.batch * p.seqlen * chunks + 255) / 256;
  int shares = (int)((1024 + blocks - 1) / blocks);
  if (shares > total) shares = total;
  int per = (total + shares - 1) / shares;
  if (per > U) per = (per + U - 1) / U * U;
  shares = (total + per - 1) / per;
  const dim3 grid = row_grid(blocks, (unsigned)shares);
  if (p.interleaved) rotary_kernel<T, true><<<grid, 256, 0, st>>>(p, chunks, shares, per);
  else rotary_kernel<T, false><<<grid, 256, 0, st>>>(p, chunks, shares, per);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryParams& p, hipStream_t st) {
  return p.dtype == DT_F32 ? run<float>(p, st) : run<bf16>(p, st);
}

}  // namespace mh
