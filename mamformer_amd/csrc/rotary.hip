// Rotary positions: channel pairs (x0, x1) turned by the angle position * inv_freq[i], (x0 c - x1 s, x1 c + x0 s) * scale,
// the pairs being channels (i, n + i) or (2 i, 2 i + 1) of the first 2 n; the rest pass.  The turn by the negative angle is
// its gradient (and its inverse where scale is 1).
//
// Bound by the rows' bytes.  Angles: position * inv_freq / (2 pi) in fp64, of which the fraction of a turn is left, exact
// to fp32 for positions beyond 2^31 turns; then the sine and cosine of that many turns in fp32.  A thread computes those of
// its 8 pairs once and runs through its share of the heads of queries and keys with them.
#include "launch.h"
#include "rows.h"

namespace mh {
namespace {

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, int chunks, int shares, int per) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
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
  }
  const int total = p.q_heads + p.k_heads, h1 = min(total, (share + 1) * per);
  for (int h = share * per; h < h1; ++h) {
    const bool isq = h < p.q_heads;
    const RotaryTensor& x = isq ? p.q : p.k;
    const int64_t hh = isq ? h : h - p.q_heads;
    const T* in = reinterpret_cast<const T*>(x.in) + b * x.in_s.b + hh * x.in_s.h + l * x.in_s.l + ch;
    T* out = reinterpret_cast<T*>(x.out) + b * x.out_s.b + hh * x.out_s.h + l * x.out_s.l + ch;
    float a[8], e[8];
    if (!turn) {
      load8(in, p.dim - ch, a);
      store8(out, p.dim - ch, a);
    } else if (INTER) {
      load8(in, 2 * n, a);
      if (n > 4) load8(in + 8, 2 * n - 8, e);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x0 = a[2 * j], x1 = a[2 * j + 1];
        a[2 * j] = x0 * cs[j] - x1 * sn[j];
        a[2 * j + 1] = x1 * cs[j] + x0 * sn[j];
      }
      store8(out, 2 * n, a);
      if (n > 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x0 = e[2 * j], x1 = e[2 * j + 1];
          e[2 * j] = x0 * cs[4 + j] - x1 * sn[4 + j];
          e[2 * j + 1] = x1 * cs[4 + j] + x0 * sn[4 + j];
        }
        store8(out + 8, 2 * n - 8, e);
      }
    } else {
      load8(in, n, a);
      load8(in + p.pairs, n, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x0 = a[j], x1 = e[j];
        a[j] = x0 * cs[j] - x1 * sn[j];
        e[j] = x1 * cs[j] + x0 * sn[j];
      }
      store8(out, n, a);
      store8(out + p.pairs, n, e);
    }
  }
}

template <typename T>
hipError_t run(const RotaryParams& p, hipStream_t st) {
  const int chunks = (p.pairs + 7) / 8 + (p.dim - 2 * p.pairs + 7) / 8, total = p.q_heads + p.k_heads;
  const int64_t blocks = ((int64_t)p.batch * p.seqlen * chunks + 255) / 256;
  int shares = (int)((1024 + blocks - 1) / blocks);
  if (shares > total) shares = total;
  const int per = (total + shares - 1) / shares;
  shares = (total + per - 1) / per;
  const dim3 grid((unsigned)blocks, (unsigned)shares);
  if (p.interleaved) rotary_kernel<T, true><<<grid, 256, 0, st>>>(p, chunks, shares, per);
  else rotary_kernel<T, false><<<grid, 256, 0, st>>>(p, chunks, shares, per);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryParams& p, hipStream_t st) {
  return p.dtype == DT_F32 ? run<float>(p, st) : run<bf16>(p, st);
}

}  // namespace mh
