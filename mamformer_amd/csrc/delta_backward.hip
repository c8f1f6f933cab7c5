// Backward of the gated delta rule (delta_scan.hip has the forward and its names).  With dS the gradient of the state
// behind a piece:
//   ddelta = scale P^T dO + (beta e^{G_end - G} K) dS,   y = T^T ddelta = dV
//   dS_before = e^{G_end} dS + scale (e^G Q)^T dO - (e^G K)^T y
// which is the forward's recurrence run backwards (delta_back_scan_kernel: the gradient of 16 columns of the state in a
// wave's registers).  What is left of a piece needs nothing of its neighbours (delta_grads_kernel):
//   A' = -y delta^T (j < t),  P' = scale dO delta^T (j <= t),  D_tj = e^{G_t - G_j}
//   dQ = scale e^G dO S^T + (P' D beta) K
//   dK = [-e^G y S^T + (A' D beta) K] + [beta e^{G_end - G} delta dS^T + (A' D beta)^T K + (P' D beta)^T Q]
//   dbeta_j = sum_t D_tj (A'_tj k_t k_j + P'_tj q_t k_j) + e^{G_end - G_j} k_j (dS delta_j)
//   dG_t = q_t dQ_t + k_t dK_t[left] - k_t dK_t[right], at the piece's end + e^{G_end} <S, dS> + sum_j k_j (right's first
//   term)_j; dg is the sum of dG from t to the end.  The pair terms of q dQ and k dK are taken from the rows and columns of
//   A' and P' themselves, in fp32.
// The forward's states are computed again rather than kept: b L H (dk dv) / 64 of them are twice the size of q, k and v.
#include "delta.h"

namespace mh {
namespace {

template <typename T, int DKP, int NW>
__global__ __launch_bounds__(64 * NW) void delta_back_scan_kernel(DeltaBwdParams q, DeltaLayout lay, int nblk, int nwg) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int NBUF = NP == 1 ? 2 : 1;
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int KQ = 2 * NP * TK::ELEMS, TP = 4 * TC::ELEMS, BUF = KQ + TP + kVecFloats * 2;
  constexpr int NS = DKP / 16, KS = DKP / 32;
  __shared__ __align__(1024) f16 smem[NBUF * BUF];
  const DeltaParams& p = q.f;

  const int lane = threadIdx.x & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  int bh, wg;
  if (!head_block(blockIdx.x, p.batch * p.heads, nwg, bh, wg)) return;
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kheads);
  const int blk = wg * NW + w, col = 16 * blk + l16;
  const bool live = blk < nblk, cv = col < p.dv;
  const int64_t kunit0 = ((int64_t)b * p.kheads + hk) * p.pieces, vunit0 = (int64_t)bh * p.pieces;

  auto fetch = [&](int c, int buf) {
    char* to = reinterpret_cast<char*>(smem + buf * BUF);
    const char* kq = p.workspace + lay.kq + (kunit0 + c) * (int64_t)(KQ * 2);
    const char* tp = p.workspace + lay.tp + (vunit0 + c) * (int64_t)(TP * 2);
    const char* vec = p.workspace + lay.vec + (vunit0 + c) * (int64_t)(kVecFloats * 4);
#pragma unroll
    for (int i = w; i < KQ / 512; i += NW) dma_lds<16>(kq + i * 1024, 16u * lane, to + i * 1024);
#pragma unroll
    for (int i = w; i < TP / 512; i += NW) dma_lds<16>(tp + i * 1024, 16u * lane, to + KQ * 2 + i * 1024);
    if (w == 0) dma_lds<16>(vec, 16u * lane, to + (KQ + TP) * 2);
  };

  f32x4 dS[NS];
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * n + 4 * g4 + r;
      dS[n][r] = q.d_final_state && cv && row < p.dk ? q.d_final_state[((int64_t)bh * p.dk + row) * p.dv + col] : 0.f;
    }
  const T* osrc = reinterpret_cast<const T*>(q.d_o) + b * q.dos.b + h * q.dos.h + col;
  T on[16];
  auto load_o = [&](int c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = c * DC + 16 * (i >> 2) + 4 * g4 + (i & 3);
      on[i] = cv && t < p.seqlen ? osrc[(int64_t)t * q.dos.l] : from_f32<T>(0.f);
    }
  };
  load_o(p.pieces - 1);
  if (NBUF == 2) fetch(p.pieces - 1, (p.pieces - 1) & 1);

  for (int c = p.pieces - 1; c >= 0; --c) {
    const f16* buf = smem + (NBUF == 2 ? (c & 1) * BUF : 0);
    if (NBUF == 2) {
      wait_vmem();
      __syncthreads();
      if (c > 0) fetch(c - 1, (c - 1) & 1);
    } else {
      __syncthreads();
      fetch(c, 0);
      wait_vmem();
      __syncthreads();
    }
    if (!live) continue;
    const f16 *Kt = buf, *Qt = buf + NP * TK::ELEMS, *Tt = buf + KQ, *Pt = Tt + 2 * TC::ELEMS;
    const float* vec = reinterpret_cast<const float*>(buf + KQ + TP);
    f32x4 U[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) U[i >> 2][i & 3] = to_f32(on[i]);
    if (c > 0) load_o(c - 1);

    const int64_t at = (vunit0 + c) * nblk + blk;
    f16* keep = reinterpret_cast<f16*>(p.workspace + lay.keep) + at * (int64_t)keep_halfs<DKP>();
    float* scales = reinterpret_cast<float*>(p.workspace + lay.scales) + at * 4;
    f16x8 sh[KS], sl[KS];
    const Scale ss(wave_max(abs_max(dS)));
    parts_of<2>(dS, ss.mult, sh, sl);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f16* to = keep + 2 * 16 * DKP + l16 * DKP + 16 * n + 4 * g4;
      *reinterpret_cast<f16x4*>(to) = n & 1 ? __builtin_shufflevector(sh[n >> 1], sh[n >> 1], 4, 5, 6, 7)
                                            : __builtin_shufflevector(sh[n >> 1], sh[n >> 1], 0, 1, 2, 3);
      *reinterpret_cast<f16x4*>(to + 16 * DKP) = n & 1 ? __builtin_shufflevector(sl[n >> 1], sl[n >> 1], 4, 5, 6, 7)
                                                       : __builtin_shufflevector(sl[n >> 1], sl[n >> 1], 0, 1, 2, 3);
    }
    if (lane == 0) scales[KEEP_DS] = ss.inv;
    // K dS
    f32x4 X[4] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f16x8 a = row_frag16<DKP>(Kt, 16 * i, 32 * s, lane);
        X[i] = mma_h(a, sh[s], X[i]);
        X[i] = mma_h(a, sl[s], X[i]);
        if constexpr (NP == 2) X[i] = mma_h(row_frag16<DKP>(Kt + TK::ELEMS, 16 * i, 32 * s, lane), sh[s], X[i]);
      }
    // P^T dO
    f16x8 oh[2], ol[2];
    const Scale so(wave_max(abs_max(U)));
    parts_of<NP>(U, so.mult, oh, ol);
    f32x4 Z[4] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 2 + 2 * s; ++i) {
        const f16x8 a = col_frag16<64>(Pt, 16 * i, 32 * s, lane);
        Z[i] = mma_h(a, oh[s], Z[i]);
        if constexpr (NP == 2) Z[i] = mma_h(a, ol[s], Z[i]);
        Z[i] = mma_h(col_frag16<64>(Pt + TC::ELEMS, 16 * i, 32 * s, lane), oh[s], Z[i]);
      }
    const float zs = p.scale * (so.inv * vec[VEC_SP]), xs = ss.inv * vec[VEC_SK];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 wt = *reinterpret_cast<const f32x4*>(vec + VEC_W + 16 * i + 4 * g4);
#pragma unroll
      for (int r = 0; r < 4; ++r) Z[i][r] = zs * Z[i][r] + wt[r] * (xs * X[i][r]);
    }
    // y = T^T ddelta
    f16x8 zh[2], zl[2];
    const Scale sz(wave_max(abs_max(Z)));
    parts_of<2>(Z, sz.mult, zh, zl);
    f32x4 Y[4] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 2 + 2 * s; ++i) {
        const f16x8 a = col_frag16<64>(Tt, 16 * i, 32 * s, lane);
        Y[i] = mma_h(a, zh[s], Y[i]);
        Y[i] = mma_h(a, zl[s], Y[i]);
        Y[i] = mma_h(col_frag16<64>(Tt + TC::ELEMS, 16 * i, 32 * s, lane), zh[s], Y[i]);
      }
    const float ysc = sz.inv * vec[VEC_ST];
    T* dv = reinterpret_cast<T*>(q.dv) + b * q.dvs.b + h * q.dvs.h + col;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float y = Y[i >> 2][i & 3] *= ysc;
      const int t = c * DC + 16 * (i >> 2) + 4 * g4 + (i & 3);
      if (cv && t < p.seqlen) dv[(int64_t)t * q.dvs.l] = from_f32<T>(y);
    }
    f16x8 yh[2], yl[2];
    const Scale sy(wave_max(abs_max(Y)));
    parts_of<2>(Y, sy.mult, yh, yl);
    {
      f16* to = keep + 2 * (2 * 16 * DKP) + 2 * 16 * DC + l16 * DC + 4 * g4;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        *reinterpret_cast<f16x4*>(to + 16 * n) = n & 1 ? __builtin_shufflevector(yh[n >> 1], yh[n >> 1], 4, 5, 6, 7)
                                                       : __builtin_shufflevector(yh[n >> 1], yh[n >> 1], 0, 1, 2, 3);
        *reinterpret_cast<f16x4*>(to + 16 * DC + 16 * n) = n & 1 ? __builtin_shufflevector(yl[n >> 1], yl[n >> 1], 4, 5, 6, 7)
                                                                 : __builtin_shufflevector(yl[n >> 1], yl[n >> 1], 0, 1, 2, 3);
      }
      if (lane == 0) scales[KEEP_Y] = sy.inv;
    }
    // the gradient before the piece: both terms on one scale, those of Q's and K's parts in it
    const float uq = p.scale * vec[VEC_SQ], uk = -vec[VEC_SK];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 eg = *reinterpret_cast<const f32x4*>(vec + 16 * i + 4 * g4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        U[i][r] *= uq * eg[r];
        Y[i][r] *= uk * eg[r];
      }
    }
    const Scale su(wave_max(abs_max(Y, abs_max(U))));
    parts_of<2>(U, su.mult, oh, ol);
    parts_of<2>(Y, su.mult, yh, yl);
    const float gamma = vec[VEC_GAMMA];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x4 u = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 a = col_frag16<DKP>(Qt, 16 * n, 32 * s, lane), k = col_frag16<DKP>(Kt, 16 * n, 32 * s, lane);
        u = mma_h(a, oh[s], u);
        u = mma_h(a, ol[s], u);
        u = mma_h(k, yh[s], u);
        u = mma_h(k, yl[s], u);
        if constexpr (NP == 2) {
          u = mma_h(col_frag16<DKP>(Qt + TK::ELEMS, 16 * n, 32 * s, lane), oh[s], u);
          u = mma_h(col_frag16<DKP>(Kt + TK::ELEMS, 16 * n, 32 * s, lane), yh[s], u);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) dS[n][r] = gamma * dS[n][r] + su.inv * u[r];
    }
  }
  if (q.d_initial_state && live && cv) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * n + 4 * g4 + r;
        if (row < p.dk) q.d_initial_state[((int64_t)bh * p.dk + row) * p.dv + col] = dS[n][r];
      }
  }
}

// One workgroup of 4 waves for a piece of a key head, its value heads one after the other (their dQ and dK are added in
// that order).  Wave w holds rows 16 w .. 16 w + 15 of the three products with the states (64 x dk) and of A' and P'.  The
// columns of v pass through LDS DVB at a time, every matrix brought to one scale on the way (the wave's 16 columns that
// made it had their own).
template <typename T, int DKP>
__global__ __launch_bounds__(256) void delta_grads_kernel(DeltaBwdParams q, DeltaLayout lay, int nblk) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int DVB = NP == 1 ? 64 : 32;
  constexpr int NS = DKP / 16;
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int SE = DVB * DKP, YE = DVB * 64;   // elements of a part of S / dS and of delta / y
  static_assert(4 * SE + 4 * YE >= 2 * NP * TC::ELEMS, "the pair terms take the place of the states, delta and y");
  __shared__ __align__(1024) f16 smem[4 * SE + 4 * YE + NP * TC::ELEMS + 2 * NP * TK::ELEMS];
  f16 *sS = smem, *sN = sS + 2 * SE, *sY = sN + 2 * SE, *sD = sY + 2 * YE, *sO = sD + 2 * YE, *sKQ = sO + NP * TC::ELEMS;
  f16 *sXa = smem, *sXp = smem + NP * TC::ELEMS;                       // where those were
  __shared__ double sG[DC];
  __shared__ float sB[DC], sEG[DC], sEnd[DC], sRow[DC], sH[DC], sB2[DC], sCol[4][DC], red[4][4];
  const DeltaParams& p = q.f;

  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  const int64_t unit = blockIdx.x;
  const int c = (int)(unit % p.pieces), bk = (int)(unit / p.pieces), hk = bk % p.kheads, b = bk / p.kheads;
  const int t0 = c * DC, len = min(DC, p.seqlen - t0), rep = p.heads / p.kheads;
  {
    const uint4* kq = reinterpret_cast<const uint4*>(p.workspace + lay.kq) + unit * (2 * NP * TK::ELEMS / 8);
    for (int i = tid; i < 2 * NP * TK::ELEMS / 8; i += 256) reinterpret_cast<uint4*>(sKQ)[i] = kq[i];
  }
  const f16 *Kt = sKQ, *Qt = sKQ + NP * TK::ELEMS;
  const float* vec0 = reinterpret_cast<const float*>(p.workspace + lay.vec) +
                      (((int64_t)b * p.heads + hk * rep) * p.pieces + c) * kVecFloats;
  const float sk = vec0[VEC_SK], sq = vec0[VEC_SQ];
  __syncthreads();
  auto value = [&](const f16* t, int r, int col) {                     // K or Q without its scale
    float v = (float)t[TK::at(r, col)];
    if constexpr (NP == 2) v += (float)t[TK::ELEMS + TK::at(r, col)];
    return v;
  };
  f32x4 kk[4] = {}, qk[4] = {};
#pragma unroll
  for (int s = 0; s < DKP / 32; ++s) {
    f16x8 ka[NP], qa[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      ka[n] = row_frag16<DKP>(Kt + n * TK::ELEMS, 16 * w, 32 * s, lane);
      qa[n] = row_frag16<DKP>(Qt + n * TK::ELEMS, 16 * w, 32 * s, lane);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w) continue;
      const f16x8 kb = row_frag16<DKP>(Kt, 16 * j, 32 * s, lane);
      kk[j] = mma_h(ka[0], kb, kk[j]);
      qk[j] = mma_h(qa[0], kb, qk[j]);
      if constexpr (NP == 2) {
        const f16x8 kl = row_frag16<DKP>(Kt + TK::ELEMS, 16 * j, 32 * s, lane);
        kk[j] = mma_h(ka[0], kl, kk[j]);
        kk[j] = mma_h(ka[1], kb, kk[j]);
        qk[j] = mma_h(qa[0], kl, qk[j]);
        qk[j] = mma_h(qa[1], kb, qk[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      kk[j][r] = kk[j][r] * sk * sk;
      qk[j][r] = qk[j][r] * sq * sk;
    }

  f32x4 tq[NS] = {}, tk[NS] = {};                // dQ and dK over the value heads
  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const int64_t vunit = ((int64_t)b * p.heads + h) * p.pieces + c;
    const T* osrc = reinterpret_cast<const T*>(q.d_o) + b * q.dos.b + h * q.dos.h + (int64_t)t0 * q.dos.l;
    // dO's largest magnitude, the matrices' scales
    float om = 0.f;
    for (int u = tid; u < len * ((p.dv + 7) / 8); u += 256) {
      const int r = u / ((p.dv + 7) / 8), c8 = u % ((p.dv + 7) / 8) * 8;
      float v[8];
      load8(osrc + r * q.dos.l + c8, p.dv - c8, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) om = fmaxf(om, fabsf(v[j]));
    }
    om = wave_max(om);
    const float* scales = reinterpret_cast<const float*>(p.workspace + lay.scales) + vunit * nblk * 4;
    float mx[4] = {};
    for (int i = 0; i < nblk; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx[j] = fmaxf(mx[j], scales[4 * i + j]);
    __syncthreads();                             // the last head's use of the LDS is over
    if (lane == 0) red[w][0] = om;
    if (w == 0) {
      float gv = 0.f, bv = 0.f;
      if (lane < len) {
        if (p.g) gv = gate_log(p.g[b * p.gs.b + h * p.gs.h + (int64_t)(t0 + lane) * p.gs.l]);
        bv = p.beta ? p.beta[b * p.bs.b + h * p.bs.h + (int64_t)(t0 + lane) * p.bs.l] : 1.f;
      }
      const double G = wave_scan64((double)gv);
      const double end = __shfl(G, 63);
      sG[lane] = G;
      sB[lane] = bv;
      sEG[lane] = expf((float)G);
      sEnd[lane] = expf((float)(end - G));
    }
    __syncthreads();
    const Scale so(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
    const float mS = mx[KEEP_S], mN = mx[KEEP_DS], mD = mx[KEEP_D], mY = mx[KEEP_Y];

    f32x4 aq[NS] = {}, al[NS] = {}, ar[NS] = {}, pA[4] = {}, pP[4] = {};
    float dot = 0.f;                             // <S, dS>
    const f16* keep0 = reinterpret_cast<const f16*>(p.workspace + lay.keep) + vunit * nblk * (int64_t)keep_halfs<DKP>();
    for (int v0 = 0; v0 < 16 * nblk; v0 += DVB) {
      if (v0) __syncthreads();
      for (int u = tid; u < SE / 8; u += 256) {
        const int r = u / (DKP / 8), c8 = u % (DKP / 8) * 8, blk = (v0 + r) / 16;
        f16x8 s0 = {}, s1 = {}, n0 = {}, n1 = {};
        if (blk < nblk) {
          const f16* from = keep0 + blk * (int64_t)keep_halfs<DKP>() + (r & 15) * DKP + c8;
          s0 = *reinterpret_cast<const f16x8*>(from);
          s1 = *reinterpret_cast<const f16x8*>(from + 16 * DKP);
          n0 = *reinterpret_cast<const f16x8*>(from + 32 * DKP);
          n1 = *reinterpret_cast<const f16x8*>(from + 48 * DKP);
          const float fs = scales[4 * blk + KEEP_S], fn = scales[4 * blk + KEEP_DS];
          float d = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) d += ((float)s0[j] + (float)s1[j]) * ((float)n0[j] + (float)n1[j]);
          dot += d * fs * fn;
          const f16 hs = (f16)(fs / mS), hn = (f16)(fn / mN);          // powers of two, at most 1
          s0 *= hs;
          s1 *= hs;
          n0 *= hn;
          n1 *= hn;
        }
        const int at = TK::at(r, c8);
        *reinterpret_cast<f16x8*>(sS + at) = s0;
        *reinterpret_cast<f16x8*>(sS + SE + at) = s1;
        *reinterpret_cast<f16x8*>(sN + at) = n0;
        *reinterpret_cast<f16x8*>(sN + SE + at) = n1;
      }
      for (int u = tid; u < YE / 8; u += 256) {
        const int r = u / 8, c8 = u % 8 * 8, blk = (v0 + r) / 16;
        f16x8 d0 = {}, d1 = {}, y0 = {}, y1 = {};
        if (blk < nblk) {
          const f16* from = keep0 + blk * (int64_t)keep_halfs<DKP>() + 64 * DKP + (r & 15) * DC + c8;
          const f16 hd = (f16)(scales[4 * blk + KEEP_D] / mD), hy = (f16)(scales[4 * blk + KEEP_Y] / mY);
          d0 = *reinterpret_cast<const f16x8*>(from) * hd;
          d1 = *reinterpret_cast<const f16x8*>(from + 16 * DC) * hd;
          y0 = *reinterpret_cast<const f16x8*>(from + 32 * DC) * hy;
          y1 = *reinterpret_cast<const f16x8*>(from + 48 * DC) * hy;
        }
        const int at = TC::at(r, c8);
        *reinterpret_cast<f16x8*>(sD + at) = d0;
        *reinterpret_cast<f16x8*>(sD + YE + at) = d1;
        *reinterpret_cast<f16x8*>(sY + at) = y0;
        *reinterpret_cast<f16x8*>(sY + YE + at) = y1;
      }
      for (int u = tid; u < DC * DVB / 8; u += 256) {
        const int r = u / (DVB / 8), c8 = u % (DVB / 8) * 8;
        float v[8] = {};
        if (r < len && v0 + c8 < p.dv) load8(osrc + r * q.dos.l + v0 + c8, p.dv - v0 - c8, v);
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hi[j] = part_hi(v[j], so.mult);
          if constexpr (NP == 2) lo[j] = part_lo(v[j], so.mult, hi[j]);
        }
        *reinterpret_cast<f16x8*>(sO + TC::at(r, c8)) = hi;
        if constexpr (NP == 2) *reinterpret_cast<f16x8*>(sO + TC::ELEMS + TC::at(r, c8)) = lo;
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < DVB / 32; ++s) {
        const f16x8 o0 = row_frag16<64>(sO, 16 * w, 32 * s, lane);
        f16x8 o1;
        if constexpr (NP == 2) o1 = row_frag16<64>(sO + TC::ELEMS, 16 * w, 32 * s, lane);
        const f16x8 y0 = col_frag16<64>(sY, 16 * w, 32 * s, lane), y1 = col_frag16<64>(sY + YE, 16 * w, 32 * s, lane);
        const f16x8 d0 = col_frag16<64>(sD, 16 * w, 32 * s, lane), d1 = col_frag16<64>(sD + YE, 16 * w, 32 * s, lane);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const f16x8 b0 = col_frag16<DKP>(sS, 16 * n, 32 * s, lane), b1 = col_frag16<DKP>(sS + SE, 16 * n, 32 * s, lane);
          aq[n] = mma_h(o0, b0, aq[n]);
          aq[n] = mma_h(o0, b1, aq[n]);
          if constexpr (NP == 2) aq[n] = mma_h(o1, b0, aq[n]);
          al[n] = mma_h(y0, b0, al[n]);
          al[n] = mma_h(y0, b1, al[n]);
          al[n] = mma_h(y1, b0, al[n]);
          const f16x8 n0 = col_frag16<DKP>(sN, 16 * n, 32 * s, lane), n1 = col_frag16<DKP>(sN + SE, 16 * n, 32 * s, lane);
          ar[n] = mma_h(d0, n0, ar[n]);
          ar[n] = mma_h(d0, n1, ar[n]);
          ar[n] = mma_h(d1, n0, ar[n]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j > w) continue;
          const f16x8 b0 = col_frag16<64>(sD, 16 * j, 32 * s, lane), b1 = col_frag16<64>(sD + YE, 16 * j, 32 * s, lane);
          pA[j] = mma_h(y0, b0, pA[j]);
          pA[j] = mma_h(y0, b1, pA[j]);
          pA[j] = mma_h(y1, b0, pA[j]);
          pP[j] = mma_h(o0, b0, pP[j]);
          pP[j] = mma_h(o0, b1, pP[j]);
          if constexpr (NP == 2) pP[j] = mma_h(o1, b0, pP[j]);
        }
      }
    }
    // A' and P', what they give dbeta and dG, and the pair terms' matrices
    const float fA = -(mY * mD), fP = p.scale * (so.inv * mD);
    float rows[4] = {}, xam = 0.f, xpm = 0.f;
    double Gt[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) Gt[r] = sG[16 * w + 4 * g4 + r];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float colb = 0.f;
      if (j <= w) {
        const double Gj = sG[16 * j + l16];
        const float bj = sB[16 * j + l16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int below = 16 * (w - j) + 4 * g4 + r - l16;
          const float d = below >= 0 ? expf((float)(Gt[r] - Gj)) : 0.f;
          const float xa = below > 0 ? fA * pA[j][r] * d : 0.f, xp = below >= 0 ? fP * pP[j][r] * d : 0.f;
          const float m = (below > 0 ? xa * kk[j][r] : 0.f) + (below >= 0 ? xp * qk[j][r] : 0.f);
          colb += m;
          rows[r] += m * bj;
          pA[j][r] = xa * bj;
          pP[j][r] = xp * bj;
          xam = fmaxf(xam, fabsf(pA[j][r]));
          xpm = fmaxf(xpm, fabsf(pP[j][r]));
        }
      }
      colb += __shfl_xor(colb, 16);
      colb += __shfl_xor(colb, 32);
      if (g4 == 0) sCol[w][16 * j + l16] = colb;
    }
    xam = wave_max(xam);
    xpm = wave_max(xpm);
    dot = group_sum<64>(dot);
    if (lane == 0) {
      red[w][1] = xam;
      red[w][2] = xpm;
      red[w][3] = dot;
    }
    const float fq = p.scale * (so.inv * mS), fl = -(mY * mS), fr = mD * mN;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * w + 4 * g4 + r;
      float dq = 0.f, dl = 0.f, dr = 0.f;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const float kv = value(Kt, t, 16 * n + l16), qv = value(Qt, t, 16 * n + l16);
        aq[n][r] *= fq * sEG[t];
        al[n][r] *= fl * sEG[t];
        ar[n][r] *= fr * sEnd[t];
        dq += qv * aq[n][r];
        dl += kv * al[n][r];
        dr += kv * ar[n][r];
        tq[n][r] += aq[n][r];
        tk[n][r] += al[n][r] + sB[t] * ar[n][r];
      }
      const float left = group_sum<16>(sq * dq + sk * dl + rows[r]), right = sk * group_sum<16>(dr);
      if (l16 == 0) {
        sRow[t] = left;
        sB2[t] = right;
        sH[t] = sB[t] * right;
      }
    }
    __syncthreads();
    if (w == 0) {                                // the gates' gradients, a token a lane
      const float col = (sCol[0][lane] + sCol[1][lane]) + (sCol[2][lane] + sCol[3][lane]);
      const float hs = group_sum<64>(sH[lane]), all = (red[0][3] + red[1][3]) + (red[2][3] + red[3][3]);
      float dG = sRow[lane] - sB[lane] * col - sH[lane];
      const double mine = (double)dG + (lane == 63 ? (double)hs + (double)(sEG[63] * all) : 0.0);
      const double upto = wave_scan64(mine);
      const double total = __shfl(upto, 63);
      if (lane < len) {
        const int64_t at = ((int64_t)b * p.heads + h) * p.seqlen + t0 + lane;
        if (q.dg) {
          const float gv = p.g ? p.g[b * p.gs.b + h * p.gs.h + (int64_t)(t0 + lane) * p.gs.l] : 0.f;
          q.dg[at] = gv < -200.f ? 0.f : (float)(total - upto + mine);
        }
        if (q.dbeta) q.dbeta[at] = col + sB2[lane];
      }
    }
    const Scale xa(fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1])));
    const Scale xp(fmaxf(fmaxf(red[0][2], red[1][2]), fmaxf(red[2][2], red[3][2])));
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {              // block row w; zeros above the diagonal
        const int at = TC::at(16 * w + 4 * g4 + r, 16 * j + l16);
        const f16 a = part_hi(pA[j][r], xa.mult), e = part_hi(pP[j][r], xp.mult);
        sXa[at] = a;
        sXp[at] = e;
        if constexpr (NP == 2) {
          sXa[TC::ELEMS + at] = part_lo(pA[j][r], xa.mult, a);
          sXp[TC::ELEMS + at] = part_lo(pP[j][r], xp.mult, e);
        }
      }
    __syncthreads();
    f16x8 ra[2][NP], rp[2][NP], ca[2][NP], cp[2][NP];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        ra[s][n] = row_frag16<64>(sXa + n * TC::ELEMS, 16 * w, 32 * s, lane);
        rp[s][n] = row_frag16<64>(sXp + n * TC::ELEMS, 16 * w, 32 * s, lane);
        ca[s][n] = col_frag16<64>(sXa + n * TC::ELEMS, 16 * w, 32 * s, lane);
        cp[s][n] = col_frag16<64>(sXp + n * TC::ELEMS, 16 * w, 32 * s, lane);
      }
    const float f1 = xp.inv * sk, f2 = xa.inv * sk, f3 = xp.inv * sq;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x4 u1 = {}, u2 = {}, u3 = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 k0 = col_frag16<DKP>(Kt, 16 * n, 32 * s, lane), q0 = col_frag16<DKP>(Qt, 16 * n, 32 * s, lane);
        u1 = mma_h(rp[s][0], k0, u1);
        u2 = mma_h(ra[s][0], k0, u2);
        u2 = mma_h(ca[s][0], k0, u2);
        u3 = mma_h(cp[s][0], q0, u3);
        if constexpr (NP == 2) {
          const f16x8 k1 = col_frag16<DKP>(Kt + TK::ELEMS, 16 * n, 32 * s, lane);
          const f16x8 q1 = col_frag16<DKP>(Qt + TK::ELEMS, 16 * n, 32 * s, lane);
          u1 = mma_h(rp[s][0], k1, u1);
          u1 = mma_h(rp[s][1], k0, u1);
          u2 = mma_h(ra[s][0], k1, u2);
          u2 = mma_h(ra[s][1], k0, u2);
          u2 = mma_h(ca[s][0], k1, u2);
          u2 = mma_h(ca[s][1], k0, u2);
          u3 = mma_h(cp[s][0], q1, u3);
          u3 = mma_h(cp[s][1], q0, u3);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        tq[n][r] += f1 * u1[r];
        tk[n][r] += f2 * u2[r] + f3 * u3[r];
      }
    }
  }
  T* dq = reinterpret_cast<T*>(q.dq) + b * q.dqs.b + hk * q.dqs.h;
  T* dk = reinterpret_cast<T*>(q.dk) + b * q.dks.b + hk * q.dks.h;
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * w + 4 * g4 + r, col = 16 * n + l16;
      if (t < len && col < p.dk) {
        dq[(int64_t)(t0 + t) * q.dqs.l + col] = from_f32<T>(tq[n][r]);
        dk[(int64_t)(t0 + t) * q.dks.l + col] = from_f32<T>(tk[n][r]);
      }
    }
}

template <typename T, int DKP>
hipError_t run_bwd(const DeltaBwdParams& q, hipStream_t st) {
  const DeltaParams& p = q.f;
  const DeltaLayout lay(p, true);
  constexpr int NW = 2;
  const int nblk = (p.dv + 15) / 16, nwg = (nblk + NW - 1) / NW;
  delta_back_scan_kernel<T, DKP, NW><<<head_block_grid(p.batch * p.heads, nwg), 64 * NW, 0, st>>>(q, lay, nblk, nwg);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  delta_grads_kernel<T, DKP><<<(unsigned)((int64_t)p.batch * p.kheads * p.pieces), 256, 0, st>>>(q, lay, nblk);
  return hipGetLastError();
}

__global__ void delta_copy_grad_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

}  // namespace

size_t delta_bwd_workspace_bytes(const DeltaParams& p) { return DeltaLayout(p, true).total; }

hipError_t launch_delta_bwd(const DeltaBwdParams& q, hipStream_t st) {
  const DeltaParams& p = q.f;
  if (p.seqlen == 0) {
    const int64_t n = (int64_t)p.batch * p.heads * p.dk * p.dv;
    if (!q.d_initial_state) return hipSuccess;
    delta_copy_grad_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(q.d_final_state, q.d_initial_state, n);
    return hipGetLastError();
  }
  hipError_t e = launch_delta_prep(p, true, st);
  if (e == hipSuccess) e = launch_delta_keep(p, st);
  if (e != hipSuccess) return e;
  if (p.dtype == DT_F32) return p.dk <= 64 ? run_bwd<float, 64>(q, st) : run_bwd<float, 128>(q, st);
  return p.dk <= 64 ? run_bwd<bf16, 64>(q, st) : run_bwd<bf16, 128>(q, st);
}

}  // namespace mh
