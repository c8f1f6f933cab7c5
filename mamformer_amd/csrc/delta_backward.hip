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
// What it reads of the forward, the pieces' systems, entering states and corrections, a forward kept for it (3 KB a token
// and head of 128 x 128 in bf16, six times q, k and v) or is computed again, which at b 2, H 16 over 8, L 4096 (bf16) takes
// 172 us beside the 420 of the two kernels here.
#include "delta.h"

namespace mh {
namespace {

// Two waves hold the gradient of 16 columns of the state as the forward's scan holds the state: half of its rows and half of
// a piece's tokens each, and (bf16) a wave fetches the fragments and another dO.  y = T^T ddelta is upper triangular, so
// that here the first wave needs the second one's ddelta.  Bound by a piece's chain as that scan is: 3.0 us for each of
// the 64 pieces of L 4096 (b 2, H 16, 128 x 128: 194 us, with two pairs a workgroup and half of the CUs idle 226; b 3, which
// takes two pairs, 246, with 27 registers spilled).
template <typename T, int DKP, int PAIRS>
__global__ __launch_bounds__((kDeltaThreads<T, PAIRS>)) void delta_back_scan_kernel(DeltaBwdParams q, DeltaLayout lay, DeltaScratch scr, int nblk, int nwg) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr bool AHEAD = NP == 1;
  constexpr int FW = AHEAD ? 1 : 4;
  constexpr int KS = DKP / 32, KSH = KS / 2, NSH = DKP / 32, F = kKFrags<DKP>;
  constexpr int GA = NP * F + 2 * kTFrags;                           // fragments of K by rows and P by columns: before barrier 1
  constexpr int GB = 2 * NP * F + 2 * kTFrags + 1;                   // K and Q by columns, T by columns, vec: after it
  constexpr int EX = (2 * 2 + 2 + 2 * 4 + 1) * FR;                   // halfs of a pair's exchange
  constexpr int IOC = kIoCols<PAIRS>, IOH = IOC * IO_PITCH, IO = AHEAD ? 2 * IOH : 0;
  __shared__ __align__(1024) f16 smem[(GA + (AHEAD ? 2 : 1) * GB) * FR + PAIRS * EX + IO];
  const DeltaParams& p = q.f;

  const int lane = threadIdx.x & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4, hf = w & 1;
  int bh, wg;
  if (!head_block(blockIdx.x, p.batch * p.heads, nwg, bh, wg)) return;
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kheads);
  const int64_t kunit0 = ((int64_t)b * p.kheads + hk) * p.pieces, vunit0 = (int64_t)bh * p.pieces;
  constexpr int DOUT = (GA + (AHEAD ? 2 : 1) * GB) * FR + PAIRS * EX;    // where dO of two pieces is

  const int fw = AHEAD ? 0 : w;
  lds_f16_t* const lds = (lds_f16_t*)smem;
  auto fetch_a = [&](int c) {
    fetch_share<NP * F, FW>(lds, p.workspace + lay.kq + (kunit0 + c) * lay.kq_unit + NP * F * 1024, fw, lane);
    fetch_share<2 * kTFrags, FW>(lds + NP * F * FR, p.workspace + lay.tp + (vunit0 + c) * lay.tp_unit + 6 * kTFrags * 1024, fw, lane);
  };
  auto fetch_b = [&](int c) {
    lds_f16_t* to = lds + (GA + (AHEAD ? (c & 1) * GB : 0)) * FR;
    fetch_share<2 * NP * F, FW>(to, p.workspace + lay.kq + (kunit0 + c) * lay.kq_unit + 2 * NP * F * 1024, fw, lane);
    fetch_share<2 * kTFrags, FW>(to + 2 * NP * F * FR, p.workspace + lay.tp + (vunit0 + c) * lay.tp_unit + 4 * kTFrags * 1024, fw, lane);
    if (fw == 0) fetch_share<1, 1>(to + (2 * NP * F + 2 * kTFrags) * FR, p.workspace + lay.vec + (vunit0 + c) * (int64_t)(kVecFloats * 4), 0, lane);
  };
  if constexpr (AHEAD) {
    if (w == 2 * PAIRS) {
      fetch_a(p.pieces - 1);
      fetch_b(p.pieces - 1);
      wait_vmem_n<GB>();
      lds_barrier();
      for (int c = p.pieces - 1; c >= 0; --c) {
        wait_vmem();
        lds_barrier();                           // 1
        if (c > 0) fetch_a(c - 1);
        lds_barrier();                           // 2
        if (c > 0) {
          fetch_b(c - 1);
          wait_vmem_n<GB>();
        }
        lds_barrier();                           // 3
      }
      return;
    }
    if (w == 2 * PAIRS + 1) {                    // dO; tokens beyond the sequence have none
      const int col0 = IOC * wg, left = p.dv - col0;
      const bf16* src = reinterpret_cast<const bf16*>(q.d_o) + b * q.dos.b + h * q.dos.h + col0;
      auto run = [&](auto full) {
        IoRows<IOC> v;
        auto load = [&](int c) {
          const int t = min(max(c, 0) * DC + lane, p.seqlen - 1);
          v.template load<decltype(full)::value>(src + t * q.dos.l, left);
        };
        load(p.pieces - 1);
        v.zero_unless((p.pieces - 1) * DC + lane < p.seqlen);
        v.to_lds(reinterpret_cast<bf16*>(smem + DOUT + ((p.pieces - 1) & 1) * IOH), lane);
        load(p.pieces - 2);
        lds_barrier();
        for (int c = p.pieces - 1; c >= 0; --c) {
          lds_barrier();                         // 1
          v.to_lds(reinterpret_cast<bf16*>(smem + DOUT + ((c + 1) & 1) * IOH), lane);
          load(c - 2);
          lds_barrier();                         // 2
          lds_barrier();                         // 3
        }
      };
      if (left >= IOC) run(std::true_type{});
      else run(std::false_type{});
      return;
    }
  }
  const int blk = PAIRS * wg + (w >> 1), col = 16 * blk + l16;
  const bool live = blk < nblk, cv = col < p.dv;
  f16* ex = smem + (GA + (AHEAD ? 2 : 1) * GB) * FR + (w >> 1) * EX;
  f32x4* const xSend = reinterpret_cast<f32x4*>(ex) + hf * 2 * 64 + lane;
  const f32x4* const xRecv = reinterpret_cast<const f32x4*>(ex) + (1 - hf) * 2 * 64 + lane;
  f16* const eZ = ex + 4 * FR;                                       // the second half's ddelta
  f16* const eU = eZ + 2 * FR;                                       // the terms of Q and K, two parts of each half
  float* const eS = reinterpret_cast<float*>(eU + 8 * FR);

  f32x4 dS[NSH];
#pragma unroll
  for (int n = 0; n < NSH; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = DKP / 2 * hf + 16 * n + 4 * g4 + r;
      dS[n][r] = q.d_final_state && cv && row < p.dk ? q.d_final_state[((int64_t)bh * p.dk + row) * p.dv + col] : 0.f;
    }
  // dO of one's own tokens; the first wave's P^T dO takes the other's too
  T on[2][8];
  auto load_o = [&](int c) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x4 v = *reinterpret_cast<const bf16x4*>(smem + DOUT + (c & 1) * IOH + ((w >> 1) * 16 + l16) * IO_PITCH + 32 * (x ? 1 - hf : hf) + 16 * i + 4 * g4);
#pragma unroll
          for (int r = 0; r < 4; ++r) on[x][4 * i + r] = v[r];
        }
    } else {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int t = c * DC + 32 * (x ? 1 - hf : hf), len = p.seqlen - t, from = min(t, p.seqlen - 1);
        const T* osrc = reinterpret_cast<const T*>(q.d_o) + b * q.dos.b + h * q.dos.h + (live ? 16 * blk : 0);
        load_rows8<T>(osrc + from * q.dos.l, q.dos.l, p.seqlen - from, cv, 16 * blk + 16 <= p.dv, l16, g4, on[x]);
        if (len < 32)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (16 * (i >> 2) + 4 * g4 + (i & 3) >= len) on[x][i] = from_f32<T>(0.f);
      }
    }
  };
  if (AHEAD) lds_barrier();

  f16x8 ka[KSH][4], p0[2], p1[2], q0[2], q1[2];  // P^T on one's own tokens; on the second half's
  auto load_a = [&](int c) {
#pragma unroll
    for (int s = 0; s < KSH; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) ka[s][i] = frag(smem, ((2 * hf + i) & 3) * KS + hf * KSH + s, lane);
    load_o(c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p0[i] = frag(smem, NP * F + tt_frag(2 * hf + i, hf), lane);
      p1[i] = frag(smem, NP * F + kTFrags + tt_frag(2 * hf + i, hf), lane);
      q0[i] = frag(smem, NP * F + tt_frag(i, 1), lane);
      q1[i] = frag(smem, NP * F + kTFrags + tt_frag(i, 1), lane);
    }
  };
  if (AHEAD) load_a(p.pieces - 1);

  for (int c = p.pieces - 1; c >= 0; --c) {
    if (!AHEAD) {
      lds_barrier();
      fetch_a(c);
      fetch_b(c);
      wait_vmem();
      lds_barrier();
      load_a(c);
    }
    const int kc0 = GA + (AHEAD ? (c & 1) * GB : 0), qc0 = kc0 + NP * F, tt0 = qc0 + NP * F;         // fragments
    const float* vec = reinterpret_cast<const float*>(smem + (tt0 + 2 * kTFrags) * FR);
    f16x8 sh[KSH], sl[KSH];
    f32x4 X[4] = {}, Z[2] = {}, U[2], V[2];
    const Scale ss(col_max(abs_max(dS)));
    parts_of<2>(dS, ss.mult, sh, sl);
#pragma unroll
    for (int s = 0; s < KSH; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) X[i] = mma_h(ka[s][i], sh[s], X[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) X[i] = mma_h(ka[s][i], sl[s], X[i]);
      if constexpr (NP == 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) X[i] = mma_h(frag(smem, F + ((2 * hf + i) & 3) * KS + hf * KSH + s, lane), sh[s], X[i]);
    }
    // P^T dO
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      U[i >> 2][i & 3] = to_f32(on[0][i]);
      V[i >> 2][i & 3] = to_f32(on[1][i]);
    }
    f16x8 oh[1], ol[1];
    const Scale so(col_max(abs_max(V, abs_max(U))));
    parts_of<NP>(U, so.mult, oh, ol);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      Z[i] = mma_h(p0[i], oh[0], Z[i]);
      if constexpr (NP == 2) Z[i] = mma_h(p0[i], ol[0], Z[i]);
      Z[i] = mma_h(p1[i], oh[0], Z[i]);
    }
    if (hf == 0) {
      parts_of<NP>(V, so.mult, oh, ol);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Z[i] = mma_h(q0[i], oh[0], Z[i]);
        if constexpr (NP == 2) Z[i] = mma_h(q0[i], ol[0], Z[i]);
        Z[i] = mma_h(q1[i], oh[0], Z[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) xSend[i * 64] = X[2 + i] * ss.inv;
    lds_barrier();                               // 1
    f32x4 xr[2], wt[2], eg[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xr[i] = xRecv[i * 64];
      wt[i] = *reinterpret_cast<const f32x4*>(vec + VEC_W + 32 * hf + 16 * i + 4 * g4);
    }
    const f32x4 cs = *reinterpret_cast<const f32x4*>(vec + VEC_GAMMA);                 // gamma, scales of T, P, K
    const float sQ = vec[VEC_SQ];
    f16x8 t0[2], t1[2], x0[2], x1[2];            // T^T on one's own tokens; on the second half's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t0[i] = frag(smem, tt0 + tt_frag(2 * hf + i, hf), lane);
      t1[i] = frag(smem, tt0 + kTFrags + tt_frag(2 * hf + i, hf), lane);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x0[i] = frag(smem, tt0 + tt_frag(i, 1), lane);
      x1[i] = frag(smem, tt0 + kTFrags + tt_frag(i, 1), lane);
      eg[i] = *reinterpret_cast<const f32x4*>(vec + 32 * hf + 16 * i + 4 * g4);
    }
    __builtin_amdgcn_sched_barrier(0);
    const float zs = so.inv * cs[2];             // a power of two, exact also below fp32's normal range, as ysc and uk
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) Z[i][r] = __builtin_fmaf(p.scale, zs * Z[i][r], wt[i][r] * (cs[3] * __builtin_fmaf(ss.inv, X[i][r], xr[i][r])));
    // y = T^T ddelta
    f16x8 zh[1], zl[1];
    const Scale sz(col_max(abs_max(Z)));
    parts_of<2>(Z, sz.mult, zh, zl);
    if (hf == 1) {
      put_frag(eZ, 0, lane, zh[0]);
      put_frag(eZ, 1, lane, zl[0]);
      eS[lane] = sz.inv;
    }
    f32x4 Yv[2] = {}, E[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) Yv[i] = mma_h(t0[i], zh[0], Yv[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) Yv[i] = mma_h(t0[i], zl[0], Yv[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) Yv[i] = mma_h(t1[i], zh[0], Yv[i]);
    lds_barrier();                               // 2
    const f16x8 z0 = frag(eZ, 0, lane), z1 = frag(eZ, 1, lane);
    const float es = eS[lane];
    f16x8 kc[NSH][2], qc[NSH][2];                // K and Q by columns, one's own tokens first
#pragma unroll
    for (int n = 0; n < NSH; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        qc[n][x] = frag(smem, qc0 + 2 * (hf * NSH + n) + (x ? 1 - hf : hf), lane);
        kc[n][x] = frag(smem, kc0 + 2 * (hf * NSH + n) + (x ? 1 - hf : hf), lane);
      }
    __builtin_amdgcn_sched_barrier(0);
    float zi = sz.inv;
    if (hf == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x0[i], z0, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x0[i], z1, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x1[i], z0, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) Yv[i][r] = zi * Yv[i][r] + es * E[i][r];
      zi = 1.f;
    }
    // both terms of the gradient before the piece on one scale, those of Q's and K's parts in it
    const float ysc = zi * cs[1], uq = p.scale * sQ, uk = -(ysc * cs[3]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        U[i][r] *= uq * eg[i][r];
        V[i][r] = uk * Yv[i][r] * eg[i][r];
      }
    f16x8 uh[1], ul[1], vh[1], vl[1], yh[1], yl[1];
    const Scale su(col_max(abs_max(V, abs_max(U))));
    parts_of<2>(U, su.mult, uh, ul);
    parts_of<2>(V, su.mult, vh, vl);
    put_frag(eU, 4 * hf, lane, uh[0]);
    put_frag(eU, 4 * hf + 1, lane, ul[0]);
    put_frag(eU, 4 * hf + 2, lane, vh[0]);
    put_frag(eU, 4 * hf + 3, lane, vl[0]);
    eS[(2 + hf) * 64 + lane] = su.inv;
    lds_barrier();                               // 3
    const f16* eO = eU + 4 * (1 - hf) * FR;
    const f16x8 o0 = frag(eO, 0, lane), o1 = frag(eO, 1, lane), o2 = frag(eO, 2, lane), o3 = frag(eO, 3, lane);
    const float other = eS[(3 - hf) * 64 + lane];
    if (AHEAD && c > 0) load_a(c - 1);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 u0[NSH] = {}, u1[NSH] = {};
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(qc[n][0], uh[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(qc[n][0], ul[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(kc[n][0], vh[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(kc[n][0], vl[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(qc[n][1], o0, u1[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(qc[n][1], o1, u1[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(kc[n][1], o2, u1[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(kc[n][1], o3, u1[n]);
    if constexpr (NP == 2)
#pragma unroll
      for (int n = 0; n < NSH; ++n) {
        const int at = F + 2 * (hf * NSH + n);
        u0[n] = mma_h(frag(smem, qc0 + at + hf, lane), uh[0], u0[n]);
        u1[n] = mma_h(frag(smem, qc0 + at + 1 - hf, lane), o0, u1[n]);
        u0[n] = mma_h(frag(smem, kc0 + at + hf, lane), vh[0], u0[n]);
        u1[n] = mma_h(frag(smem, kc0 + at + 1 - hf, lane), o2, u1[n]);
      }
#pragma unroll
    for (int n = 0; n < NSH; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) dS[n][r] = __builtin_fmaf(other, u1[n][r], __builtin_fmaf(su.inv, u0[n][r], cs[0] * dS[n][r]));
    if (live) {
      const Scale sy(col_max(abs_max(Yv)));
      parts_of<2>(Yv, sy.mult, yh, yl);
      const int64_t at = (vunit0 + c) * nblk + blk;
      f16* keep = reinterpret_cast<f16*>(q.scratch + scr.keep) + at * (int64_t)keep_halfs<DKP>();
      float* scales = reinterpret_cast<float*>(q.scratch + scr.scales) + at * kGradScales + 32 * hf + l16;
      keep_parts<KS>(keep, hf * KSH, sh, sl, lane);
      keep_parts<2>(keep + kTokens<DKP>, hf, yh, yl, lane);
      if (g4 == 0) {
        scales[0] = ss.inv;
        scales[16] = sy.inv * ysc;
        if (hf == 0) scales[64] = so.inv;       // over all tokens in either half
      }
    }
  }
  if (q.d_initial_state && cv) {
#pragma unroll
    for (int n = 0; n < NSH; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = DKP / 2 * hf + 16 * n + 4 * g4 + r;
        if (row < p.dk) q.d_initial_state[((int64_t)bh * p.dk + row) * p.dv + col] = dS[n][r];
      }
  }
}

// A lane's 8 values of a k-step (keep_parts): columns c .. c + 3 and c + 16 .. c + 19 of row r.
template <int W>
__device__ __forceinline__ void put_halves(f16* t, int r, int c, f16x8 v) {
  *reinterpret_cast<f16x4*>(t + HTile<W>::at(r, c)) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
  *reinterpret_cast<f16x4*>(t + HTile<W>::at(r, c + 16)) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
}

// One workgroup of 8 waves for a piece of a key head, its value heads one after the other (their dQ and dK are added in
// that order).  Waves w and w + 4 hold rows 16 w .. 16 w + 15: of the three products with the states (64 x dk) half of the
// channels each, of A' and P' every other tile (four waves with all of it spilled 150 registers: 407 us against 300 when
// this was split).  The columns of v pass through LDS DVB at a time, every matrix brought to one scale on the way (its
// columns have their own), a stage's loads under way during the one before.  Now 225 us at b 2, H 16 over 8, L 4096: 400 MB
// of states, corrections and their gradients, which at a copy's rate take 70; one workgroup fits a CU, two waves a SIMD, which
// issue vector instructions in 41% of the cycles, matrix products in 11%, and wait for one another at the stages' barriers.
// Stages of 64 columns (fewer barriers) took 252.
template <typename T, int DKP>
__global__ __launch_bounds__(512) void delta_grads_kernel(DeltaBwdParams q, DeltaLayout lay, DeltaScratch scr, int nblk) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int DVB = 32;
  constexpr int NSH = DKP / 32, KS = DKP / 32, F = kKFrags<DKP>;
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int SE = DVB * DKP, YE = DVB * 64;   // elements of a part of S / dS and of delta / y
  static_assert(4 * SE + 4 * YE >= 4 * TC::ELEMS, "the pair terms take the place of the states, delta and y");
  __shared__ __align__(1024) f16 smem[4 * SE + 4 * YE + NP * TC::ELEMS + 2 * NP * F * FR];
  f16 *sS = smem, *sN = sS + 2 * SE, *sY = sN + 2 * SE, *sD = sY + 2 * YE, *sO = sD + 2 * YE, *sK = sO + NP * TC::ELEMS, *sQ = sK + NP * F * FR;
  f16 *sXa = smem, *sXp = smem + 2 * TC::ELEMS;                        // where those were
  __shared__ double sG[DC];
  __shared__ float sB[DC], sEG[DC], sEnd[DC], sRow[2][DC], sB2[2][DC], sCol[4][DC], red[8][4];
  const DeltaParams& p = q.f;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), w = wave & 3, hf = wave >> 2, l16 = lane & 15, g4 = lane >> 4;
  const int unit = blockIdx.x;
  const int c = unit % p.pieces, bk = unit / p.pieces, hk = bk % p.kheads, b = bk / p.kheads;
  const int t0 = c * DC, len = min(DC, p.seqlen - t0), rep = p.heads / p.kheads;
  const f16* kq = reinterpret_cast<const f16*>(p.workspace + lay.kq + unit * lay.kq_unit);       // Q, K by rows
  {
    f16x8 v[2 * NP * F / 8];                     // K, Q by columns
#pragma unroll
    for (int i = 0; i < 2 * NP * F / 8; ++i) v[i] = frag(kq, 2 * NP * F + 8 * i + wave, lane);
#pragma unroll
    for (int i = 0; i < 2 * NP * F / 8; ++i) put_frag(sK, 8 * i + wave, lane, v[i]);
  }
  const float* vec0 = reinterpret_cast<const float*>(p.workspace + lay.vec) +
                      (((int64_t)b * p.heads + hk * rep) * p.pieces + c) * kVecFloats;
  const float sk = vec0[VEC_SK], sq = vec0[VEC_SQ];
  __syncthreads();
  f32x4 kk[2] = {}, qk[2] = {};                  // tiles 2 m + hf of A' and P'
#pragma unroll
  for (int n = 0; n < NP; ++n) {                 // with part n of K's rows j
    f16x8 kb[2][KS], ka[NP][KS], qa[NP][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int m = 0; m < 2; ++m) kb[m][s] = frag(kq, (NP + n) * F + min(2 * m + hf, w) * KS + s, lane);
#pragma unroll
      for (int x = 0; x < NP - n; ++x) {         // lo lo is left out
        ka[x][s] = frag(kq, (NP + x) * F + w * KS + s, lane);
        qa[x][s] = frag(kq, x * F + w * KS + s, lane);
      }
    }
    __builtin_amdgcn_sched_barrier(0);           // all of it under way before the first product
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int x = 0; x < NP - n; ++x) {
          kk[m] = mma_h(ka[x][s], kb[m][s], kk[m]);
          qk[m] = mma_h(qa[x][s], kb[m][s], qk[m]);
        }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      kk[m][r] = kk[m][r] * sk * sk;
      qk[m][r] = qk[m][r] * sq * sk;
    }

  // What a stage (DVB columns of v of a head) has to load, under way while the one before it is multiplied: a lane's 8
  // values of a k-step (rows 4 g .. and 16 + 4 g .. of 32, of column l % 16) of S, dS, delta and y, 8 columns of dO's row.
  constexpr int SU = (SE / 8 + 511) / 512, YU = YE / 8, OU = DC * DVB / 8;
  static_assert(YU <= 512 && OU <= 512, "one unit a thread");
  f16x8 ps[SU][4], pd[4];
  Raw8<T> po;
  float fs[SU][2], fd[2], mx = 0.f, mg = 0.f, mo = 0.f;     // scales of the units' columns; a head's largest, lanes as the scales
  auto vunit_of = [&](int hr) { return ((int64_t)b * p.heads + hk * rep + hr) * p.pieces + c; };
  auto scales_of = [&](int hr) { return reinterpret_cast<const float*>(p.workspace + lay.scales) + vunit_of(hr) * nblk * kScales; };
  auto grad_scales_of = [&](int hr) { return reinterpret_cast<const float*>(q.scratch + scr.scales) + vunit_of(hr) * nblk * kGradScales; };
  auto load_stage = [&](int hr, int v0) {
    const int lane = lane_id_here(), tid = 64 * wave + lane;           // addresses formed here, not held for the loops
    const int64_t at0 = vunit_of(hr) * nblk * (int64_t)keep_halfs<DKP>();
    const f16 *keep0 = reinterpret_cast<const f16*>(p.workspace + lay.keep) + at0, *grad0 = reinterpret_cast<const f16*>(q.scratch + scr.keep) + at0;
    const float *scales = scales_of(hr), *grad_scales = grad_scales_of(hr);
#pragma unroll
    for (int i = 0; i < SU; ++i) {
      const int u = tid + 512 * i, blk = v0 / 16 + u / (16 * DKP / 8), k = u / 64 % KS;
#pragma unroll
      for (int j = 0; j < 4; ++j) ps[i][j] = f16x8{};
      fs[i][0] = fs[i][1] = 0.f;
      if (u < SE / 8 && blk < nblk) {
        const int at = blk * keep_halfs<DKP>() + (k * 64 + lane) * 8, f = (k >= KS / 2 ? 32 : 0) + (lane & 15);
        ps[i][0] = *reinterpret_cast<const f16x8*>(keep0 + at);
        ps[i][1] = *reinterpret_cast<const f16x8*>(keep0 + at + 16 * DKP);
        ps[i][2] = *reinterpret_cast<const f16x8*>(grad0 + at);
        ps[i][3] = *reinterpret_cast<const f16x8*>(grad0 + at + 16 * DKP);
        fs[i][0] = scales[kScales * blk + f];
        fs[i][1] = grad_scales[kGradScales * blk + f];
      }
    }
    {
      const int blk = v0 / 16 + tid / 128, k = tid / 64 % 2;
#pragma unroll
      for (int j = 0; j < 4; ++j) pd[j] = f16x8{};
      fd[0] = fd[1] = 0.f;
      if (tid < YU && blk < nblk) {
        const int at = blk * keep_halfs<DKP>() + kTokens<DKP> + (k * 64 + lane) * 8, f = 32 * k + 16 + (lane & 15);
        pd[0] = *reinterpret_cast<const f16x8*>(keep0 + at);
        pd[1] = *reinterpret_cast<const f16x8*>(keep0 + at + 16 * DC);
        pd[2] = *reinterpret_cast<const f16x8*>(grad0 + at);
        pd[3] = *reinterpret_cast<const f16x8*>(grad0 + at + 16 * DC);
        fd[0] = scales[kScales * blk + f];
        fd[1] = grad_scales[kGradScales * blk + f];
      }
    }
    const int r = tid / (DVB / 8), c8 = v0 + tid % (DVB / 8) * 8;
    po.clear();
    if (tid < OU && r < len && c8 < p.dv)
      load_raw(po, reinterpret_cast<const T*>(q.d_o) + b * q.dos.b + (hk * rep + hr) * q.dos.h + (int64_t)(t0 + r) * q.dos.l + c8, p.dv - c8);
  };
  auto load_scales = [&](int hr) {
    const int lane = lane_id_here();
    const float *scales = scales_of(hr), *grad_scales = grad_scales_of(hr);
    mx = mg = mo = 0.f;
#pragma unroll 4
    for (int i = 0; i < nblk; ++i) {
      mx = fmaxf(mx, scales[kScales * i + lane]);
      mg = fmaxf(mg, grad_scales[kGradScales * i + lane]);
      mo = fmaxf(mo, grad_scales[kGradScales * i + 64 + (lane & 15)]);
    }
  };
  float gv = 0.f, bv = 0.f;                      // wave 0: of the lane's token
  auto load_gates = [&](int hr) {
    if (wave != 0) return;
    const int h = hk * rep + hr, t = t0 + min(lane, len - 1);
    gv = p.g ? p.g[b * p.gs.b + h * p.gs.h + t * p.gs.l] : 0.f;
    bv = p.beta ? p.beta[b * p.bs.b + h * p.bs.h + t * p.bs.l] : 1.f;
  };
  load_stage(0, 0);
  load_scales(0);
  load_gates(0);

  f32x4 tq[NSH] = {}, tk[NSH] = {};              // dQ and dK over the value heads, channels 16 (hf NSH + n) ..
  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    T* dvo = reinterpret_cast<T*>(q.dv) + b * q.dvs.b + h * q.dvs.h + (int64_t)t0 * q.dvs.l;
    __syncthreads();                             // the last head's use of the LDS is over
    const float raw_g = gv;
    if (wave == 0) {
      const double G = wave_scan64(lane < len ? (double)gate_log(gv) * kLog2e64 : 0.), end = last_lane64(G);
      sG[lane] = G;
      sB[lane] = lane < len ? bv : 0.f;
      sEG[lane] = exp_of(G);
      sEnd[lane] = exp_of(end - G);
    }
    if (hr + 1 < rep) load_gates(hr + 1);
    mx = row16_max(mx);
    mg = row16_max(mg);
    const float mS = fmaxf(lane_val(mx, 0), lane_val(mx, 32)), mD = fmaxf(lane_val(mx, 16), lane_val(mx, 48)),
                mN = fmaxf(lane_val(mg, 0), lane_val(mg, 32)), mY = fmaxf(lane_val(mg, 16), lane_val(mg, 48));
    const float so_inv = row16_max(mo), so_mult = 1.f / so_inv;        // a power of two
    auto most = [&](int i) {
      return fmaxf(fmaxf(fmaxf(red[0][i], red[1][i]), fmaxf(red[2][i], red[3][i])), fmaxf(fmaxf(red[4][i], red[5][i]), fmaxf(red[6][i], red[7][i])));
    };

    f32x4 aq[NSH] = {}, al[NSH] = {}, ar[NSH] = {}, pA[2] = {}, pP[2] = {};
    float dot = 0.f;                             // <S, dS>
    for (int v0 = 0; v0 < 16 * nblk; v0 += DVB) {
      if (v0) __syncthreads();
      const int lane = lane_id_here(), tid = 64 * wave + lane;
#pragma unroll
      for (int i = 0; i < SU; ++i) {
        const int u = tid + 512 * i, r = u / (16 * DKP / 8) * 16 + (lane & 15), ch = u / 64 % KS * 32 + 4 * (lane >> 4);
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) d += ((float)ps[i][0][j] + (float)ps[i][1][j]) * ((float)ps[i][2][j] + (float)ps[i][3][j]);
        dot += d * fs[i][0] * fs[i][1];
        const f16 hs = (f16)(fs[i][0] / mS), hn = (f16)(fs[i][1] / mN);  // powers of two, at most 1
        if (u < SE / 8) {
          put_halves<DKP>(sS, r, ch, ps[i][0] * hs);
          put_halves<DKP>(sS + SE, r, ch, ps[i][1] * hs);
          put_halves<DKP>(sN, r, ch, ps[i][2] * hn);
          put_halves<DKP>(sN + SE, r, ch, ps[i][3] * hn);
        }
      }
      if (tid < YU) {
        const int r = tid / 128 * 16 + (lane & 15), ch = tid / 64 % 2 * 32 + 4 * (lane >> 4);
        const f16 hd = (f16)(fd[0] / mD), hy = (f16)(fd[1] / mY);
        put_halves<64>(sD, r, ch, pd[0] * hd);
        put_halves<64>(sD + YE, r, ch, pd[1] * hd);
        put_halves<64>(sY, r, ch, pd[2] * hy);
        put_halves<64>(sY + YE, r, ch, pd[3] * hy);
        if (v0 + r < p.dv)                       // dV
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int t = ch + (j & 3) + 4 * (j & 4);
            if (t < len) dvo[t * q.dvs.l + v0 + r] = from_f32<T>(((float)pd[2][j] + (float)pd[3][j]) * fd[1]);
          }
      }
      if (tid < OU) {
        const int r = tid / (DVB / 8), c8 = tid % (DVB / 8) * 8;
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hi[j] = part_hi(po.get(j), so_mult);
          if constexpr (NP == 2) lo[j] = part_lo(po.get(j), so_mult, hi[j]);
        }
        *reinterpret_cast<f16x8*>(sO + TC::at(r, c8)) = hi;
        if constexpr (NP == 2) *reinterpret_cast<f16x8*>(sO + TC::ELEMS + TC::at(r, c8)) = lo;
      }
      __syncthreads();
      if (v0 + DVB < 16 * nblk) {
        load_stage(hr, v0 + DVB);
      } else if (hr + 1 < rep) {
        load_stage(hr + 1, 0);
        load_scales(hr + 1);
      }
#pragma unroll
      for (int s = 0; s < DVB / 32; ++s) {
        const f16x8 o0 = row_frag16<64>(sO, 16 * w, 32 * s, lane);
        f16x8 o1;
        if constexpr (NP == 2) o1 = row_frag16<64>(sO + TC::ELEMS, 16 * w, 32 * s, lane);
        const f16x8 y0 = col_frag16<64>(sY, 16 * w, 32 * s, lane), y1 = col_frag16<64>(sY + YE, 16 * w, 32 * s, lane);
        const f16x8 d0 = col_frag16<64>(sD, 16 * w, 32 * s, lane), d1 = col_frag16<64>(sD + YE, 16 * w, 32 * s, lane);
#pragma unroll
        for (int n = 0; n < NSH; ++n) {
          const int at = 16 * (hf * NSH + n);
          const f16x8 b0 = col_frag16<DKP>(sS, at, 32 * s, lane), b1 = col_frag16<DKP>(sS + SE, at, 32 * s, lane);
          const f16x8 n0 = col_frag16<DKP>(sN, at, 32 * s, lane), n1 = col_frag16<DKP>(sN + SE, at, 32 * s, lane);
          aq[n] = mma_h(o0, b0, aq[n]);
          al[n] = mma_h(y0, b0, al[n]);
          ar[n] = mma_h(d0, n0, ar[n]);
          aq[n] = mma_h(o0, b1, aq[n]);
          al[n] = mma_h(y0, b1, al[n]);
          ar[n] = mma_h(d0, n1, ar[n]);
          if constexpr (NP == 2) aq[n] = mma_h(o1, b0, aq[n]);
          al[n] = mma_h(y1, b0, al[n]);
          ar[n] = mma_h(d1, n0, ar[n]);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int j = 2 * m + hf;
          if (j > w) continue;
          const f16x8 b0 = col_frag16<64>(sD, 16 * j, 32 * s, lane), b1 = col_frag16<64>(sD + YE, 16 * j, 32 * s, lane);
          pA[m] = mma_h(y0, b0, pA[m]);
          pP[m] = mma_h(o0, b0, pP[m]);
          pA[m] = mma_h(y0, b1, pA[m]);
          pP[m] = mma_h(o0, b1, pP[m]);
          pA[m] = mma_h(y1, b0, pA[m]);
          if constexpr (NP == 2) pP[m] = mma_h(o1, b0, pP[m]);
        }
      }
    }
    // A' and P', what they give dbeta and dG, and the pair terms' matrices.  The operands' scales, powers of two, go to the
    // sums one after the other, as their products alone may leave fp32's range where those do not.
    const int lane = lane_id_here(), l16 = lane & 15, g4 = lane >> 4;
    float rows[4] = {}, xam = 0.f, xpm = 0.f;
    double Gt[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) Gt[r] = sG[16 * w + 4 * g4 + r];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int j = 2 * m + hf;
      float colb = 0.f;
      if (j <= w) {
        const double Gj = sG[16 * j + l16];
        const float bj = sB[16 * j + l16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int below = 16 * (w - j) + 4 * g4 + r - l16;
          const float d = below >= 0 ? exp_of(Gt[r] - Gj) : 0.f;
          const float xa = below > 0 ? pA[m][r] * -mY * mD * d : 0.f, xp = below >= 0 ? pP[m][r] * so_inv * mD * (p.scale * d) : 0.f;
          const float v = (below > 0 ? xa * kk[m][r] : 0.f) + (below >= 0 ? xp * qk[m][r] : 0.f);
          colb += v;
          rows[r] += v * bj;
          pA[m][r] = xa * bj;
          pP[m][r] = xp * bj;
          xam = fmaxf(xam, fabsf(pA[m][r]));
          xpm = fmaxf(xpm, fabsf(pP[m][r]));
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
      red[wave][1] = xam;
      red[wave][2] = xpm;
      red[wave][3] = dot;
    }
    float dots[4] = {}, rights[4] = {};
#pragma unroll
    for (int n = 0; n < NSH; ++n) {
      // rows 16 w + 4 g + r of channel l % 16 of tile hf NSH + n: half of a fragment by columns
      f16x8 kf[NP], qf[NP];
#pragma unroll
      for (int m = 0; m < NP; ++m) {
        kf[m] = frag(sK, m * F + 2 * (hf * NSH + n) + (w >> 1), lane);
        qf[m] = frag(sQ, m * F + 2 * (hf * NSH + n) + (w >> 1), lane);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * w + 4 * g4 + r;
        float kv = (float)(w & 1 ? kf[0][4 + r] : kf[0][r]), qv = (float)(w & 1 ? qf[0][4 + r] : qf[0][r]);
        if constexpr (NP == 2) {
          kv += (float)(w & 1 ? kf[1][4 + r] : kf[1][r]);
          qv += (float)(w & 1 ? qf[1][4 + r] : qf[1][r]);
        }
        const float q1 = aq[n][r] * so_inv * mS * (p.scale * sEG[t]), l1 = al[n][r] * -mY * mS * sEG[t], r1 = ar[n][r] * mD * mN * sEnd[t];
        dots[r] += (sq * qv) * q1 + (sk * kv) * l1;
        rights[r] += (sk * kv) * r1;
        tq[n][r] += q1;
        tk[n][r] += l1 + sB[t] * r1;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * w + 4 * g4 + r;
      const float left = group_sum<16>(dots[r] + rows[r]), right = group_sum<16>(rights[r]);
      if (l16 == 0) {
        sRow[hf][t] = left;
        sB2[hf][t] = right;
      }
    }
    __syncthreads();
    if (wave == 0) {                             // the gates' gradients, a token a lane
      const float col = (sCol[0][lane] + sCol[1][lane]) + (sCol[2][lane] + sCol[3][lane]);
      const float b2 = sB2[0][lane] + sB2[1][lane], H = sB[lane] * b2;
      const float hs = group_sum<64>(H);
      float all = 0.f;
      for (int i = 0; i < 8; ++i) all += red[i][3];
      const double mine = (double)(sRow[0][lane] + sRow[1][lane] - sB[lane] * col - H) +
                          (lane == 63 ? (double)hs + (double)(sEG[63] * all) : 0.0);
      const double upto = wave_scan64(mine);
      const double total = last_lane64(upto);
      if (lane < len) {
        const int64_t at = ((int64_t)b * p.heads + h) * p.seqlen + t0 + lane;
        if (q.dg) q.dg[at] = raw_g < -200.f ? 0.f : (float)(total - upto + mine);
        if (q.dbeta) q.dbeta[at] = col + b2;
      }
    }
    const Scale xa(most(1)), xp(most(2));
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {              // block row w; zeros above the diagonal
        const int at = TC::at(16 * w + 4 * g4 + r, 16 * (2 * m + hf) + l16);
        const f16 a = part_hi(pA[m][r], xa.mult), e = part_hi(pP[m][r], xp.mult);
        sXa[at] = a;
        sXp[at] = e;
        sXa[TC::ELEMS + at] = part_lo(pA[m][r], xa.mult, a);
        sXp[TC::ELEMS + at] = part_lo(pP[m][r], xp.mult, e);
      }
    __syncthreads();
    f16x8 ra[2][2], rp[2][2], ca[2][2], cp[2][2]; // both parts also for bf16: rows of dQ and dK may cancel far below them
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        ra[s][n] = row_frag16<64>(sXa + n * TC::ELEMS, 16 * w, 32 * s, lane);
        rp[s][n] = row_frag16<64>(sXp + n * TC::ELEMS, 16 * w, 32 * s, lane);
        ca[s][n] = col_frag16<64>(sXa + n * TC::ELEMS, 16 * w, 32 * s, lane);
        cp[s][n] = col_frag16<64>(sXp + n * TC::ELEMS, 16 * w, 32 * s, lane);
      }
    const float f1 = xp.inv * sk, f2 = xa.inv * sk, f3 = xp.inv * sq;
#pragma unroll
    for (int n = 0; n < NSH; ++n) {
      f32x4 u1 = {}, u2 = {}, u3 = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 k0 = frag(sK, 2 * (hf * NSH + n) + s, lane), q0 = frag(sQ, 2 * (hf * NSH + n) + s, lane);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u1 = mma_h(rp[s][x], k0, u1);
          u2 = mma_h(ra[s][x], k0, u2);
          u2 = mma_h(ca[s][x], k0, u2);
          u3 = mma_h(cp[s][x], q0, u3);
        }
        if constexpr (NP == 2) {
          const f16x8 k1 = frag(sK, F + 2 * (hf * NSH + n) + s, lane);
          const f16x8 q1 = frag(sQ, F + 2 * (hf * NSH + n) + s, lane);
          u1 = mma_h(rp[s][0], k1, u1);
          u2 = mma_h(ra[s][0], k1, u2);
          u2 = mma_h(ca[s][0], k1, u2);
          u3 = mma_h(cp[s][0], q1, u3);
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
  for (int n = 0; n < NSH; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * w + 4 * g4 + r, col = 16 * (hf * NSH + n) + l16;
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
  const DeltaScratch scr(p);
  const int nblk = (p.dv + 15) / 16, nwg = (nblk + 1) / 2;
  if (sizeof(T) == 2 && delta_one_pair(p, 1)) {
    if constexpr (sizeof(T) == 2)
      delta_back_scan_kernel<T, DKP, 1><<<head_block_grid(p.batch * p.heads, nblk), kDeltaThreads<T, 1>, 0, st>>>(q, lay, scr, nblk, nblk);
  } else {
    delta_back_scan_kernel<T, DKP, 2><<<head_block_grid(p.batch * p.heads, nwg), kDeltaThreads<T, 2>, 0, st>>>(q, lay, scr, nblk, nwg);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  delta_grads_kernel<T, DKP><<<(unsigned)((int64_t)p.batch * p.kheads * p.pieces), 512, 0, st>>>(q, lay, scr, nblk);
  return hipGetLastError();
}

__global__ void delta_copy_grad_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = grid_row() * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

}  // namespace

size_t delta_scratch_bytes(const DeltaParams& p) { return DeltaScratch(p).total; }

hipError_t launch_delta_bwd(const DeltaBwdParams& q, hipStream_t st) {
  const DeltaParams& p = q.f;
  if (p.seqlen == 0) {
    const int64_t n = (int64_t)p.batch * p.heads * p.dk * p.dv;
    if (!q.d_initial_state) return hipSuccess;
    delta_copy_grad_kernel<<<row_grid((n + 255) / 256, 1), 256, 0, st>>>(q.d_final_state, q.d_initial_state, n);
    return hipGetLastError();
  }
  if (!q.kept) {
    hipError_t e = launch_delta_prep(p, true, st);
    if (e == hipSuccess) e = launch_delta_keep(p, st);
    if (e != hipSuccess) return e;
  }
  if (p.dtype == DT_F32) return p.dk <= 64 ? run_bwd<float, 64>(q, st) : run_bwd<float, 128>(q, st);
  return p.dk <= 64 ? run_bwd<bf16, 64>(q, st) : run_bwd<bf16, 128>(q, st);
}

}  // namespace mh
