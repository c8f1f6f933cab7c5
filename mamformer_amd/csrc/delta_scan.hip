// Gated delta rule over sequences:
//   S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - e^{g_t} S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t.
// In pieces of 64 tokens, G the inclusive sum of g in the piece and S the state that enters it:
//   delta = T (V - e^G K S),   T = (I + A)^-1,  A_tj = e^{G_t - G_j} (k_t k_j) beta_j for j < t
//   O     = scale (e^G Q S + P delta),          P_tj = e^{G_t - G_j} (q_t k_j) beta_j for j <= t
//   S'    = e^{G_end} S + (beta e^{G_end - G} K)^T delta
// delta is what each token corrects before its beta, so that beta = 0 divides nothing.  delta_prep_kernel makes T and P of
// every piece side by side; delta_scan_kernel walks the pieces with the state in registers.
// o takes both parts of S, P and delta also where it is rounded to bf16: its terms may cancel far below what enters them, and
// one part, 2^-12 of that, would show (12 of 141 us at b 4, H 16, L 2048).
#include "delta.h"

namespace mh {
namespace {

// ------------------------------------------------------------------ pieces side by side
// One workgroup of 4 waves for a piece of a key head: K and Q into their fp16 parts and fragments (kept for the scans), K K^T
// and K Q^T once, then for each value head that shares them A, its inverse and P.  Everything is transposed: wave w has the
// tokens t = 16 w + l % 16 as columns and the tokens j <= t as rows of its accumulators, which are then the fragments of T
// and P by rows as they stand.  The inverse in fp32: every wave solves one 16 x 16 diagonal block by substitution, a column
// a lane, then wave w builds block row w of T from the diagonal outwards, T_wj = -(sum over j < k <= w of T_wk A_kj) T_jj,
// with fp32 matrix instructions, T_wk staying in accumulators, which are the B operand of the next product.
// Workgroups on one CU hide each other's latencies (LDS, substitution); what they write, 73 KB a piece of one value head,
// is what bounds them: b 4, H 16, L 2048 (bf16, 128): 57 us for 2048 pieces, 220 MB read and written, 3.9 TB/s.
template <typename T, int DKP>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) void delta_prep_kernel(DeltaParams p, DeltaLayout lay, int backward) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int CPR = DKP / 8;                   // threads of 8 channels for a row
  constexpr int RPP = 256 / CPR;                 // rows of a pass
  constexpr int F = kKFrags<DKP>, KS = DKP / 32;
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int AP = 68;                         // pitch of A
  constexpr int HALFS = 2 * NP * TK::ELEMS > 4 * TC::ELEMS ? 2 * NP * TK::ELEMS : 4 * TC::ELEMS;
  static_assert(HALFS * 2 >= DC * AP * 4, "A takes the tiles' place");
  __shared__ __align__(16) f16 tiles[HALFS];     // K and Q, then A, then T and P for the fragments by columns
  __shared__ __align__(16) float sD[4 * 16 * 20];
  __shared__ __align__(16) double sG[DC];        // sums of gates times log2 e
  __shared__ __align__(16) float sB[DC], sVec[2 * DC];
  __shared__ float red[4][2];
  float* const sA = reinterpret_cast<float*>(tiles);                   // A^T: row j, column t

  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  const int unit = blockIdx.x;                   // (batch, key head, piece)
  const int c = unit % p.pieces, bk = unit / p.pieces, hk = bk % p.kheads, b = bk / p.kheads;
  const int t0 = c * DC, len = min(DC, p.seqlen - t0), rep = p.heads / p.kheads;

  float gv = 0.f, bv = 0.f;                      // wave 0: of the lane's token, a head ahead
  auto load_gates = [&](int h) {
    if (w != 0) return;
    const int t = t0 + min(lane, len - 1);
    gv = p.g ? p.g[b * p.gs.b + h * p.gs.h + t * p.gs.l] : 0.f;
    bv = p.beta ? p.beta[b * p.bs.b + h * p.bs.h + t * p.bs.l] : 1.f;
  };

  // K and Q: largest magnitudes, then parts into the tiles.  Rows and channels beyond the last are read within the tensor
  // and cleared, so that all loads are under way at once.
  Raw8<T> raw[2][DC / RPP];
  const int cc = tid % CPR, rr = tid / CPR;
  const bool cok = cc * 8 < p.dk;
  const T* src[2] = {reinterpret_cast<const T*>(p.k) + b * p.ks.b + hk * p.ks.h + t0 * p.ks.l,
                     reinterpret_cast<const T*>(p.q) + b * p.qs.b + hk * p.qs.h + t0 * p.qs.l};
  const int64_t sl[2] = {p.ks.l, p.qs.l};
  if (p.dk % 8 == 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < DC / RPP; ++i) raw[x][i].load(src[x] + min(i * RPP + rr, len - 1) * sl[x] + (cok ? cc * 8 : 0));
    load_gates(hk * rep);
  } else {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < DC / RPP; ++i) {
        raw[x][i].clear();
        if (cok) load_raw(raw[x][i], src[x] + min(i * RPP + rr, len - 1) * sl[x] + cc * 8, p.dk - cc * 8);
      }
    load_gates(hk * rep);
  }
  float amax[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int i = 0; i < DC / RPP; ++i) {
      if (!cok || i * RPP + rr >= len) raw[x][i].clear();
#pragma unroll
      for (int j = 0; j < 8; ++j) amax[x] = fmaxf(amax[x], fabsf(raw[x][i].get(j)));
    }
    amax[x] = wave_max(amax[x]);
    if (lane == 0) red[w][x] = amax[x];
  }
  __syncthreads();
  const Scale sk(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
  const Scale sq(fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1])));
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < DC / RPP; ++i) {
      const float mult = x ? sq.mult : sk.mult;
      f16x8 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = raw[x][i].get(j);
        hi[j] = part_hi(v, mult);
        if constexpr (NP == 2) lo[j] = part_lo(v, mult, hi[j]);
      }
      f16* to = tiles + x * NP * TK::ELEMS + TK::at(i * RPP + rr, cc * 8);
      *reinterpret_cast<f16x8*>(to) = hi;
      if constexpr (NP == 2) *reinterpret_cast<f16x8*>(to + TK::ELEMS) = lo;
    }
  __syncthreads();
  f32x4 kk[4] = {}, qk[4] = {};                  // rows j = 16 n + 4 g4 + r, column t = 16 w + l16
  {
    f16* out = reinterpret_cast<f16*>(p.workspace + lay.kq + unit * lay.kq_unit);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      f16x8 kb[NP], qb[NP];
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        qb[n] = row_frag16<DKP>(tiles + (NP + n) * TK::ELEMS, 16 * w, 32 * s, lane);
        kb[n] = row_frag16<DKP>(tiles + n * TK::ELEMS, 16 * w, 32 * s, lane);
        put_frag(out, n * F + w * KS + s, lane, qb[n]);
        put_frag(out, (NP + n) * F + w * KS + s, lane, kb[n]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > w) continue;
        const f16x8 a0 = row_frag16<DKP>(tiles, 16 * j, 32 * s, lane);
        kk[j] = mma_h(a0, kb[0], kk[j]);
        qk[j] = mma_h(a0, qb[0], qk[j]);
        if constexpr (NP == 2) {
          const f16x8 a1 = row_frag16<DKP>(tiles + TK::ELEMS, 16 * j, 32 * s, lane);
          kk[j] = mma_h(a1, kb[0], kk[j]);
          kk[j] = mma_h(a0, kb[1], kk[j]);
          qk[j] = mma_h(a1, qb[0], qk[j]);
          qk[j] = mma_h(a0, qb[1], qk[j]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int m = 0; m < DKP / 64; ++m)         // channels 16 (4 m + w) ..
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int at = 2 * (4 * m + w) + s;
          put_frag(out, (2 * NP + n) * F + at, lane, col_frag16<DKP>(tiles + n * TK::ELEMS, 16 * (4 * m + w), 32 * s, lane));
          if (backward) put_frag(out, (3 * NP + n) * F + at, lane, col_frag16<DKP>(tiles + (NP + n) * TK::ELEMS, 16 * (4 * m + w), 32 * s, lane));
        }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      kk[j][r] = kk[j][r] * sk.inv * sk.inv;
      qk[j][r] = qk[j][r] * sq.inv * sk.inv;
    }

  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const int64_t vunit = ((int64_t)b * p.heads + h) * p.pieces + c;
    if (w == 0) {
      const double G = wave_scan64(lane < len ? (double)gate_log(gv) * kLog2e64 : 0.);
      const double end = last_lane64(G);
      const float beta = lane < len ? bv : 0.f;
      sG[lane] = G;
      sB[lane] = beta;
      sVec[lane] = exp_of(G);
      sVec[DC + lane] = beta * exp_of(end - G);
      if (hr + 1 < rep) load_gates(h + 1);
    }
    __syncthreads();                             // and the tiles or the last head's parts have been read
    const double Gt = sG[16 * w + l16];
    f32x4 P[4] = {};
    float pmax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w) continue;
      const f32x4 bj = *reinterpret_cast<const f32x4*>(sB + 16 * j + 4 * g4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int below = 16 * (w - j) + l16 - 4 * g4 - r;               // t - j
        const float d = below >= 0 ? exp_of(Gt - sG[16 * j + 4 * g4 + r]) * bj[r] : 0.f;
        P[j][r] = below >= 0 ? qk[j][r] * d : 0.f;
        pmax = fmaxf(pmax, fabsf(P[j][r]));
        sA[(16 * j + 4 * g4 + r) * AP + 16 * w + l16] = below > 0 ? kk[j][r] * d : 0.f;
      }
    }
    __syncthreads();
    // T^T of diagonal block w, a column a lane (the four groups of 16 lanes do the same), from the last row up
    {
      const float* at = sA + (16 * w) * AP + 16 * w;
      float x[16];
#pragma unroll
      for (int i = 15; i >= 0; --i) {
        float s0 = i == l16 ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j4 = (i + 1) / 4; j4 < 4; ++j4) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(at + i * AP + 4 * j4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * j4 + j > i) (j & 1 ? s1 : s0) -= a[j] * x[4 * j4 + j];
        }
        x[i] = s0 + s1;
        if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);             // the rows' reads in four lots, not all held at once
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (g4 == i >> 2) sD[(w * 16 + i) * 20 + l16] = x[i];
    }
    __syncthreads();
    // block row w of T, transposed, from the diagonal outwards
    f32x4 t[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i == w)
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i][r] = sD[(w * 16 + 4 * g4 + r) * 20 + l16];
#pragma unroll
    for (int j = 2; j >= 0; --j) {
      if (j >= w) continue;
      f32x4 m0 = {}, m1 = {};
#pragma unroll
      for (int k = j + 1; k < 4; ++k) {
        if (k > w) continue;
        const f32x4 a = *reinterpret_cast<const f32x4*>(sA + (16 * j + l16) * AP + 16 * k + 4 * g4);
#pragma unroll
        for (int s = 0; s < 4; ++s) (s & 1 ? m1 : m0) = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], t[k][s], s & 1 ? m1 : m0, 0, 0, 0);
      }
      const f32x4 d = *reinterpret_cast<const f32x4*>(sD + (j * 16 + l16) * 20 + 4 * g4);
      f32x4 y0 = {}, y1 = {};
#pragma unroll
      for (int s = 0; s < 4; ++s) (s & 1 ? y1 : y0) = __builtin_amdgcn_mfma_f32_16x16x4f32(d[s], m0[s] + m1[s], s & 1 ? y1 : y0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) t[j][r] = -(y0[r] + y1[r]);
    }
    const float tm = wave_max(abs_max(t)), pm = wave_max(pmax);
    if (lane == 0) {
      red[w][0] = tm;
      red[w][1] = pm;
    }
    __syncthreads();
    const Scale st(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
    const Scale sp(fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1])));
    f16x8 th[2], tl[2], ph[2], pl[2];
    parts_of<2>(t, st.mult, th, tl);
    parts_of<2>(P, sp.mult, ph, pl);
    f16* out = reinterpret_cast<f16*>(p.workspace + lay.tp + vunit * lay.tp_unit);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (w >= 2 * s) {
        put_frag(out, t_frag(w, s), lane, th[s]);
        put_frag(out, kTFrags + t_frag(w, s), lane, tl[s]);
        put_frag(out, 2 * kTFrags + t_frag(w, s), lane, ph[s]);
        put_frag(out, 3 * kTFrags + t_frag(w, s), lane, pl[s]);
      }
    if (backward) {                              // by columns: through LDS, as T^T and P^T (row j, column t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = TC::at(16 * j + 4 * g4 + r, 16 * w + l16), e = 4 * (j & 1) + r;
          tiles[at] = th[j >> 1][e];
          tiles[TC::ELEMS + at] = tl[j >> 1][e];
          tiles[2 * TC::ELEMS + at] = ph[j >> 1][e];
          tiles[3 * TC::ELEMS + at] = pl[j >> 1][e];
        }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (w < 2 + 2 * s) {
            put_frag(out, (4 + n) * kTFrags + tt_frag(w, s), lane, row_frag16<64>(tiles + n * TC::ELEMS, 16 * w, 32 * s, lane));
            put_frag(out, (6 + n) * kTFrags + tt_frag(w, s), lane, row_frag16<64>(tiles + (2 + n) * TC::ELEMS, 16 * w, 32 * s, lane));
          }
    }
    float* vec = reinterpret_cast<float*>(p.workspace + lay.vec) + vunit * kVecFloats;
    if (tid < 2 * DC) vec[tid] = sVec[tid];
    if (tid == 2 * DC) {
      vec[VEC_GAMMA] = sVec[DC - 1];
      vec[VEC_ST] = st.inv;
      vec[VEC_SP] = sp.inv;
      vec[VEC_SK] = sk.inv;
      vec[VEC_SQ] = sq.inv;
    }
    if (hr + 1 < rep) __syncthreads();           // sVec and the parts have been read
  }
}

// ------------------------------------------------------------------ the state from piece to piece
// Two waves hold 16 columns of the state, half of its rows each (fp32), and half of a piece's tokens; a workgroup has two
// such pairs, which read the same fragments, or one where the pairs are no more than the CUs (b 2, H 16, L 4096, o and what
// a backward keeps: 204 us against 224 when it was chosen, 188 now; b 3, which takes two pairs, 254), or four for a segment
// without o, whose exchange takes less LDS.  For a piece:
//   each wave multiplies K (and Q) by its rows of S and gives the other its part of the other's tokens;   [barrier 1]
//   R = V - e^G K S of its tokens; T is lower triangular, so that the second wave needs the first one's R;  [barrier 2]
//   U = beta e^{G_end - G} delta of its tokens goes to the other, each adds K^T U to its rows.              [barrier 3]
// bf16: one more wave fetches the next piece's fragments by LDS DMA and another one v, and stores o: a wave that issues such
// loads stands still while they drain (2000 of the 8000 cycles that a piece took before), which those two may.
// KEEP: the entering states and delta are stored for the backward.  OUT: o is computed.  What is multiplied and added in
// one instruction is written out, so that all variants give the same bits.
//
// Bound by the chain of one piece on waves that have a SIMD to themselves: 3.0 us (b 4, H 16, L 2048, 128 x 128: 95 us; b 2,
// H 16, L 4096 with what a backward keeps 188).  Of its 6000 cycles a wave issues vector instructions in 2400 (about 500, 66
// of them matrix products), the matrix units work in 1060 and the CU's LDS in 1360; the rest are waits for one another, for
// operands and at the three barriers, which nothing on the SIMD fills.  Operands that no other wave has to finish first are
// read from LDS right behind a barrier, ahead of what they are needed for.
template <typename T, int DKP, bool OUT, bool KEEP, int PAIRS>
__global__ __launch_bounds__((kDeltaThreads<T, PAIRS>)) void delta_scan_kernel(DeltaParams p, DeltaLayout lay, int nblk, int nwg) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr bool AHEAD = NP == 1;                // fp32: the fragments of a piece fill the LDS
  constexpr bool MOVE = !OUT && !KEEP;           // what a segment makes of the state, and of any other
  constexpr int IOW = kIoWaves<PAIRS>, IOC = kIoCols<PAIRS>, IOH = IOC * IO_PITCH;
  constexpr int FW = AHEAD ? 1 : 2 * PAIRS;      // waves that fetch
  constexpr int KS = DKP / 32, KSH = KS / 2, NSH = DKP / 32, F = kKFrags<DKP>;
  constexpr int GA = (OUT ? 2 : 1) * NP * F;                         // fragments of (Q and) K by rows: before barrier 1
  constexpr int TPF = (OUT ? 4 : 2) * kTFrags;                       // of T (and P)
  constexpr int GB = NP * F + TPF + 1;                               // with K by columns and vec: after it
  constexpr int XF = OUT ? 4 : 2;
  constexpr int EX = (2 * XF + 2 + 4 + 1) * FR;                      // halfs of a pair's exchange
  constexpr int IO = AHEAD ? (OUT ? 3 : 2) * IOW * IOH : 0;           // v of two pieces, o of one
  // Pieces of which K and Q by rows have room.  A second one's took 4% off the chain (175 -> 168 us at b 2, H 16, L 4096,
  // where P had one part); with o of 128 channels the two parts of P leave none for it.
  constexpr int AB = AHEAD && PAIRS == 1 && !(OUT && DKP == 128) ? 2 : 1;
  __shared__ __align__(1024) f16 smem[(AB * GA + (AHEAD ? 2 : 1) * GB) * FR + PAIRS * EX + IO];

  const int lane = threadIdx.x & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4, hf = w & 1;
  int part, wg;
  const int segs = MOVE ? lay.segs - 1 : lay.segs;
  if (!head_block(blockIdx.x, p.batch * p.heads * segs, nwg, part, wg)) return;
  const int bh = part / segs, seg = part % segs, c0 = seg * lay.per, c1 = min(c0 + lay.per, p.pieces);
  const int nv = (nblk + PAIRS - 1) / PAIRS;     // workgroups behind them: the columns of the identity, without v
  const bool unit = MOVE && wg >= nv;
  if (unit && seg == 0) return;                  // its state is known
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kheads);
  const int64_t kunit0 = ((int64_t)b * p.kheads + hk) * p.pieces, vunit0 = (int64_t)bh * p.pieces;
  bf16* const sV = reinterpret_cast<bf16*>(smem + (AB * GA + (AHEAD ? 2 : 1) * GB) * FR + PAIRS * EX);
  bf16* const sO = sV + 2 * IOW * IOH;

  const int fw = AHEAD ? 0 : w;
  lds_f16_t* const lds = (lds_f16_t*)smem;
  auto fetch_a = [&](int c) { fetch_share<GA, FW>(lds + (AB == 2 ? (c & 1) * GA * FR : 0), p.workspace + lay.kq + (kunit0 + c) * lay.kq_unit + (OUT ? 0 : NP * F * 1024), fw, lane); };
  // The second kind in two parts: K by columns at the top of a piece, T and P behind its barrier 2, so that the next piece's
  // first kind, which has to have landed by barrier 3, waits for less (one part: 89 us against 86 when it was chosen, b 4, H 16, L 2048).
  constexpr int GB1 = NP * F + 1, GB2 = TPF;
  auto b_of = [&](int c) { return lds + (AB * GA + (AHEAD ? (c & 1) * GB : 0)) * FR; };
  auto fetch_b2 = [&](int c) {
    if (FW < 8 || fw < 4) fetch_share<TPF, (FW < 4 ? FW : 4)>(b_of(c) + NP * F * FR, p.workspace + lay.tp + (vunit0 + c) * lay.tp_unit, fw, lane);
  };
  auto fetch_b1 = [&](int c) {
    lds_f16_t* to = b_of(c);
    fetch_share<NP * F, FW>(to, p.workspace + lay.kq + (kunit0 + c) * lay.kq_unit + 2 * NP * F * 1024, fw, lane);
    if (fw == 0) fetch_share<1, 1>(to + (NP * F + TPF) * FR, p.workspace + lay.vec + (vunit0 + c) * (int64_t)(kVecFloats * 4), 0, lane);
  };
  if constexpr (AHEAD) {
    if (w == 2 * PAIRS) {
      fetch_a(c0);
      fetch_b1(c0);
      fetch_b2(c0);
      wait_vmem_n<GB>();
      lds_barrier();
      for (int c = c0; c < c1; ++c) {            // the next piece's, each where what was there has been read
        const bool more = c + 1 < c1;
        if (more) {
          if (AB == 2) fetch_a(c + 1);
          fetch_b1(c + 1);
          wait_vmem_n<(AB == 2 ? GA : 0) + GB1>();                     // T, P and K by columns of this piece
        } else {
          wait_vmem();
        }
        lds_barrier();                           // 1
        if (AB == 1 && more) fetch_a(c + 1);
        lds_barrier();                           // 2
        if (more) {
          fetch_b2(c + 1);
          wait_vmem_n<(AB == 2 ? GB1 : 0) + GB2>();                    // K and Q by rows of the next piece
        }
        lds_barrier();                           // 3
      }
      lds_barrier();
      return;
    }
    if (w > 2 * PAIRS) {
      const int io = w - 2 * PAIRS - 1, col0 = IOC * (IOW * wg + io), left = unit ? 0 : p.dv - col0;
      const bf16* vs = reinterpret_cast<const bf16*>(p.v) + b * p.vs.b + h * p.vs.h + col0;
      bf16* os = reinterpret_cast<bf16*>(p.o) + b * p.os.b + h * p.os.h + col0;
      bf16* const to = sV + io * IOH;
      auto run = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        IoRows<IOC> v, o;
        auto load_v = [&](int c) {               // tokens beyond the sequence as its last: their gates are zero
          const int t = min(c * DC + lane, p.seqlen - 1);
          v.template load<FULL>(vs + t * p.vs.l, left);
        };
        auto store_o = [&](int c, bool row) {
          o.from_lds(sO + io * IOH, lane);
          o.template store<FULL>(os + (c * DC + lane) * p.os.l, row, left);
        };
        Warm warm;
        auto warm_up = [&](int c) {
          c = min(c, c1 - 1);
          warm.template load<(OUT ? 3 : 2) * F, TPF>(p.workspace + lay.kq + (kunit0 + c) * lay.kq_unit + (OUT ? 0 : F * 1024),
                                                     p.workspace + lay.tp + (vunit0 + c) * lay.tp_unit,
                                                     p.workspace + lay.vec + (vunit0 + c) * (int64_t)(kVecFloats * 4), wg, nwg, lane);
        };
        if (PAIRS == 1) warm_up(c0 + 2);
        load_v(c0);
        v.to_lds(to + (c0 & 1) * IOW * IOH, lane);
        load_v(c0 + 1);
        lds_barrier();
        for (int c = c0; c < c1; ++c) {
          lds_barrier();                         // 1
          v.to_lds(to + ((c + 1) & 1) * IOW * IOH, lane);
          load_v(c + 2);
          if (PAIRS == 1) {
            warm.done();
            warm_up(c + 3);
          }
          if (OUT && c > c0) store_o(c - 1, true);
          lds_barrier();                         // 2
          lds_barrier();                         // 3
        }
        lds_barrier();                           // the last piece's o is whole
        if (OUT) store_o(c1 - 1, (c1 - 1) * DC + lane < p.seqlen);
      };
      if (left >= IOC) run(std::true_type{});
      else run(std::false_type{});
      return;
    }
  }
  const int blk = PAIRS * (unit ? wg - nv : wg) + (w >> 1), col = 16 * blk + l16, cols = unit ? p.dk : p.dv;
  const bool live = 16 * blk < cols, cv = col < cols;                // a pair beyond the last columns has zeros
  f16* ex = smem + (AB * GA + (AHEAD ? 2 : 1) * GB) * FR + (w >> 1) * EX;
  f32x4* const xSend = reinterpret_cast<f32x4*>(ex) + hf * XF * 64 + lane;             // X (and Y) of the other's tokens
  const f32x4* const xRecv = reinterpret_cast<const f32x4*>(ex) + (1 - hf) * XF * 64 + lane;
  f16* const eR = ex + 2 * XF * FR;                                                    // the first half's R
  f16* const eU = eR + 2 * FR;                                                         // U, two parts of each half
  // the first half's delta, where the second wave's X was: the first one has read that before barrier 2, and the second
  // one, which reads delta behind barrier 3, writes its next X itself
  f16* const eD = ex + XF * FR;
  float* const eS = reinterpret_cast<float*>(eU + 4 * FR);                             // scales: R, D, U of each half

  const int64_t states = (int64_t)p.dk * p.dv;   // elements of a state
  float* const seg_states = reinterpret_cast<float*>(p.workspace + lay.seg_states) + (int64_t)bh * lay.segs * states;
  const float* entry = seg > 0 ? (MOVE ? nullptr : seg_states + (seg - 1) * states) : p.initial_state ? p.initial_state + bh * states : nullptr;
  f32x4 S[NSH];                                  // rows DKP / 2 hf + 16 n + 4 g4 + r, column col
#pragma unroll
  for (int n = 0; n < NSH; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = DKP / 2 * hf + 16 * n + 4 * g4 + r;
      if (unit) S[n][r] = row == col && cv ? 1.f : 0.f;
      else S[n][r] = entry && cv && row < p.dk ? entry[(int64_t)row * p.dv + col] : 0.f;
    }
  T vn[8];
  auto load_v = [&](int c) {                     // a half that lies beyond the sequence reads the last token
    const int t = min(c * DC + 32 * hf, p.seqlen - 1);
    const T* vsrc = reinterpret_cast<const T*>(p.v) + b * p.vs.b + h * p.vs.h + (live && !unit ? 16 * blk : 0);
    load_rows8<T>(vsrc + t * p.vs.l, p.vs.l, p.seqlen - t, cv && !unit, !unit && 16 * blk + 16 <= p.dv, l16, g4, vn);
  };
  if (AHEAD) lds_barrier();
  else load_v(c0);

  const f16 *Qr = smem, *Kr = smem + (OUT ? NP * F * FR : 0);        // AB == 1: of the one piece there is
  f16x8 ka[KSH][4], qa[OUT ? KSH : 1][4];        // the next piece's; tiles 0, 1: one's own tokens, 2, 3: the other's
  auto load_a = [&](int c) {
    const int at = AB == 2 ? (c & 1) * GA : 0;
#pragma unroll
    for (int s = 0; s < KSH; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) ka[s][i] = frag(Kr, at + ((2 * hf + i) & 3) * KS + hf * KSH + s, lane);
    if constexpr (OUT)
#pragma unroll
      for (int s = 0; s < KSH; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) qa[s][i] = frag(Qr, at + ((2 * hf + i) & 3) * KS + hf * KSH + s, lane);
  };
  if (AHEAD) load_a(c0);

  for (int c = c0; c < c1; ++c) {
    if (!AHEAD) {
      lds_barrier();
      fetch_a(c);
      fetch_b1(c);
      fetch_b2(c);
      wait_vmem();
      lds_barrier();
      load_a(c);
    }
    const f16 *Kc = smem + (AB * GA + (AHEAD ? (c & 1) * GB : 0)) * FR, *Tt = Kc + NP * F * FR, *Pt = Tt + 2 * kTFrags * FR;
    const float* vec = reinterpret_cast<const float*>(Tt + TPF * FR);
    f16x8 sh[KSH], sl[KSH];
    f32x4 X[4] = {}, Y[4] = {};
    const Scale ss(col_max(abs_max(S)));
    parts_of<2>(S, ss.mult, sh, sl);
#pragma unroll
    for (int s = 0; s < KSH; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) X[i] = mma_h(ka[s][i], sh[s], X[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) X[i] = mma_h(ka[s][i], sl[s], X[i]);
      if constexpr (NP == 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) X[i] = mma_h(frag(Kr, F + ((2 * hf + i) & 3) * KS + hf * KSH + s, lane), sh[s], X[i]);
    }
    if constexpr (OUT)
#pragma unroll
      for (int s = 0; s < KSH; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          Y[i] = mma_h(qa[s][i], sh[s], Y[i]);
          Y[i] = mma_h(qa[s][i], sl[s], Y[i]);
          if constexpr (NP == 2) Y[i] = mma_h(frag(Qr, F + ((2 * hf + i) & 3) * KS + hf * KSH + s, lane), sh[s], Y[i]);
        }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xSend[i * 64] = X[2 + i] * ss.inv;
      if constexpr (OUT) xSend[(2 + i) * 64] = Y[2 + i] * ss.inv;
    }
    f16* keep = nullptr;
    float* scales = nullptr;
    if constexpr (KEEP) {                        // stored where they are made: held to the end they would spill
      const int64_t at = (vunit0 + c) * nblk + blk;
      keep = reinterpret_cast<f16*>(p.workspace + lay.keep) + at * keep_halfs<DKP>();
      scales = reinterpret_cast<float*>(p.workspace + lay.scales) + at * kScales + 32 * hf + l16;
      if (live) {
        keep_parts<KS>(keep, hf * KSH, sh, sl, lane);
        if (g4 == 0) scales[0] = ss.inv;
      }
    }
    lds_barrier();                               // 1
    f32x4 xr[2], yr[2], eg[2], wt[2];
    bf16x4 vb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xr[i] = xRecv[i * 64];
      eg[i] = *reinterpret_cast<const f32x4*>(vec + 32 * hf + 16 * i + 4 * g4);
      if constexpr (AHEAD)
        vb[i] = *reinterpret_cast<const bf16x4*>(sV + (c & 1) * IOW * IOH + ((w >> 1) * 16 + l16) * IO_PITCH + 32 * hf + 16 * i + 4 * g4);
    }
    const f32x4 cs = *reinterpret_cast<const f32x4*>(vec + VEC_GAMMA);                 // gamma, scales of T, P, K
    f16x8 t0[2], t1[2], x0[2], x1[2];            // T on one's own tokens; on the first half's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t0[i] = frag(Tt, t_frag(2 * hf + i, hf), lane);
      t1[i] = frag(Tt, kTFrags + t_frag(2 * hf + i, hf), lane);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x0[i] = frag(Tt, t_frag(2 + i, 0), lane);
      x1[i] = frag(Tt, kTFrags + t_frag(2 + i, 0), lane);
      wt[i] = *reinterpret_cast<const f32x4*>(vec + VEC_W + 32 * hf + 16 * i + 4 * g4);
      if constexpr (OUT) yr[i] = xRecv[(2 + i) * 64];
    }
    const float sQ = vec[VEC_SQ];
    __builtin_amdgcn_sched_barrier(0);
    f32x4 R[2], D[2] = {}, E[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = AHEAD ? (float)vb[i][r] : to_f32(vn[4 * i + r]);
        R[i][r] = __builtin_fmaf(-eg[i][r], cs[3] * __builtin_fmaf(ss.inv, X[i][r], xr[i][r]), v);
      }
    if (!AHEAD && c + 1 < c1) load_v(c + 1);
    // delta = T R: one's own tokens, and for the second wave those of the first
    f16x8 rh[1], rl[1];
    const Scale sr(col_max(abs_max(R)));
    parts_of<2>(R, sr.mult, rh, rl);
    if (hf == 0) {
      put_frag(eR, 0, lane, rh[0]);
      put_frag(eR, 1, lane, rl[0]);
      eS[lane] = sr.inv;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) D[i] = mma_h(t0[i], rh[0], D[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) D[i] = mma_h(t0[i], rl[0], D[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) D[i] = mma_h(t1[i], rh[0], D[i]);
    lds_barrier();                               // 2
    float rs = sr.inv;
    const f16x8 r0 = frag(eR, 0, lane), r1 = frag(eR, 1, lane);
    const float es = eS[lane];
    f16x8 kc[NSH][2], pa[2], px[2];              // K by columns, one's own tokens first; P as T
#pragma unroll
    for (int n = 0; n < NSH; ++n) {
      kc[n][0] = frag(Kc, 2 * (hf * NSH + n) + hf, lane);
      kc[n][1] = frag(Kc, 2 * (hf * NSH + n) + 1 - hf, lane);
    }
    if constexpr (OUT)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        pa[i] = frag(Pt, t_frag(2 * hf + i, hf), lane);
        px[i] = frag(Pt, t_frag(2 + i, 0), lane);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (hf == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x0[i], r0, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x0[i], r1, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] = mma_h(x1[i], r0, E[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) D[i][r] = __builtin_fmaf(es, E[i][r], rs * D[i][r]);
      rs = 1.f;
    }
    const float ds = rs * cs[1];                 // of D, and of U until it leaves its own scale
    f32x4 U[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) U[i][r] = wt[i][r] * D[i][r];
    f16x8 wh[1], wl[1], dh[1], dl[1];
    const Scale su(col_max(abs_max(U)));
    parts_of<2>(U, su.mult, wh, wl);
    const float own_us = su.inv * ds * cs[3];
    put_frag(eU, 2 * hf, lane, wh[0]);
    put_frag(eU, 2 * hf + 1, lane, wl[0]);
    eS[(2 + hf) * 64 + lane] = own_us;
    const Scale sd(col_max(abs_max(D)));
    parts_of<KEEP || OUT ? 2 : 1>(D, sd.mult, dh, dl);
    if constexpr (KEEP)
      if (live) {
        keep_parts<2>(keep + kTokens<DKP>, hf, dh, dl, lane);
        if (g4 == 0) scales[16] = sd.inv * ds;
      }
    if constexpr (OUT)
      if (hf == 0) {
        put_frag(eD, 0, lane, dh[0]);
        put_frag(eD, 1, lane, dl[0]);
        eS[64 + lane] = sd.inv * ds;
      }
    lds_barrier();                               // 3
    const f16x8 oh = frag(eU, 2 - 2 * hf, lane), ol = frag(eU, 3 - 2 * hf, lane);
    const float other_us = eS[(3 - hf) * 64 + lane];
    f16x8 d0, d1;
    float od = 0.f;
    if constexpr (OUT) {
      d0 = frag(eD, 0, lane);
      d1 = frag(eD, 1, lane);
      od = eS[64 + lane];
    }
    if (AHEAD && c + 1 < c1) load_a(c + 1);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 u0[NSH] = {}, u1[NSH] = {};
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(kc[n][0], wh[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u0[n] = mma_h(kc[n][0], wl[0], u0[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(kc[n][1], oh, u1[n]);
#pragma unroll
    for (int n = 0; n < NSH; ++n) u1[n] = mma_h(kc[n][1], ol, u1[n]);
    if constexpr (NP == 2)
#pragma unroll
      for (int n = 0; n < NSH; ++n) {
        u0[n] = mma_h(frag(Kc, F + 2 * (hf * NSH + n) + hf, lane), wh[0], u0[n]);
        u1[n] = mma_h(frag(Kc, F + 2 * (hf * NSH + n) + 1 - hf, lane), oh, u1[n]);
      }
#pragma unroll
    for (int n = 0; n < NSH; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[n][r] = __builtin_fmaf(other_us, u1[n][r], __builtin_fmaf(own_us, u0[n][r], cs[0] * S[n][r]));
    if constexpr (OUT) {
      f32x4 O[2] = {}, OX[2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        O[i] = mma_h(pa[i], dh[0], O[i]);
        O[i] = mma_h(pa[i], dl[0], O[i]);
        O[i] = mma_h(frag(Pt, kTFrags + t_frag(2 * hf + i, hf), lane), dh[0], O[i]);
      }
      if (hf == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          OX[i] = mma_h(px[i], d0, OX[i]);
          OX[i] = mma_h(px[i], d1, OX[i]);
          OX[i] = mma_h(frag(Pt, kTFrags + t_frag(2 + i, 0), lane), d0, OX[i]);
        }
      }
      const float os = sd.inv * ds * cs[2], ox = od * cs[2];           // powers of two, exact also below fp32's normal range
      float o[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          o[4 * i + r] = __builtin_fmaf(eg[i][r], sQ * __builtin_fmaf(ss.inv, Y[i][r], yr[i][r]), os * O[i][r]);
          if (hf == 1) o[4 * i + r] = __builtin_fmaf(ox, OX[i][r], o[4 * i + r]);
          o[4 * i + r] *= p.scale;
        }
      if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<bf16x4*>(sO + ((w >> 1) * 16 + l16) * IO_PITCH + 32 * hf + 16 * i + 4 * g4) =
              bf16x4{(bf16)o[4 * i], (bf16)o[4 * i + 1], (bf16)o[4 * i + 2], (bf16)o[4 * i + 3]};
      } else {
        const int t = c * DC + 32 * hf;
        store_rows8<T>(reinterpret_cast<T*>(p.o) + b * p.os.b + h * p.os.h + t * p.os.l + 16 * blk, p.os.l, p.seqlen - t, cv, l16, g4, o);
      }
    }
  }
  if (AHEAD) lds_barrier();
  float* out = MOVE ? seg_states + seg * states : seg == lay.segs - 1 && p.final_state ? p.final_state + bh * states : nullptr;
  if (unit) {                                    // by columns, as the segments' kernel reads it
    float* trans = reinterpret_cast<float*>(p.workspace + lay.seg_trans) + ((int64_t)bh * lay.segs + seg) * DKP * DKP + (int64_t)col * DKP;
    if (cv)
#pragma unroll
      for (int n = 0; n < NSH; ++n) *reinterpret_cast<f32x4*>(trans + DKP / 2 * hf + 16 * n + 4 * g4) = S[n];
  } else if (out && cv) {
#pragma unroll
    for (int n = 0; n < NSH; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = DKP / 2 * hf + 16 * n + 4 * g4 + r;
        if (row < p.dk) out[(int64_t)row * p.dv + col] = S[n][r];
      }
  }
}

// The states that the segments begin with, S_{s+1} = M_s S_s + N_s, where the scan has left N_s (segment 0: S_1 itself) and
// M_s: a workgroup takes 16 columns from segment to segment, a wave 16 rows of them by fp32 matrix instructions.  M_s does
// not wait for a state: those of the next two segments are under way (8 heads of 128 x 128, 8 segments: 55 us with the rows
// a thread each and M read where it is used, 33 with one segment under way, now 24).
template <int DKP>
__global__ __launch_bounds__(4 * DKP) void delta_segments_kernel(DeltaParams p, DeltaLayout lay) {
  __shared__ float sS[2][DKP][16];
  const int lane = threadIdx.x & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  const int nblk = (p.dv + 15) / 16, bh = blockIdx.x / nblk, col = blockIdx.x % nblk * 16 + l16;
  const int64_t states = (int64_t)p.dk * p.dv;
  const int row0 = 16 * w + 4 * g4;
  float* const at = reinterpret_cast<float*>(p.workspace + lay.seg_states) + (int64_t)bh * lay.segs * states + (int64_t)row0 * p.dv + col;
  const float* const M = reinterpret_cast<const float*>(p.workspace + lay.seg_trans) + (int64_t)bh * lay.segs * DKP * DKP + g4 * DKP + 16 * w + l16;
  auto state_of = [&](int s) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = s < lay.segs - 1 && col < p.dv && row0 + r < p.dk ? at[s * states + r * p.dv] : 0.f;
    return v;
  };
  float m[2][DKP / 4];                           // k = 4 i + g4; of this segment and the next
  f32x4 N[2], S = state_of(0);
  auto load = [&](int s, int x) {
#pragma unroll
    for (int i = 0; i < DKP / 4; ++i) m[x][i] = s < lay.segs - 1 && 4 * i + g4 < p.dk ? M[(int64_t)s * DKP * DKP + 4 * i * DKP] : 0.f;
    N[x] = state_of(s);
  };
  auto step = [&](int s, int x) {
    float(*t)[16] = sS[x];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[row0 + r][l16] = S[r];
    __syncthreads();
    float b[DKP / 4];
#pragma unroll
    for (int i = 0; i < DKP / 4; ++i) b[i] = t[4 * i + g4][l16];
    f32x4 acc[2] = {N[x], {}};
#pragma unroll
    for (int i = 0; i < DKP / 4; ++i) acc[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[x][i], b[i], acc[i & 1], 0, 0, 0);
    S = acc[0] + acc[1];
    load(s + 2, x);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col < p.dv && row0 + r < p.dk) at[s * states + r * p.dv] = S[r];
  };
  load(1, 0);
  load(2, 1);
  for (int s = 1; s < lay.segs - 1; s += 2) {
    step(s, 0);
    if (s + 1 < lay.segs - 1) step(s + 1, 1);
  }
}

template <typename T, int DKP, bool OUT, bool KEEP, int PAIRS>
hipError_t launch_scan_of(const DeltaParams& p, const DeltaLayout& lay, hipStream_t st) {
  const int nblk = (p.dv + 15) / 16, nwg = (nblk + PAIRS - 1) / PAIRS + (OUT || KEEP ? 0 : ((p.dk + 15) / 16 + PAIRS - 1) / PAIRS);
  const int parts = p.batch * p.heads * (OUT || KEEP ? lay.segs : lay.segs - 1);
  delta_scan_kernel<T, DKP, OUT, KEEP, PAIRS><<<head_block_grid(parts, nwg), kDeltaThreads<T, PAIRS>, 0, st>>>(p, lay, nblk, nwg);
  return hipGetLastError();
}
template <typename T, int DKP, bool OUT, bool KEEP>
hipError_t launch_scan(const DeltaParams& p, const DeltaLayout& lay, hipStream_t st) {
  if constexpr (!OUT && !KEEP) return launch_scan_of<T, DKP, false, false, 4>(p, lay, st);       // without o four pairs fit the LDS
  else if constexpr (sizeof(T) == 2)
    if (delta_one_pair(p, lay.segs)) return launch_scan_of<T, DKP, OUT, KEEP, 1>(p, lay, st);
  return launch_scan_of<T, DKP, OUT, KEEP, (OUT || KEEP ? 2 : 4)>(p, lay, st);
}
template <typename T, int DKP>
hipError_t launch_segments(const DeltaParams& p, const DeltaLayout& lay, hipStream_t st) {
  if (lay.segs == 1) return hipSuccess;
  const hipError_t e = launch_scan<T, DKP, false, false>(p, lay, st);
  if (e != hipSuccess) return e;
  delta_segments_kernel<DKP><<<(unsigned)(p.batch * p.heads * ((p.dv + 15) / 16)), 4 * DKP, 0, st>>>(p, lay);
  return hipGetLastError();
}
template <typename T, int DKP>
hipError_t run_scan(const DeltaParams& p, const DeltaLayout& lay, bool out, bool keep, hipStream_t st) {
  const hipError_t e = launch_segments<T, DKP>(p, lay, st);
  if (e != hipSuccess) return e;
  return !out ? launch_scan<T, DKP, false, true>(p, lay, st) : keep ? launch_scan<T, DKP, true, true>(p, lay, st) : launch_scan<T, DKP, true, false>(p, lay, st);
}
hipError_t scan(const DeltaParams& p, bool out, bool keep, hipStream_t st) {
  const DeltaLayout lay(p, keep);
  if (p.dtype == DT_F32) return p.dk <= 64 ? run_scan<float, 64>(p, lay, out, keep, st) : run_scan<float, 128>(p, lay, out, keep, st);
  return p.dk <= 64 ? run_scan<bf16, 64>(p, lay, out, keep, st) : run_scan<bf16, 128>(p, lay, out, keep, st);
}

template <typename T>
hipError_t run_prep(const DeltaParams& p, const DeltaLayout& lay, bool backward, hipStream_t st) {
  const unsigned grid = (unsigned)((int64_t)p.batch * p.kheads * p.pieces);
  if (p.dk <= 64) delta_prep_kernel<T, 64><<<grid, 256, 0, st>>>(p, lay, backward);
  else delta_prep_kernel<T, 128><<<grid, 256, 0, st>>>(p, lay, backward);
  return hipGetLastError();
}

// A sequence of no tokens: the state goes through.
__global__ void delta_copy_state_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = grid_row() * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

}  // namespace

// A sequence of few heads leaves most CUs idle while it goes from piece to piece.  It is then cut into segments: a scan
// without o finds what each makes of no state (N) and of the identity's columns (M), delta_segments_kernel goes from segment
// to segment, and the scan with o takes all segments at once.  The segments' number is the one with the least time by this
// count, in tenths of a piece's time (o and all: 10, without o: 9; a segment's product: 10); a gain of less than a fifth is
// left.  H 8, L 32768 of 128 x 128 (bf16): 8 segments, 180 + 24 + 198 us where the scan in one went 1205.
int delta_segments(const DeltaParams& p) {
  const int64_t heads = (int64_t)p.batch * p.heads, nblk = (p.dv + 15) / 16, kblk = (p.dk + 15) / 16;
  const int64_t whole = heads * ((nblk + 1) / 2), move = heads * ((nblk + 3) / 4 + (kblk + 3) / 4);
  auto rounds = [](int64_t n) { return (n + kCUs - 1) / kCUs; };
  int64_t best = 1, least = p.pieces * rounds(whole) * 8;
  for (int64_t n = 2; n <= 64 && 4 * n <= p.pieces; ++n) {
    const int64_t per = (p.pieces + n - 1) / n;
    if ((p.pieces + per - 1) / per != n) continue;
    const int64_t cost = per * (9 * rounds(move * (n - 1)) + 10 * rounds(whole * n)) + 10 * n + 40;
    if (cost < least) least = cost, best = n;
  }
  return (int)best;
}

size_t delta_workspace_bytes(const DeltaParams& p) { return DeltaLayout(p, p.keep).total; }

hipError_t launch_delta_prep(const DeltaParams& p, bool backward, hipStream_t st) {
  const DeltaLayout lay(p, backward);
  return p.dtype == DT_F32 ? run_prep<float>(p, lay, backward, st) : run_prep<bf16>(p, lay, backward, st);
}

hipError_t launch_delta_keep(const DeltaParams& p, hipStream_t st) { return scan(p, false, true, st); }

hipError_t launch_delta(const DeltaParams& p, hipStream_t st) {
  if (p.seqlen == 0) {
    const int64_t n = (int64_t)p.batch * p.heads * p.dk * p.dv;
    if (!p.final_state) return hipSuccess;
    delta_copy_state_kernel<<<row_grid((n + 255) / 256, 1), 256, 0, st>>>(p.initial_state, p.final_state, n);
    return hipGetLastError();
  }
  const hipError_t e = launch_delta_prep(p, p.keep, st);
  if (e != hipSuccess) return e;
  return scan(p, true, p.keep, st);
}

}  // namespace mh
