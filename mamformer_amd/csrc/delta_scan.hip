// Gated delta rule over sequences:
//   S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - e^{g_t} S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t.
// In pieces of 64 tokens, G the inclusive sum of g in the piece and S the state that enters it:
//   delta = T (V - e^G K S),   T = (I + A)^-1,  A_tj = e^{G_t - G_j} (k_t k_j) beta_j for j < t
//   O     = scale (e^G Q S + P delta),          P_tj = e^{G_t - G_j} (q_t k_j) beta_j for j <= t
//   S'    = e^{G_end} S + (beta e^{G_end - G} K)^T delta
// delta is what each token corrects before its beta, so that beta = 0 divides nothing.  delta_prep_kernel makes T and P of
// every piece side by side; delta_scan_kernel walks the pieces with the state in registers.
#include "delta.h"

namespace mh {
namespace {

// ------------------------------------------------------------------ pieces side by side
// One workgroup of 4 waves for a piece of a key head: K and Q into their fp16 parts (kept for the scan), K K^T and Q K^T
// once (wave w: rows 16 w .. 16 w + 15, tiles up to the diagonal), then for each value head that shares them A, its
// inverse and P.  The inverse in fp32: every wave solves one 16 x 16 diagonal block by substitution, a column a lane, then
// wave j builds block column j downwards, T_ij = -T_ii sum_k A_ik T_kj, with fp32 matrix instructions, T_kj staying in
// accumulators, which are the B operand of the next product.
template <typename T, int DKP>
__global__ __launch_bounds__(256) void delta_prep_kernel(DeltaParams p, DeltaLayout lay, int p_planes) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int CPR = DKP / 8;                   // threads of 8 channels for a row
  constexpr int RPP = 256 / CPR;                 // rows of a pass
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int AP = 68;                         // pitch of A and of the diagonal blocks' inverses
  __shared__ __align__(16) f16 tiles[2 * NP * TK::ELEMS > 4 * TC::ELEMS ? 2 * NP * TK::ELEMS : 4 * TC::ELEMS];
  __shared__ __align__(16) float sA[DC * AP];
  __shared__ __align__(16) float sD[4 * 16 * 20];
  __shared__ double sG[DC];
  __shared__ float sB[DC], sVec[2 * DC], red[4][2];

  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  const int64_t unit = blockIdx.x;               // (batch, key head, piece)
  const int c = (int)(unit % p.pieces), bk = (int)(unit / p.pieces), hk = bk % p.kheads, b = bk / p.kheads;
  const int t0 = c * DC, len = min(DC, p.seqlen - t0), rep = p.heads / p.kheads;

  // K and Q: largest magnitudes, then parts into the tiles
  Raw8<T> raw[2][DC / RPP];
  const int cc = tid % CPR, rr = tid / CPR;
  const T* src[2] = {reinterpret_cast<const T*>(p.k) + b * p.ks.b + hk * p.ks.h + (int64_t)t0 * p.ks.l + cc * 8,
                     reinterpret_cast<const T*>(p.q) + b * p.qs.b + hk * p.qs.h + (int64_t)t0 * p.qs.l + cc * 8};
  const int64_t sl[2] = {p.ks.l, p.qs.l};
  float amax[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < DC / RPP; ++i) {
      const int r = i * RPP + rr;
      if (r < len && cc * 8 < p.dk) load_raw(raw[x][i], src[x] + r * sl[x], p.dk - cc * 8);
      else raw[x][i].clear();
    }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int i = 0; i < DC / RPP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) amax[x] = fmaxf(amax[x], fabsf(raw[x][i].get(j)));
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
      const int r = i * RPP + rr;
      const float mult = x ? sq.mult : sk.mult;
      f16x8 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = raw[x][i].get(j);
        hi[j] = part_hi(v, mult);
        if constexpr (NP == 2) lo[j] = part_lo(v, mult, hi[j]);
      }
      f16* to = tiles + x * NP * TK::ELEMS + TK::at(r, cc * 8);
      *reinterpret_cast<f16x8*>(to) = hi;
      if constexpr (NP == 2) *reinterpret_cast<f16x8*>(to + TK::ELEMS) = lo;
    }
  __syncthreads();
  {
    uint4* out = reinterpret_cast<uint4*>(p.workspace + lay.kq) + unit * (2 * NP * TK::ELEMS / 8);
    for (int i = tid; i < 2 * NP * TK::ELEMS / 8; i += 256) out[i] = reinterpret_cast<const uint4*>(tiles)[i];
  }
  // rows 16 w .. of K K^T and Q K^T, tiles j <= w
  f32x4 kk[4] = {}, qk[4] = {};
#pragma unroll
  for (int s = 0; s < DKP / 32; ++s) {
    f16x8 ka[NP], qa[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      ka[n] = row_frag16<DKP>(tiles + n * TK::ELEMS, 16 * w, 32 * s, lane);
      qa[n] = row_frag16<DKP>(tiles + (NP + n) * TK::ELEMS, 16 * w, 32 * s, lane);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w) continue;
      const f16x8 kb = row_frag16<DKP>(tiles, 16 * j, 32 * s, lane);
      kk[j] = mma_h(ka[0], kb, kk[j]);
      qk[j] = mma_h(qa[0], kb, qk[j]);
      if constexpr (NP == 2) {
        const f16x8 kl = row_frag16<DKP>(tiles + TK::ELEMS, 16 * j, 32 * s, lane);
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
      kk[j][r] = kk[j][r] * sk.inv * sk.inv;
      qk[j][r] = qk[j][r] * sq.inv * sk.inv;
    }

  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const int64_t vunit = ((int64_t)b * p.heads + h) * p.pieces + c;
    __syncthreads();                             // the tiles and the last head's parts have been read
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
      sVec[lane] = expf((float)G);
      sVec[DC + lane] = bv * expf((float)(end - G));
    }
    __syncthreads();
    double Gt[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) Gt[r] = sG[16 * w + 4 * g4 + r];
    f32x4 P[4] = {};
    float pmax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w) continue;
      const double Gj = sG[16 * j + l16];
      const float bj = sB[16 * j + l16];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int below = 16 * (w - j) + 4 * g4 + r - l16;               // t - j
        const float d = below >= 0 ? expf((float)(Gt[r] - Gj)) * bj : 0.f;
        P[j][r] = below >= 0 ? qk[j][r] * d : 0.f;
        pmax = fmaxf(pmax, fabsf(P[j][r]));
        sA[(16 * w + 4 * g4 + r) * AP + 16 * j + l16] = below > 0 ? kk[j][r] * d : 0.f;
      }
    }
    __syncthreads();
    // diagonal block w, a column a lane (the four groups of 16 lanes do the same)
    {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == l16 ? 1.f : 0.f;
#pragma unroll
        for (int j4 = 0; j4 < (i + 3) / 4; ++j4) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(sA + (16 * w + i) * AP + 16 * w + 4 * j4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * j4 + j < i) s -= a[j] * x[4 * j4 + j];
        }
        x[i] = s;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (g4 == i >> 2) sD[(w * 16 + i) * 20 + l16] = x[i];
    }
    __syncthreads();
    // block column w downwards
    f32x4 t[4] = {};
#pragma unroll
    for (int r = 0; r < 4; ++r) t[0][r] = sD[(w * 16 + 4 * g4 + r) * 20 + l16];      // t[n]: block row w + n
#pragma unroll
    for (int n = 1; n < 4; ++n) {
      if (w + n > 3) continue;
      f32x4 m = {};
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(sA + (16 * (w + n) + l16) * AP + 16 * (w + k) + 4 * g4);
#pragma unroll
        for (int s = 0; s < 4; ++s) m = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], t[k][s], m, 0, 0, 0);
      }
      const f32x4 d = *reinterpret_cast<const f32x4*>(sD + ((w + n) * 16 + l16) * 20 + 4 * g4);
      f32x4 y = {};
#pragma unroll
      for (int s = 0; s < 4; ++s) y = __builtin_amdgcn_mfma_f32_16x16x4f32(d[s], m[s], y, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) t[n][r] = -y[r];
    }
    const float tm = wave_max(abs_max(t)), pm = wave_max(pmax);
    if (lane == 0) {
      red[w][0] = tm;
      red[w][1] = pm;
    }
    __syncthreads();
    const Scale st(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
    const Scale sp(fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1])));
#pragma unroll
    for (int i = 0; i < 4; ++i)                  // T: block rows i of block column w; P: block columns i of block row w
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (i == w + n) v = t[n][r];
        const int at = TC::at(16 * i + 4 * g4 + r, 16 * w + l16), pt = TC::at(16 * w + 4 * g4 + r, 16 * i + l16);
        const f16 th = part_hi(v, st.mult), ph = part_hi(P[i][r], sp.mult);
        tiles[at] = th;
        tiles[TC::ELEMS + at] = part_lo(v, st.mult, th);
        tiles[2 * TC::ELEMS + pt] = ph;
        if (p_planes == 2) tiles[3 * TC::ELEMS + pt] = part_lo(P[i][r], sp.mult, ph);
      }
    __syncthreads();
    uint4* out = reinterpret_cast<uint4*>(p.workspace + lay.tp) + vunit * (4 * TC::ELEMS / 8);
    for (int i = tid; i < (2 + p_planes) * TC::ELEMS / 8; i += 256) out[i] = reinterpret_cast<const uint4*>(tiles)[i];
    float* vec = reinterpret_cast<float*>(p.workspace + lay.vec) + vunit * kVecFloats;
    if (tid < 2 * DC) vec[tid] = sVec[tid];
    if (tid == 2 * DC) {
      vec[VEC_W + DC] = sVec[DC - 1];
      vec[VEC_ST] = st.inv;
      vec[VEC_SP] = sp.inv;
      vec[VEC_SK] = sk.inv;
      vec[VEC_SQ] = sq.inv;
    }
  }
}

// ------------------------------------------------------------------ the state from piece to piece
// A wave holds 16 columns of the state (dk x 16, fp32) and runs the whole recurrence for them without exchanging anything
// with another; the NW waves of a workgroup read the same tiles, fetched by LDS DMA one piece ahead (NBUF = 2).
// KEEP: the entering states and delta are stored for the backward.  OUT: o is computed.
template <typename T, int DKP, int NW, bool OUT, bool KEEP>
__global__ __launch_bounds__(64 * NW) void delta_scan_kernel(DeltaParams p, DeltaLayout lay, int nblk, int nwg) {
  constexpr int NP = sizeof(T) == 4 ? 2 : 1;
  constexpr int NBUF = NP == 1 ? 2 : 1;
  using TK = HTile<DKP>;
  using TC = HTile<64>;
  constexpr int KQ = (OUT ? 2 : 1) * NP * TK::ELEMS;                 // halfs of K (and Q)
  constexpr int TP = (2 + (OUT ? NP : 0)) * TC::ELEMS;               // halfs of T (and P)
  constexpr int BUF = KQ + TP + kVecFloats * 2;                      // halfs of a buffer
  constexpr int NS = DKP / 16, KS = DKP / 32;
  __shared__ __align__(1024) f16 smem[NBUF * BUF];

  const int lane = threadIdx.x & 63, w = wave_id(), l16 = lane & 15, g4 = lane >> 4;
  int bh, wg;
  if (!head_block(blockIdx.x, p.batch * p.heads, nwg, bh, wg)) return;
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kheads);
  const int blk = wg * NW + w, col = 16 * blk + l16;
  const bool live = blk < nblk, cv = col < p.dv;
  const int64_t kunit0 = ((int64_t)b * p.kheads + hk) * p.pieces, vunit0 = (int64_t)bh * p.pieces;

  auto fetch = [&](int c, int buf) {             // 1 KB blocks, the waves in turn
    char* to = reinterpret_cast<char*>(smem + buf * BUF);
    const char* kq = p.workspace + lay.kq + (kunit0 + c) * (int64_t)(2 * NP * TK::ELEMS * 2);
    const char* tp = p.workspace + lay.tp + (vunit0 + c) * (int64_t)(4 * TC::ELEMS * 2);
    const char* vec = p.workspace + lay.vec + (vunit0 + c) * (int64_t)(kVecFloats * 4);
#pragma unroll
    for (int q = w; q < KQ / 512; q += NW) dma_lds<16>(kq + q * 1024, 16u * lane, to + q * 1024);
#pragma unroll
    for (int q = w; q < TP / 512; q += NW) dma_lds<16>(tp + q * 1024, 16u * lane, to + KQ * 2 + q * 1024);
    if (w == 0) dma_lds<16>(vec, 16u * lane, to + (KQ + TP) * 2);
  };

  f32x4 S[NS];                                   // rows 16 n + 4 g4 + r, column col
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * n + 4 * g4 + r;
      S[n][r] = p.initial_state && cv && row < p.dk ? p.initial_state[((int64_t)bh * p.dk + row) * p.dv + col] : 0.f;
    }
  const T* vsrc = reinterpret_cast<const T*>(p.v) + b * p.vs.b + h * p.vs.h + col;
  T vn[16];
  auto load_v = [&](int c) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = c * DC + 16 * (i >> 2) + 4 * g4 + (i & 3);
      vn[i] = cv && t < p.seqlen ? vsrc[(int64_t)t * p.vs.l] : from_f32<T>(0.f);
    }
  };
  load_v(0);
  if (NBUF == 2) fetch(0, 0);

  for (int c = 0; c < p.pieces; ++c) {
    const f16* buf = smem + (NBUF == 2 ? (c & 1) * BUF : 0);
    if (NBUF == 2) {
      wait_vmem();
      __syncthreads();                           // the piece has arrived, the other buffer has been read
      if (c + 1 < p.pieces) fetch(c + 1, (c + 1) & 1);
    } else {
      __syncthreads();
      fetch(c, 0);
      wait_vmem();
      __syncthreads();
    }
    if (!live) continue;
    const f16 *Kt = buf, *Qt = buf + NP * TK::ELEMS, *Tt = buf + KQ, *Pt = Tt + 2 * TC::ELEMS;
    const float* vec = reinterpret_cast<const float*>(buf + KQ + TP);
    f32x4 R[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) R[i >> 2][i & 3] = to_f32(vn[i]);
    if (c + 1 < p.pieces) load_v(c + 1);

    f16x8 sh[KS], sl[KS];
    const Scale ss(wave_max(abs_max(S)));
    parts_of<2>(S, ss.mult, sh, sl);
    f16* keep = nullptr;
    float* scales = nullptr;
    if constexpr (KEEP) {
      const int64_t at = (vunit0 + c) * nblk + blk;
      keep = reinterpret_cast<f16*>(p.workspace + lay.keep) + at * (int64_t)keep_halfs<DKP>();
      scales = reinterpret_cast<float*>(p.workspace + lay.scales) + at * 4;
#pragma unroll
      for (int n = 0; n < NS; ++n) {             // [column][row]: 4 rows of a column a lane
        f16* to = keep + l16 * DKP + 16 * n + 4 * g4;
        *reinterpret_cast<f16x4*>(to) = n & 1 ? __builtin_shufflevector(sh[n >> 1], sh[n >> 1], 4, 5, 6, 7)
                                              : __builtin_shufflevector(sh[n >> 1], sh[n >> 1], 0, 1, 2, 3);
        *reinterpret_cast<f16x4*>(to + 16 * DKP) = n & 1 ? __builtin_shufflevector(sl[n >> 1], sl[n >> 1], 4, 5, 6, 7)
                                                         : __builtin_shufflevector(sl[n >> 1], sl[n >> 1], 0, 1, 2, 3);
      }
      if (lane == 0) scales[KEEP_S] = ss.inv;
    }
    // K S, and Q S for the output
    f32x4 X[4] = {}, Y[4] = {};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f16x8 a = row_frag16<DKP>(Kt, 16 * i, 32 * s, lane);
        X[i] = mma_h(a, sh[s], X[i]);
        X[i] = mma_h(a, sl[s], X[i]);
        if constexpr (NP == 2) X[i] = mma_h(row_frag16<DKP>(Kt + TK::ELEMS, 16 * i, 32 * s, lane), sh[s], X[i]);
        if constexpr (OUT) {
          const f16x8 q = row_frag16<DKP>(Qt, 16 * i, 32 * s, lane);
          Y[i] = mma_h(q, sh[s], Y[i]);          // o is rounded to T: one part is enough for bf16
          if constexpr (NP == 2) {
            Y[i] = mma_h(q, sl[s], Y[i]);
            Y[i] = mma_h(row_frag16<DKP>(Qt + TK::ELEMS, 16 * i, 32 * s, lane), sh[s], Y[i]);
          }
        }
      }
    const float xs = ss.inv * vec[VEC_SK];
    f32x4 eg[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      eg[i] = *reinterpret_cast<const f32x4*>(vec + 16 * i + 4 * g4);
#pragma unroll
      for (int r = 0; r < 4; ++r) R[i][r] -= eg[i][r] * (xs * X[i][r]);
    }
    // delta = T R; T is lower triangular
    f16x8 rh[2], rl[2];
    const Scale sr(wave_max(abs_max(R)));
    parts_of<2>(R, sr.mult, rh, rl);
    f32x4 D[4] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 2 * s; i < 4; ++i) {
        const f16x8 a = row_frag16<64>(Tt, 16 * i, 32 * s, lane);
        D[i] = mma_h(a, rh[s], D[i]);
        D[i] = mma_h(a, rl[s], D[i]);
        D[i] = mma_h(row_frag16<64>(Tt + TC::ELEMS, 16 * i, 32 * s, lane), rh[s], D[i]);
      }
    const float ds = sr.inv * vec[VEC_ST];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) D[i][r] *= ds;
    if constexpr (OUT || KEEP) {
      f16x8 dh[2], dl[2];
      const Scale sd(wave_max(abs_max(D)));
      parts_of<(KEEP || NP == 2) ? 2 : 1>(D, sd.mult, dh, dl);
      if constexpr (KEEP) {
        f16* to = keep + 2 * (2 * 16 * DKP) + l16 * DC + 4 * g4;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          *reinterpret_cast<f16x4*>(to + 16 * n) = n & 1 ? __builtin_shufflevector(dh[n >> 1], dh[n >> 1], 4, 5, 6, 7)
                                                         : __builtin_shufflevector(dh[n >> 1], dh[n >> 1], 0, 1, 2, 3);
          *reinterpret_cast<f16x4*>(to + 16 * DC + 16 * n) = n & 1 ? __builtin_shufflevector(dl[n >> 1], dl[n >> 1], 4, 5, 6, 7)
                                                                   : __builtin_shufflevector(dl[n >> 1], dl[n >> 1], 0, 1, 2, 3);
        }
        if (lane == 0) scales[KEEP_D] = sd.inv;
      }
      if constexpr (OUT) {
        f32x4 O[4] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 2 * s; i < 4; ++i) {
            const f16x8 a = row_frag16<64>(Pt, 16 * i, 32 * s, lane);
            O[i] = mma_h(a, dh[s], O[i]);
            if constexpr (NP == 2) {
              O[i] = mma_h(a, dl[s], O[i]);
              O[i] = mma_h(row_frag16<64>(Pt + TC::ELEMS, 16 * i, 32 * s, lane), dh[s], O[i]);
            }
          }
        const float ys = ss.inv * vec[VEC_SQ], os = sd.inv * vec[VEC_SP];
        T* out = reinterpret_cast<T*>(p.o) + b * p.os.b + h * p.os.h + col;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int t = c * DC + 16 * (i >> 2) + 4 * g4 + (i & 3);
          const float o = p.scale * (eg[i >> 2][i & 3] * (ys * Y[i >> 2][i & 3]) + os * O[i >> 2][i & 3]);
          if (cv && t < p.seqlen) out[(int64_t)t * p.os.l] = from_f32<T>(o);
        }
      }
    }
    // the state behind the piece
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 wt = *reinterpret_cast<const f32x4*>(vec + VEC_W + 16 * i + 4 * g4);
#pragma unroll
      for (int r = 0; r < 4; ++r) D[i][r] *= wt[r];
    }
    f16x8 wh[2], wl[2];
    const Scale sw(wave_max(abs_max(D)));
    parts_of<2>(D, sw.mult, wh, wl);
    const float gamma = vec[VEC_GAMMA], us = sw.inv * vec[VEC_SK];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x4 u = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 a = col_frag16<DKP>(Kt, 16 * n, 32 * s, lane);
        u = mma_h(a, wh[s], u);
        u = mma_h(a, wl[s], u);
        if constexpr (NP == 2) u = mma_h(col_frag16<DKP>(Kt + TK::ELEMS, 16 * n, 32 * s, lane), wh[s], u);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) S[n][r] = gamma * S[n][r] + us * u[r];
    }
  }
  if (p.final_state && live && cv) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * n + 4 * g4 + r;
        if (row < p.dk) p.final_state[((int64_t)bh * p.dk + row) * p.dv + col] = S[n][r];
      }
  }
}

template <typename T, int DKP, bool OUT, bool KEEP>
hipError_t launch_scan(const DeltaParams& p, const DeltaLayout& lay, hipStream_t st) {
  constexpr int NW = 2;
  const int nblk = (p.dv + 15) / 16, nwg = (nblk + NW - 1) / NW;
  delta_scan_kernel<T, DKP, NW, OUT, KEEP><<<head_block_grid(p.batch * p.heads, nwg), 64 * NW, 0, st>>>(p, lay, nblk, nwg);
  return hipGetLastError();
}

template <typename T>
hipError_t run_prep(const DeltaParams& p, const DeltaLayout& lay, bool backward, hipStream_t st) {
  const unsigned grid = (unsigned)((int64_t)p.batch * p.kheads * p.pieces);
  const int planes = sizeof(T) == 4 || backward ? 2 : 1;
  if (p.dk <= 64) delta_prep_kernel<T, 64><<<grid, 256, 0, st>>>(p, lay, planes);
  else delta_prep_kernel<T, 128><<<grid, 256, 0, st>>>(p, lay, planes);
  return hipGetLastError();
}

// A sequence of no tokens: the state goes through.
__global__ void delta_copy_state_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}

}  // namespace

size_t delta_workspace_bytes(const DeltaParams& p) { return DeltaLayout(p, false).total; }

hipError_t launch_delta_prep(const DeltaParams& p, bool backward, hipStream_t st) {
  const DeltaLayout lay(p, backward);
  return p.dtype == DT_F32 ? run_prep<float>(p, lay, backward, st) : run_prep<bf16>(p, lay, backward, st);
}

hipError_t launch_delta_keep(const DeltaParams& p, hipStream_t st) {
  const DeltaLayout lay(p, true);
  if (p.dtype == DT_F32) return p.dk <= 64 ? launch_scan<float, 64, false, true>(p, lay, st) : launch_scan<float, 128, false, true>(p, lay, st);
  return p.dk <= 64 ? launch_scan<bf16, 64, false, true>(p, lay, st) : launch_scan<bf16, 128, false, true>(p, lay, st);
}

hipError_t launch_delta(const DeltaParams& p, hipStream_t st) {
  if (p.seqlen == 0) {
    const int64_t n = (int64_t)p.batch * p.heads * p.dk * p.dv;
    if (!p.final_state) return hipSuccess;
    delta_copy_state_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p.initial_state, p.final_state, n);
    return hipGetLastError();
  }
  const hipError_t e = launch_delta_prep(p, false, st);
  if (e != hipSuccess) return e;
  const DeltaLayout lay(p, false);
  if (p.dtype == DT_F32) return p.dk <= 64 ? launch_scan<float, 64, true, false>(p, lay, st) : launch_scan<float, 128, true, false>(p, lay, st);
  return p.dk <= 64 ? launch_scan<bf16, 64, true, false>(p, lay, st) : launch_scan<bf16, 128, true, false>(p, lay, st);
}

}  // namespace mh
