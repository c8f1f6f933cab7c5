// One token of the gated delta rule for every (batch, head):
//   S' = e^g S + k d^T,  d = beta (v - e^g S^T k),  o = scale S'^T q = scale (e^g S^T q + (k q) d)
// so one reading of S, held in registers between the products and the update, gives both.  Bound by the state's bytes
// (dk dv fp32 read and written); columns of S are independent, so a workgroup takes all rows of 4 CW columns.  64 sequences
// of 32 heads of 128 x 128: 46 us for 270 MB, 5.9 TB/s; one sequence of 16 heads: 5 us, a launch and one round trip.
#include "launch.h"
#include "rows.h"

namespace mh {
namespace {

constexpr int kStepMaxDk = 128;

template <typename T, int CW>                    // CW lanes of 4 columns, 256 / CW rows at once
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaStepParams p, int blocks) {
  constexpr int RG = 256 / CW, R = kStepMaxDk / RG;
  __shared__ float sk[kStepMaxDk], sq[kStepMaxDk];
  __shared__ float part[4][CW][9];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cw = tid % CW, rg = tid / CW;
  const int at = (int)grid_row(), bh = at / blocks, blk = at % blocks;
  if (bh >= p.batch * p.heads) return;
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kheads);
  const int col = (blk * CW + cw) * 4, left = p.dv - col;
  const float* src = p.state_in + (int64_t)bh * p.dk * p.dv + col;
  f32x4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = i * RG + rg;
    s[i] = f32x4{};
    if (row < p.dk && left > 0) {
      const float* at = src + (int64_t)row * p.dv;
      if (left >= 4) s[i] = get_vec<false>(at);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = j < left ? at[j] : 0.f;
    }
  }
  if (tid < p.dk) {
    sk[tid] = to_f32(reinterpret_cast<const T*>(p.k)[b * p.k_sb + hk * p.k_sh + tid]);
    sq[tid] = to_f32(reinterpret_cast<const T*>(p.q)[b * p.q_sb + hk * p.q_sh + tid]);
  }
  const float decay = p.g ? expf(p.g[b * p.g_sb + h * p.g_sh]) : 1.f;
  const float beta = p.beta ? p.beta[b * p.b_sb + h * p.b_sh] : 1.f;
  f32x4 v = {};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) v[j] = to_f32(reinterpret_cast<const T*>(p.v)[b * p.v_sb + h * p.v_sh + col + j]);
  __syncthreads();
  f32x4 a = {}, c = {};
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = i * RG + rg;
    if (row < p.dk) {
      const float kv = sk[row], qv = sq[row];
      s[i] *= decay;
      a += kv * s[i];
      c += qv * s[i];
      kq += kv * qv;
    }
  }
  // over the rows: lanes of a wave that share columns, then the waves in order
  float red[9] = {a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3], kq};
#pragma unroll
  for (int off = CW; off < 64; off <<= 1)
#pragma unroll
    for (int j = 0; j < 9; ++j) red[j] += __shfl_xor(red[j], off);
  if (lane < CW)
#pragma unroll
    for (int j = 0; j < 9; ++j) part[w][cw][j] = red[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 9; ++j) red[j] = (part[0][cw][j] + part[1][cw][j]) + (part[2][cw][j] + part[3][cw][j]);
  f32x4 d, o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    d[j] = beta * (v[j] - red[j]);
    o[j] = p.scale * (red[4 + j] + red[8] * d[j]);
  }
  float* dst = p.state_out + (int64_t)bh * p.dk * p.dv + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = i * RG + rg;
    if (row < p.dk && left > 0) {
      const f32x4 n = s[i] + sk[row] * d;
      float* at = dst + (int64_t)row * p.dv;
      if (left >= 4) put_vec<false>(at, n);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) at[j] = n[j];
    }
  }
  if (rg == 0) {
    T* out = reinterpret_cast<T*>(p.o) + b * p.o_sb + h * p.o_sh + col;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) out[j] = from_f32<T>(o[j]);
  }
}

template <typename T>
hipError_t run(const DeltaStepParams& p, hipStream_t st) {
  const int blocks = (p.dv + 31) / 32;
  delta_step_kernel<T, 8><<<row_grid((int64_t)p.batch * p.heads * blocks, 1), 256, 0, st>>>(p, blocks);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_delta_step(const DeltaStepParams& p, hipStream_t st) {
  return p.dtype == DT_F32 ? run<float>(p, st) : run<bf16>(p, st);
}

}  // namespace mh
