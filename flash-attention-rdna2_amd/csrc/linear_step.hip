// linear_step.hip — linear attention of one new token or a few: the state of each sequence and head read once, taken
// through the tokens in registers, written once.
//
// 8 DK DV bytes per state against 6 DK DV operations and token: bound by HBM. A workgroup takes CT columns of a state: 32 where
// there are few states (the latency of the loads is the time: more workgroups, fewer loads each), 128 else. A thread holds
// four columns of R consecutive rows. q, k and v pass through LDS in fp32, TB tokens at a time; the products with q are summed
// over a wave by lane exchanges and over the four waves through LDS, in a fixed order.
//   Measured, bf16, states of 128 x 128: 48 sequences x 64 heads (403 MB) 80 us, 5.0 TB/s; one sequence x 32 heads 5 us, its latency.
#include "linear_kernel.hpp"

namespace fa {

template <typename T, int CT, int R>
__global__ __launch_bounds__(256) void la_step_kernel(LaArgs p) {
  constexpr int CL = CT / 4, RG = 256 / CL, TB = 4;
  __shared__ float qs[TB][RG * R], ks[TB][RG * R], vs[TB][CT], red[TB][4][CT];
  const int tid = threadIdx.x, cl = tid % CL, rg = tid / CL, wave = tid / 64;
  const int tiles = (p.db + CT - 1) / CT;
  int w = blockIdx.x;
  const int ct = w % tiles;
  w /= tiles;
  const int h = w % p.NH, b = w / p.NH;
  const LaSeq sq = la_seq(p, b);
  const int c0 = ct * CT, nc = min(CT, p.db - c0);
  const long long obase = (p.cu ? 0 : b * p.so.b) + h * p.so.h;
  if (p.cu && b == 0) la_zero_rows<T>(p, obase, 0, sq.row0, c0, nc, tid, 256);
  if (p.cu && b == p.batch - 1) la_zero_rows<T>(p, obase, sq.row0 + sq.len, p.total, c0, nc, tid, 256);
  if (sq.slot < 0) {
    la_zero_rows<T>(p, obase, sq.row0, sq.row0 + sq.len, c0, nc, tid, 256);
    return;
  }
  const long long state = ((long long)sq.slot * p.NH + h) * p.da * p.db + c0 + 4 * cl;
  const bool cin = 4 * cl < nc;
  f32x4 S[R];
#pragma unroll
  for (int i = 0; i < R; i++) {
    const int a = rg * R + i;
    S[i] = cin && a < p.da ? *(const f32x4*)(p.first + state + (long long)a * p.db) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const LaFade fade(la_decay(p, b, h), 1.0f);
  const T* const gq = (const T*)p.x + (p.cu ? 0 : b * p.sx.b) + (h / p.hx) * p.sx.h + sq.row0 * p.sx.s;
  const T* const gk = (const T*)p.y + (p.cu ? 0 : b * p.sy.b) + (h / p.hy) * p.sy.h + sq.row0 * p.sy.s;
  const T* const gv = (const T*)p.z + (p.cu ? 0 : b * p.sz.b) + (h / p.hz) * p.sz.h + sq.row0 * p.sz.s + c0;
  for (int t0 = 0; t0 < sq.len; t0 += TB) {
    const int nt = min(TB, sq.len - t0);
    if (t0) __syncthreads();
#pragma unroll
    for (int t = 0; t < TB; t++) {
      if (t >= nt) break;
      if (tid < RG * R) {
        qs[t][tid] = tid < p.da ? (float)gq[(t0 + t) * p.sx.s + tid] : 0.0f;
        ks[t][tid] = tid < p.da ? (float)gk[(t0 + t) * p.sy.s + tid] : 0.0f;
      }
      if (tid < CT) vs[t][tid] = tid < nc ? (float)gv[(t0 + t) * p.sz.s + tid] : 0.0f;
    }
    __syncthreads();
    for (int t = 0; t < nt; t++) {
      const f32x4 v = *(const f32x4*)&vs[t][4 * cl];
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < R; i++) {
        const float k = ks[t][rg * R + i], q = qs[t][rg * R + i];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          S[i][j] = fmaf(k, v[j], fade(S[i][j]));
          acc[j] = fmaf(q, S[i][j], acc[j]);
        }
      }
#pragma unroll
      for (int m = CL; m < 64; m *= 2)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] += __shfl_xor(acc[j], m);
      if (tid % 64 < CL) *(f32x4*)&red[t][wave][4 * cl] = acc;
    }
    __syncthreads();
    for (int i = tid; i < nt * CT; i += 256) {
      const int t = i / CT, c = i % CT;
      if (c < nc)
        ((T*)p.o)[obase + (sq.row0 + t0 + t) * p.so.s + c0 + c] = (T)(p.iscale * ((red[t][0][c] + red[t][1][c]) + (red[t][2][c] + red[t][3][c])));
    }
  }
  if (sq.len > 0 || p.first != p.last) {
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int a = rg * R + i;
      if (cin && a < p.da) *(f32x4*)(p.last + state + (long long)a * p.db) = S[i];
    }
  }
}

namespace {

template <typename T, int CT>
void la_step_rows(const LaArgs& p, hipStream_t st) {
  constexpr int RG = 256 / (CT / 4);
  const dim3 grid((unsigned)(p.batch * p.NH * ((p.db + CT - 1) / CT)));
  if (p.da <= 64) hipLaunchKernelGGL((la_step_kernel<T, CT, 64 / RG>), grid, dim3(256), 0, st, p);
  else if (p.da <= 128) hipLaunchKernelGGL((la_step_kernel<T, CT, 128 / RG>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((la_step_kernel<T, CT, 256 / RG>), grid, dim3(256), 0, st, p);
}

// Columns of a workgroup. Heads of 128, 32 columns against 128, us on the device one call after another: 32 states 4.6 / 5.2, 128 6.0 / 6.2,
// 256 8.5 / 7.6, 512 12.4 / 10.5, 48 x 64 62.7 / 64.8; 128 heads of 64 4.2 / 5.2, 1024 10.3 / 9.0; 256 heads of 256 (512 tiles) 24.1 / 27.1.
template <typename T>
void la_step_type(const LaArgs& p, hipStream_t st) {
  if ((long long)p.batch * p.NH * ((p.db + 127) / 128) < 512 || p.db <= 32) la_step_rows<T, 32>(p, st);
  else la_step_rows<T, 128>(p, st);
}

}  // namespace

void la_step(const LaArgs& p, int dtype, hipStream_t st) {
  if (dtype == FA_F16) la_step_type<_Float16>(p, st);
  else if (dtype == FA_BF16) la_step_type<__bf16>(p, st);
  else la_step_type<float>(p, st);
}

}  // namespace fa
