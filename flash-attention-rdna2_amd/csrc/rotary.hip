// rotary.hip — queries and keys turned by their positions, and the tables of cosines and sines.
//
// The rotation reads and writes every value once: bound by HBM, by latency for a few tokens. A wave takes one token; its
// lanes are (head, unit of columns) and walk over the token's heads, so a lane loads its cosines and sines once for all of
// them. A unit is 16 bytes of a head and, where pairs are half the rotated columns apart, the 16 bytes it is paired with.
// Few tokens spread their heads over several waves. Measured, bf16, 8192 tokens x 40 heads of 128 (168 MB): 36 us, 4.7 TB/s
// (a dense copy of as much 33); the heads in batches of four with their loads ahead, and stores past the caches, 42.
#include <math.h>

#include "attn_device.hpp"
#include "status.hpp"

namespace fa {

namespace {

struct RotArgs {
  FableRotaryParams p;
  int units, split;      // units of a head, waves of a token
  long long tokens;
};

// The table row of token `tok`, -1 for one of no sequence.
__device__ __forceinline__ int rot_row(const FableRotaryParams& p, long long tok, int& b, long long& t) {
  if (p.cu) {
    // the last b with cu[b] <= tok (sequences without tokens share their first row with the next)
    int lo = 0, hi = p.batch;
    while (lo < hi) {
      const int m = (lo + hi + 1) / 2;
      if ((long long)p.cu[m] <= tok) lo = m;
      else hi = m - 1;
    }
    b = lo;
    if (p.batch == 0 || lo >= p.batch || tok < (long long)p.cu[0]) return -1;
    t = tok - p.cu[lo];
  } else {
    b = (int)(tok / p.n);
    t = tok % p.n;
  }
  const long long row = t + (p.start ? p.start[b] : 0);
  return (int)min(max(row, 0LL), (long long)p.rotary_rows - 1);
}

// The pair (a, b) turned, its first and second value: one product rounded, the other in the sum, the same in all kernels.
__device__ __forceinline__ float rot_first(float a, float b, float c, float s) { return fmaf(a, c, -(b * s)); }
__device__ __forceinline__ float rot_second(float a, float b, float c, float s) { return fmaf(b, c, a * s); }

template <typename T>
struct RotVec {
  static constexpr int N = 16 / sizeof(T);
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
};

// PAIR 1: halves, 2: neighbours. Units [0, rotating) turn, the others are copied.
template <typename T, int PAIR>
__global__ __launch_bounds__(256) void rot_kernel(RotArgs a) {
  const FableRotaryParams& p = a.p;
  constexpr int N = RotVec<T>::N;
  using V = typename RotVec<T>::V;
  const int lane = threadIdx.x % 64;
  const long long w = (long long)blockIdx.x * 4 + threadIdx.x / 64;
  const long long tok = w / a.split;
  if (tok >= a.tokens) return;
  const int part = (int)(w % a.split);
  int b;
  long long t;
  const int row = rot_row(p, tok, b, t);
  const int half = p.rotary_dim / 2;
  const int rotating = PAIR == 1 ? half / N : p.rotary_dim / N;
  const long long qi = p.cu ? tok * p.sq.s : b * p.sq.b + t * p.sq.s, qo = p.cu ? tok * p.sqo.s : b * p.sqo.b + t * p.sqo.s;
  const long long ki = p.cu ? tok * p.sk.s : b * p.sk.b + t * p.sk.s, ko = p.cu ? tok * p.sko.s : b * p.sko.b + t * p.sko.s;
  const int heads = p.NH + (p.k ? p.NKV : 0);
  // lanes over (head, unit); a lane keeps its unit
  const int per = a.units >= 64 ? 1 : 64 / a.units;
  for (int u = lane % a.units; u < a.units; u += 64) {
    if (a.units < 64 && lane >= per * a.units) break;
    const bool turn = u < rotating;
    const int col = turn ? u * N : p.rotary_dim + (u - rotating) * N;
    float c[N], s[N];
    if (turn && row >= 0) {
      const int first = PAIR == 1 ? col : col / 2;
      const float* cp = p.cos + (long long)row * half + first;
      const float* sp = p.sin + (long long)row * half + first;
      constexpr int M = PAIR == 1 ? N : N / 2;
#pragma unroll
      for (int j = 0; j < M; j++) {
        c[j] = cp[j];
        s[j] = p.conj ? -sp[j] : sp[j];
      }
    }
    const int h0 = a.units < 64 ? lane / a.units + per * part : part;
#pragma unroll 4
    for (int h = h0; h < heads; h += per * a.split) {
      const bool isq = h < p.NH;
      const T* in = isq ? (const T*)p.q + qi + h * p.sq.h + col : (const T*)p.k + ki + (h - p.NH) * p.sk.h + col;
      T* out = isq ? (T*)p.q_out + qo + h * p.sqo.h + col : (T*)p.k_out + ko + (h - p.NH) * p.sko.h + col;
      V x, y;
      if (row < 0) {
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = y[j] = (T)0.0f;
      } else {
        x = *(const V*)in;
        if constexpr (PAIR == 1) {
          if (turn) {
            y = *(const V*)(in + half);
#pragma unroll
            for (int j = 0; j < N; j++) {
              const float e = (float)x[j], f = (float)y[j];
              x[j] = (T)rot_first(e, f, c[j], s[j]);
              y[j] = (T)rot_second(e, f, c[j], s[j]);
            }
          }
        } else if (turn) {
#pragma unroll
          for (int j = 0; j < N / 2; j++) {
            const float e = (float)x[2 * j], f = (float)x[2 * j + 1];
            x[2 * j] = (T)rot_first(e, f, c[j], s[j]);
            x[2 * j + 1] = (T)rot_second(e, f, c[j], s[j]);
          }
        }
      }
      *(V*)out = x;
      if (PAIR == 1 && turn) *(V*)(out + half) = y;
    }
  }
}

// Any head dim, rotated part and alignment: a thread per value.
template <typename T>
__global__ __launch_bounds__(256) void rot_any_kernel(RotArgs a) {
  const FableRotaryParams& p = a.p;
  const int heads = p.NH + (p.k ? p.NKV : 0);
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.tokens * heads * p.HD) return;
  const int col = (int)(i % p.HD), h = (int)(i / p.HD % heads);
  const long long tok = i / p.HD / heads;
  int b;
  long long t;
  const int row = rot_row(p, tok, b, t);
  const bool isq = h < p.NH;
  const fa_strides si = isq ? p.sq : p.sk, so = isq ? p.sqo : p.sko;
  const int hh = isq ? h : h - p.NH;
  const T* in = (const T*)(isq ? p.q : p.k) + (p.cu ? tok * si.s : b * si.b + t * si.s) + hh * si.h;
  T* out = (T*)(isq ? p.q_out : p.k_out) + (p.cu ? tok * so.s : b * so.b + t * so.s) + hh * so.h;
  T v = (T)0.0f;
  if (row >= 0) {
    v = in[col];
    if (col < p.rotary_dim) {
      const int half = p.rotary_dim / 2;
      const int pair = p.rotary == 1 ? col % half : col / 2;
      const bool second = p.rotary == 1 ? col >= half : col % 2;
      const float o = (float)in[p.rotary == 1 ? (second ? col - half : col + half) : col ^ 1];
      const float c = p.cos[(long long)row * half + pair];
      float s = p.sin[(long long)row * half + pair];
      if (p.conj) s = -s;
      v = (T)(second ? rot_second(o, (float)v, c, s) : rot_first((float)v, o, c, s));
    }
  }
  out[col] = v;
}

template <typename T>
void rot_launch(RotArgs a, bool wide, hipStream_t st) {
  const FableRotaryParams& p = a.p;
  constexpr int N = RotVec<T>::N;
  const int heads = p.NH + (p.k ? p.NKV : 0);
  if (!wide) {
    const long long items = a.tokens * heads * p.HD;
    hipLaunchKernelGGL(rot_any_kernel<T>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, a);
    return;
  }
  a.units = (p.rotary == 1 ? p.rotary_dim / 2 / N : p.rotary_dim / N) + (p.HD - p.rotary_dim) / N;
  const int per = a.units >= 64 ? 1 : 64 / a.units, turns = (heads + per - 1) / per;
  // Waves of a token: up to one per turn of the loop while the chip has fewer than 2048 waves. bf16, 64 + 8 heads of 128, us on the device with
  // one wave a token / 1024 / 2048 / 4096 in all / one per turn: 48 tokens 8.1 / 3.5 / 3.5 / 3.5 / 3.5, 512 8.9 / 6.7 / 6.0 / 6.0 / 7.1,
  // 1024 12.1 / 12.2 / 8.9 / 8.4 / 11.4, 2048 16.6 / 17.0 / 16.6 / 14.8 / 18.8.
  long long split = a.tokens > 0 ? 2048 / a.tokens : 1;
  a.split = (int)(split < 1 ? 1 : split > turns ? turns : split);
  const dim3 grid((unsigned)((a.tokens * a.split + 3) / 4));
  if (p.rotary == 1) hipLaunchKernelGGL((rot_kernel<T, 1>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rot_kernel<T, 2>), grid, dim3(256), 0, st, a);
}

// Angles are counted in turns, in 64 bits, and reduced to half a turn; what rounding that to fp32 leaves goes into the first order of
// sine and cosine, so the tables are exact to about their own rounding at any position. A thread keeps V neighbouring pairs, forms
// their frequencies once, and walks over the rows: bound by the bytes written at 10^5 rows.
struct RotTable {
  FableRotaryTableParams p;
  double step;            // log2(base) / pairs
  int columns;            // threads of a row: pairs / V, at most 256; the others of a workgroup take further rows
};
template <int V>
__global__ __launch_bounds__(256) void rot_table_kernel(RotTable a) {
  const FableRotaryTableParams& p = a.p;
  const int rows = 256 / a.columns, sub = threadIdx.x / a.columns;
  if (sub >= rows) return;
  const float amp = (float)p.amplitude;
  for (int c = V * (threadIdx.x % a.columns); c < p.pairs; c += V * a.columns) {
    double freq[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
      const double f = exp2(-(double)(c + j) * a.step) * 0.15915494309189533577;   // turns per position
      freq[j] = f;
      if (p.factor != 1.0) {
        double keep = p.original > 0.0 ? (p.original * f - p.low) / (p.high - p.low) : 0.0;
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        freq[j] = f * (keep + (1.0 - keep) / p.factor);
      }
    }
    typedef float FV __attribute__((ext_vector_type(V)));
    for (long long row = (long long)blockIdx.x * rows + sub; row < p.rows; row += (long long)gridDim.x * rows) {
      FV co, si;
#pragma unroll
      for (int j = 0; j < V; j++) {
        double x = (double)(row + p.first) * freq[j];
        x = 2.0 * (x - rint(x));
        const float hi = (float)x, lo = (float)(x - (double)hi) * 3.14159265358979f;
        float s, k;
        sincospif(hi, &s, &k);
        co[j] = amp * fmaf(-lo, s, k);
        si[j] = amp * fmaf(lo, k, s);
      }
      *(FV*)(p.cos + row * p.pairs + c) = co;
      *(FV*)(p.sin + row * p.pairs + c) = si;
    }
  }
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int fable_attn_rotary(FableRotaryParams p, int dtype, void* stream) {
  const char* what = "fable_attn_rotary";
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return fail(FA_ERR_DTYPE, "%s: unknown dtype %d", what, dtype);
  if (p.batch < 0 || p.n < 0 || p.total < 0 || p.NH < 1 || (p.k && p.NKV < 1) || p.HD < 1)
    return fail(FA_ERR_ARG, "%s: batch=%d n=%d NH=%d NKV=%d HD=%d", what, p.batch, p.n, p.NH, p.NKV, p.HD);
  if (p.rotary < 1 || p.rotary > 2 || p.rotary_dim < 2 || p.rotary_dim % 2 || p.rotary_dim > p.HD || p.rotary_rows < 1)
    return fail(FA_ERR_ARG, "%s: rotary=%d rotary_dim=%d rotary_rows=%d", what, p.rotary, p.rotary_dim, p.rotary_rows);
  RotArgs a;
  a.p = p;
  a.units = a.split = 1;
  a.tokens = p.cu ? p.total : (long long)p.batch * p.n;
  if (a.tokens == 0) return FA_OK;
  if (!p.q || !p.q_out || !p.cos || !p.sin || (p.k && !p.k_out)) return fail(FA_ERR_ARG, "%s: null tensor", what);
  const int e = dtype == FA_F32 ? 4 : 2;
  auto bits = [&](const void* t, const fa_strides& s) { return (uintptr_t)t | (uintptr_t)(s.b * e) | (uintptr_t)(s.h * e) | (uintptr_t)(s.s * e); };
  uintptr_t x = bits(p.q, p.sq) | bits(p.q_out, p.sqo);
  if (p.k) x |= bits(p.k, p.sk) | bits(p.k_out, p.sko);
  // 16-byte accesses; else a thread per value
  const int N = 16 / e;
  const bool wide = (x & 15) == 0 && p.HD % N == 0 && p.rotary_dim % N == 0 && (p.rotary == 2 || p.rotary_dim / 2 % N == 0);
  // a grid has fewer than 2^32 threads
  if (wide ? a.tokens >= (1LL << 25) : a.tokens * (p.NH + (p.k ? p.NKV : 0)) >= (1LL << 31) / p.HD)
    return fail(FA_ERR_ARG, "%s: %lld tokens", what, a.tokens);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == FA_F16) rot_launch<_Float16>(a, wide, st);
  else if (dtype == FA_BF16) rot_launch<__bf16>(a, wide, st);
  else rot_launch<float>(a, wide, st);
  return launch_status(what);
}

extern "C" int fable_attn_rotary_tables(FableRotaryTableParams p, void* stream) {
  const char* what = "fable_attn_rotary_tables";
  if (p.rows < 0 || p.first < 0 || p.pairs < 1 || p.pairs > 4096) return fail(FA_ERR_ARG, "%s: rows=%lld first=%lld pairs=%d", what, (long long)p.rows, (long long)p.first, p.pairs);
  if (!(p.base > 0.0 && p.base <= 1.7e308) || !(p.factor > 0.0) || !(p.original >= 0.0) || (p.original > 0.0 && !(p.high > p.low)))
    return fail(FA_ERR_ARG, "%s: base=%g factor=%g original=%g low=%g high=%g", what, p.base, p.factor, p.original, p.low, p.high);
  if (p.rows == 0) return FA_OK;
  if (!p.cos || !p.sin) return fail(FA_ERR_ARG, "%s: null tensor", what);
  const bool wide = p.pairs % 4 == 0 && (((uintptr_t)p.cos | (uintptr_t)p.sin) & 15) == 0;
  RotTable a;
  a.p = p;
  a.step = log2(p.base) / p.pairs;
  const int columns = wide ? p.pairs / 4 : p.pairs;
  a.columns = columns < 256 ? columns : 256;
  // Eight rows a thread at least where there are enough of them to fill the chip, for the frequencies formed once. 64 pairs, us on the
  // device, this rule / at most 1024 workgroups / a row a thread: 32768 positions 7.7 / 7.6 / 8.6, 131072 16.0 / 15.7 / 22.0, 1048576
  // 120 / 119 / 157.
  const long long groups = (p.rows + 256 / a.columns - 1) / (256 / a.columns);
  const unsigned grid = (unsigned)(groups < 1024 ? groups : groups / 8 < 1024 ? 1024 : groups / 8 < 4096 ? groups / 8 : 4096);
  if (wide) hipLaunchKernelGGL(rot_table_kernel<4>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(rot_table_kernel<1>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  return launch_status(what);
}
