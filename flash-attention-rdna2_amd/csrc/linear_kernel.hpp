// linear_kernel.hpp — causal linear attention with a decay for each head, by chunks.
//
// One kernel serves the forward pass and the three products of the backward pass. With lambda = exp(-decay[h])
//   out_i = pscale sum_{j<=i} lambda^(i-j) (x_i . y_j) z_j + iscale lambda^(i+1) S x_i,
//   S     = the state before the first row,  S' = lambda^n S + uscale sum_j lambda^(n-1-j) y_j z_j^T,
// over rows i of the sequence in processing order. The forward pass is x, y, z = q, k, v. With the state's
// gradient G_t = lambda G_{t+1} + scale q_t dout_t^T, dq is x, y, z = dout, v, k in the same order, and dv
// (k, q, dout) and dk (v, dout, q) run over the rows from the last one to the first.
//
// A workgroup of NW waves takes a segment of one head of one sequence, a chunk of C rows at a time, and a tile of
// 32 NW columns of z; a wave owns 32 of them. It keeps S (DA x 32 of its columns) in accumulators, in 32 bits, for the
// whole segment, so a chunk reads its rows of x, y and z once and writes its rows of out once: 1 KB per row and head of
// 128 in 16 bits against some 100 kFLOP.
//   Scores are formed transposed (y x^T), so that a lane holds all keys of one query: weighted and rounded, they are the
// operand of the product with z as they are. S is DA x 32 with z's columns across the lanes, which is the operand
// layout of the product with x. x is read from LDS once for both. out is formed transposed too: a lane holds 32 columns
// of one row.
//   Roundings to 16 bits: the weighted scores and S once each as operands, as attention rounds its probabilities (each
// is as large as the rounding of out itself). The weighted z of the state's update is split into PIECES parts, each
// the rounding of what the ones before left: in bf16 three parts, which hold its 24 bits, where a state is a result or
// runs into one, and two (16 bits) where only rounded outputs follow; in fp32 it is itself.
//   fp16 has too few exponents for what a chunk puts together: a score of 2^-24 may meet a value of 2^15 (in the backward pass scores
// are products of dout and v), a row weighted by 2^-40 may be all that there is, columns may be 2^24 apart. There every operand
// that carries a weight is taken in bf16, whose range is fp32's: the rows of y, weighted as they are put into LDS (once for all waves), in PIECES
// parts, z in two (all of its 11 bits), a weighted score in two. Products of parts that the result does not resolve are left out: three a
// product remain, five where a state is a result. S alone is an fp16 operand, each of its columns brought to a power of two of its own
// before: what is under 2^-27 of the column's largest value loses bits there (2^-38 of that value is the most it is off by).
//   The decay of S is put off: the accumulators hold S lambda^-lag, `lag` the rows since they were last brought up to
// date, and what a chunk adds is weighted up by as much, until lambda^lag leaves 2^+-kLaLag. Each rounding of such a factor
// then touches what is about to be forgotten only, where one for each chunk would add up over all that a slow decay
// remembers; and for all but fast decays that spares most of the DA / 2 multiplications per lane and chunk.
//
// Measured, bf16, heads of 128: B2 S4096 H32 (268 MB) 54 to 60 us, 4.5 to 5.0 TB/s, of the 5.2 that a large copy reaches
// here; the states of its segments beside that 35 us, and 11 to chain them; a whole call 103, in fp16 124 to 131. What bounds it
// is the bytes and, as much, the issue of vector and matrix instructions, which are busy 80% of a CU's cycles together. Where a
// SIMD has one wave, the chain of a chunk's steps
// does: 1.9 us per chunk, 60 ns per row. Not kept, because slower or no faster: three waves per SIMD (387 against 371 us forward
// and backward: fewer loads of operands in flight), two chunks' tiles ahead in registers, two LDS buffers, the operands of
// four steps read ahead, C = 64 (registers spill).
#pragma once
#include <type_traits>

#include "attn_device.hpp"

namespace fa {

// What a launch takes. Strides in elements. Rows of sequence b: [cu[b], cu[b+1]) of [0, total) of the packed tensors, or n of batch element b.
struct LaArgs {
  const void *x, *y, *z;
  void* o;
  fa_strides sx, sy, sz, so;
  int hx, hy, hz;            // heads of the item's head h: h / hx, ...
  int da, db;                // columns of x and y, of z and out
  const float* decay;
  long long decay_b;         // stride over the batch
  const float* first;        // states before the first row in processing order, [slot][NH][da][db] by ...
  float* last;               // ... and behind the last one; NULL: zeros, not wanted
  int sa, sb;                // strides of a state's element (a, b)
  const int32_t* slots;      // a sequence's state; NULL: its own number. Outside [0, nslots): no sequence
  int nslots;
  float* ws;                 // the states before the segments (nseg > 1), [la_ws_row() + segment][NH] ...
  int wa, wb;                // ... and the strides of their elements
  const int32_t* cu;
  long long total;
  int batch, n, NH;
  int nseg, seg;             // segments of `seg` rows, a multiple of C; the last one takes all rows left
  int span;                  // rows, a multiple of C, over which no tensor spans more than 2^29 bytes
  float pscale, iscale, uscale;
  int rev;                   // rows from the last to the first
  int inplace;               // last may be first (segments then find the first state in ws)
  int enter;                 // first is not to decay before the first row (the gradient of the final state)
  int leave;                 // last decays once more behind the last row (the gradient of the initial state)
  int o32;                   // out is fp32 (partial gradients of shared heads)
};

// Passes of one launch over the same rows: the backward pass's three, that share the reading of theirs through the caches.
struct LaPasses {
  LaArgs p[3];
  int n;
};

// A fragment: lane (r, g) = (l % 32, l / 32) holds the contraction indices 16 s + 4 g + {0..3} and 16 s + 8 + 4 g + {0..3} of
// its row or column r, the rows of a 32 x 32 accumulator that its registers 8 (s % 2) .. + 7 hold.
template <typename T>
struct La {
  using F = typename Dt<T>::V8;
  using H = typename Dt<T>::V4;
  static __device__ __forceinline__ f32x16 mma(F a, F b, f32x16 c) { return Dt<T>::mma32(a, b, c); }
};
typedef float f32x8 __attribute__((ext_vector_type(8)));
template <>
struct La<float> {
  using F = f32x8;
  using H = f32x4;
  static __device__ __forceinline__ f32x16 mma(F a, F b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// LDS tiles, rows of LD values. Rows of x and y are read by 32 lanes at one column (8 bytes each) and y by columns, 4 rows
// x 32 columns at a time: a row is 7 units of 8 bytes longer than a multiple of the 64 banks (or of half of them), so the
// first meets every bank once and the second nearly so; z, and fp16's weighted y, are read by columns only and 8 units longer. (fp32: one unit of
// 16 bytes.) Padding, not a turned order within the row, because then all addresses are one register and constants.
template <typename T, int W>
constexpr int kLaRow = W + (sizeof(T) == 2 ? 28 : 4);
template <typename T, int W>
constexpr int kLaRowZ = W + (sizeof(T) == 2 ? 32 : 4);

// rows row (per lane), columns 16 s .. 16 s + 15
template <typename T, int LD>
__device__ __forceinline__ typename La<T>::F la_rows(const T* tile, int row, int s, int g) {
  using H = typename La<T>::H;
  const T* at = tile + row * LD + 4 * g + 16 * s;
  const H a = *(const H*)at, b = *(const H*)(at + 8);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// column 32 ct + r, rows 16 s .. 16 s + 15
template <typename T, int LD>
__device__ __forceinline__ typename La<T>::F la_cols(const T* tile, int ct, int s, int lane) {
  using H = typename La<T>::H;
  const int g = lane / 32;
  if constexpr (sizeof(T) == 2) {
    const T* at = tile + (4 * g + (lane % 16) / 4) * LD + 16 * ((lane / 16) % 2) + 4 * (lane % 4) + 16 * s * LD + 32 * ct;
    const H a = lds_read_tr<T>(at), b = lds_read_tr<T>(at + 8 * LD);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const T* at = tile + 4 * g * LD + lane % 32 + 16 * s * LD + 32 * ct;
    typename La<T>::F f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = at[(8 * (j / 4) + j % 4) * LD];
    return f;
  }
}

// The power of two that brings a largest magnitude m into [2^13, 2^14), its inverse in `inv`; 1 for zero, and for what is no number.
__device__ __forceinline__ float la_norm(float m, float& inv) {
  const int e = (int)((__float_as_uint(m) >> 23) & 255);
  const int k = (e == 0 || e == 255) ? 0 : min(max(140 - e, -120), 120);
  inv = __uint_as_float((uint32_t)(127 - k) << 23);
  return __uint_as_float((uint32_t)(127 + k) << 23);
}

// The larger magnitude, as bits, of `top` (0 at first) and a fragment's values; what is no number is above all that are.
template <typename F>
__device__ __forceinline__ uint32_t la_top(uint32_t top, F f) {
  if constexpr (sizeof(f[0]) == 2) {
    typedef unsigned short U2 __attribute__((ext_vector_type(2)));
    U2 t = bitcast<U2>(top);
    const u32x4 w = bitcast<u32x4>(f);
#pragma unroll
    for (int j = 0; j < 4; j++) t = __builtin_elementwise_max(t, bitcast<U2>(w[j] & 0x7fff7fffu));
    return bitcast<uint32_t>(t);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
    return top;
  }
}
// the magnitude that la_top() came to, in the lane; the bits from which on it is no number
template <typename T>
__device__ __forceinline__ uint32_t la_top_bits(uint32_t top) {
  return sizeof(T) == 2 ? max(top & 0xffffu, top >> 16) : top;
}
template <typename T>
constexpr uint32_t kLaNone = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;

constexpr float kLaLag = 8.0f;

// Two values split into parts of T, each the rounding of what the ones before left.
template <typename T, int PIECES, typename F>
__device__ __forceinline__ void la_split2(float a, float b, F* parts, int j) {
  if constexpr (sizeof(T) == 4) {
    parts[0][j] = a;
    parts[0][j + 1] = b;
  } else {
    using V2 = typename Dt<T>::V2;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
      // (The empty asm keeps the compiler from forming a product twice, once fused with its rounding, and from converting a value
      // once for the operand and once for the difference.)
      asm("" : "+v"(a), "+v"(b));
      uint32_t u = bitcast<uint32_t>(V2{(T)a, (T)b});
      asm("" : "+v"(u));
      const V2 h = bitcast<V2>(u);
      parts[i][j] = h[0];
      parts[i][j + 1] = h[1];
      if (i + 1 < PIECES) {
        a -= (float)h[0];
        b -= (float)h[1];
      }
    }
  }
}

// Eight values of fp16 times w, in PARTS tiles `part` values apart of their parts in bf16.
template <int PARTS, int part>
__device__ __forceinline__ void la_put(__bf16* at, u32x4 v, float w) {
  const f16x8 h = bitcast<f16x8>(v);
  bf16x8 parts[PARTS];
#pragma unroll
  for (int j = 0; j < 8; j += 2) la_split2<__bf16, PARTS>((float)h[j] * w, (float)h[j + 1] * w, parts, j);
#pragma unroll
  for (int i = 0; i < PARTS; i++) *(bf16x8*)(at + i * part) = parts[i];
}

// A state carried over `rows` rows, S <- keep S + by S: keep 1 and by = lambda^rows - 1 where that is near 1 (the factor itself, rounded
// to 32 bits, is off by up to 2^-25 in the same direction each time), else 0 and the factor.
struct LaFade {
  float by, keep;
  __device__ __forceinline__ LaFade(float d, float rows) {
    by = expm1f(-d * rows);
    keep = 1.0f;
    if (by < -0.5f) {
      by = expf(-d * rows);
      keep = 0.0f;
    }
  }
  __device__ __forceinline__ float operator()(float s) const { return fmaf(s, by, keep * s); }
};

// lambda^k as 2^(-k d log2 e)
__device__ __forceinline__ float la_pow(float dl2, float k) { return exp2f(-dl2 * k); }

// A decay too large for products with a row count is one that nothing survives; 0 times it has to stay 0.
__device__ __forceinline__ float la_decay(const LaArgs& p, int b, int h) {
  const float d = p.decay[b * p.decay_b + h];
  return d > 1e25f ? 1e25f : d < -1e25f ? -1e25f : d;
}

// A value that all lanes have, in scalar registers.
__device__ __forceinline__ const char* la_uniform(const char* at) {
  const unsigned long long u = (unsigned long long)at;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
  return (const char*)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned la_uniform(unsigned n) { return __builtin_amdgcn_readfirstlane(n); }

struct LaSeq {
  int row0;                  // first row in the tensors
  int len;
  int slot;                  // -1: no sequence
};
// cu[b], kept within the rows that there are
__device__ __forceinline__ int la_row(const LaArgs& p, int b) { return (int)min((long long)max(p.cu[b], 0), p.total); }
__device__ __forceinline__ LaSeq la_seq(const LaArgs& p, int b) {
  LaSeq s;
  if (p.cu) {
    s.row0 = la_row(p, b);
    s.len = max(la_row(p, b + 1), s.row0) - s.row0;
  } else {
    s.row0 = 0;
    s.len = p.n;
  }
  s.slot = p.slots ? p.slots[b] : b;
  if (p.slots && (s.slot < 0 || s.slot >= p.nslots)) s.slot = -1;
  return s;
}
__device__ __forceinline__ int la_segments(const LaArgs& p, int len) {
  const int k = (int)(((long long)len + p.seg - 1) / p.seg);
  return k < 1 ? 1 : k > p.nseg ? p.nseg : k;
}
// Where the states of a sequence's segments start in ws. A packed sequence of more than one segment ends at least one
// multiple of `seg` rows further than it starts, so twice that count leaves room for its segments ahead of the next such
// sequence's.
__device__ __forceinline__ long long la_ws_row(const LaArgs& p, int b, const LaSeq& sq) {
  return p.cu ? 2LL * (sq.row0 / p.seg) : (long long)b * p.nseg;
}
// (sequence, segment) of an item. Packed sequence b has its items from cu[b] / seg + b on, which leaves room for all its
// segments without a grid of the longest sequence's count for each: the threads of a workgroup look for it side by side.
__device__ __forceinline__ void la_item(const LaArgs& p, int i, int segs, int tid, int nt, int& b, int& sg) {
  if (!p.cu || p.nseg == 1) {
    b = i / segs;
    sg = i % segs;
    return;
  }
  int at = 0;
  for (int b0 = 0; b0 < p.batch; b0 += nt) {
    const int j = b0 + tid;
    at += __syncthreads_count(j < p.batch && la_row(p, j) / p.seg + j <= i);
  }
  b = __builtin_amdgcn_readfirstlane(max(at - 1, 0));
  sg = __builtin_amdgcn_readfirstlane(i - b - la_row(p, b) / p.seg);
}
// how many items a launch has
inline long long la_items(const LaArgs& p, bool state) {
  if (p.nseg == 1) return p.batch;
  return p.cu ? p.total / p.seg + p.batch : (long long)p.batch * (state ? p.nseg - 1 : p.nseg);
}

// Zeros in rows [lo, hi) of out for the item's columns (at most 512 bytes of a row), 32 threads to a row.
template <typename O>
__device__ __forceinline__ void la_zero_rows(const LaArgs& p, long long base, long long lo, long long hi, int c0, int nc, int tid, int nt) {
  constexpr int E = 16 / sizeof(O);
  const int c = E * (tid % 32);
  if (c >= nc) return;
  for (long long row = lo + tid / 32; row < hi; row += nt / 32) *(u32x4*)((O*)p.o + base + row * p.so.s + c0 + c) = u32x4{0, 0, 0, 0};
}

// An offset past every descriptor (those span 2^29 bytes at most), also with up to 2^30 added or taken off.
constexpr int kLaOut = (int)0xC0000000u;

// A 32-column block of a row, laid out as store_cblock's, through a buffer descriptor: `at` is the byte offset of the row's block, kLaOut
// where nothing is to be stored. No branch around a store: the waits for the loads ahead of it then need not
// wait for the store as well.
template <typename O>
__device__ __forceinline__ void la_store(__amdgpu_buffer_rsrc_t to, int at, const f32x16& acc, int hh, int ncols) {
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int c = 8 * j + 4 * hh;
      const f32x4 v = {acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]};
      __builtin_amdgcn_raw_buffer_store_b128(bitcast<u32x4>(v), to, (c < ncols ? at : kLaOut) + 4 * c, 0, 0);
    }
  } else {
    typedef O O4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < 2; j++) {
      O4 x, y;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        x[c] = (O)acc[8 * j + c];
        y[c] = (O)acc[8 * j + 4 + c];
      }
      const u32x2 xd = bitcast<u32x2>(x), yd = bitcast<u32x2>(y);
      const auto r0 = __builtin_amdgcn_permlane32_swap(xd[0], yd[0], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(xd[1], yd[1], false, false);
      const int c = 16 * j + 8 * hh;
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{r0[0], r1[0], r0[1], r1[1]}, to, (c < ncols ? at : kLaOut) + 2 * c, 0, 0);
    }
  }
}

// Waves per SIMD that the registers are to allow; S takes DA / 2 of them.
constexpr int la_waves(int DA) { return DA <= 128 ? 2 : 1; }

template <typename T, typename O, int DA, int NW, int C, int PIECES, bool STATE>
__global__ __launch_bounds__(NW * 64, la_waves(DA)) void la_kernel(LaPasses) {
  using F = typename La<T>::F;
  constexpr int NT = NW * 64, DB = NW * 32, NB = C / 32, KT = DA / 32, E = 16 / sizeof(T);
  constexpr int CA = DA / E, CB = DB / E;                     // 16-byte chunks of a row
  constexpr int LA = C * CA / NT, LB = C * CB / NT;           // chunks per thread
  static_assert(NT % CA == 0 && C * CA % NT == 0 && NT % CB == 0 && C * CB % NT == 0, "tile loads");
  // fp16: y with its rows weighted, in PIECES parts, and z, in two, lie beside x and y in tiles of their own
  constexpr bool HALF = __is_same(T, _Float16);
  using U = typename std::conditional<HALF, __bf16, T>::type;
  using FU = typename La<U>::F;
  constexpr int PZ = HALF ? 2 : PIECES;
  constexpr int LDA = kLaRow<T, DA>, LDW = kLaRowZ<U, DA>, LDZ = kLaRowZ<U, DB>;
  constexpr int NX = STATE ? 0 : C * LDA, NY = HALF && STATE ? 0 : C * LDA, NV = HALF ? C * LDW : 0, NZ = C * LDZ;
  __shared__ __align__(16) T lds[NX + NY + PIECES * NV + (HALF ? 2 : 1) * NZ];
  __shared__ float pw[STATE ? 1 : C + 32];                    // pscale lambda^k at k + 31; zeros for k < 0
  __shared__ __align__(16) float pu[HALF ? 4 : C];            // weights of the rows in the update
  __shared__ __align__(16) float pn[HALF && !STATE ? DB : 4]; // fp16: what undoes the powers of two of S's columns
  T* const tx = lds;
  T* const ty = lds + NX;
  U* const tw = (U*)(ty + NY);
  U* const tz = tw + PIECES * NV;

  const int tid = threadIdx.x, lane = tid % 64, r = lane % 32, g = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  // The argument, where it lies: one of its passes is picked by a scalar, which no copy of it in registers allows.
  const LaPasses& all = *(const LaPasses*)(const __attribute__((address_space(4))) LaPasses*)__builtin_amdgcn_kernarg_segment_ptr();
  const int ndb = (all.p[0].db + DB - 1) / DB;
  // Items in the order (sequence, segment, head, column tile, pass). What shares rows (the passes and tiles of a head, the
  // heads of a group) runs on one XCD; such groups are dealt to the XCDs in turn, because neighbours may differ in length (in
  // contiguous ranges a prompt of 32768 rows beside 255 single tokens ran on one XCD: 1958 us, 675 dealt).
  const int G = all.n * ndb * max(all.p[0].hx, max(all.p[0].hy, all.p[0].hz));
  int w = blockIdx.x;
  if (w < (int)(gridDim.x / G / 8) * 8 * G) w = ((w / 8) / G * 8 + w % 8) * G + (w / 8) % G;
  const LaArgs& p = all.p[w % all.n];
  w /= all.n;
  const int segs = STATE ? p.nseg - 1 : p.nseg;
  const int dbt = w % ndb;
  w /= ndb;
  const int h = w % p.NH;
  int b, sg;
  la_item(p, w / p.NH, segs, tid, NT, b, sg);
  if (sg < 0) return;
  const LaSeq sq = la_seq(p, b);
  const int nseg = la_segments(p, sq.len);
  const int col0 = dbt * DB + 32 * wave;                      // the wave's first column

  const long long obase = (p.cu ? 0 : b * p.so.b) + h * p.so.h;
  if constexpr (!STATE) {
    // rows of no sequence in front of the first one and behind the last one
    const int c0 = dbt * DB, nc = min(DB, p.db - c0);
    if (p.cu && sg == 0 && b == 0) la_zero_rows<O>(p, obase, 0, sq.row0, c0, nc, tid, NT);
    if (p.cu && sg == 0 && b == p.batch - 1) la_zero_rows<O>(p, obase, sq.row0 + sq.len, p.total, c0, nc, tid, NT);
    if (sq.slot < 0) {
      if (sg == 0) la_zero_rows<O>(p, obase, sq.row0, sq.row0 + sq.len, c0, nc, tid, NT);
      return;
    }
  }
  if (sq.slot < 0 || sg >= nseg || (STATE && sg >= nseg - 1)) return;
  const bool tail = sg == nseg - 1;
  // the segment's rows, counted in processing order
  const int p0 = sg * p.seg, p1 = tail ? sq.len : p0 + p.seg;
  const int nch = (p1 - p0 + C - 1) / C;

  const float d = la_decay(p, b, h), dl2 = d * kLog2e;
  const float* const weight = pw + 31 + r - 4 * g;
  if constexpr (!STATE)
    for (int i = tid; i < C + 32; i += NT) pw[i] = i < 31 ? 0.0f : p.pscale * la_pow(dl2, (float)(i - 31));
  if constexpr (!HALF)
    for (int i = tid; i < C; i += NT) pu[i] = p.uscale * la_pow(dl2, (float)(C - 1 - i));

  // byte offset of a state's element in the lane's column
  auto state_at = [&](int a, int ra, int rb) { return a < p.da && col0 + r < p.db ? 4 * (a * ra + (col0 + r) * rb) : kLaOut; };
  f32x16 S[KT];
  const long long state = ((long long)sq.slot * p.NH + h) * p.da * p.db;
#pragma unroll
  for (int t = 0; t < KT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) S[t][i] = 0.0f;
  if (!STATE) {
    const float* from = nullptr;
    int ra = p.sa, rb = p.sb;
    if (nseg == 1 || (sg == 0 && !p.inplace)) {                // (one segment has no ws)
      if (p.first) from = p.first + state;
    } else {
      from = p.ws + ((la_ws_row(p, b, sq) + sg) * p.NH + h) * p.da * p.db;
      ra = p.wa;
      rb = p.wb;
    }
    if (from) {
      const auto rs = buf_rsrc32(from, (unsigned)(p.da * p.db * 4));
      if (ra == 1) {                                           // four elements of the lane's side by side
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 v = bitcast<f32x4>(buf_load16(rs, state_at(32 * t + 2 * i + 4 * g, 1, rb)));
#pragma unroll
            for (int j = 0; j < 4; j++) S[t][i + j] = v[j];
          }
      } else
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          S[t][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, state_at(32 * t + 8 * (i / 4) + 4 * g + i % 4, ra, rb), 0, 0));
    }
  }

  // Tile loads. A thread's 16-byte column and its rows of the tile are fixed. Buffer descriptors span `span` rows of the
  // segment, so that offsets within them are 32 bits wide and move by the same step from chunk to chunk. Rows behind the
  // segment's last one fall outside (past the descriptor's end, or in reverse below its start: negative) and read as zeros or
  // are not stored; columns past the head dim start from an offset so large that no row brings it back.
  const int xr = tid / CA, xc = tid % CA, zr = tid / CB, zc = tid % CB;
  const int bx = (int)p.sx.s * (int)sizeof(T), by = (int)p.sy.s * (int)sizeof(T), bz = (int)p.sz.s * (int)sizeof(T), bo = (int)p.so.s * (int)sizeof(O);
  const char* const gx = (const char*)p.x + ((p.cu ? 0 : b * p.sx.b) + (h / p.hx) * p.sx.h + sq.row0 * p.sx.s) * (long long)sizeof(T);
  const char* const gy = (const char*)p.y + ((p.cu ? 0 : b * p.sy.b) + (h / p.hy) * p.sy.h + sq.row0 * p.sy.s) * (long long)sizeof(T);
  const char* const gz = (const char*)p.z + ((p.cu ? 0 : b * p.sz.b) + (h / p.hz) * p.sz.h + sq.row0 * p.sz.s + dbt * DB) * (long long)sizeof(T);
  const char* const go = (const char*)p.o + (obase + sq.row0 * p.so.s + col0) * (long long)sizeof(O);
  // the lowest row of the span that starts at row q0 in processing order, and its number of rows
  auto span = [&](int q0, int& rows) -> long long {
    rows = max(0, min(p.span, p1 - q0));
    return p.rev ? sq.len - q0 - rows : q0;
  };
  auto bytes = [&](int rows, int stride, int width) { return rows > 0 ? (unsigned)((rows - 1) * stride + width) : 0u; };
  // the offset of row i of a span
  auto place = [&](int i, int rows, int stride) { return (p.rev ? rows - 1 - i : i) * stride; };
  const int sign = p.rev ? -1 : 1, per = p.span / C;                     // chunks of a span
  const int jx = xc * E < p.da ? xc * 16 : kLaOut, jz = dbt * DB + zc * E < p.db ? zc * 16 : kLaOut;
  // (start and size, not descriptors: those went through vector registers and a loop around each store)
  const char *fx = nullptr, *fy = nullptr, *fz = nullptr, *fo = nullptr;
  unsigned nx = 0, ny = 0, nz = 0, no = 0;
  int vox = 0, voy = 0, voz = 0, voo[STATE ? 1 : NB];
  u32x4 vx[STATE ? 1 : LA], vy[LA], vz[LB];
  int next = p0, left = 0, oleft = 0;                                    // the row to fetch, chunks left of the spans
  auto fetch = [&]() {
    if (left == 0) {
      left = per;
      int rows;
      const long long row = span(next, rows);
      fx = la_uniform(gx + row * bx), nx = la_uniform(bytes(rows, bx, p.da * (int)sizeof(T)));
      fy = la_uniform(gy + row * by), ny = la_uniform(bytes(rows, by, p.da * (int)sizeof(T)));
      fz = la_uniform(gz + row * bz), nz = la_uniform(bytes(rows, bz, (p.db - dbt * DB) * (int)sizeof(T)));
      vox = jx + place(xr, rows, bx);
      voy = jx + place(xr, rows, by);
      voz = jz + place(zr, rows, bz);
    }
    left--;
    next += C;
    const auto rx = buf_rsrc32(fx, nx), ry = buf_rsrc32(fy, ny), rz = buf_rsrc32(fz, nz);
#pragma unroll
    for (int i = 0; i < LA; i++) {
      if constexpr (!STATE) vx[i] = buf_load16(rx, vox + i * (sign * (NT / CA) * bx));
      vy[i] = buf_load16(ry, voy + i * (sign * (NT / CA) * by));
    }
#pragma unroll
    for (int i = 0; i < LB; i++) vz[i] = buf_load16(rz, voz + i * (sign * (NT / CB) * bz));
    vox += sign * C * bx;
    voy += sign * C * by;
    voz += sign * C * bz;
  };
  T* const px = tx + xr * LDA + xc * E;
  T* const py = ty + xr * LDA + xc * E;
  U* const py2 = tw + xr * LDW + xc * E;
  U* const pz = tz + zr * LDZ + zc * E;
  float wy[LA];                                               // fp16: the weights of the thread's rows of y
#pragma unroll
  for (int i = 0; i < LA; i++) wy[i] = HALF ? p.uscale * la_pow(dl2, (float)(C - 1 - xr - i * (NT / CA))) : 0.0f;
  auto put = [&](T* at, u32x4 v) {                            // rows of x and y are 8-byte aligned in 16 bits
    if constexpr (sizeof(T) == 2) {
      ((u32x2*)at)[0] = u32x2{v[0], v[1]};
      ((u32x2*)at)[1] = u32x2{v[2], v[3]};
    } else {
      *(u32x4*)at = v;
    }
  };

  // the state's gradient enters the first row as it is, any other state decayed once
  int lag = p.enter && sg == 0 ? -1 : 0;

  fetch();
  if constexpr (!STATE) {
    // Stores to nowhere, as many as a chunk has behind the next one's loads: a wait for loads counts what was issued since, and the
    // compiler takes the lowest count of all ways into the loop.
    f32x16 none;
#pragma unroll
    for (int i = 0; i < 16; i++) none[i] = 0.0f;
    const auto ro = buf_rsrc32(p.o, 0u);
#pragma unroll
    for (int q = 0; q < NB; q++) la_store<O>(ro, kLaOut, none, g, 32);
  }
  for (int c = 0; c < nch; c++) {
    const int n = min(C, p1 - p0 - c * C);                    // rows of the chunk; zeros behind them
    // the decay that S is behind by, and whether it is made up for now
    const int behind = lag + n;
    const bool due = fabsf(dl2 * (float)behind) > kLaLag;
    const float weigh = due ? 1.0f : exp2_fast(dl2 * (float)behind);
    if constexpr (HALF)
      if (n < C)
#pragma unroll
        for (int i = 0; i < LA; i++) wy[i] = p.uscale * la_pow(dl2, (float)max(n - 1 - xr - i * (NT / CA), 0));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LA; i++) {
      if constexpr (!STATE) put(px + i * (NT / CA) * LDA, vx[i]);
      if constexpr (!STATE || !HALF) put(py + i * (NT / CA) * LDA, vy[i]);
      if constexpr (HALF) la_put<PIECES, NV>(py2 + i * (NT / CA) * LDW, vy[i], wy[i] * weigh);
    }
#pragma unroll
    for (int i = 0; i < LB; i++) {
      if constexpr (HALF) la_put<2, NZ>(pz + i * (NT / CB) * LDZ, vz[i], 1.0f);
      else *(u32x4*)(pz + i * (NT / CB) * LDZ) = vz[i];
    }
    if constexpr (!HALF)
      if (n < C && tid < C) pu[tid] = p.uscale * la_pow(dl2, (float)max(n - 1 - tid, 0));
    fetch();
    __syncthreads();

    // What follows alternates matrix and vector instructions that do not wait for one another: the scores and the product
    // with S beside the splitting of z, the state's update beside the weighting of the scores.
    FU zf[2 * NB], z[2 * NB][PZ];                              // fp16: z is its two parts, and zf the first
    f32x8 wu[2 * NB];
#pragma unroll
    for (int s = 0; s < 2 * NB; s++) {
      zf[s] = la_cols<U, LDZ>(tz, wave, s, lane);
      if constexpr (HALF) {
        z[s][0] = zf[s];
        z[s][1] = la_cols<U, LDZ>(tz + NZ, wave, s, lane);
      } else {
        wu[s] = la_rows<float, 0>(pu, 0, s, g);
      }
    }
    // A value of z that is no number reaches the rows that see it, not those whose weight for it is 0: a wave that has one (rare)
    // leaves it out of the product and sets those rows after.
    bool none = false;
    if constexpr (!STATE) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < 2 * NB; s++) top = la_top(top, zf[s]);
      none = __builtin_amdgcn_ballot_w64(la_top_bits<U>(top) >= kLaNone<U>) != 0;
    }
    auto split = [&](int k) {                                  // the k-th of 8 NB pairs of weighted z
      if constexpr (!HALF) {
        const int s = k / 4, j = 2 * (k % 4);
        la_split2<T, PIECES>((float)zf[s][j] * (wu[s][j] * weigh), (float)zf[s][j + 1] * (wu[s][j + 1] * weigh), z[s], j);
      }
    };

    f32x16 sc[NB][NB], o[NB];                                  // [key block][query block], transposed
    float norm = 1.0f;
    f32x4 undo[4];                                             // for the lane's rows of o
    if constexpr (!STATE) {
#pragma unroll
      for (int q = 0; q < NB; q++) {
#pragma unroll
        for (int i = 0; i < 16; i++) o[q][i] = 0.0f;
#pragma unroll
        for (int k = 0; k <= q; k++)
#pragma unroll
          for (int i = 0; i < 16; i++) sc[k][q][i] = 0.0f;
      }
      if constexpr (HALF) {
        float m = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int i = 0; i < 16; i++) m = fmaxf(m, fabsf(S[t][i]));
        float inv;
        norm = la_norm(half_max(m), inv);
        pn[32 * wave + r] = inv;
        __builtin_amdgcn_wave_barrier();                       // (a wave's own LDS accesses are in order)
#pragma unroll
        for (int i = 0; i < 4; i++) undo[i] = *(const f32x4*)(pn + 32 * wave + 8 * i + 4 * g);
      }
#pragma unroll
      for (int s = 0; s < DA / 16; s++) {
        F xf[NB], yf[NB], sf;
#pragma unroll
        for (int q = 0; q < NB; q++) xf[q] = la_rows<T, LDA>(tx, 32 * q + r, s, g);
#pragma unroll
        for (int k = 0; k < NB; k++) yf[k] = la_rows<T, LDA>(ty, 32 * k + r, s, g);
#pragma unroll
        for (int j = 0; j < 8; j++) sf[j] = (T)(S[s / 2][8 * (s % 2) + j] * norm);
#pragma unroll
        for (int q = 0; q < NB; q++) {
#pragma unroll
          for (int k = 0; k <= q; k++) sc[k][q] = La<T>::mma(yf[k], xf[q], sc[k][q]);
          o[q] = La<T>::mma(sf, xf[q], o[q]);
        }
#pragma unroll
        for (int k = s * 8 * NB / (DA / 16); k < (s + 1) * 8 * NB / (DA / 16); k++) split(k);
      }
    }

    // the state's update
    if (due) {
      const float f = exp2_fast(-dl2 * (float)behind);
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) S[t][i] *= f;
    }
    if constexpr (STATE)
#pragma unroll
      for (int k = 0; k < 4; k++) split(k);
    // the lane's rows of the scores and of the product with S, a quarter for each quarter of the tiles
    float lw[NB];
    if constexpr (!STATE)
#pragma unroll
      for (int q = 0; q < NB; q++) lw[q] = p.iscale * exp2_fast(-dl2 * (float)(32 * q + r + 1 + lag));
    auto weighted = [&](int part, int parts) {
#pragma unroll
      for (int q = 0; q < NB; q++)
#pragma unroll
        for (int i = 16 * part / parts; i < 16 * (part + 1) / parts; i++) {
          o[q][i] *= HALF ? lw[q] * undo[i / 4][i % 4] : lw[q];
#pragma unroll
          for (int k = 0; k <= q; k++) {
            const float w = weight[32 * (q - k) - (8 * (i / 4) + i % 4)];
            sc[k][q][i] = w == 0.0f ? 0.0f : sc[k][q][i] * w;  // (a masked score that is no number stays out)
          }
        }
    };
#pragma unroll
    for (int s = 0; s < 2 * NB; s++) {
#pragma unroll
      for (int t = 0; t < KT; t++) {
        if constexpr (HALF) {
          FU y[PIECES];
#pragma unroll
          for (int i = 0; i < PIECES; i++) y[i] = la_cols<U, LDW>(tw + i * NV, t, s, lane);
          // from the smallest on; left out are 2^-16 of the product for two parts of y, 2^-24 for three
          if constexpr (PIECES == 3) {
            S[t] = La<U>::mma(y[2], z[s][0], S[t]);
            S[t] = La<U>::mma(y[1], z[s][1], S[t]);
          }
          S[t] = La<U>::mma(y[1], z[s][0], S[t]);
          S[t] = La<U>::mma(y[0], z[s][1], S[t]);
          S[t] = La<U>::mma(y[0], z[s][0], S[t]);
        } else {
          const F yt = la_cols<T, LDA>(ty, t, s, lane);
#pragma unroll
          for (int i = PIECES - 1; i >= 0; i--) S[t] = La<T>::mma(yt, z[s][i], S[t]);
        }
        if constexpr (STATE) {
          if (s + 1 < 2 * NB)
#pragma unroll
            for (int k = 4 * t / KT; k < 4 * (t + 1) / KT; k++) split(4 * (s + 1) + k);
        } else {
          weighted(s * KT + t, 2 * NB * KT);
        }
      }
    }
    lag = due ? 0 : behind;

    if constexpr (!STATE) {
      if (oleft == 0) {
        oleft = per;
        int rows;
        const long long row = span(p0 + c * C, rows);
        fo = la_uniform(go + row * bo), no = la_uniform(bytes(rows, bo, min(32, max(p.db - col0, 0)) * (int)sizeof(O)));
#pragma unroll
        for (int q = 0; q < NB; q++) voo[q] = place(32 * q + r, rows, bo);
      }
      oleft--;
      const auto ro = buf_rsrc32(fo, no);
#pragma unroll
      for (int q = 0; q < NB; q++) {
        if (none) {
#pragma unroll
          for (int s = 0; s < 2 * NB; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const bool ok = fabsf((float)zf[s][j]) < __builtin_inff();
              zf[s][j] = ok ? zf[s][j] : (U)0.0f;
              if constexpr (HALF) z[s][1][j] = ok ? z[s][1][j] : (U)0.0f;
            }
        }
#pragma unroll
        for (int s = 0; s < 2 * (q + 1); s++) {
          if constexpr (HALF) {                                // 16 bits of the score, in any range
            FU pf[2];
#pragma unroll
            for (int j = 0; j < 8; j += 2) la_split2<U, 2>(sc[s / 2][q][8 * (s % 2) + j], sc[s / 2][q][8 * (s % 2) + j + 1], pf, j);
            o[q] = La<U>::mma(z[s][1], pf[0], o[q]);
            o[q] = La<U>::mma(zf[s], pf[1], o[q]);
            o[q] = La<U>::mma(zf[s], pf[0], o[q]);
          } else {
            F pf;
#pragma unroll
            for (int j = 0; j < 8; j++) pf[j] = (T)sc[s / 2][q][8 * (s % 2) + j];
            o[q] = La<T>::mma(zf[s], pf, o[q]);
          }
        }
        if (none)
          for (int j = 0; j <= 32 * q + r && j < n; j++) {
            const U* const row = tz + j * LDZ + 32 * wave + 4 * g;
#pragma unroll
            for (int i = 0; i < 16; i++)
              if (!(fabsf((float)row[8 * (i / 4) + i % 4]) < __builtin_inff())) o[q][i] = __builtin_nanf("");
          }
        la_store<O>(ro, voo[q], o[q], g, p.db - col0);
        voo[q] += sign * C * bo;
      }
    }
  }

  float* to = nullptr;
  int ra = p.sa, rb = p.sb;
  float f = 1.0f;
  if constexpr (STATE) {
    to = p.ws + ((la_ws_row(p, b, sq) + sg + 1) * p.NH + h) * p.da * p.db;
    ra = p.db;
    rb = 1;
  } else if (tail && p.last) {
    to = p.last + state;
    if (p.leave && sq.len > 0) f = la_pow(dl2, 1.0f);
  }
  if (to) {
    if (nch > 0) f *= exp2_fast(-dl2 * (float)lag);
    const auto rs = buf_rsrc32(to, (unsigned)(p.da * p.db * 4));
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[t][i] * f), rs, state_at(32 * t + 8 * (i / 4) + 4 * g + i % 4, ra, rb), 0, 0);
  }
}

// one new token or a few of each sequence (linear_step.hip)
void la_step(const LaArgs& p, int dtype, hipStream_t stream);

// The states that the segments add (`state`), or everything; exact: the states are results, or run into such. The passes of a
// launch have da, db and o32 in common, and all that makes their items.
template <typename T>
void la_launch(const LaPasses& p, bool state, bool exact, hipStream_t stream);

constexpr int kLaChunk = 32;   // rows of a chunk; segments are multiples of it

template <typename T, typename O, int DA, int NW, int PIECES, bool STATE>
inline void la_run(const LaPasses& a, hipStream_t st) {
  const LaArgs& p = a.p[0];
  const long long items = la_items(p, STATE) * p.NH * ((p.db + NW * 32 - 1) / (NW * 32)) * a.n;
  hipLaunchKernelGGL((la_kernel<T, O, DA, NW, kLaChunk, PIECES, STATE>), dim3((unsigned)items), dim3(NW * 64), 0, st, a);
}

template <typename T, typename O, int NW, int PIECES, bool STATE>
inline void la_depth(const LaPasses& a, hipStream_t st) {
  const int da = a.p[0].da;
  if (da <= 64) la_run<T, O, 64, NW, PIECES, STATE>(a, st);
  else if (da <= 128) la_run<T, O, 128, NW, PIECES, STATE>(a, st);
  else la_run<T, O, 256, NW, PIECES, STATE>(a, st);
}

template <typename T, typename O, int PIECES, bool STATE>
inline void la_pick(const LaPasses& a, hipStream_t st) {
  if (a.p[0].db <= 64) la_depth<T, O, 2, PIECES, STATE>(a, st);
  else la_depth<T, O, 4, PIECES, STATE>(a, st);
}

template <typename T, int PIECES>
inline void la_all(const LaPasses& a, bool state, hipStream_t st) {
  if (state) return la_pick<T, T, PIECES, true>(a, st);
  if constexpr (sizeof(T) == 2)
    if (a.p[0].o32) return la_pick<T, float, PIECES, false>(a, st);
  la_pick<T, T, PIECES, false>(a, st);
}

}  // namespace fa
