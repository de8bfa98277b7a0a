// linear.hip — entry points of linear attention: argument checks, the split of long sequences into segments, the passes of
// forward and backward, and the kernels between them.
//
// Segments. A workgroup per head and 128 columns leaves CUs idle where batch x heads is small, so long sequences are cut:
// one launch forms what each segment adds to the state (reading y and z), la_scan_kernel turns these into the state before
// each segment, and the main launch runs all segments side by side. The backward pass takes the forward pass's states
// for dq; dv and dk share theirs.
#include <string.h>

#include "linear_kernel.hpp"
#include "status.hpp"

namespace fa {

// Segment sg's addition to the state stands where the state before segment sg + 1 is to be; the state before the first is written
// where the call overwrites it. A thread carries four elements along; its loads of the next four segments do not wait for
// the sum (B2 S4096 H32 D128, 8 segments: 11 us, 64 MB).
__global__ __launch_bounds__(256) void la_scan_kernel(LaArgs p) {
  const int n = p.da * p.db, nb = (n / 4 + 255) / 256;
  const int e = 4 * ((blockIdx.x % nb) * 256 + threadIdx.x);
  const int i = blockIdx.x / nb / p.NH, h = blockIdx.x / nb % p.NH;
  int b = i;
  if (p.cu) {
    // item i: the one sequence of several segments that starts in rows [i seg, (i + 1) seg)
    __shared__ int found;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int j = threadIdx.x; j < p.batch; j += 256) {
      const LaSeq sq = la_seq(p, j);
      if (sq.row0 / p.seg == i && la_segments(p, sq.len) > 1) found = j;
    }
    __syncthreads();
    b = found;
    if (b < 0) return;
  }
  const LaSeq sq = la_seq(p, b);
  if (e >= n || sq.slot < 0) return;
  const int nseg = la_segments(p, sq.len);
  const long long step = (long long)p.NH * n;
  float* const ws = p.ws + (la_ws_row(p, b, sq) * p.NH + h) * n + e;
  f32x4 cur = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.first) cur = *(const f32x4*)(p.first + ((long long)sq.slot * p.NH + h) * n + e);
  const float d = la_decay(p, b, h);
  const LaFade whole(d, (float)p.seg), first(d, (float)(p.seg - 1));
  if (p.inplace) *(f32x4*)ws = cur;
  for (int s = 1; s < nseg; s += 4) {
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = *(const f32x4*)(ws + min(s + j, nseg - 1) * step);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const LaFade& fade = p.enter && s + j == 1 ? first : whole;
#pragma unroll
      for (int k = 0; k < 4; k++) cur[k] = fade(cur[k]) + v[j][k];
      if (s + j < nseg) *(f32x4*)(ws + (s + j) * step) = cur;
    }
  }
}

// The gradients of a head of keys or values that `gqa` heads of queries share: their sum, in the heads' order, rounded once.
struct LaGroup {
  const float* part;
  void* out;
  fa_strides so;
  int D;
};
template <typename T>
__global__ __launch_bounds__(256) void la_group_kernel(LaGroup one, LaGroup two, unsigned blocks, long long rows, int n, int NKV, int gqa) {
  const bool other = blockIdx.x >= blocks;
  const float* const part = other ? two.part : one.part;
  T* const out = (T*)(other ? two.out : one.out);
  const fa_strides so = other ? two.so : one.so;
  const int D = other ? two.D : one.D, d4 = D / 4;
  const long long i = (long long)(blockIdx.x - (other ? blocks : 0)) * 256 + threadIdx.x;
  if (i >= rows * NKV * d4) return;
  const int c = (int)(i % d4), hk = (int)(i / d4 % NKV);
  const long long row = i / d4 / NKV;
  const float* from = part + ((row * NKV + hk) * gqa) * (long long)D + 4 * c;
  f32x4 sum = *(const f32x4*)from;
  for (int j = 1; j < gqa; j++) sum += *(const f32x4*)(from + (long long)j * D);
  T* to = out + (row / n) * so.b + (row % n) * so.s + hk * so.h + 4 * c;
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 v;
#pragma unroll
  for (int j = 0; j < 4; j++) v[j] = (T)sum[j];
  *(T4*)to = v;
}

namespace {

int la_elt(int dtype) { return dtype == FA_F32 ? 4 : 2; }

// The stride of a single row is anything; the kernel takes it for a distance.
void la_single(LaArgs& a) {
  if ((a.cu ? a.total : a.n) > 1) return;
  a.sx.s = a.sy.s = a.da;
  a.sz.s = a.so.s = a.db;
}

// Segments of a call, the same for all its passes. A wave per 32 columns of a head has a row's work in about 60 ns, whatever the others do, so
// the longest sequence takes n of those; spread evenly over the 1024 SIMDs the rows of all heads take n * 1024 / (waves' rows) times
// less. Below 1.8 that does not pay for a second reading of k and v and the states' traffic (8 prompts of up to 2048 rows, 32 heads
// of 128, ratio 1.44: 131 us in one piece, 190 cut; 24 documents H16 D64, ratio 2.6: forward and backward 448 against 365). Two waves per
// SIMD then, but no segment under `least` rows (fp32, B2 S1000 H16 of 64 and 128 wide, forward and backward: 64 rows 165 us,
// 128 rows 153; 16 bits, heads of 256: 128 rows 93, 256 rows 71). Packed sequences leave parts of segments at their ends: with them
// counted the 24 documents take 295 us, 303 without, prompts of 8 such documents H16 D128 93 and 113.
void la_split(LaArgs& a, const FableLinearParams& p, int dtype) {
  la_single(a);
  const int D = p.DK > p.DV ? p.DK : p.DV;
  const long long rows = p.cu ? p.total : (long long)a.batch * a.n;
  const long long work = rows * a.NH * ((D + 31) / 32);
  const long long least = dtype == FA_F32 ? 128 : 256;
  long long seg = a.n;
  long long waves = 2048;
  if (p.cu) {                                                  // each packed sequence ends in a part of a segment, half of one on average
    waves -= (long long)a.batch * a.NH * ((D + 31) / 32) / 2;
    if (waves < 1024) waves = 1024;
  }
  if ((long long)a.n * 10240 > 18 * work) seg = (work + waves - 1) / waves;
  seg = seg < least ? least : seg;
  seg = (seg + kLaChunk - 1) / kLaChunk * kLaChunk;
  a.seg = (int)(seg < (1 << 30) ? seg : (1 << 30));
  a.nseg = (int)(((long long)a.n + a.seg - 1) / a.seg);
  if (a.nseg < 1) a.nseg = 1;
  a.wa = p.DV, a.wb = 1;
}

// the rows that la_ws_row() counts on
long long la_ws(const LaArgs& a) {
  const long long rows = a.cu ? 2 * (a.total / a.seg + 2) : (long long)a.batch * a.nseg;
  return a.nseg > 1 ? rows * a.NH * a.da * a.db * 4 : 0;
}

LaArgs la_base(const FableLinearParams& p) {
  LaArgs a;
  memset(&a, 0, sizeof(a));
  a.decay = p.decay;
  a.decay_b = p.decay_b;
  a.cu = p.cu;
  a.total = p.total;
  a.batch = p.batch;
  a.n = p.cu && p.n > p.total ? (int)p.total : p.n;
  a.NH = p.NH;
  a.pscale = p.scale;
  a.hx = a.hy = a.hz = 1;
  return a;
}

LaArgs la_forward(const FableLinearParams& p, int dtype) {
  LaArgs a = la_base(p);
  a.x = p.q, a.y = p.k, a.z = p.v, a.o = p.o;
  a.sx = p.sq, a.sy = p.sk, a.sz = p.sv, a.so = p.so;
  a.hy = a.hz = p.gqa;
  a.da = p.DK, a.db = p.DV;
  a.first = p.state_in, a.last = p.state_out;
  a.sa = p.DV, a.sb = 1;
  a.slots = p.slots, a.nslots = p.num_slots;
  a.inplace = p.state_in && p.state_in == p.state_out;
  a.iscale = p.scale, a.uscale = 1.0f;
  la_split(a, p, dtype);
  return a;
}

// dq_t = scale S_t dout_t
LaArgs la_dq(const FableLinearParams& p, int dtype) {
  LaArgs a = la_base(p);
  a.x = p.dout, a.y = p.v, a.z = p.k, a.o = p.dq;
  a.sx = p.sdo, a.sy = p.sv, a.sz = p.sk, a.so = p.sdq;
  a.hy = a.hz = p.gqa;
  a.da = p.DV, a.db = p.DK;
  a.first = p.state_in;
  a.sa = 1, a.sb = p.DV;
  a.iscale = p.scale, a.uscale = 1.0f;
  la_split(a, p, dtype);
  a.wa = 1, a.wb = p.DV;   // the states as they are for k, v (q, dout)
  return a;
}

// dv_t = G_t^T k_t; G is DK x DV
LaArgs la_dv(const FableLinearParams& p, int dtype) {
  LaArgs a = la_base(p);
  a.x = p.k, a.y = p.q, a.z = p.dout, a.o = p.dv;
  a.sx = p.sk, a.sy = p.sq, a.sz = p.sdo, a.so = p.sdv;
  a.hx = p.gqa;
  a.da = p.DK, a.db = p.DV;
  a.first = p.dstate_out, a.last = p.dstate_in;
  a.sa = p.DV, a.sb = 1;
  a.iscale = 1.0f, a.uscale = p.scale;
  a.rev = 1, a.enter = p.dstate_out != nullptr, a.leave = 1;
  la_split(a, p, dtype);
  return a;
}

// dk_t = G_t v_t, on G^T
LaArgs la_dk(const FableLinearParams& p, int dtype) {
  LaArgs a = la_base(p);
  a.x = p.v, a.y = p.dout, a.z = p.q, a.o = p.dk;
  a.sx = p.sv, a.sy = p.sdo, a.sz = p.sq, a.so = p.sdk;
  a.hx = p.gqa;
  a.da = p.DV, a.db = p.DK;
  a.first = p.dstate_out;
  a.sa = 1, a.sb = p.DV;
  a.iscale = 1.0f, a.uscale = p.scale;
  a.rev = 1, a.enter = p.dstate_out != nullptr;
  la_split(a, p, dtype);
  a.wa = 1, a.wb = p.DV;   // the states as they are for k, v (q, dout)
  return a;
}

void la_go(const LaArgs* first, int n, int dtype, bool state, bool exact, hipStream_t st) {
  LaPasses all;
  all.n = n;
  for (int i = 0; i < 3; i++) {
    LaArgs& a = all.p[i] = first[i < n ? i : 0];
    long long row = (state ? 0 : a.so.s * (a.o32 ? 4 : la_elt(dtype)));
    for (const fa_strides* s : {&a.sx, &a.sy, &a.sz}) row = s->s * la_elt(dtype) > row ? s->s * la_elt(dtype) : row;
    const long long span = row > 0 ? (1LL << 29) / row / kLaChunk * kLaChunk : kLaChunk;
    a.span = (int)(span < kLaChunk ? kLaChunk : span > (1 << 29) ? (1 << 29) : span);
  }
  if (dtype == FA_F16) la_launch<_Float16>(all, state, exact, st);
  else if (dtype == FA_BF16) la_launch<__bf16>(all, state, exact, st);
  else la_launch<float>(all, state, exact, st);
}

// The states before all segments, into a.ws, for arguments whose states are as the caller has them (DK x DV).
void la_states(const LaArgs& a, int dtype, bool exact, hipStream_t st) {
  if (a.nseg < 2) return;
  la_go(&a, 1, dtype, true, exact, st);
  const long long items = (a.cu ? a.total / a.seg + 1 : a.batch) * a.NH * ((a.da * a.db / 4 + 255) / 256);
  hipLaunchKernelGGL(la_scan_kernel, dim3((unsigned)items), dim3(256), 0, st, a);
}

// What every call has to satisfy; the tensors' own checks follow in the entry points.
int la_check(const FableLinearParams& p, int dtype, const char* what) {
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return fail(FA_ERR_DTYPE, "%s: unknown dtype %d", what, dtype);
  if (p.DK < 8 || p.DK > 256 || p.DK % 8 || p.DV < 8 || p.DV > 256 || p.DV % 8)
    return fail(FA_ERR_HEADDIM, "%s: head dims %d and %d: multiples of 8 up to 256", what, p.DK, p.DV);
  if (p.batch < 0 || p.n < 0 || p.NH < 1 || p.gqa < 1 || p.NH % p.gqa || p.total < 0 || p.n > (1 << 30) || p.total > (1 << 30))
    return fail(FA_ERR_ARG, "%s: batch=%d n=%d total=%lld NH=%d gqa=%d", what, p.batch, p.n, (long long)p.total, p.NH, p.gqa);
  if (((uintptr_t)p.state_in | (uintptr_t)p.state_out | (uintptr_t)p.dstate_out | (uintptr_t)p.dstate_in | (uintptr_t)p.seg_states) & 15)
    return fail(FA_ERR_ARG, "%s: states must be 16-byte aligned", what);
  // (64 workgroups of 256 threads for each state in the scan; a grid has fewer than 2^32 threads)
  if ((long long)p.batch * p.NH >= (1 << 18)) return fail(FA_ERR_ARG, "%s: batch x heads = %lld", what, (long long)p.batch * p.NH);
  return FA_OK;
}

int la_tensor(const char* what, const char* name, const void* t, const fa_strides& s, int width, const FableLinearParams& p, int dtype) {
  const int e = la_elt(dtype);
  if (!t) return fail(FA_ERR_ARG, "%s: null %s", what, name);
  if (((uintptr_t)t | (uintptr_t)(s.b * e) | (uintptr_t)(s.h * e) | (uintptr_t)(s.s * e)) & 15)
    return fail(FA_ERR_ARG, "%s: %s: rows must be 16-byte aligned", what, name);
  // Offsets within 32 rows or more are 32 bits wide, and rows must not overlap: one of no token is known by its offset.
  if ((p.cu ? p.total : p.n) > 1 && (s.s >= (1LL << 29) / (e * kLaChunk) || s.s < width))
    return fail(FA_ERR_ARG, "%s: %s: a row stride of %lld values", what, name, (long long)s.s);
  return FA_OK;
}

// q, k, v and o, or in the backward pass dout and the gradients
int la_tensors(const char* what, const FableLinearParams& p, int dtype, bool backward) {
  int rc;
  if ((p.cu ? p.total : p.n) == 0) return FA_OK;
  if ((rc = la_tensor(what, "q", p.q, p.sq, p.DK, p, dtype)) || (rc = la_tensor(what, "k", p.k, p.sk, p.DK, p, dtype)) ||
      (rc = la_tensor(what, "v", p.v, p.sv, p.DV, p, dtype)))
    return rc;
  if (!backward) return la_tensor(what, "o", p.o, p.so, p.DV, p, dtype);
  if ((rc = la_tensor(what, "dout", p.dout, p.sdo, p.DV, p, dtype)) || (rc = la_tensor(what, "dq", p.dq, p.sdq, p.DK, p, dtype)) ||
      (rc = la_tensor(what, "dk", p.dk, p.sdk, p.DK, p, dtype)))
    return rc;
  return la_tensor(what, "dv", p.dv, p.sdv, p.DV, p, dtype);
}

long long la_group_bytes(const FableLinearParams& p) {
  const long long rows = p.cu ? p.total : (long long)p.batch * p.n;
  return p.gqa > 1 ? rows * p.NH * (p.DK + p.DV) * 4 : 0;
}

long long la_round(long long x) { return (x + 255) / 256 * 256; }

// Forward: the segments' states. Backward: those of q and dout, before them the ones of k and v, if the forward pass's are not
// given, and behind them the partial gradients of shared heads.
long long la_need(const FableLinearParams& p, int dtype, bool backward) {
  const long long w = la_ws(la_forward(p, dtype));
  return backward ? la_round(w) * (p.seg_states ? 1 : 2) + la_group_bytes(p) : w;
}

template <typename T>
void la_group(const LaGroup& one, const LaGroup& two, const FableLinearParams& p, hipStream_t st) {
  const long long rows = p.cu ? p.total : (long long)p.batch * p.n;
  const int n = p.cu ? (int)rows : p.n, NKV = p.NH / p.gqa;
  if (rows == 0) return;
  const long long blocks = (rows * NKV * (one.D / 4) + 255) / 256, more = (rows * NKV * (two.D / 4) + 255) / 256;
  hipLaunchKernelGGL(la_group_kernel<T>, dim3((unsigned)(blocks + more)), dim3(256), 0, st, one, two, (unsigned)blocks, rows, n, NKV, p.gqa);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int64_t fable_linear_attn_ws_bytes(FableLinearParams p, int dtype, int backward) {
  if (la_check(p, dtype, "fable_linear_attn_ws_bytes") != FA_OK) return -1;
  return la_need(p, dtype, backward != 0);
}

extern "C" int fable_linear_attn_fwd(FableLinearParams p, int dtype, void* ws, int64_t ws_bytes, void* stream) {
  const char* what = "fable_linear_attn_fwd";
  int rc = la_check(p, dtype, what);
  if (rc != FA_OK) return rc;
  if (!p.decay) return fail(FA_ERR_ARG, "%s: null decay", what);
  if (p.slots && (p.num_slots < 0 || (!p.state_in && !p.state_out))) return fail(FA_ERR_ARG, "%s: slots without states", what);
  if ((rc = la_tensors(what, p, dtype, false)) != FA_OK) return rc;
  const long long need = la_need(p, dtype, false);
  if (need > 0 && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return fail(FA_ERR_ARG, "%s: a workspace of %lld bytes is needed, %lld given", what, need, (long long)ws_bytes);
  if (p.batch == 0) return FA_OK;
  LaArgs a = la_forward(p, dtype);
  a.ws = (float*)ws;
  const bool exact = a.last != nullptr;
  la_states(a, dtype, exact, (hipStream_t)stream);
  la_go(&a, 1, dtype, false, exact, (hipStream_t)stream);
  return launch_status(what);
}

extern "C" int fable_linear_attn_step(FableLinearParams p, int dtype, void* stream) {
  const char* what = "fable_linear_attn_step";
  int rc = la_check(p, dtype, what);
  if (rc != FA_OK) return rc;
  if (!p.decay || !p.state_in || !p.state_out) return fail(FA_ERR_ARG, "%s: null decay or state", what);
  if (p.slots && p.num_slots < 0) return fail(FA_ERR_ARG, "%s: num_slots=%d", what, p.num_slots);
  if ((rc = la_tensors(what, p, dtype, false)) != FA_OK) return rc;
  if (p.batch == 0) return FA_OK;
  la_step(la_forward(p, dtype), dtype, (hipStream_t)stream);
  return launch_status(what);
}

extern "C" int fable_linear_attn_bwd(FableLinearParams p, int dtype, void* ws, int64_t ws_bytes, void* stream) {
  const char* what = "fable_linear_attn_bwd";
  int rc = la_check(p, dtype, what);
  if (rc != FA_OK) return rc;
  if (!p.decay) return fail(FA_ERR_ARG, "%s: null decay", what);
  if (p.slots) return fail(FA_ERR_ARG, "%s: states of a pool have no gradient", what);
  if (p.gqa > 1 && (long long)p.NH * (p.DK > p.DV ? p.DK : p.DV) >= (1LL << 29) / (4 * kLaChunk)) return fail(FA_ERR_ARG, "%s: NH=%d", what, p.NH);
  if ((rc = la_tensors(what, p, dtype, true)) != FA_OK) return rc;
  const long long need = la_need(p, dtype, true);
  if (need > 0 && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return fail(FA_ERR_ARG, "%s: a workspace of %lld bytes is needed, %lld given", what, need, (long long)ws_bytes);
  if (p.batch == 0) return FA_OK;
  hipStream_t st = (hipStream_t)stream;
  // dq runs over the states of k and v, dv and dk over those of q and dout, from the last row on
  LaArgs pass[3] = {la_dq(p, dtype), la_dk(p, dtype), la_dv(p, dtype)};
  LaArgs &dq = pass[0], &dk = pass[1], &dv = pass[2];
  const bool exact = dv.last != nullptr;
  char* at = (char*)ws;
  if (p.seg_states) {
    dq.ws = (float*)p.seg_states;
  } else {
    LaArgs a = la_forward(p, dtype);
    a.ws = dq.ws = (float*)at;
    at += la_round(la_ws(a));
    la_states(a, dtype, false, st);
  }
  dv.ws = dk.ws = (float*)at;
  la_states(dv, dtype, exact, st);
  LaGroup sum[2];
  if (p.gqa > 1) {
    float* part = (float*)((char*)ws + (need - la_group_bytes(p)));
    for (int i = 0; i < 2; i++) {
      LaArgs& a = pass[1 + i];
      const int D = a.db;
      sum[i] = {part, a.o, a.so, D};
      a.o = part;
      a.o32 = 1;
      a.so.b = p.cu ? 0 : (long long)p.n * p.NH * D;
      a.so.s = (long long)p.NH * D;
      a.so.h = D;
      part += (p.cu ? p.total : (long long)p.batch * p.n) * p.NH * D;
    }
  }
  // Passes of one kernel go together: they read the same rows (B2 S4096 H32 D128 bf16: 162 us, 171 one by one; 24 documents
  // H16 D64 fp16: 151 and 195).
  const bool wide = dtype == FA_F32 || p.gqa == 1;             // dq is written as dv and dk are
  const bool square = p.DK == p.DV;
  for (int i = 0; i < 3;) {
    const int n = square ? (i == 0 ? (wide ? 3 : 1) : 3 - i) : i == 0 && wide ? 2 : 1;
    la_go(pass + i, n, dtype, false, exact && i + n == 3, st);
    i += n;
  }
  if (p.gqa > 1) {
    if (dtype == FA_F16) la_group<_Float16>(sum[0], sum[1], p, st);
    else if (dtype == FA_BF16) la_group<__bf16>(sum[0], sum[1], p, st);
    else la_group<float>(sum[0], sum[1], p, st);
  }
  return launch_status(what);
}
