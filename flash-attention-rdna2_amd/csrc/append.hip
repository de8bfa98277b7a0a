// append.hip — new tokens into a K/V cache (fable_attn_append) and cached rows back out of it
// (fable_attn_gather): the packed or padded batch, rotary, paged or dense caches in 16 or 32 bits or in 8 with
// scales (cache8.hpp).
//
// No counterpart in the reference, whose append takes one count of tokens for every sequence and 16-bit
// caches (kernels/fa_decode.hip:275-302) and which refuses ragged ones.
#include "cache8.hpp"

namespace fa {

// eight consecutive values of a row in fp32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    const auto v = bitcast<typename Dt<T>::V8>(*(const u32x4*)p);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)v[e];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    typename Dt<T>::V8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (T)x[e];
    *(u32x4*)p = bitcast<u32x4>(v);
  }
}

// Rotation (AppendArgs::rot): none; halves or pairs in whole chunks of eight (half a multiple of 8, or the
// width for pairs, tables 16-byte aligned); halves or pairs element by element (any even width).
enum { kRotNone = 0, kRotHalves = 1, kRotPairs = 2, kRotHalvesAny = 3, kRotPairsAny = 4 };

struct AppendArgs : FableAppendParams {
  int page_shift, gshift, tshift, rot, rdim, tiles, nunits, nkv;   // nkv: NKV, or 0 where only q is rotated
};

// A lane's two chunks of eight values of a row: with halves in whole chunks, one of the first half and its
// partner, so a rotation needs no other lane; else two neighbours.
struct Chunks {
  int c[2];
  bool ok[2];
};
__device__ __forceinline__ Chunks chunks_of(const AppendArgs& p, int u, bool rotated) {
  Chunks k;
  const int half = p.rdim / 2;
  if (rotated && p.rot == kRotHalves) {
    const int n = half / 8;
    k.c[0] = u < n ? u : 2 * n + 2 * (u - n);
    k.c[1] = u < n ? u + n : k.c[0] + 1;
  } else {
    k.c[0] = 2 * u;
    k.c[1] = 2 * u + 1;
  }
  k.ok[0] = 8 * k.c[0] < p.HD;
  k.ok[1] = 8 * k.c[1] < p.HD;
  return k;
}

// the lane's values of one row, rotated at row rp of the tables if asked (row: in bounds, rp too)
template <typename T>
__device__ __forceinline__ void load_row(const AppendArgs& p, const T* row, const Chunks& k, bool rotated, int rp, float (&x)[2][8]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if (k.ok[i]) {
      load8(row + 8 * k.c[i], x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
    }
  }
  if (!rotated || p.rot == kRotNone) return;
  const int half = p.rdim / 2;
  const float* cos = p.cos + (long long)rp * half;
  const float* sin = p.sin + (long long)rp * half;
  if (p.rot == kRotHalves) {
    if (8 * k.c[0] < half) {
      float c[8], s[8];
      load8(cos + 8 * k.c[0], c);
      load8(sin + 8 * k.c[0], s);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float a = x[0][e], b = x[1][e];
        x[0][e] = a * c[e] - b * s[e];
        x[1][e] = b * c[e] + a * s[e];
      }
    }
  } else if (p.rot == kRotPairs) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (k.ok[i] && 8 * k.c[i] < p.rdim) {
        const f32x4 c = *(const f32x4*)(cos + 4 * k.c[i]), s = *(const f32x4*)(sin + 4 * k.c[i]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float a = x[i][2 * e], b = x[i][2 * e + 1];
          x[i][2 * e] = a * c[e] - b * s[e];
          x[i][2 * e + 1] = b * c[e] + a * s[e];
        }
      }
    }
  } else {
    const bool halves = p.rot == kRotHalvesAny;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int d = 8 * k.c[i] + e;
        if (k.ok[i] && d < p.rdim) {
          const int j = halves ? (d < half ? d : d - half) : d / 2;
          const bool first = halves ? d < half : (d & 1) == 0;
          const int other = halves ? (first ? d + half : d - half) : d ^ 1;
          const float a = x[i][e], b = (float)row[other];
          x[i][e] = first ? a * cos[j] - b * sin[j] : a * cos[j] + b * sin[j];
        }
      }
  }
}

// A wave takes a tile of 2^tshift consecutive positions of one sequence, aligned to the tile, and one head of
// the keys, values or queries; LPR lanes share a row (16 values each), so a pass covers 64 / LPR rows. In 8
// bits a tile holds whole blocks of `group` rows, which no other wave touches: their largest value is a
// reduction within the wave, and older rows of a block whose scale grew are rewritten by the same lanes.
// NP: passes of a tile, whose rows stay in registers between the search for the largest value and the
// rounding; 0: any number, read twice (the second time from L2).
// What bounds it: a step of few tokens the launch and two dependent memory latencies (lengths, then rows);
// prompts the bytes read and written.
template <typename T, bool Q8, int NP, int LPR>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs p) {
  constexpr int R = 64 / LPR, NH = NP > 0 ? NP : 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / p.tiles, tile = blockIdx.x - b * p.tiles;
  const int unit = blockIdx.y * 4 + wave;
  if (unit >= p.nunits) return;
  // units: the key heads, the value heads, the query heads
  const int kind = unit < p.nkv ? 0 : (unit < 2 * p.nkv ? 1 : 2), head = unit - kind * p.nkv;
  const int ctx = p.ctx_len[b], c0 = p.cu ? p.cu[b] : 0, n = p.cu ? p.cu[b + 1] - c0 : p.n;
  const long long base = (((long long)max(ctx, 0) >> p.tshift) + tile) << p.tshift, stop = (long long)ctx + n;
  if (base >= stop) return;
  const int r = lane / LPR;
  const bool rotated = kind != 1;
  const Chunks ch = chunks_of(p, lane % LPR, rotated);
  const fa_strides st = kind == 0 ? p.sk : (kind == 1 ? p.sv : p.sq);
  const T* src = (const T*)(kind == 0 ? p.k : (kind == 1 ? p.v : p.q)) + (long long)head * st.h + (p.cu ? (long long)c0 * st.s : (long long)b * st.b);
  const long long rp0 = (p.rotary_pos && p.rot ? p.rotary_pos[b] : ctx);
  const int passes = NP > 0 ? NP : max((1 << p.tshift) / R, 1);
  const long long room = (long long)p.max_blocks << p.page_shift;
  // row of pass i: its token, whether there is one (queries have no place in the table)
  auto pos_of = [&](int i) { return base + i * R + r; };
  auto live = [&](long long pos) { return pos >= ctx && pos < stop && (kind == 2 || pos < room); };
  auto fetch = [&](int i, float (&x)[2][8]) {
    const long long pos = pos_of(i), t = pos - ctx;
    if (live(pos)) {
      const int rp = (int)min(max(rp0 + t, 0LL), (long long)max(p.rotary_rows - 1, 0));
      load_row<T>(p, src + t * st.s, ch, rotated, rp, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[0][e] = x[1][e] = 0.0f;
    }
  };
  // the page of a position, or -1
  auto page_of = [&](long long pos) {
    const long long j = pos >> p.page_shift;
    const int blk = p.block_table ? p.block_table[(long long)b * p.max_blocks + j] : (int)(b * (long long)p.max_blocks + j);
    return (unsigned)blk < (unsigned)p.num_blocks ? blk : -1;
  };

  if (kind == 2) {
    for (int i = 0; i < passes; i++) {
      const long long pos = pos_of(i);
      if (!live(pos)) continue;
      float x[2][8];
      fetch(i, x);
      const long long o = (((long long)(p.cu ? c0 : b * (long long)p.n) + pos - ctx) * p.NH + head) * p.HD;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        if (!ch.ok[u]) continue;
        store8((T*)p.q_out + o + 8 * ch.c[u], x[u]);
        if (p.q_lo) {
#pragma unroll
          for (int e = 0; e < 8; e++) x[u][e] -= (float)(T)x[u][e];
          store8((T*)p.q_lo + o + 8 * ch.c[u], x[u]);
        }
      }
    }
    return;
  }
  const fa_strides cs = kind == 0 ? p.kc : p.vc;
  if constexpr (!Q8) {
    T* cache = (T*)(kind == 0 ? p.Kc : p.Vc) + (long long)head * cs.h;
    for (int i = 0; i < passes; i++) {
      const long long pos = pos_of(i);
      if (!live(pos)) continue;
      float x[2][8];
      fetch(i, x);
      const int blk = page_of(pos);
      if (blk < 0) continue;
      T* dst = cache + (long long)blk * cs.b + (pos & ((1 << p.page_shift) - 1)) * cs.s;
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (ch.ok[u]) store8(dst + 8 * ch.c[u], x[u]);
    }
  } else {
    uint8_t* cache = (uint8_t*)(kind == 0 ? p.Kc : p.Vc) + (long long)head * cs.h;
    float x[NH][2][8];
    auto hold = [&](float (&v)[2][8], float& top) {
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          // the largest value a code stands for in T's range (fp16: 65504 would round to 65536)
          constexpr float kMost = std::is_same<T, _Float16>::value ? 61440.0f : 448.0f * 6.646139978924579e35f /* 2^119 */;
          if (fabsf(v[u][e]) <= 3.4028234e38f) v[u][e] = fminf(fmaxf(v[u][e], -kMost), kMost);
          const float a = fabsf(v[u][e]);
          top = a <= 3.4028234e38f ? fmaxf(top, a) : top;
        }
    };
    float top = 0.0f;
    if constexpr (NP > 0) {
#pragma unroll
      for (int i = 0; i < NP; i++) fetch(i, x[i]);
#pragma unroll
      for (int i = 0; i < NP; i++) hold(x[i], top);
    } else {
      for (int i = 0; i < passes; i++) {
        fetch(i, x[0]);
        hold(x[0], top);
      }
    }
    // the block's lanes: rows of one block in this pass
    const int group = 1 << p.gshift, span = min(group, R) * LPR;
    for (int m = 1; m < span; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    const long long bs = pos_of(0) & ~(long long)(group - 1), f = max(bs, (long long)ctx);   // the block, its first new row
    const bool touched = f < min(min(bs + group, stop), room);
    const int blk = touched ? page_of(f) : -1;
    if (blk < 0) return;
    const int in = (int)(bs & ((1 << p.page_shift) - 1)), subs = 1 << (p.page_shift - p.gshift);
    uint8_t* sc = (kind == 0 ? p.k_scale : p.v_scale) + ((long long)blk * p.NKV + head) * subs + (in >> p.gshift);
    uint8_t* rows = cache + (long long)blk * cs.b + (long long)in * cs.s;
    const long long old = max(bs, (long long)(p.leftpad ? p.leftpad[b] : 0));   // the first row the sequence holds
    int e = code_exponent(top);
    if (f > old) {
      const int was = min((int)*sc, 253) - 127;
      if (e > was) {   // rows [old, f) under the scale that grew
        const float down = exp2i(max(was - e, -126));
        for (int i = 0; i < passes; i++) {
          const long long pos = pos_of(i);
          if (pos < old || pos >= f) continue;
          uint8_t* row = rows + (pos - bs) * cs.s;
#pragma unroll
          for (int u = 0; u < 2; u++) {
            if (!ch.ok[u]) continue;
            const u32x2 c = *(const u32x2*)(row + 8 * ch.c[u]);
            float v[8];
#pragma unroll
            for (int w = 0; w < 2; w++) {
              const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[w], true);
              v[4 * w] = lo[0];
              v[4 * w + 1] = lo[1];
              v[4 * w + 2] = hi[0];
              v[4 * w + 3] = hi[1];
            }
            *(u32x2*)(row + 8 * ch.c[u]) = to_codes(v, down);
          }
        }
      } else {
        e = was;
      }
    }
    const float inv = exp2i(-e);
    if constexpr (NP > 0) {
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const long long pos = pos_of(i);
        if (!live(pos)) continue;
#pragma unroll
        for (int u = 0; u < 2; u++)
          if (ch.ok[u]) *(u32x2*)(rows + (pos - bs) * cs.s + 8 * ch.c[u]) = to_codes(x[i][u], inv);
      }
    } else {
      for (int i = 0; i < passes; i++) {
        const long long pos = pos_of(i);
        if (!live(pos)) continue;
        fetch(i, x[0]);
        hold(x[0], top);
#pragma unroll
        for (int u = 0; u < 2; u++)
          if (ch.ok[u]) *(u32x2*)(rows + (pos - bs) * cs.s + 8 * ch.c[u]) = to_codes(x[0][u], inv);
      }
    }
    if ((lane & (span - 1)) == 0) *sc = (uint8_t)(e + 127);
  }
}

template <typename T, bool Q8, int LPR>
static int launch_append_lpr(AppendArgs& a, hipStream_t st) {
  constexpr int R = 64 / LPR;
  constexpr int rshift = __builtin_ctz(R);
  // tiles: a pass, or a block that is longer; without scales 4 passes where the tokens fill them
  a.tshift = Q8 && a.gshift > rshift ? a.gshift : rshift;
  if (!Q8 && a.n >= 16 * R) a.tshift = rshift + 2;
  const long long tiles = ((long long)a.n - 1 >> a.tshift) + 2, grid = tiles * a.batch;
  if (grid > 0x7FFFFFFF || a.nunits > 4 * 65535) return fail(FA_ERR_ARG, "fable_attn_append: grid too large");
  a.tiles = (int)tiles;
  const dim3 g((unsigned)grid, (unsigned)((a.nunits + 3) / 4));
  auto go = [&](auto np) { hipLaunchKernelGGL((append_kernel<T, Q8, decltype(np)::value, LPR>), g, dim3(256), 0, st, a); };
  if constexpr (Q8) {
    switch (a.tshift - rshift) {
      case 0: go(std::integral_constant<int, 1>{}); break;
      case 1: go(std::integral_constant<int, 2>{}); break;
      case 2: go(std::integral_constant<int, 4>{}); break;
      default: go(std::integral_constant<int, 0>{}); break;
    }
  } else {
    go(std::integral_constant<int, 0>{});
  }
  return launch_status("fable_attn_append");
}
template <typename T, bool Q8>
static int launch_append(AppendArgs& a, hipStream_t st) {
  if (a.HD <= 64) return launch_append_lpr<T, Q8, 4>(a, st);
  if (a.HD <= 128) return launch_append_lpr<T, Q8, 8>(a, st);
  return launch_append_lpr<T, Q8, 16>(a, st);
}

static bool strides_ok(const fa_strides& s, int el) { return (s.b * el | s.h * el | s.s * el) % 16 == 0; }

}  // namespace fa

int fa::append_rows(const FableAppendParams& p, int dtype, hipStream_t st) {
  const char* what = "fable_attn_append";
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return fail(FA_ERR_DTYPE, "%s: dtype %d not implemented (fp16/bf16/fp32)", what, dtype);
  const int el = dtype == FA_F32 ? 4 : 2;
  const bool q8 = p.k_scale != nullptr;
  if (!p.Kc || !p.Vc || !p.ctx_len) return fail(FA_ERR_ARG, "%s: null pointer", what);
  if ((p.k_scale == nullptr) != (p.v_scale == nullptr)) return fail(FA_ERR_ARG, "%s: k_scale and v_scale go together", what);
  if ((p.q == nullptr) != (p.q_out == nullptr)) return fail(FA_ERR_ARG, "%s: q and q_out go together", what);
  if (q8 && dtype == FA_F32) return fail(FA_ERR_DTYPE, "%s: 8-bit caches take fp16 and bf16 tokens", what);
  if (p.NKV <= 0 || (p.q && p.NH <= 0)) return fail(FA_ERR_ARG, "%s: NKV=%d NH=%d", what, p.NKV, p.NH);
  if (p.batch < 0 || p.n < 0 || p.max_blocks < 0) return fail(FA_ERR_ARG, "%s: batch=%d n=%d max_blocks=%d", what, p.batch, p.n, p.max_blocks);
  if (q8) {
    const FableCache8 c{p.k_scale, p.v_scale, p.kc, p.vc, p.group, p.num_blocks};
    if (int rc = cache8_check(what, c, p.HD, p.page)) return rc;
  } else {
    if (p.HD <= 0 || p.HD > 256 || p.HD % 8) return fail(FA_ERR_HEADDIM, "%s: head_dim=%d has no kernel (multiples of 8 up to 256)", what, p.HD);
    if (p.page <= 0 || (p.page & (p.page - 1))) return fail(FA_ERR_ARG, "%s: page=%d is not a power of two", what, p.page);
    if (p.num_blocks < 1 || !strides_ok(p.kc, el) || !strides_ok(p.vc, el)) return fail(FA_ERR_ARG, "%s: num_blocks=%d, or rows not 16-byte aligned", what, p.num_blocks);
  }
  if (!strides_ok(p.sk, el) || !strides_ok(p.sv, el) || (p.q && !strides_ok(p.sq, el)))
    return fail(FA_ERR_ARG, "%s: rows of the new tokens are not 16-byte aligned", what);
  AppendArgs a;
  (FableAppendParams&)a = p;
  a.rdim = p.rotary ? (p.rotary_dim > 0 ? p.rotary_dim : p.HD) : 0;
  a.rot = kRotNone;
  if (p.rotary) {
    if (!p.cos || !p.sin) return fail(FA_ERR_ARG, "%s: rotary needs cos and sin", what);
    if (p.rotary < 1 || p.rotary > 2 || a.rdim > p.HD || a.rdim % 2 || p.rotary_rows < 1)
      return fail(FA_ERR_ARG, "%s: rotary=%d rotary_dim=%d rotary_rows=%d", what, p.rotary, p.rotary_dim, p.rotary_rows);
    const bool aligned = ((uintptr_t)p.cos | (uintptr_t)p.sin) % 16 == 0;
    if (p.rotary == 1)
      a.rot = aligned && a.rdim % 16 == 0 ? kRotHalves : kRotHalvesAny;
    else
      a.rot = aligned && a.rdim % 8 == 0 ? kRotPairs : kRotPairsAny;
  }
  if (p.batch == 0 || p.n == 0) return FA_OK;
  a.page_shift = __builtin_ctz((unsigned)p.page);
  a.gshift = q8 ? __builtin_ctz((unsigned)p.group) : 0;
  a.nkv = p.k ? p.NKV : 0;
  a.nunits = 2 * a.nkv + (p.q ? p.NH : 0);
  switch (dtype) {
    case FA_F16: return q8 ? launch_append<_Float16, true>(a, st) : launch_append<_Float16, false>(a, st);
    case FA_BF16: return q8 ? launch_append<__bf16, true>(a, st) : launch_append<__bf16, false>(a, st);
    default: return launch_append<float, false>(a, st);
  }
}

extern "C" int fable_attn_append(FableAppendParams p, int dtype, void* stream) {
  if (!p.k || !p.v) return fa::fail(FA_ERR_ARG, "fable_attn_append: null pointer");
  return fa::append_rows(p, dtype, (hipStream_t)stream);
}

namespace fa {

struct GatherArgs : FableGatherParams {
  int page_shift, gshift;
};

// One wave per row of the output, its keys and values; the row's sequence by bisection of cu.
template <typename T, bool Q8>
__global__ __launch_bounds__(256) void gather_kernel(GatherArgs p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row = (long long)blockIdx.x * 4 + wave;
  if (row >= p.total) return;
  int lo = 0, hi = p.batch;   // the last sequence that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  const long long j = row - p.cu[lo];
  int blk = -1;
  if (p.batch > 0 && j >= 0 && row < p.cu[lo + 1] && j < ((long long)p.max_blocks << p.page_shift)) {
    const long long at = (long long)lo * p.max_blocks + (j >> p.page_shift);
    blk = p.block_table ? p.block_table[at] : (int)at;
    if ((unsigned)blk >= (unsigned)p.num_blocks) blk = -1;
  }
  const int in = (int)(j & ((1 << p.page_shift) - 1));
  const int per = p.HD / 8, chunks = p.NKV * per;
  for (int i = lane; i < 2 * chunks; i += 64) {
    const int kv = i >= chunks, c = i - kv * chunks, h = c / per, d = 8 * (c - h * per);
    const fa_strides s = kv ? p.vc : p.kc;
    T* dst = (T*)(kv ? p.v_out : p.k_out) + (row * p.NKV + h) * p.HD + d;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (blk >= 0) {
      const long long off = (long long)blk * s.b + (long long)in * s.s + (long long)h * s.h + d;
      if constexpr (Q8) {
        const int subs = 1 << (p.page_shift - p.gshift);
        const unsigned e = (kv ? p.v_scale : p.k_scale)[((long long)blk * p.NKV + h) * subs + (in >> p.gshift)];
        const auto v = codes_to<T>(*(const u32x2*)((const uint8_t*)(kv ? p.Vc : p.Kc) + off), e8_f32(e));
        *(u32x4*)dst = bitcast<u32x4>(v);
        continue;
      } else {
        load8((const T*)(kv ? p.Vc : p.Kc) + off, x);
      }
    }
    store8(dst, x);
  }
}

template <typename T, bool Q8>
static int launch_gather(const GatherArgs& a, hipStream_t st) {
  const long long grid = (a.total + 3) / 4;
  if (grid > 0x7FFFFFFF) return fail(FA_ERR_ARG, "fable_attn_gather: grid too large");
  hipLaunchKernelGGL((gather_kernel<T, Q8>), dim3((unsigned)grid), dim3(256), 0, st, a);
  return launch_status("fable_attn_gather");
}

}  // namespace fa

extern "C" int fable_attn_gather(FableGatherParams p, int dtype, void* stream) {
  using namespace fa;
  const char* what = "fable_attn_gather";
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return fail(FA_ERR_DTYPE, "%s: dtype %d not implemented (fp16/bf16/fp32)", what, dtype);
  const int el = dtype == FA_F32 ? 4 : 2;
  const bool q8 = p.k_scale != nullptr;
  if (!p.Kc || !p.Vc || !p.k_out || !p.v_out || !p.cu) return fail(FA_ERR_ARG, "%s: null pointer", what);
  if ((p.k_scale == nullptr) != (p.v_scale == nullptr)) return fail(FA_ERR_ARG, "%s: k_scale and v_scale go together", what);
  if (q8 && dtype == FA_F32) return fail(FA_ERR_DTYPE, "%s: 8-bit caches come back in fp16 or bf16", what);
  if (p.NKV <= 0 || p.batch < 0 || p.total < 0 || p.max_blocks < 0)
    return fail(FA_ERR_ARG, "%s: NKV=%d batch=%d total=%lld max_blocks=%d", what, p.NKV, p.batch, (long long)p.total, p.max_blocks);
  if (q8) {
    const FableCache8 c{p.k_scale, p.v_scale, p.kc, p.vc, p.group, p.num_blocks};
    if (int rc = cache8_check(what, c, p.HD, p.page)) return rc;
  } else {
    if (p.HD <= 0 || p.HD > 256 || p.HD % 8) return fail(FA_ERR_HEADDIM, "%s: head_dim=%d has no kernel (multiples of 8 up to 256)", what, p.HD);
    if (p.page <= 0 || (p.page & (p.page - 1))) return fail(FA_ERR_ARG, "%s: page=%d is not a power of two", what, p.page);
    if (p.num_blocks < 1 || !strides_ok(p.kc, el) || !strides_ok(p.vc, el)) return fail(FA_ERR_ARG, "%s: num_blocks=%d, or rows not 16-byte aligned", what, p.num_blocks);
  }
  if (p.total == 0) return FA_OK;
  GatherArgs a;
  (FableGatherParams&)a = p;
  a.page_shift = __builtin_ctz((unsigned)p.page);
  a.gshift = q8 ? __builtin_ctz((unsigned)p.group) : 0;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case FA_F16: return q8 ? launch_gather<_Float16, true>(a, st) : launch_gather<_Float16, false>(a, st);
    case FA_BF16: return q8 ? launch_gather<__bf16, true>(a, st) : launch_gather<__bf16, false>(a, st);
    default: return launch_gather<float, false>(a, st);
  }
}
