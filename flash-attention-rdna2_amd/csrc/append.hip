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
constexpr int kHeadsPerWave = 4;   // heads of a unit whose rows need no scale

struct AppendArgs : FableAppendParams {
  int page_shift, gshift, tshift, rot, rdim, tiles, wgs;   // tiles of a sequence, workgroups of a tile
  int ukv, uq;   // units (waves) of a tile: of K, and as many of V, and of q
};

// A lane's two chunks of eight values of a row: with halves in whole chunks, one of the first half and its
// partner, so a rotation needs no other lane; else two neighbours. (Chunks past the head dim: chunk 0, not ok.)
struct Chunks {
  int c[2];
  bool ok[2], turn;   // turn: halves, and this lane's chunks are in the rotated columns
};
__device__ __forceinline__ Chunks chunks_of(const AppendArgs& p, int u, bool rotated) {
  Chunks k;
  k.c[0] = 2 * u;
  k.c[1] = 2 * u + 1;
  k.turn = false;
  if (rotated && p.rot == kRotHalves) {
    const int n = p.rdim / 16;
    k.turn = u < n;
    k.c[0] = u < n ? u : 2 * u;   // (past the rotated columns: 2n + 2(u - n))
    k.c[1] = u < n ? u + n : 2 * u + 1;
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    k.ok[i] = 8 * k.c[i] < p.HD;
    k.c[i] = k.ok[i] ? k.c[i] : 0;
  }
  return k;
}

// cosines and sines for a lane's chunks at row rp of the tables (in bounds; only p.rot < kRotHalvesAny)
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ void load_angles(const AppendArgs& p, const Chunks& k, int rp, Angles& a) {
  const int half = p.rdim / 2;
  const float* cos = p.cos + (long long)rp * half;
  const float* sin = p.sin + (long long)rp * half;
  if (p.rot == kRotHalves) {
    const int at = k.turn ? 8 * k.c[0] : 0;
    load8(cos + at, a.c);
    load8(sin + at, a.s);
  } else if (p.rot == kRotPairs) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int at = 8 * k.c[i] < p.rdim ? 4 * k.c[i] : 0;
      const f32x4 c = *(const f32x4*)(cos + at), s = *(const f32x4*)(sin + at);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        a.c[4 * i + e] = c[e];
        a.s[4 * i + e] = s[e];
      }
    }
  }
}
// (ANY: the element-by-element forms only, which read the partner from the row)
template <bool ANY, typename T>
__device__ __forceinline__ void turn(const AppendArgs& p, const Chunks& k, const Angles& an, const T* row, int rp, float (&x)[2][8]) {
  if constexpr (!ANY) {
    if (p.rot == kRotHalves) {
      if (k.turn) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float a = x[0][e], b = x[1][e];
          x[0][e] = a * an.c[e] - b * an.s[e];
          x[1][e] = b * an.c[e] + a * an.s[e];
        }
      }
    } else if (p.rot == kRotPairs) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (8 * k.c[i] < p.rdim) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float a = x[i][2 * e], b = x[i][2 * e + 1], c = an.c[4 * i + e], s = an.s[4 * i + e];
            x[i][2 * e] = a * c - b * s;
            x[i][2 * e + 1] = b * c + a * s;
          }
        }
      }
    }
  } else {
    const int half = p.rdim / 2;
    const float* cos = p.cos + (long long)rp * half;
    const float* sin = p.sin + (long long)rp * half;
    const bool halves = p.rot == kRotHalvesAny;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int d = 8 * k.c[i] + e;
        if (d < p.rdim) {
          const int j = halves ? (d < half ? d : d - half) : d / 2;
          const bool first = halves ? d < half : (d & 1) == 0;
          const int other = halves ? (first ? d + half : d - half) : d ^ 1;
          const float a = x[i][e], b = (float)row[other];
          x[i][e] = first ? a * cos[j] - b * sin[j] : a * cos[j] + b * sin[j];
        }
      }
  }
}

// A unit takes a tile of 2^tshift consecutive positions of one sequence, aligned to the tile; LPR lanes share a
// row (16 values each), so a pass of a wave covers 64 / LPR rows. In 8 bits a tile holds whole blocks of `group`
// rows, which no other unit touches: their largest value is a reduction over the unit, and older rows of a block
// whose scale grew are rewritten by the same lanes. A unit is WB waves of NP passes each, whose rows stay in
// registers between the search for the largest value and the rounding (NP 0: any number of passes, read twice,
// the second time from L2), and HB heads of the keys or values, which share their angles: a head of 128 has half as many
// bytes as its angles, which came from L2 for every head before (8192 tokens of 8 heads, blocks of 16: 24.3 us,
// 17.3 without a rotation, the angles' way through scratch, below, included). Rows that need no scale (queries, caches of 16 and 32 bits) go four heads to a unit of
// one wave and one pass. The units of a tile follow one another in the grid, so that the heads of a token are
// read together (rather than the tiles of a head one after another).
// Loads carry no lane condition (a row that is not there reads the sequence's first or last token). Those of one pass
// of one head are in flight together; the next pass or head is asked for when this one has been turned. The two forms of
// load_angles fill one array from different loads, which the compiler joins through memory: 28 bytes of scratch per lane in every
// instance that takes whole chunks, written and read back between the angles and the rows. What bounds it: a step of few tokens
// the launch and a chain of latencies (lengths, table, then angles, scratch and rows of each pass and head, and the older codes of a block
// whose scale grows): 48 tokens of 64 + 8 heads of 128, rotated, 9.0 us (a gather of few rows, four latencies, 3.3); prompts that chain
// beside the bytes: 11400 tokens of 32 + 8 heads of 128, rotated, blocks of 64, 71 us for 262 MB (3.7 TB/s: the angles of every
// two heads' keys come from L2 beside them); 24 of 64 to 2048 tokens of 8 heads in 16 bits 50 us for 232 MB (4.6 TB/s, a copy's).
template <typename T, bool Q8, int NP, int HB, int WB, int LPR, bool ANY>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs p) {
  constexpr int R = 64 / LPR, NH = NP > 0 ? NP : 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bt = blockIdx.x / p.wgs, wg = blockIdx.x - bt * p.wgs;
  const int b = bt / p.tiles, tile = bt - b * p.tiles;
  // units of K and V (of one wave, or of a workgroup's four, which meet at a barrier), then those of q
  static_assert(WB == 1 || WB == 4, "waves of a unit");
  const int kvw = 2 * p.ukv * WB, at = wg * 4 + wave;
  const int unit = at < kvw ? at / WB : 2 * p.ukv + at - kvw;
  if (unit >= 2 * p.ukv + p.uq) return;
  const int kind = at >= kvw ? 2 : (unit < p.ukv ? 0 : 1);   // q, K, V
  const int ctx = p.ctx_len[b], c0 = p.cu ? p.cu[b] : 0, n = p.cu ? p.cu[b + 1] - c0 : p.n;
  const long long base = (((long long)max(ctx, 0) >> p.tshift) + tile) << p.tshift, stop = (long long)ctx + n;
  if (n <= 0 || base >= stop) return;
  const int r = lane / LPR;
  const bool rotated = kind != 1 && p.rot != kRotNone;
  const Chunks ch = chunks_of(p, lane % LPR, rotated);
  const fa_strides st = kind == 0 ? p.sk : (kind == 1 ? p.sv : p.sq);
  const T* src = (const T*)(kind == 0 ? p.k : (kind == 1 ? p.v : p.q)) + (p.cu ? (long long)c0 * st.s : (long long)b * st.b);
  const long long rp0 = rotated && p.rotary_pos ? p.rotary_pos[b] : ctx;
  const int passes = NP > 0 ? NP : max((1 << p.tshift) / R, 1);   // of a wave
  const int part = WB > 1 && kind != 2 ? at % WB : 0;             // of the unit's waves (queries: one)
  const long long room = (long long)p.max_blocks << p.page_shift;
  auto pos_of = [&](int i) { return base + (part * NH + i) * R + r; };
  auto token_of = [&](int i) { return min(max(pos_of(i) - ctx, 0LL), (long long)n - 1); };   // in bounds
  auto row_of = [&](int i) { return (int)min(max(rp0 + token_of(i), 0LL), (long long)p.rotary_rows - 1); };
  // (queries have no place in the table)
  auto live = [&](long long pos) { return pos >= ctx && pos < stop && (kind == 2 || pos < room); };
  // the page of a position in the table, or -1
  auto page_of = [&](long long pos) {
    const long long j = pos >> p.page_shift;
    const int blk = p.block_table ? p.block_table[(long long)b * p.max_blocks + j] : (int)(b * (long long)p.max_blocks + j);
    return (unsigned)blk < (unsigned)p.num_blocks ? blk : -1;
  };

  if (!Q8 || kind == 2) {
    // (a wave of queries takes one pass of the tile, whatever the block's length)
    const int nheads = kind == 2 ? p.NH : p.NKV, per = (nheads + kHeadsPerWave - 1) / kHeadsPerWave;
    const int mine = unit - kind * p.ukv, i = mine / per, h0 = (mine - i * per) * kHeadsPerWave;
    const fa_strides cs = kind == 0 ? p.kc : p.vc;
    T* cache = (T*)(kind == 0 ? p.Kc : p.Vc);
    const long long pos = pos_of(i);
    const T* row = src + token_of(i) * st.s;
    const int rp = rotated ? row_of(i) : 0;
    Angles an;
    if (!ANY && rotated) load_angles(p, ch, rp, an);
    float x[kHeadsPerWave][2][8];
#pragma unroll
    for (int g = 0; g < kHeadsPerWave; g++) {
      const T* q = row + (long long)min(h0 + g, nheads - 1) * st.h;
      load8(q + 8 * ch.c[0], x[g][0]);
      load8(q + 8 * ch.c[1], x[g][1]);
    }
    bool ok = live(pos);
    long long o = 0, step = p.HD;
    T* dst = (T*)p.q_out;
    if (kind == 2) {
      o = ((p.cu ? c0 : b * (long long)p.n) + token_of(i)) * p.NH * p.HD;
    } else if (ok) {
      const int blk = page_of(pos);
      ok = blk >= 0;
      o = (long long)blk * cs.b + (pos & ((1 << p.page_shift) - 1)) * cs.s;
    }
    if (kind != 2) {
      dst = cache;
      step = cs.h;
    }
#pragma unroll
    for (int g = 0; g < kHeadsPerWave; g++) {
      const int h = h0 + g;
      if (rotated) turn<ANY, T>(p, ch, an, row + (long long)min(h, nheads - 1) * st.h, rp, x[g]);
      if (!ok || h >= nheads) continue;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        if (!ch.ok[u]) continue;
        const long long at = o + h * step + 8 * ch.c[u];
        store8(dst + at, x[g][u]);
        if (kind == 2 && p.q_lo) {   // what the rounding left
#pragma unroll
          for (int e = 0; e < 8; e++) x[g][u][e] -= (float)(T)x[g][u][e];
          store8((T*)p.q_lo + at, x[g][u]);
        }
      }
    }
    return;
  }
  if constexpr (Q8) {
    const int h0 = (unit - kind * p.ukv) * HB;
    const fa_strides cs = kind == 0 ? p.kc : p.vc;
    // this lane's block, its first new row, and what is there already: looked up while the rows come
    const int group = 1 << p.gshift, span = min(group, R) * LPR;
    const long long bs = pos_of(0) & ~(long long)(group - 1), f = max(bs, (long long)ctx);
    const bool touched = f < min(min(bs + group, stop), room);
    const int blk = touched && h0 < p.NKV ? page_of(f) : -1;
    const int in = (int)(bs & ((1 << p.page_shift) - 1)), subs = 1 << (p.page_shift - p.gshift);
    const long long old = max(bs, (long long)(p.leftpad ? p.leftpad[b] : 0));   // the first row the sequence holds
    uint8_t* sc[HB];
    int was[HB];
#pragma unroll
    for (int g = 0; g < HB; g++) {
      sc[g] = (kind == 0 ? p.k_scale : p.v_scale) + ((long long)max(blk, 0) * p.NKV + min(h0 + g, p.NKV - 1)) * subs + (in >> p.gshift);
      was[g] = min((int)*sc[g], 254) - 127;   // (255 is no number: as the largest)
    }
    float x[HB][NH][2][8], top[HB];
    auto fetch = [&](int i, int j) {   // pass i of all heads, to x[.][j]
      const T* row = src + token_of(i) * st.s;
      const int rp = rotated ? row_of(i) : 0;
      Angles an;
      if (!ANY && rotated) load_angles(p, ch, rp, an);
#pragma unroll
      for (int g = 0; g < HB; g++) {
        const T* q = row + (long long)min(h0 + g, p.NKV - 1) * st.h;
        load8(q + 8 * ch.c[0], x[g][j][0]);
        load8(q + 8 * ch.c[1], x[g][j][1]);
        if (rotated) turn<ANY, T>(p, ch, an, q, rp, x[g][j]);
      }
    };
    auto hold = [&](int i, int j) {
      const bool ok = live(pos_of(i));
#pragma unroll
      for (int g = 0; g < HB; g++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            // the largest value a code stands for in T's range (fp16: 65504 would round to 65536)
            constexpr float kMost = std::is_same<T, _Float16>::value ? 61440.0f : 448.0f * 6.646139978924579e35f /* 2^119 */;
            float& v = x[g][j][u][e];
            if (fabsf(v) <= 3.4028234e38f) v = fminf(fmaxf(v, -kMost), kMost);
            const float a = fabsf(v);
            top[g] = ok && ch.ok[u] && a <= 3.4028234e38f ? fmaxf(top[g], a) : top[g];
          }
    };
#pragma unroll
    for (int g = 0; g < HB; g++) top[g] = 0.0f;
    if constexpr (NP > 0) {
#pragma unroll
      for (int i = 0; i < NP; i++) fetch(i, i);
#pragma unroll
      for (int i = 0; i < NP; i++) hold(i, i);
    } else {
      for (int i = 0; i < passes; i++) {
        fetch(i, 0);
        hold(i, 0);
      }
    }
#pragma unroll
    for (int g = 0; g < HB; g++)
      for (int m = 1; m < span; m <<= 1) top[g] = fmaxf(top[g], __shfl_xor(top[g], m));   // over the block's lanes
    if constexpr (WB > 1) {   // and its waves
      __shared__ float tops[HB][4];
      if (lane == 0)
#pragma unroll
        for (int g = 0; g < HB; g++) tops[g][wave] = top[g];
      __syncthreads();
#pragma unroll
      for (int g = 0; g < HB; g++)
#pragma unroll
        for (int w = 0; w < WB; w++) top[g] = fmaxf(top[g], tops[g][w]);
    }
    if (blk < 0) return;
#pragma unroll
    for (int g = 0; g < HB; g++) {
      if (h0 + g >= p.NKV) break;
      uint8_t* rows = (uint8_t*)(kind == 0 ? p.Kc : p.Vc) + (long long)(h0 + g) * cs.h + (long long)blk * cs.b + (long long)in * cs.s;
      int e = code_exponent(top[g]);
      if (f > old) {
        if (e > was[g]) {   // rows [old, f) under the scale that grew
          const float down = exp2i(max(was[g] - e, -126));
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
          e = was[g];
        }
      }
      const float inv = exp2i(-e);
      auto put = [&](int i, int j) {
        const long long pos = pos_of(i);
        if (!live(pos)) return;
#pragma unroll
        for (int u = 0; u < 2; u++)
          if (ch.ok[u]) *(u32x2*)(rows + (pos - bs) * cs.s + 8 * ch.c[u]) = to_codes(x[g][j][u], inv);
      };
      if constexpr (NP > 0) {
#pragma unroll
        for (int i = 0; i < NP; i++) put(i, i);
      } else {
        for (int i = 0; i < passes; i++) {
          fetch(i, 0);
          hold(i, 0);
          put(i, 0);
        }
      }
      if (part == 0 && (lane & (span - 1)) == 0) *sc[g] = (uint8_t)(e + 127);
    }
  }
}

template <typename T, bool Q8, int LPR>
static int launch_append_lpr(AppendArgs& a, hipStream_t st) {
  constexpr int R = 64 / LPR;
  constexpr int rshift = __builtin_ctz(R);
  // tiles: a pass, or a block that is longer
  a.tshift = Q8 && a.gshift > rshift ? a.gshift : rshift;
  const long long tiles = ((a.n - 2LL + (1LL << a.tshift)) >> a.tshift) + 1;   // (wherever the first token is)
  auto go = [&](auto np, auto hb, auto wb, auto any) -> int {
    constexpr int NP = decltype(np)::value, HB = decltype(hb)::value, WB = decltype(wb)::value;
    auto units = [](int heads, int per) { return (heads + per - 1) / per; };
    a.ukv = a.k ? units(a.NKV, Q8 ? HB : kHeadsPerWave) : 0;
    a.uq = a.q ? units(a.NH, kHeadsPerWave) << (a.tshift - rshift) : 0;
    const int waves = 2 * a.ukv * WB + a.uq;
    a.wgs = (waves + 3) / 4;
    if (tiles > 0x7FFFFFFF / a.batch / a.wgs) return fail(FA_ERR_ARG, "fable_attn_append: grid too large");
    a.tiles = (int)tiles;
    hipLaunchKernelGGL((append_kernel<T, Q8, NP, HB, WB, LPR, decltype(any)::value>), dim3((unsigned)(tiles * a.batch * a.wgs)), dim3(256), 0, st, a);
    return launch_status("fable_attn_append");
  };
  using N = std::integral_constant<bool, false>;
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  using I8 = std::integral_constant<int, 8>;
  if (a.rot >= kRotHalvesAny) return go(I0{}, I1{}, I1{}, std::integral_constant<bool, true>{});
  if constexpr (Q8) {
    // (four passes at most, but for the longest blocks: with eight in one wave the instance held 200 registers, and a
    // prompt of 11400 tokens with 32 query heads of 128, blocks of 64, took 85 us; 67 with four in each of two waves, 62 with two
    // passes of two heads in each of four, which halves the angles read: eight passes go so. Two of four heads 107, and the
    // sixteen passes of blocks of 128 as four of two heads 116 for 66, both out of registers.)
    // Heads share a wave only where there are waves enough without (a chip holds some 2000 of these): 32 tokens of 4
    // heads of 256 took 10.1 us with four heads to a wave, 5.5 with one.
    const bool few = tiles * a.batch * 2 * a.NKV <= 2048;
    switch (a.tshift - rshift) {
      case 0: return few ? go(I1{}, I1{}, I1{}, N{}) : go(I1{}, I4{}, I1{}, N{});
      case 1: return few ? go(I2{}, I1{}, I1{}, N{}) : go(I2{}, I2{}, I1{}, N{});
      case 2: return go(I4{}, I1{}, I1{}, N{});
      case 3: return go(I2{}, I2{}, I4{}, N{});
      case 4: return go(I4{}, I1{}, I4{}, N{});
      case 5: return go(I8{}, I1{}, I4{}, N{});
      default: return go(I0{}, I1{}, I1{}, N{});   // (blocks of 256 rows wider than 128)
    }
  } else {
    return go(I1{}, I1{}, I1{}, N{});
  }
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
    for (const fa_strides& s : {p.kc, p.vc}) {
      const FableCache8 c{p.k_scale, p.v_scale, s, p.group, p.num_blocks, 0, nullptr};
      if (int rc = cache8_check(what, c, p.HD, p.page)) return rc;
    }
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

// One wave per row of the output, its keys and values, eight per lane and pass. The row's sequence is found by 64
// entries of cu at a time (a bisection took a memory latency for every doubling of the batch), the loads of kPasses
// passes are in flight together, and a row that is not there reads page 0. What bounds it: a few rows the launch and
// four dependent latencies (cu, table, rows and scales): 300 rows of 8 heads of 64 3.3 us; many the bytes: 16 requests of
// 500 to 8000 rows, 8 heads of 128, 507 MB in 97 us (5.2 TB/s, written at twice the bytes it is read at); over 16-bit pages 557 MB
// of as many requests in 109 us, in 32 bits 1114 MB in 217 (5.1 TB/s both).
template <typename T, bool Q8>
__global__ __launch_bounds__(256) void gather_kernel(GatherArgs p) {
  constexpr int kPasses = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row = (long long)blockIdx.x * 4 + wave;
  if (row >= p.total) return;
  int lo = 0;   // the last sequence that starts at or before the row
  for (int n = p.batch; n > 1;) {
    const int step = (n + 63) / 64, at = lo + lane * step;
    const bool before = lane * step < n && p.cu[min(at, p.batch)] <= row;
    const int k = max(__popcll(__builtin_amdgcn_ballot_w64(before)) - 1, 0) * step;
    lo += k;
    n = min(step, n - k);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const long long j = row - p.cu[lo];
  if (p.used && (p.batch <= 0 || j < 0 || j >= p.used[lo])) return;
  int blk = -1;
  if (p.batch > 0 && j >= 0 && row < p.cu[lo + 1] && j < ((long long)p.max_blocks << p.page_shift)) {
    const long long at = (long long)lo * p.max_blocks + (j >> p.page_shift);
    blk = p.block_table ? p.block_table[at] : (int)at;
    if ((unsigned)blk >= (unsigned)p.num_blocks) blk = -1;
  }
  const int in = (int)(j & ((1 << p.page_shift) - 1)), in0 = blk >= 0 ? in : 0;
  const int per = p.HD / 8, chunks = p.NKV * per, subs = Q8 ? 1 << (p.page_shift - p.gshift) : 0;
  const long long page = max(blk, 0);
  for (int i0 = lane; i0 < 2 * chunks; i0 += 64 * kPasses) {
    u32x2 code[kPasses];
    unsigned scale[kPasses];
    float x[kPasses][8];
    int col[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; u++) {
      const int i = min(i0 + 64 * u, 2 * chunks - 1), kv = i >= chunks, c = i - kv * chunks, h = c / per, d = 8 * (c - h * per);
      const fa_strides s = kv ? p.vc : p.kc;
      const long long off = page * s.b + (long long)in0 * s.s + (long long)h * s.h + d;
      const void* cache = kv ? p.Vc : p.Kc;
      col[u] = h * p.HD + d;
      if constexpr (Q8) {
        scale[u] = (kv ? p.v_scale : p.k_scale)[(page * p.NKV + h) * subs + (in0 >> p.gshift)];
        code[u] = *(const u32x2*)((const uint8_t*)cache + off);
      } else {
        load8((const T*)cache + off, x[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kPasses; u++) {
      if (i0 + 64 * u >= 2 * chunks) break;
      T* dst = (T*)(i0 + 64 * u >= chunks ? p.v_out : p.k_out) + row * p.NKV * p.HD + col[u];
      if constexpr (Q8) {
        const auto v = codes_to<T>(code[u], e8_f32(scale[u]));
        *(u32x4*)dst = blk >= 0 ? bitcast<u32x4>(v) : u32x4{0, 0, 0, 0};
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[u][e] = blk >= 0 ? x[u][e] : 0.0f;
        store8(dst, x[u]);
      }
    }
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
    for (const fa_strides& s : {p.kc, p.vc}) {
      const FableCache8 c{p.k_scale, p.v_scale, s, p.group, p.num_blocks, 0, nullptr};
      if (int rc = cache8_check(what, c, p.HD, p.page)) return rc;
    }
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
