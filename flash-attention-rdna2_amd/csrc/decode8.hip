// decode8.hip — decode over a K/V cache held in 8 bits (fable_attn_dec8; the format: cache8.hpp).
//
// The split of the work, the records and the combine are the 16-bit decode's (decode.hip): one workgroup of
// four waves per (K/V head, group of 16 rows, run of a sequence's keys), each wave with its own chunks and
// online softmax, merged in LDS. Large calls give a workgroup two or four K/V heads, waves and all (dec8_heads). What differs:
//  * a chunk is 32 keys, so as many bytes are in flight per wave as there with 16. A SIMD has one wave, whose
//    instructions per chunk are what bounds it next to HBM, so the rest is about having few;
//  * codes stay codes in LDS (half the LDS traffic) and become fp16/bf16 between the LDS read and the matrix
//    instruction: K by 16-byte reads of a key's row, V by the transposing 8-bit reads (ds_read_b64_tr_b8: a lane
//    gets one column of eight rows, the A operand of v_mfma_f32_16x16x32 as it is);
//  * they are converted without their scales, which are exact powers of two: a key's K scale multiplies its fp32
//    scores, its V scale the fp32 probability ahead of the rounding to 16 bits. The scales of a chunk come
//    in one byte load per lane and reach the lanes that need them through LDS;
//  * chunks are aligned to 32 keys, so one lies in one page (two of 16 rows): a buffer descriptor for a
//    page makes the lanes' offsets loop invariant and rows past the end zero;
//  * the accumulators are rescaled only in chunks that raise a row's maximum, and only chunks that some row does not
//    see in full are masked (scalar branches).
// fp16: a scaled probability can leave fp16's range (and V's codes need no more than bf16 holds), so P goes
// as two bf16 parts, high and low, into two products: 16 bits of it, as many as fp16's own rounding left.
// What bounds it: HBM. 16 x 32768 keys of 8 heads, D 128, 1.07 GB: 158 us and 5 for the merge of the splits (6.6 TB/s; reads alone
// in this pattern 151), 48 requests of 64 to 8192 keys under pages of 16, 428 MB: 74 and 5.5 (5.4 TB/s; the shares and the prologue
// of their segments are the rest). Small calls wait for a chain of latencies (lengths, table, rows, merge): 2000 keys 7.2
// and 3.7 us, 8 x 4 drafted tokens in a window of 512, D 256, 12 and 4.
// An append is a launch ahead of this one. A share or split starts at a multiple of 32 keys, and a chunk of 32 is one wave's,
// so with one row group and blocks of at most 32 tokens the wave that reads a new token's block could also write
// it (where no other sequence names its page); it does not yet. Nor is a row asked for before q has been rotated, though
// only the lengths and the table are needed for it.
// Not taken: the products of e4m3 operands with e8m0 scales (v_mfma_scale_f32_16x16x128_f8f6f4), K as it is and q as
// a sum of e4m3 parts. They need no conversion of K, but add their 128 products aligned to the largest: with one
// dimension of q and k 30 times the others, scores of size 100 were off by up to 0.1.
#include "cache8.hpp"
#include "dec_common.hpp"
#include "fwd_common.hpp"

namespace fa {

constexpr int kKeys8 = 32;                       // keys per wave iteration
constexpr int kDec8Append = 1, kDec8Final = 2;   // new keys were appended; one split, no combine launch

struct Dec8Args : FableDecParams {
  FableCache8 c;
  const int* table;   // as DecArgs::table (decode.hip): the block table, or any readable address and tmask 0
  int tmask, page_shift, gshift, ngrp, flags, parts, nkv, bshift;
};

__device__ __forceinline__ float lane16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float lane16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int HD>
struct Dec8Lds {
  // rows of codes padded by 16 bytes: the 16-byte K reads of 16 rows and the transposing V reads of 16 rows both
  // touch every bank once. Scales: 32 of K, 32 of V, fp32.
  static constexpr int STR = HD + 16;
  static constexpr int WAVE = 2 * kKeys8 * STR + 64 * 4;   // K, V, scales
  // rows of q (fp32) and of the merge's accumulators, padded likewise: 16 lanes write or read a column of them
  static constexpr int FSTR = HD + 4;
  static constexpr int ACC = kDecWaves * 16 * FSTR * 4;     // (q's rows are as many at most)
  static constexpr int BYTES = kDecWaves * WAVE > ACC ? kDecWaves * WAVE : ACC;
};

typedef int i32x2 __attribute__((ext_vector_type(2)));

// P16: pages of 16 rows (two to a chunk); WH: heads of a workgroup
template <typename T, int HD, bool FEAT, bool SHARE, bool P16, int WH>
__global__ __launch_bounds__(256) void dec8_partial_kernel(Dec8Args p) {
  using V8 = typename Dt<T>::V8;
  using L = Dec8Lds<HD>;
  constexpr bool kTwoP = std::is_same<T, _Float16>::value;   // P in two bf16 parts
  constexpr int NDB = HD / 16, RB = HD / 16, NV = kKeys8 * RB / 64, NDS = HD / 32;
  constexpr int NPG = P16 ? 2 : 1;
  constexpr int WR = kDecWaves / WH, kUnit8 = kKeys8 * WR;   // waves on the keys of a head; keys of a unit of a share
  // Chunks whose rows are in flight. One left a wave waiting for most of the memory latency (32000 keys of one sequence
  // in 4 splits, D 128: 78 us, 66 with two; 16 x 32768 keys, D 64: 178 and 119; D 192 96 and 72 in 3 splits); rows of
  // 256 bytes fill the same bytes with one, and two cost registers (8 x 4000 keys 23.4 and 25.4).
  constexpr int DEPTH = HD <= 192 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) char raw[L::BYTES];
  __shared__ float red_m[kDecWaves][16], red_l[kDecWaves][16];
  float (*qsh)[L::FSTR] = (float (*)[L::FSTR])raw;

  const int append = p.flags & kDec8Append, page_shift = p.page_shift;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = lane >> 4, lh = lane & 15;
  const int NKV = p.nkv, HDr = p.HD, nq = p.nq, gqa = p.gqa, NH = p.NH;
  const int X = gridDim.x;
  int hgl = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
  if (p.bshift) {   // 2^bshift heads whose rows share 128-byte lines: one after another on one XCD (launch_dec8)
    const unsigned l = (bz * gridDim.y + by) * X + hgl, k = l / 8, bundle = (k >> p.bshift) * 8 + l % 8, w = bundle / ((unsigned)X >> p.bshift);
    hgl = (int)(((bundle - w * ((unsigned)X >> p.bshift)) << p.bshift) + (k & ((1u << p.bshift) - 1)));
    bz = (int)(w / gridDim.y);
    by = (int)w - bz * gridDim.y;
  }
  const int hw = wave % WH, rw = wave / WH;   // this wave's head of the workgroup's, and place among its waves
  const int grp = p.ngrp > 1 ? hgl / (NKV / WH) : 0, head0 = (hgl - grp * (NKV / WH)) * WH, kvh = head0 + hw;
  const int r0 = 16 * grp, hg = min(16, nq * gqa - r0);  // rows of this group
  auto row_tok = [&](int g) { return nq > 1 ? (int)((unsigned)(r0 + g) / (unsigned)gqa) : 0; };
  auto row_of = [&](int b, int head, int g) {
    const int tok = row_tok(g);
    return (long long)(b * nq + tok) * NH + head * gqa + (r0 + g - tok * gqa);
  };
  auto args = [&]() -> Dec8Args {   // (as in decode.hip: the phases that only some workgroups run read it again)
    if constexpr (SHARE) return dec_reload<Dec8Args>();
    return p;
  };
  DecShare<kUnit8, kKeys8> str;
  int at = 0, at_end = 0, sq = 0, first = 0;  // (units; sq: the sequence that holds `at`, first: its first)
  if constexpr (SHARE) {
    const Dec8Args p = dec_reload<Dec8Args>();
    str.init(p, append, p.parts, lane);
    const int part = by;
    if (str.even) {
      sq = str.seek(p, append, part, lane, first);
      if (sq >= p.batch) return;
      at = (part - first) * str.per;
      at_end = at + str.per;
      first = 0;
    } else {
      at = part * str.per;
      at_end = min(at + str.per, str.total);
      if (at >= at_end) return;
      sq = str.seek(p, append, at, lane, first);
    }
  }
  for (bool more = true; more;) {
    const int b = SHARE ? sq : by;
    // Q^T as the B operand, loaded while the lengths are on their way. A 16-byte read of a K row holds dims 64m + 16lg ..
    // +15 and feeds steps 2m and 2m + 1, so step 2m + s takes dims 64m + 16lg + 8s + e of row lh.
    auto dim = [&](int ds) { return 64 * (ds / 2) + 16 * lg + 8 * (ds % 2); };
    u32x4 qraw[NDS];
    {
      const Dec8Args p = args();
      const T* row = (const T*)p.q + row_of(b, kvh, min(lh, hg - 1)) * HDr;
#pragma unroll
      for (int ds = 0; ds < NDS; ds++) qraw[ds] = *(const u32x4*)(row + (dim(ds) < HDr ? dim(ds) : 0));
    }
    DecSpan sp;
    int start, end;
    float* rec = nullptr;  // record of row 0 (rows rec_step apart); null: the final output
    long long rec_step = HDr + 2;
    if constexpr (SHARE) {
      const Dec8Args p = dec_reload<Dec8Args>();
      if (b >= str.base + 64) str.load(p, append, b, lane);
      sp = str.span(b);
      const int units = dec_units<kUnit8>(sp), stop = min(at_end, first + units);
      start = sp.lo + (at - first) * kUnit8;
      end = min(sp.lo + (stop - first) * kUnit8, sp.hi);
      const bool begins = at == first;
      const int part = by;
      if (begins && hgl == 0 && tid == 0) {   // where the combine finds this sequence's records (decode.hip)
        const int n = str.even ? str.items(units) : (int)((unsigned)(first + units - 1) / (unsigned)str.per) - part + 1;
        ((int*)p.scratch)[2 * b] = 2 * part + (str.even ? 0 : 1);
        ((int*)p.scratch)[2 * b + 1] = str.even ? n : -n;
      }
      if (!(begins && stop == first + units))
        rec = p.scratch + dec_meta_floats(p) + ((2ll * part + (begins && !str.even ? 1 : 0)) * X * WH + grp * NKV + head0) * 16 * (HDr + 2);
      at = stop;
      first += units;
      sq++;
      more = !str.even && at < at_end;
    } else {
      sp = dec_span(p, b, append);
      sp.lo &= -kKeys8;
      const int n = max(sp.hi - sp.lo, 0);
      const int share = p.nsplit > 1 ? (int)((unsigned)(n + p.nsplit - 1) / (unsigned)p.nsplit) : n;
      const int chunk = (share + kKeys8 - 1) / kKeys8 * kKeys8;
      start = sp.lo + bz * chunk;
      end = min(start + chunk, sp.hi);
      if (!(p.flags & kDec8Final)) {
        rec = p.scratch + (long long)bz * (HDr + 2);
        rec_step = (long long)p.nsplit * (HDr + 2);   // rows are indexed as in q
      }
      more = false;
    }
    const int ctx = sp.ctx;
    start = __builtin_amdgcn_readfirstlane(start);   // a multiple of 32
    end = __builtin_amdgcn_readfirstlane(end);
    // the first key some row of the call sees: nothing ahead of it is read; and the keys that every row sees
    int klo, slo, shi;
    int rlo, rspan;   // this lane's row (lh)
    const int tok = row_tok(min(lh, hg - 1)), qpos = ctx + tok;
    float slope = 0.0f, c_log2;
    {
      const Dec8Args p = args();
      const int lo0 = dec_lo(p, b, ctx, 0);
      klo = __builtin_amdgcn_readfirstlane(max(append ? max(min(lo0, ctx), 0) : lo0, start));
      slo = __builtin_amdgcn_readfirstlane(max(dec_lo(p, b, ctx, nq - 1), start));
      shi = __builtin_amdgcn_readfirstlane(min(dec_hi(p, ctx, 0, append), end));
      rlo = max(dec_lo(p, b, ctx, tok), start);
      rspan = max(min(dec_hi(p, ctx, tok, append), end) - rlo, 0);
      if (FEAT && p.alibi && lh < hg) slope = p.alibi[kvh * gqa + (r0 + lh - tok * gqa)];
      c_log2 = p.scale * kLog2e;
    }

    // ---- zero columns past the head dim; a rotated q goes through LDS in fp32 and is carried as hi + lo
    V8 qb[NDS], ql[NDS];
#pragma unroll
    for (int ds = 0; ds < NDS; ds++) {
      qb[ds] = bitcast<V8>(dim(ds) < HDr ? qraw[ds] : u32x4{0, 0, 0, 0});
      ql[ds] = bitcast<V8>(u32x4{0, 0, 0, 0});
    }
    bool qsplit;
    {
      const Dec8Args p = args();
      qsplit = p.rotary != 0;
      if (p.rotary) {
        if (rw == 0) {
#pragma unroll
          for (int ds = 0; ds < NDS; ds++)
#pragma unroll
            for (int e = 0; e < 8; e++) qsh[16 * hw + lh][dim(ds) + e] = (float)qb[ds][e];
        }
        __syncthreads();
        const int rdim = p.rotary_dim > 0 ? p.rotary_dim : HDr, half = rdim / 2;
        const int rbase = p.rotary_pos ? p.rotary_pos[b] : ctx;
        for (int i = tid; i < WH * 16 * half; i += 256) {
          const int g = i / half, j = i % half;
          if (g % 16 >= hg) continue;
          const int rp = min(max(rbase + row_tok(g % 16), 0), p.c.rotary_rows - 1);
          const float c = p.cos[(long long)rp * half + j], s = p.sin[(long long)rp * half + j];
          const int ia = p.rotary == 1 ? j : 2 * j, ib = p.rotary == 1 ? j + half : 2 * j + 1;
          const float x = qsh[g][ia], y = qsh[g][ib];
          qsh[g][ia] = x * c - y * s;
          qsh[g][ib] = y * c + x * s;
        }
        __syncthreads();
#pragma unroll
        for (int ds = 0; ds < NDS; ds++)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float x = qsh[16 * hw + lh][dim(ds) + e];
            qb[ds][e] = (T)x;
            ql[ds][e] = (T)(x - (float)(T)x);
          }
        __syncthreads();  // q staging is dead from here on
      }
    }

    f32x4 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) oacc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.0f;
    const int* bt = p.table + (long long)b * (p.max_blocks & p.tmask);
    const int blk0 = b * p.max_blocks, tmask = p.tmask, pmask = p.page - 1, subs = 1 << (page_shift - p.gshift);
    const unsigned rstep = (unsigned)p.c.s.s, pstep = (unsigned)p.c.s.b, top_blk = (unsigned)p.c.num_blocks - 1;
    const uint8_t* Kc = (const uint8_t*)p.Kc + (long long)kvh * p.c.s.h;
    const uint8_t* Vc = (const uint8_t*)p.Vc + (long long)kvh * p.c.s.h;
    const uint8_t* scales = (lane < 32 ? p.c.k_scale : p.c.v_scale) + (long long)kvh * subs;
    const unsigned sstep = (unsigned)NKV * (unsigned)subs;   // scales of a page
    uint8_t* kb = (uint8_t*)raw + wave * L::WAVE;
    uint8_t* vb = kb + kKeys8 * L::STR;
    float* sb = (float*)(vb + kKeys8 * L::STR);

    // Load i of a lane covers chunk f = 64i + lane of the tile: row f / RB, 16 bytes at f % RB, consecutive
    // lanes on whole rows. K's rows go to the slots that make them the rows of the two S products with eight
    // consecutive keys per lane: row 8a + 4h + r to slot 16h + 4a + r.
    const int last = end - 1;
    int off[NV], lk[NV], lv[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int f = 64 * i + lane, row = f / RB, ch = f % RB;
      off[i] = 16 * ch < HDr ? (P16 ? row & 15 : row) * (int)rstep + 16 * ch : kBufZero;
      lk[i] = (16 * ((row >> 2) & 1) + 4 * (row >> 3) + (row & 3)) * L::STR + 16 * ch;
      lv[i] = row * L::STR + 16 * ch;
    }
    // Pages of the wave's chunks, 64 at a time: lane l of `page` has those of chunk c (c % 64 = l), which reach the scalar
    // unit by a readlane; the next 64 are fetched meanwhile. (By scalar loads, one chunk ahead, an entry
    // held up the LDS reads it shares a counter with.)
    const int kfirst = start + kKeys8 * rw;
    int page[NPG], next[NPG];   // (next: the entries as read)
    auto index = [&](int c0, int h) {   // lane's page of its sequence, among those with keys of it
      const unsigned key = (unsigned)kfirst + min((unsigned)(c0 + lane) * kUnit8, (unsigned)end) + 16u * h;
      return (int)min(max(key, (unsigned)klo), (unsigned)last) >> page_shift;
    };
    auto fetch = [&](int c0) {
#pragma unroll
      for (int h = 0; h < NPG; h++) next[h] = bt[index(c0, h) & tmask];
    };
    auto take = [&](int c0) {
#pragma unroll
      for (int h = 0; h < NPG; h++) page[h] = (int)min((unsigned)((next[h] & tmask) | ((blk0 + index(c0, h)) & ~tmask)), top_blk);
    };
    struct Rows {
      u32x4 k[NV], v[NV];
      unsigned s;
    };
    Rows set[DEPTH];
    // (chunks past the end load nothing: their descriptors have no bytes. No condition around the loads, which would
    // have every wait be for all of them.)
    auto load = [&](int kc0, int c, bool front, Rows& r) {
      __amdgpu_buffer_rsrc_t kr[NPG], vr[NPG];
      unsigned blk[NPG];
#pragma unroll
      for (int h = 0; h < NPG; h++) {
        blk[h] = (unsigned)__builtin_amdgcn_readlane(page[h], c & 63);
        const int k0 = kc0 + 16 * h;
        const unsigned bytes = (unsigned)max(min(end - k0, 32 / NPG), 0) * rstep;
        const uint64_t o = (uint64_t)blk[h] * pstep + (unsigned)(k0 & pmask) * rstep;
        kr[h] = buf_rsrc32(Kc + o, (unsigned)__builtin_amdgcn_readfirstlane((int)bytes));
        vr[h] = buf_rsrc32(Vc + o, (unsigned)__builtin_amdgcn_readfirstlane((int)bytes));
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int f = 64 * i + lane;
        // (rows ahead of klo in a run's first chunk: zeros too)
        const int o = front && kc0 + f / RB < klo ? kBufZero : off[i];
        // (a load of the wave lies in one page: 16 rows are HD chunks, whole loads)
        static_assert(HD % 64 == 0, "loads of a page of 16 rows");
        constexpr int kLo = 16 * RB;   // chunks of the first page
        const int pg = P16 && 64 * i >= kLo ? NPG - 1 : 0;
        r.k[i] = buf_load16_nt(kr[pg], o);
        r.v[i] = buf_load16_nt(vr[pg], o);
      }
      // scale of key kc0 + (lane & 31): K's for the first 32 lanes, V's for the others
      const unsigned pg = P16 && (lane & 16) ? blk[NPG - 1] : blk[0];
      r.s = scales[(uint64_t)pg * sstep + (unsigned)(((kc0 + (lane & 31)) & pmask) >> p.gshift)];
    };

    // chunk c at key kc0: its rows from r to LDS, and the loads of the rows DEPTH chunks on to r
    auto stage = [&](int kc0, int c, Rows& r) {
      // codes and scales -> this wave's own LDS (its operations complete in order: no barrier). A scale of a key
      // that is not there is no number to multiply zeros by.
      const int skey = kc0 + (lane & 31);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        *(u32x4*)(kb + lk[i]) = r.k[i];
        *(u32x4*)(vb + lv[i]) = r.v[i];
      }
      sb[lane] = skey >= klo && skey < end ? e8_f32(r.s) : 0.0f;
      if (((c + DEPTH) & 63) == 0) {
        take(c + DEPTH);
        fetch(c + DEPTH + 64);
      }
      load(kc0 + DEPTH * kUnit8, c + DEPTH, false, r);
    };
    auto chunk = [&](int kc0) {
      // S^T = K . Q^T of the keys in slots 0..15 and 16..31: lane (lg, lh) gets keys kc0 + 8lg + 4h + r of row lh
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      V8 ka[2][NDS];
#pragma unroll
      for (int m = 0; m < NDS / 2; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const u32x4 c = *(const u32x4*)(kb + (16 * h + lh) * L::STR + 64 * m + 16 * lg);
          ka[h][2 * m] = codes_to<T>(u32x2{c[0], c[1]}, 1.0f);
          ka[h][2 * m + 1] = codes_to<T>(u32x2{c[2], c[3]}, 1.0f);
        }
#pragma unroll
      for (int d = 0; d < NDS; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) s[h] = Dt<T>::mma16(ka[h][d], qb[d], s[h]);
      if (qsplit) {
#pragma unroll
        for (int d = 0; d < NDS; d++)
#pragma unroll
          for (int h = 0; h < 2; h++) s[h] = Dt<T>::mma16(ka[h][d], ql[d], s[h]);
      }
      // logits (log2 domain) and masking
      const f32x4 ks0 = *(const f32x4*)(sb + 8 * lg), ks1 = *(const f32x4*)(sb + 8 * lg + 4);
      float t[8], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        float x = s[e >> 2][e & 3] * (e < 4 ? ks0[e & 3] : ks1[e & 3]);
        if (FEAT) {
          x = x * p.scale;
          if (p.softcap > 0.0f) x = p.softcap * tanh_exp(x / p.softcap);
          x += slope * (float)(kc0 + 8 * lg + e - qpos);
          t[e] = x * kLog2e;
        } else {
          t[e] = x * c_log2;
        }
      }
      if (kc0 < slo || kc0 + kKeys8 > shi) {
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = (unsigned)(kc0 + 8 * lg + e - rlo) < (unsigned)rspan ? t[e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) mx = fmaxf(mx, t[e]);
      mx = half_max(lane16_max(mx));
      const float m_new = fmaxf(m_run, mx);
      const float m_use = m_new == -INFINITY ? 0.0f : m_new;
      if (__builtin_amdgcn_readfirstlane((int)(__builtin_amdgcn_ballot_w64(m_new > m_run) != 0))) {
        const float corr = exp2_fast(m_run - m_use);
        l_run *= corr;
#pragma unroll
        for (int db = 0; db < NDB; db++) oacc[db] *= corr;
        m_run = m_new;
      }
      float rs = 0.0f;
      bf16x8 pb, pl;     // P^T times V's scales, the B operand: keys 8lg + e, row lh
      const f32x4 vs0 = *(const f32x4*)(sb + 32 + 8 * lg), vs1 = *(const f32x4*)(sb + 36 + 8 * lg);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float w = exp2_fast(t[e] - m_use), z = w * (e < 4 ? vs0[e & 3] : vs1[e & 3]);
        rs += w;
        pb[e] = (__bf16)z;
        if constexpr (kTwoP) pl[e] = (__bf16)(z - (float)pb[e]);
      }
      l_run += rs;
      // O^T += V^T . P^T: lane lh of group lg addresses row 8lg + lh/2, column 16db + 8(lh%2), and receives
      // column 16db + lh of rows 8lg .. 8lg+7
#pragma unroll
      for (int db = 0; db < NDB; db++) {
        const uint8_t* a = vb + (8 * lg + (lh >> 1)) * L::STR + 16 * db + 8 * (lh & 1);
        const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)((__attribute__((address_space(3))) uint8_t*)a));
        const bf16x8 av = codes_to<__bf16>(u32x2{(unsigned)c[0], (unsigned)c[1]}, 1.0f);
        oacc[db] = Dt<__bf16>::mma16(av, pb, oacc[db]);
        if constexpr (kTwoP) oacc[db] = Dt<__bf16>::mma16(av, pl, oacc[db]);
      }
    };
    if (kfirst < end) {
      fetch(0);
      take(0);
      fetch(64);
#pragma unroll
      for (int d = 0; d < DEPTH; d++) {
        load(kfirst + d * kUnit8, d, d == 0, set[d]);
        // (in this order: the loop's waits count the loads behind the ones they need, whichever way it was entered)
        __builtin_amdgcn_sched_barrier(0);
      }
      // (no way out in the middle: with one, the compiler's waits at the top of the loop are for every load)
      for (int kc0 = kfirst, c = 0; kc0 < end; kc0 += DEPTH * kUnit8, c += DEPTH) {
        stage(kc0, c, set[0]);
        chunk(kc0);
        if constexpr (DEPTH == 2) {
          stage(kc0 + kUnit8, c + 1, set[1]);
          if (kc0 + kUnit8 < end) chunk(kc0 + kUnit8);
        }
      }
    }

    // ---- merge the four waves: per row max, sum and O^T accumulators through LDS
    const float l_grp = half_sum(lane16_sum(l_run));
    __syncthreads();
    float* red_o = (float*)raw;  // [wave][16 rows][FSTR]
    if (lg == 0) {
      red_m[wave][lh] = dec_row_max(m_run, l_grp);
      red_l[wave][lh] = l_grp;
    }
#pragma unroll
    for (int db = 0; db < NDB; db++) *(f32x4*)(red_o + (wave * 16 + lh) * L::FSTR + 16 * db + 4 * lg) = oacc[db];
    __syncthreads();
    const Dec8Args pe = args();
    const int quads = HDr / 4;
    for (int i = tid; i < WH * hg * quads; i += 256) {
      const int r = i / quads, d = 4 * (i - r * quads), h = WH > 1 ? r / hg : 0, g = r - h * hg;
      float gm = -INFINITY;
#pragma unroll
      for (int w = 0; w < WR; w++) gm = fmaxf(gm, red_m[WH * w + h][g]);
      float l = 0.0f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      if (gm != -INFINITY) {
#pragma unroll
        for (int w = 0; w < WR; w++) {
          const float f = exp2_fast(red_m[WH * w + h][g] - gm);
          l += f * red_l[WH * w + h][g];
          acc += f * *(const f32x4*)(red_o + ((WH * w + h) * 16 + g) * L::FSTR + d);
        }
      }
      const long long row = row_of(b, head0 + h, g);
      if (!rec) {
        const bool ok = gm != -INFINITY;
        typedef T V4 __attribute__((ext_vector_type(4)));
        V4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (T)(ok ? acc[e] / l : 0.0f);
        *(V4*)((T*)pe.o + row * HDr + d) = v;
        if (pe.lse_out && d == 0) pe.lse_out[row] = ok ? gm * kLn2 + __logf(l) : -INFINITY;
        continue;
      }
      float* out = rec + (SHARE ? 16 * h + g : row) * rec_step;   // (8-byte aligned: HDr is even)
      if (d == 0) *(f32x2*)out = f32x2{gm, l};
      *(f32x2*)(out + 2 + d) = f32x2{acc[0], acc[1]};
      *(f32x2*)(out + 4 + d) = f32x2{acc[2], acc[3]};
    }
    if (more) __syncthreads();  // the merge has read the LDS regions before the next segment fills them
  }
}

// Heads of a workgroup. One wave per head makes what the CUs read at a time runs of 4 * D bytes in place of D, which HBM
// gives faster (rows of 128 bytes at 1 KiB: 6.24 TB/s alone, 7.1 in fours); but a wave then walks four times the keys, and there
// are four times the records, so it takes a large call: 16 x 32768 keys of 8 heads, D 128: 199 -> 172 us, 48 of up to 8192 98 -> 80,
// 16 x 8000 (262 MB) 55 -> 49, 64 x 1000 (134 MB) 31 -> 29, 64 x 2000 of 4 heads (134 MB) 26.1 and 27.0; 16 x 2000 (67 MB)
// 18.6 and 18.3, 64 x 1000 of 4 heads 15.8 and 17.5, one of 500 8.4 and 13.3. The size is the table's, however full: 32 of 300
// keys in tables of 8192 14.5 and 15.8, of 1000 19.1 and 20.7, of 3000 41.2 and 40.8.
// Two where there are no four (6 heads of 64, 64 x 4000 keys: 70 -> 53), and at D 192 (32 x 4000 keys of 16 heads: 169 -> 158,
// 154 with four; of 4 heads 41.7 and 42.7, 45.7 with four). Rows of 256 bytes gain nothing (32 x 4000, 8 heads: 97, 99, 98).
// (Split counts the caller sets are for one head to a workgroup.) A row must not get more than 32 records (one of 64000
// keys, 16 heads 54.8, 52.4 in twos, 56.0 in fours; 8 heads in a table of 131072 33.7, 44.3 in fours).
constexpr long long kHeadBytes8 = 112LL << 20, kHeadGroups8 = 8;
static int dec8_heads(const FableDecParams& p) {
  const int nkv = p.NH / p.gqa;
  if (p.nsplit > 0 || p.HD > 192 || (long long)p.batch * p.max_blocks * p.page * nkv * p.HD * 2 < kHeadBytes8) return 1;
  int wh = p.HD <= 128 && nkv % 4 == 0 ? 4 : nkv % 2 == 0 ? 2 : 1;
  while (wh > 1 && (long long)p.batch * (nkv / wh) * dec_groups(p) < kHeadGroups8) wh /= 2;
  return wh;
}
static int dec8_unit(int wh) { return kKeys8 * (kDecWaves / wh); }   // keys of a unit of a share
template <typename T, int HD>
static int launch_dec8(const FableDecParams& p, const FableCache8& c, int parts, int wh, hipStream_t st, bool append) {
  Dec8Args a;
  (FableDecParams&)a = p;
  a.c = c;
  a.table = p.block_table ? p.block_table : p.ctx_len;
  a.tmask = p.block_table ? -1 : 0;
  a.page_shift = __builtin_ctz((unsigned)p.page);
  a.gshift = __builtin_ctz((unsigned)c.group);
  a.ngrp = dec_groups(p);
  a.nkv = p.NH / p.gqa;
  a.parts = parts;
  a.flags = (append ? kDec8Append : 0) | (parts == 0 && p.nsplit == 1 ? kDec8Final : 0);
  const bool feat = p.softcap > 0.0f || p.alibi != nullptr;
  const unsigned X = (unsigned)(a.nkv / wh * a.ngrp);
  const dim3 grid = parts > 0 ? dim3(X, (unsigned)dec_share_wgs(p, dec8_unit(wh), wh)) : dim3(X, (unsigned)p.batch, (unsigned)p.nsplit);
  // Heads whose rows share 128-byte lines (D 64: two, D 96: four) run one after another on one XCD, whose L2 then
  // fetches a line once: dealt out like the others, every XCD fetched them for itself (16 x 32768 keys of 8 heads,
  // D 64: 171 -> 118 us; D 192, 1.1x; at 128 and 256 nothing is shared, and the order measured the same).
  a.bshift = 0;
  while ((p.HD * wh << a.bshift) % 128 && a.bshift < 3) a.bshift++;
  if (a.nkv / wh % (1 << a.bshift) || ((long long)grid.x * grid.y * grid.z >> a.bshift) % 8) a.bshift = 0;
  auto go = [&](auto ft, auto sh, auto w) {
    if (p.page == 16)
      hipLaunchKernelGGL((dec8_partial_kernel<T, HD, decltype(ft)::value, decltype(sh)::value, true, decltype(w)::value>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((dec8_partial_kernel<T, HD, decltype(ft)::value, decltype(sh)::value, false, decltype(w)::value>), grid, dim3(256), 0, st, a);
  };
  using Y = std::integral_constant<bool, true>;
  using N = std::integral_constant<bool, false>;
  auto with = [&](auto w) {
    if (parts > 0)
      feat ? go(Y{}, Y{}, w) : go(N{}, Y{}, w);
    else
      feat ? go(Y{}, N{}, w) : go(N{}, N{}, w);
  };
  if constexpr (HD <= 128)
    if (wh == 4) with(std::integral_constant<int, 4>{});
  if constexpr (HD <= 192)
    if (wh == 2) with(std::integral_constant<int, 2>{});
  if (wh == 1) with(std::integral_constant<int, 1>{});
  return launch_status("fable_attn_dec8 (partial)");
}
// kernel widths 64, 128, 192 and 256 (a row of codes is read in 64-byte steps); a head dim below its width runs with zero columns
template <typename T>
static int dec8_dispatch(const FableDecParams& p, const FableCache8& c, int parts, int wh, hipStream_t st, bool append) {
  if (p.HD <= 64) return launch_dec8<T, 64>(p, c, parts, wh, st, append);
  if (p.HD <= 128) return launch_dec8<T, 128>(p, c, parts, wh, st, append);
  if (p.HD <= 192) return launch_dec8<T, 192>(p, c, parts, wh, st, append);
  return launch_dec8<T, 256>(p, c, parts, wh, st, append);
}

// ------------------------------------------------------------------ which path a call takes
// Many new tokens run on the tile kernel of the forward (FwdPaged8), from kTileRows rows of a K/V head on
// where there are more than kTileStreams (sequence, K/V head, 16 rows): the rule of the 16-bit decode.
constexpr int kTileRows8 = 64, kTileStreams8 = 16;
static bool dec8_uses_tiles(const FableDecParams& p, const FableCache8& c) {
  return c.s.b <= 0x7FFFFFFF && p.page * c.s.s <= 0x7FFFFFFF && (long long)c.num_blocks * (p.NH / p.gqa) * (p.page / c.group) <= 0x7FFFFFFF &&
         (long long)p.batch * (p.NH / p.gqa) * dec_groups(p) > kTileStreams8 && (long long)p.nq * p.gqa >= kTileRows8 &&
         (long long)p.batch * p.max_blocks <= 0x7FFFFFFF && p.max_blocks < (1 << 29) && p.window != 0;
}
// Shares worked out on the device for batches that equal splits would not spread evenly, as in decode.hip
constexpr long long kShareBytes8 = 64LL << 20;
static bool dec8_shares(const FableDecParams& p, int wh) {
  if (p.nsplit > 0 || p.batch < 2) return false;
  if ((long long)p.batch * p.max_blocks * p.page * (p.NH / p.gqa) * p.HD * 2 < kShareBytes8) return false;
  const int parts = dec_parts(p, dec8_unit(wh), wh);
  return p.batch > parts || parts % p.batch != 0;
}
static int dec8_fixed_splits(const FableDecParams& p, int wh) {
  return fa_decode_num_splits(p.batch, dec_groups(p), p.NH / p.gqa / wh, 1, (int64_t)p.max_blocks * p.page, p.nsplit);
}
static long long align256(long long x) { return (x + 255) / 256 * 256; }
static long long dec8_q_bytes(const FableDecParams& p) {   // one part of a rotated q
  return p.rotary ? align256((long long)p.batch * p.nq * p.NH * p.HD * 2) : 0;
}
// the forward's parameters of a call on the tile kernel
static void dec8_tile_params(const FableDecParams& p, const FableCache8& c, bool append, FableFwdParams& f, FwdPaged8& pg) {
  const int64_t D = p.HD;
  f = FableFwdParams{};
  f.Q = p.q;
  f.K = p.Kc;
  f.V = p.Vc;
  f.O = p.o;
  f.LSE = p.lse_out;
  f.sQ = f.sO = fa_strides{p.nq * p.NH * D, D, p.NH * D};
  f.sK = fa_strides{0, c.s.h, c.s.s};
  f.sV = fa_strides{0, c.s.h, c.s.s};
  f.SQ = p.nq;
  const long long room = (long long)p.max_blocks * p.page;
  f.SK = room < 0x7FFFFFFF ? (int)room : 0x7FFFFFFF;
  f.HD = p.HD;
  f.NH = p.NH;
  f.gqa = p.gqa;
  f.scale = p.scale;
  f.softcap = p.softcap;
  f.win_left = p.window >= 0 ? p.window - 1 : -1;
  f.win_right = -1;
  f.alibi_slopes = p.alibi;
  f.causal = append;
  f.batch = p.batch;
  f.lse_sb = (int64_t)p.nq * p.NH;
  f.lse_sh = 1;
  (FwdPaged&)pg = FwdPaged{p.block_table ? p.block_table : p.ctx_len, p.block_table ? -1 : 0, p.max_blocks,
                           __builtin_ctz((unsigned)p.page), c.s.b, c.s.b, p.ctx_len, append ? 1 : 0, p.leftpad, nullptr, p.NH};
  fwd_paged8_scales(pg, c, p.page);
}

// the argument checks of the two entry points (nq below 1 becomes 1)
static int dec8_check(FableDecParams& p, const FableCache8& c, int dtype) {
  const char* what = "fable_attn_dec8";
  if (dtype != FA_F16 && dtype != FA_BF16) return fail(FA_ERR_DTYPE, "%s: dtype %d not implemented (fp16/bf16)", what, dtype);
  if (p.NH <= 0 || p.gqa <= 0 || p.NH % p.gqa) return fail(FA_ERR_ARG, "%s: NH=%d gqa=%d", what, p.NH, p.gqa);
  if (p.nq < 1) p.nq = 1;
  if (p.nsplit < 0 || p.nsplit > 512) return fail(FA_ERR_ARG, "%s: nsplit=%d", what, p.nsplit);
  if (p.max_blocks < 1 || (long long)p.max_blocks * p.page > 0x7FFF0000)
    return fail(FA_ERR_ARG, "%s: max_blocks=%d page=%d", what, p.max_blocks, p.page);
  // (rows of q, and the heads of a sequence's tokens, are counted in 32 bits)
  if (p.batch > 65535 || (long long)p.nq * p.gqa > (1 << 24) || (long long)p.batch * p.nq > 0x7FFFFFFF || (long long)p.nq * p.NH > 0x7FFFFFFF)
    return fail(FA_ERR_ARG, "%s: batch=%d nq=%d", what, p.batch, p.nq);
  if (p.rotary && (p.rotary_dim < 0 || p.rotary_dim > p.HD || p.rotary_dim % 2)) return fail(FA_ERR_ARG, "%s: rotary_dim=%d", what, p.rotary_dim);
  if (p.rotary && (p.rotary > 2 || c.rotary_rows < 1)) return fail(FA_ERR_ARG, "%s: rotary=%d rotary_rows=%d", what, p.rotary, c.rotary_rows);
  if (c.s.b > 0xFFFFFFFFll || p.page * c.s.s > 0xFFFFFFFFll) return fail(FA_ERR_ARG, "%s: pages of 4 GiB", what);
  return cache8_check(what, c, p.HD, p.page);
}

}  // namespace fa

extern "C" int64_t fable_attn_dec8_ws_bytes(FableDecParams p, FableCache8 c, int dtype, int append) {
  using namespace fa;
  if (dec8_check(p, c, dtype) != FA_OK) return -1;
  if (p.batch <= 0) return 0;
  if (dec8_uses_tiles(p, c)) {
    FableFwdParams f;
    FwdPaged8 pg;
    dec8_tile_params(p, c, append != 0, f, pg);
    FwdWs fw{nullptr, 0, true, 0, p.nsplit};
    if (launch_fwd_paged8(f, pg, dtype, p.rotary != 0, nullptr, fw) != FA_OK) return -1;
    return 2 * dec8_q_bytes(p) + fw.need;
  }
  const int wh = dec8_heads(p);
  if (dec8_shares(p, wh)) return dec_share_bytes(p, dec8_unit(wh), wh);
  p.nsplit = dec8_fixed_splits(p, wh);
  return p.nsplit != 1 ? (int64_t)p.batch * p.nq * p.NH * p.nsplit * (p.HD + 2) * 4 : 0;
}

extern "C" int fable_attn_dec8(FableDecParams p, FableCache8 c, int dtype, void* ws, int64_t ws_bytes, void* stream,
                               const void* new_k, const void* new_v) {
  using namespace fa;
  const char* what = "fable_attn_dec8";
  if (!p.q || !p.Kc || !p.Vc || !p.o || !p.ctx_len || !c.k_scale || !c.v_scale) return fail(FA_ERR_ARG, "%s: null pointer", what);
  if ((new_k == nullptr) != (new_v == nullptr)) return fail(FA_ERR_ARG, "%s: new_k and new_v go together", what);
  if (p.rotary && (!p.cos || !p.sin)) return fail(FA_ERR_ARG, "%s: rotary needs cos and sin", what);
  if (int rc = dec8_check(p, c, dtype)) return rc;
  if (p.batch <= 0) return FA_OK;
  const int64_t need = fable_attn_dec8_ws_bytes(p, c, dtype, new_k != nullptr);
  if (need < 0) return FA_ERR_ARG;
  if (need > 0 && (!ws || ws_bytes < need)) return fail(FA_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)need);
  hipStream_t st = (hipStream_t)stream;
  const bool tiles = dec8_uses_tiles(p, c);
  const long long qb = tiles ? dec8_q_bytes(p) : 0;
  if (new_k || (tiles && p.rotary)) {
    // the new rows into the cache; for the tile kernel also q, rotated, in two parts
    const int64_t NKV = p.NH / p.gqa, D = p.HD;
    FableAppendParams a{};
    a.sk = a.sv = fa_strides{p.nq * NKV * D, D, NKV * D};
    a.sq = fa_strides{p.nq * p.NH * D, D, p.NH * D};
    a.k = new_k;
    a.v = new_v;
    if (tiles && p.rotary) {
      a.q = p.q;
      a.q_out = ws;
      a.q_lo = (char*)ws + qb;
    }
    a.Kc = const_cast<void*>(p.Kc);
    a.Vc = const_cast<void*>(p.Vc);
    a.k_scale = const_cast<uint8_t*>(c.k_scale);
    a.v_scale = const_cast<uint8_t*>(c.v_scale);
    a.kc = a.vc = c.s;
    a.block_table = p.block_table;
    a.ctx_len = p.ctx_len;
    a.leftpad = c.held;
    a.rotary_pos = p.rotary_pos;
    a.cos = p.cos;
    a.sin = p.sin;
    a.batch = p.batch;
    a.n = p.nq;
    a.NH = p.NH;
    a.NKV = (int)NKV;
    a.HD = p.HD;
    a.page = p.page;
    a.max_blocks = p.max_blocks;
    a.num_blocks = c.num_blocks;
    a.group = c.group;
    a.rotary = p.rotary;
    a.rotary_dim = p.rotary_dim;
    a.rotary_rows = c.rotary_rows;
    if (int rc = append_rows(a, dtype, st)) return rc;
  }
  if (tiles) {
    // (q in two parts, as in the 16-bit decode. Rounded to bf16 once the call takes 163 us instead of 217 (512 tokens of
    // two requests over up to 7000 keys, D 128), but is 3.5e-3 off instead of 1.7e-3 with keys of size 2.)
    FableFwdParams f;
    FwdPaged8 pg;
    dec8_tile_params(p, c, new_k != nullptr, f, pg);
    if (p.rotary) {
      f.Q = ws;
      pg.qlo = (char*)ws + qb;
    }
    FwdWs fw{ws ? (char*)ws + 2 * qb : nullptr, ws_bytes - 2 * qb, false, 0, p.nsplit};
    return launch_fwd_paged8(f, pg, dtype, p.rotary != 0, st, fw);
  }
  p.scratch = (float*)ws;
  const int wh = dec8_heads(p);
  const bool share = dec8_shares(p, wh);
  const int parts = share ? dec_parts(p, dec8_unit(wh), wh) : 0;
  p.nsplit = share ? 0 : dec8_fixed_splits(p, wh);
  const int rc = dtype == FA_F16 ? dec8_dispatch<_Float16>(p, c, parts, wh, st, new_k != nullptr) : dec8_dispatch<__bf16>(p, c, parts, wh, st, new_k != nullptr);
  if (rc != FA_OK || (!share && p.nsplit == 1)) return rc;
  return dec_combine(p, dtype, st, share);
}
