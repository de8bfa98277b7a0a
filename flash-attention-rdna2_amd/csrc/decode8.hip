// decode8.hip — decode over a K/V cache held in 8 bits (fable_attn_dec8; the format: cache8.hpp).
//
// The split of the work, the records and the combine are the 16-bit decode's (decode.hip): one workgroup of
// four waves per (K/V head, group of 16 rows, run of a sequence's keys), each wave with its own chunks and
// online softmax, merged in LDS. What differs:
//  * a chunk is 32 keys, so as many bytes are in flight per wave as there with 16;
//  * codes stay codes in LDS (half the LDS traffic) and become fp16/bf16 between the LDS read and the matrix
//    instruction: K by 16-byte reads of a key's row, V by the transposing 8-bit reads (ds_read_b64_tr_b8: a lane
//    gets one column of eight rows, the A operand of v_mfma_f32_16x16x32 as it is);
//  * codes are converted without their scales, which are exact powers of two: a key's K scale multiplies its fp32
//    scores, its V scale the fp32 probability ahead of the rounding to 16 bits. The scales of a chunk come
//    in one byte load per lane and reach the lanes that need them through LDS;
//  * chunks are aligned to 32 keys, so each half of one lies in one page (of 16 rows at least): a buffer
//    descriptor per half makes the lanes' offsets loop invariant and rows past the end zero.
// fp16: a scaled probability can leave fp16's range (and V's codes need no more than bf16 holds), so P goes
// as two bf16 parts, high and low, into two products: 16 bits of it, as many as fp16's own rounding left.
#include "cache8.hpp"
#include "dec_common.hpp"
#include "fwd_common.hpp"

namespace fa {

constexpr int kKeys8 = 32;                       // keys per wave iteration
constexpr int kUnit8 = kKeys8 * kDecWaves;       // keys of a unit of a share (DecShare)
constexpr int kDec8Append = 1, kDec8Final = 2;   // new keys were appended; one split, no combine launch

struct Dec8Args : FableDecParams {
  FableCache8 c;
  const int* table;   // as DecArgs::table (decode.hip): the block table, or any readable address and tmask 0
  int tmask, page_shift, gshift, ngrp, flags, parts, nkv;
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
  // touch every bank once
  static constexpr int STR = HD + 16;
  static constexpr int WAVE = 2 * kKeys8 * STR + 64 * 4;   // K, V, scales
  static constexpr int ACC = kDecWaves * 16 * HD * 4;       // the merge's accumulators (q staging is smaller)
  static constexpr int BYTES = kDecWaves * WAVE > ACC ? kDecWaves * WAVE : ACC;
};

template <typename T, int HD, bool FEAT, bool SHARE>
__global__ __launch_bounds__(256) void dec8_partial_kernel(Dec8Args p) {
  using V8 = typename Dt<T>::V8;
  using L = Dec8Lds<HD>;
  constexpr bool kTwoP = std::is_same<T, _Float16>::value;   // P in two bf16 parts
  constexpr int NDS = HD / 32, NDB = HD / 16, RB = HD / 16, NV = kKeys8 * RB / 64;
  __shared__ __attribute__((aligned(16))) char raw[L::BYTES];
  __shared__ float red_m[kDecWaves][16], red_l[kDecWaves][16];
  float (*qsh)[HD] = (float (*)[HD])raw;

  const int append = p.flags & kDec8Append, page_shift = p.page_shift;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lg = lane >> 4, lh = lane & 15;
  const int NKV = p.nkv, HDr = p.HD, nq = p.nq, gqa = p.gqa, NH = p.NH;
  const int X = gridDim.x, hgl = blockIdx.x, grp = p.ngrp > 1 ? hgl / NKV : 0, kvh = hgl - grp * NKV;
  const int r0 = 16 * grp, hg = min(16, nq * gqa - r0);  // rows of this group
  auto row_tok = [&](int g) { return nq > 1 ? (int)((unsigned)(r0 + g) / (unsigned)gqa) : 0; };
  auto row_of = [&](int b, int g) {
    const int tok = row_tok(g);
    return (long long)(b * nq + tok) * NH + kvh * gqa + (r0 + g - tok * gqa);
  };
  DecShare<kUnit8, kKeys8> str;
  int at = 0, at_end = 0, sq = 0, first = 0;  // (units; sq: the sequence that holds `at`, first: its first)
  if constexpr (SHARE) {
    str.init(p, append, p.parts, lane);
    const int part = blockIdx.y;
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
    const int b = SHARE ? sq : (int)blockIdx.y;
    // q rows of this group, loaded while the lengths are on their way
    constexpr int RCH = HD / 8, NQI = (16 * RCH + 255) / 256;
    u32x4 qraw[NQI];
#pragma unroll
    for (int u = 0; u < NQI; u++) {
      const int i = min(tid + 256 * u, 16 * RCH - 1), g = i / RCH, c = i % RCH;
      qraw[u] = *(const u32x4*)((const T*)p.q + row_of(b, min(g, hg - 1)) * HDr + (8 * c < HDr ? 8 * c : 0));
    }
    DecSpan sp;
    int start, end;
    float* rec = nullptr;  // record of row 0 (rows rec_step apart); null: the final output
    long long rec_step = HDr + 2;
    if constexpr (SHARE) {
      if (b >= str.base + 64) str.load(p, append, b, lane);
      sp = str.span(b);
      const int units = dec_units<kUnit8>(sp), stop = min(at_end, first + units);
      start = sp.lo + (at - first) * kUnit8;
      end = min(sp.lo + (stop - first) * kUnit8, sp.hi);
      const bool begins = at == first;
      const int part = blockIdx.y;
      if (begins && hgl == 0 && tid == 0) {   // where the combine finds this sequence's records (decode.hip)
        const int n = str.even ? str.items(units) : (int)((unsigned)(first + units - 1) / (unsigned)str.per) - part + 1;
        ((int*)p.scratch)[2 * b] = 2 * part + (str.even ? 0 : 1);
        ((int*)p.scratch)[2 * b + 1] = str.even ? n : -n;
      }
      if (!(begins && stop == first + units))
        rec = p.scratch + dec_meta_floats(p) + ((2ll * part + (begins && !str.even ? 1 : 0)) * X + hgl) * 16 * (HDr + 2);
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
      start = sp.lo + (int)blockIdx.z * chunk;
      end = min(start + chunk, sp.hi);
      if (!(p.flags & kDec8Final)) {
        rec = p.scratch + (long long)blockIdx.z * (HDr + 2);
        rec_step = (long long)p.nsplit * (HDr + 2);   // rows are indexed as in q
      }
      more = false;
    }
    const int ctx = sp.ctx;
    start = __builtin_amdgcn_readfirstlane(start);   // a multiple of 32
    end = __builtin_amdgcn_readfirstlane(end);
    // the first key some row of the call sees: nothing ahead of it is read
    const int klo = __builtin_amdgcn_readfirstlane(max(append ? max(min(dec_lo(p, b, ctx, 0), ctx), 0) : dec_lo(p, b, ctx, 0), start));

    // ---- q rows -> LDS (fp32), rotated; zero columns past the head dim
#pragma unroll
    for (int u = 0; u < NQI; u++) {
      const int i = tid + 256 * u, g = i / RCH, c = i % RCH;
      const bool cok = 8 * c < HDr;
      const V8 v = bitcast<V8>(qraw[u]);
      if (i < 16 * RCH)
#pragma unroll
        for (int e = 0; e < 8; e++) qsh[g][8 * c + e] = g < hg && cok ? (float)v[e] : 0.0f;
    }
    __syncthreads();
    if (p.rotary) {
      const int rdim = p.rotary_dim > 0 ? p.rotary_dim : HDr, half = rdim / 2;
      const int rbase = p.rotary_pos ? p.rotary_pos[b] : ctx;
      for (int i = tid; i < hg * half; i += 256) {
        const int g = i / half, j = i % half, rp = min(max(rbase + row_tok(g), 0), p.c.rotary_rows - 1);
        const float c = p.cos[(long long)rp * half + j], s = p.sin[(long long)rp * half + j];
        const int ia = p.rotary == 1 ? j : 2 * j, ib = p.rotary == 1 ? j + half : 2 * j + 1;
        const float x = qsh[g][ia], y = qsh[g][ib];
        qsh[g][ia] = x * c - y * s;
        qsh[g][ib] = y * c + x * s;
      }
      __syncthreads();
    }
    // Q^T as the B operand: a 16-byte read of a K row holds dims 64m + 16lg .. +15 and feeds steps 2m and 2m + 1,
    // so step 2m + s takes dims 64m + 16lg + 8s + e. A rotated q is carried as hi + lo.
    V8 qb[NDS], ql[NDS];
#pragma unroll
    for (int ds = 0; ds < NDS; ds++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float x = qsh[lh][64 * (ds / 2) + 16 * lg + 8 * (ds % 2) + e];
        const T hi = (T)x;
        qb[ds][e] = hi;
        ql[ds][e] = (T)(x - (float)hi);
      }
    __syncthreads();  // q staging is dead from here on

    f32x4 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; db++) oacc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.0f;
    const float c_log2 = p.scale * kLog2e;
    const int tok = row_tok(min(lh, hg - 1)), qpos = ctx + tok;  // this lane's row (lh)
    const int rlo = max(dec_lo(p, b, ctx, tok), start), rspan = max(min(dec_hi(p, ctx, tok, append), end) - rlo, 0);
    const float slope = (FEAT && p.alibi && lh < hg) ? p.alibi[kvh * gqa + (r0 + lh - tok * gqa)] : 0.0f;
    const cint_ptr bt = cmem(p.table) + (long long)b * (p.max_blocks & p.tmask);
    const int blk0 = b * p.max_blocks, pmask = p.page - 1, subs = 1 << (page_shift - p.gshift);
    const int krow = (int)p.c.k.s, vrow = (int)p.c.v.s;
    const uint8_t* Kc = (const uint8_t*)p.Kc + (long long)kvh * p.c.k.h;
    const uint8_t* Vc = (const uint8_t*)p.Vc + (long long)kvh * p.c.v.h;
    const uint8_t* scales = (lane < 32 ? p.c.k_scale : p.c.v_scale) + (long long)kvh * subs;
    uint8_t* kb = (uint8_t*)raw + wave * L::WAVE;
    uint8_t* vb = kb + kKeys8 * L::STR;
    float* sb = (float*)(vb + kKeys8 * L::STR);

    // Load i of a lane covers chunk f = 64i + lane of the tile: row f / RB, 16 bytes at f % RB, consecutive
    // lanes on whole rows. K's rows go to the slots that make them the rows of the two S products with eight
    // consecutive keys per lane: row 8a + 4h + r to slot 16h + 4a + r.
    const int last = end - 1;
    int koff[NV], voff[NV], lk[NV], lv[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const int f = 64 * i + lane, row = f / RB, ch = f % RB;
      const bool cok = 16 * ch < HDr;
      koff[i] = cok ? (row & 15) * krow + 16 * ch : kBufZero;
      voff[i] = cok ? (row & 15) * vrow + 16 * ch : kBufZero;
      lk[i] = (16 * ((row >> 2) & 1) + 4 * (row >> 3) + (row & 3)) * L::STR + 16 * ch;
      lv[i] = row * L::STR + 16 * ch;
    }
    // pages of the two halves of a chunk, one chunk ahead (raw entries; made pages where the rows are loaded)
    int ent[2], eidx[2];
    auto table = [&](int kc0) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        eidx[h] = min(max(kc0 + 16 * h, klo), last) >> page_shift;
        ent[h] = bt[eidx[h] & p.tmask];
      }
    };
    u32x4 kreg[NV], vreg[NV];
    unsigned sreg = 0;
    auto load = [&](int kc0, bool front) {
      __amdgpu_buffer_rsrc_t kr[2], vr[2];
      unsigned blk[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int raw_e = (ent[h] & p.tmask) | ((blk0 + eidx[h]) & ~p.tmask);
        blk[h] = __builtin_amdgcn_readfirstlane((int)min((unsigned)raw_e, (unsigned)p.c.num_blocks - 1));
        const int k0 = kc0 + 16 * h, rows = __builtin_amdgcn_readfirstlane(max(min(end - k0, 16), 0)), in = k0 & pmask;
        kr[h] = buf_rsrc32(Kc + (long long)blk[h] * p.c.k.b + (long long)in * krow, (unsigned)(rows * krow));
        vr[h] = buf_rsrc32(Vc + (long long)blk[h] * p.c.v.b + (long long)in * vrow, (unsigned)(rows * vrow));
      }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const int f = 64 * i + lane, row = f / RB;
        // (rows ahead of klo in a run's first chunk: zeros too)
        const bool hide = front && kc0 + row < klo;
        const int ko = hide ? kBufZero : koff[i], vo = hide ? kBufZero : voff[i];
        constexpr int kLo = 16 * RB;   // chunks of the first half
        if (64 * i + 63 < kLo) {
          kreg[i] = buf_load16_nt(kr[0], ko);
          vreg[i] = buf_load16_nt(vr[0], vo);
        } else if (64 * i >= kLo) {
          kreg[i] = buf_load16_nt(kr[1], ko);
          vreg[i] = buf_load16_nt(vr[1], vo);
        } else {   // rows of both halves (head dims over 64 with an odd chunk count): each lane from its own
          const u32x4 ka = buf_load16_nt(kr[0], f < kLo ? ko : kBufZero), kc = buf_load16_nt(kr[1], f < kLo ? kBufZero : ko);
          const u32x4 va = buf_load16_nt(vr[0], f < kLo ? vo : kBufZero), vc = buf_load16_nt(vr[1], f < kLo ? kBufZero : vo);
          kreg[i] = ka | kc;
          vreg[i] = va | vc;
        }
      }
      // scale of key kc0 + (lane & 31): K's for the first 32 lanes, V's for the others
      const int key = kc0 + (lane & 31);
      const unsigned pg = (lane & 16) ? blk[1] : blk[0];
      sreg = scales[(long long)pg * NKV * subs + ((key & pmask) >> p.gshift)];
    };

    const int kfirst = start + kKeys8 * wave;
    if (kfirst < end) {
      table(kfirst);
      load(kfirst, true);
      table(kfirst + kUnit8);
    }
    for (int kc0 = kfirst; kc0 < end; kc0 += kUnit8) {
      // codes and scales -> this wave's own LDS (its operations complete in order: no barrier). A scale of a key
      // that is not there is no number to multiply zeros by.
      const int skey = kc0 + (lane & 31);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        *(u32x4*)(kb + lk[i]) = kreg[i];
        *(u32x4*)(vb + lv[i]) = vreg[i];
      }
      sb[lane] = skey >= klo && skey < end ? e8_f32(sreg) : 0.0f;
      if (kc0 + kUnit8 < end) {   // the next chunk's rows are in flight during this chunk's products
        load(kc0 + kUnit8, false);
        table(kc0 + 2 * kUnit8);
      }
      // S^T = K . Q^T of the keys in slots 0..15 and 16..31: lane (lg, lh) gets keys kc0 + 8lg + 4h + r of row lh
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int m = 0; m < NDS / 2; m++) {
          const u32x4 c = *(const u32x4*)(kb + (16 * h + lh) * L::STR + 64 * m + 16 * lg);
          const V8 a0 = codes_to<T>(u32x2{c[0], c[1]}, 1.0f), a1 = codes_to<T>(u32x2{c[2], c[3]}, 1.0f);
          s[h] = Dt<T>::mma16(a0, qb[2 * m], s[h]);
          s[h] = Dt<T>::mma16(a1, qb[2 * m + 1], s[h]);
          if (p.rotary) {
            s[h] = Dt<T>::mma16(a0, ql[2 * m], s[h]);
            s[h] = Dt<T>::mma16(a1, ql[2 * m + 1], s[h]);
          }
        }
      }
      // logits (log2 domain) and masking
      float t[8], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int key = kc0 + 8 * lg + e;
        const float ks = sb[8 * lg + e];
        float x = s[e >> 2][e & 3];
        if (FEAT) {
          x = x * ks * p.scale;
          if (p.softcap > 0.0f) x = p.softcap * tanh_exp(x / p.softcap);
          x += slope * (float)(key - qpos);
          x *= kLog2e;
        } else {
          x = x * ks * c_log2;
        }
        t[e] = (unsigned)(key - rlo) < (unsigned)rspan ? x : -INFINITY;
        mx = fmaxf(mx, t[e]);
      }
      mx = half_max(lane16_max(mx));
      const float m_new = fmaxf(m_run, mx);
      const float m_use = m_new == -INFINITY ? 0.0f : m_new;
      const float corr = exp2_fast(m_run - m_use);
      float rs = 0.0f;
      bf16x8 pb, pl;     // P^T times V's scales, the B operand: keys 8lg + e, row lh
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float w = exp2_fast(t[e] - m_use), z = w * sb[32 + 8 * lg + e];
        rs += w;
        pb[e] = (__bf16)z;
        if constexpr (kTwoP) pl[e] = (__bf16)(z - (float)pb[e]);
      }
      l_run = l_run * corr + rs;
      m_run = m_new;
#pragma unroll
      for (int db = 0; db < NDB; db++) oacc[db] *= corr;
      // O^T += V^T . P^T: lane lh of group lg addresses row 8lg + lh/2, column 16db + 8(lh%2), and receives
      // column 16db + lh of rows 8lg .. 8lg+7
#pragma unroll
      for (int db = 0; db < NDB; db++) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        const uint8_t* a = vb + (8 * lg + (lh >> 1)) * L::STR + 16 * db + 8 * (lh & 1);
        const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)((__attribute__((address_space(3))) uint8_t*)a));
        const bf16x8 av = codes_to<__bf16>(u32x2{(unsigned)c[0], (unsigned)c[1]}, 1.0f);
        oacc[db] = Dt<__bf16>::mma16(av, pb, oacc[db]);
        if constexpr (kTwoP) oacc[db] = Dt<__bf16>::mma16(av, pl, oacc[db]);
      }
    }

    // ---- merge the four waves: per row max, sum and O^T accumulators through LDS
    const float l_grp = half_sum(lane16_sum(l_run));
    __syncthreads();
    float* red_o = (float*)raw;  // [wave][16 rows][HD]
    if (lg == 0) {
      red_m[wave][lh] = m_run;
      red_l[wave][lh] = l_grp;
    }
#pragma unroll
    for (int db = 0; db < NDB; db++) *(f32x4*)(red_o + (wave * 16 + lh) * HD + 16 * db + 4 * lg) = oacc[db];
    __syncthreads();
    for (int i = tid; i < hg * HDr; i += 256) {
      const int g = i / HDr, d = i % HDr;
      float gm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kDecWaves; w++) gm = fmaxf(gm, red_m[w][g]);
      float l = 0.0f, acc = 0.0f;
      if (gm != -INFINITY) {
#pragma unroll
        for (int w = 0; w < kDecWaves; w++) {
          const float f = exp2_fast(red_m[w][g] - gm);
          l += f * red_l[w][g];
          acc += f * red_o[(w * 16 + g) * HD + d];
        }
      }
      const long long row = row_of(b, g);
      if (!rec) {
        const bool ok = gm != -INFINITY && l > 0.0f;
        ((T*)p.o)[row * HDr + d] = (T)(ok ? acc / l : 0.0f);
        if (p.lse_out && d == 0) p.lse_out[row] = ok ? gm * kLn2 + __logf(l) : -INFINITY;
        continue;
      }
      float* out = rec + (SHARE ? g : row) * rec_step;
      if (d == 0) {
        out[0] = gm;
        out[1] = l;
      }
      out[2 + d] = acc;
    }
    if (more) __syncthreads();  // the merge has read the LDS regions before the next segment fills them
  }
}

template <typename T, int HD>
static int launch_dec8(const FableDecParams& p, const FableCache8& c, int parts, hipStream_t st, bool append) {
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
  const unsigned X = (unsigned)(a.nkv * a.ngrp);
  const dim3 grid = parts > 0 ? dim3(X, (unsigned)dec_share_wgs(p, kUnit8)) : dim3(X, (unsigned)p.batch, (unsigned)p.nsplit);
  auto go = [&](auto ft, auto sh) {
    hipLaunchKernelGGL((dec8_partial_kernel<T, HD, decltype(ft)::value, decltype(sh)::value>), grid, dim3(256), 0, st, a);
  };
  using Y = std::integral_constant<bool, true>;
  using N = std::integral_constant<bool, false>;
  if (parts > 0)
    feat ? go(Y{}, Y{}) : go(N{}, Y{});
  else
    feat ? go(Y{}, N{}) : go(N{}, N{});
  return launch_status("fable_attn_dec8 (partial)");
}
// kernel widths 64, 128, 192 and 256 (a row of codes is read in 64-byte steps); a head dim below its width runs with zero columns
template <typename T>
static int dec8_dispatch(const FableDecParams& p, const FableCache8& c, int parts, hipStream_t st, bool append) {
  if (p.HD <= 64) return launch_dec8<T, 64>(p, c, parts, st, append);
  if (p.HD <= 128) return launch_dec8<T, 128>(p, c, parts, st, append);
  if (p.HD <= 192) return launch_dec8<T, 192>(p, c, parts, st, append);
  return launch_dec8<T, 256>(p, c, parts, st, append);
}

// ------------------------------------------------------------------ which path a call takes
// Many new tokens run on the tile kernel of the forward (FwdPaged8), from kTileRows rows of a K/V head on
// where there are more than kTileStreams (sequence, K/V head, 16 rows): the rule of the 16-bit decode.
constexpr int kTileRows8 = 64, kTileStreams8 = 16;
static bool dec8_uses_tiles(const FableDecParams& p, const FableCache8& c) {
  return c.k.b <= 0x7FFFFFFF && c.v.b <= 0x7FFFFFFF && (long long)p.batch * (p.NH / p.gqa) * dec_groups(p) > kTileStreams8 && (long long)p.nq * p.gqa >= kTileRows8 &&
         (long long)p.batch * p.max_blocks <= 0x7FFFFFFF && p.max_blocks < (1 << 29) && p.window != 0;
}
// Shares worked out on the device for batches that equal splits would not spread evenly, as in decode.hip
constexpr long long kShareBytes8 = 64LL << 20;
static bool dec8_shares(const FableDecParams& p) {
  if (p.nsplit > 0 || p.batch < 2) return false;
  if ((long long)p.batch * p.max_blocks * p.page * (p.NH / p.gqa) * p.HD * 2 < kShareBytes8) return false;
  const int parts = dec_parts(p, kUnit8);
  return p.batch > parts || parts % p.batch != 0;
}
static int dec8_fixed_splits(const FableDecParams& p) {
  return fa_decode_num_splits(p.batch, dec_groups(p), p.NH / p.gqa, 1, (int64_t)p.max_blocks * p.page, p.nsplit);
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
  f.sK = fa_strides{0, c.k.h, c.k.s};
  f.sV = fa_strides{0, c.v.h, c.v.s};
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
                           __builtin_ctz((unsigned)p.page), c.k.b, c.v.b, p.ctx_len, append ? 1 : 0, p.leftpad, nullptr, p.NH};
  fwd_paged8_scales(pg, c, p.page);
}

// the argument checks of the two entry points (nq below 1 becomes 1)
static int dec8_check(FableDecParams& p, const FableCache8& c, int dtype) {
  const char* what = "fable_attn_dec8";
  if (dtype != FA_F16 && dtype != FA_BF16) return fail(FA_ERR_DTYPE, "%s: dtype %d not implemented (fp16/bf16)", what, dtype);
  if (p.NH <= 0 || p.gqa <= 0 || p.NH % p.gqa) return fail(FA_ERR_ARG, "%s: NH=%d gqa=%d", what, p.NH, p.gqa);
  if (p.nq < 1) p.nq = 1;
  if (p.nsplit < 0 || p.nsplit > 512) return fail(FA_ERR_ARG, "%s: nsplit=%d", what, p.nsplit);
  if (p.max_blocks < 1 || (long long)p.max_blocks * p.page > 0x7FFFFFFF)
    return fail(FA_ERR_ARG, "%s: max_blocks=%d page=%d", what, p.max_blocks, p.page);
  if (p.batch > 65535 || (long long)p.nq * p.gqa > (1 << 24)) return fail(FA_ERR_ARG, "%s: batch=%d nq=%d", what, p.batch, p.nq);
  if (p.rotary && (p.rotary_dim < 0 || p.rotary_dim > p.HD || p.rotary_dim % 2)) return fail(FA_ERR_ARG, "%s: rotary_dim=%d", what, p.rotary_dim);
  if (p.rotary && (p.rotary > 2 || c.rotary_rows < 1)) return fail(FA_ERR_ARG, "%s: rotary=%d rotary_rows=%d", what, p.rotary, c.rotary_rows);
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
  if (dec8_shares(p)) return dec_share_bytes(p, kUnit8);
  p.nsplit = dec8_fixed_splits(p);
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
    a.kc = c.k;
    a.vc = c.v;
    a.block_table = p.block_table;
    a.ctx_len = p.ctx_len;
    a.leftpad = p.leftpad;
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
  const bool share = dec8_shares(p);
  const int parts = share ? dec_parts(p, kUnit8) : 0;
  p.nsplit = share ? 0 : dec8_fixed_splits(p);
  const int rc = dtype == FA_F16 ? dec8_dispatch<_Float16>(p, c, parts, st, new_k != nullptr) : dec8_dispatch<__bf16>(p, c, parts, st, new_k != nullptr);
  if (rc != FA_OK || (!share && p.nsplit == 1)) return rc;
  return dec_combine(p, dtype, st, share);
}
