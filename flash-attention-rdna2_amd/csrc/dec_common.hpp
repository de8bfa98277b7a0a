// dec_common.hpp — what the decode kernels over 16-bit (decode.hip) and 8-bit caches (decode8.hip)
// share: the key span of a sequence, the shares of a call worked out on the device, the row groups and
// the sizes of the partial records.
#pragma once
#include "attn_device.hpp"

namespace fa {

constexpr int kDecWaves = 4;

__device__ __forceinline__ float xor16_max(float x) {
  return fmaxf(x, __shfl_xor(x, 16));
}
__device__ __forceinline__ float xor16_sum(float x) { return x + __shfl_xor(x, 16); }

// The maximum that a wave hands on of a row whose weights sum to l. A score that is no number (of a query or key with
// a NaN, or of infinities) drops out of the running maximum but not out of l, which is then no number either. Such a
// row goes on with a maximum of +inf: every merge gives it the weight 2^(inf - inf), so its output and LSE are NaN,
// whatever the row's other waves and splits saw. (Its running maximum may still be -inf, that of a row without keys.)
__device__ __forceinline__ float dec_row_max(float m, float l) { return l == l ? m : INFINITY; }

// Rows of a (sequence, K/V head): its nq new tokens x the gqa q heads of its group, token first;
// workgroups take them in groups of 16. The keys of a sequence some row sees are [lo, hi); row
// masks cut them down (a row of token tk sees [max(leftpad, pos - window + 1), ctx + (append ? tk +
// 1 : 0))). With `append` the span reaches down to ctx, so that it holds every new key.
struct DecSpan {
  int ctx, lo, hi;
};
// The lengths and tables are read as constant memory, which no kernel here writes: uniform entries
// then come by scalar loads (the kernels' own stores otherwise turn them into vector loads, whose
// in-order counter they would share with the row loads: C4 311 -> 319 us).
typedef const __attribute__((address_space(4))) int* cint_ptr;
__device__ __forceinline__ cint_ptr cmem(const int* p) { return (cint_ptr)(uintptr_t)p; }
__device__ __forceinline__ int dec_room(const FableDecParams& p) {
  return (int)min((long long)p.max_blocks * p.page, 0x7FFFFFFFLL);
}
__device__ __forceinline__ int dec_lo(const FableDecParams& p, int b, int ctx, int tk) {
  int lo = p.leftpad ? cmem(p.leftpad)[b] : 0;
  if (p.window >= 0) lo = max(lo, ctx + tk - p.window + 1);
  return max(lo, 0);
}
__device__ __forceinline__ int dec_hi(const FableDecParams& p, int ctx, int tk, int append) {
  return min(ctx + (append ? tk + 1 : 0), dec_room(p));
}
__device__ __forceinline__ DecSpan dec_span(const FableDecParams& p, int b, int append) {
  DecSpan r;
  r.ctx = cmem(p.ctx_len)[b];
  r.lo = dec_lo(p, b, r.ctx, 0);
  if (append) r.lo = max(min(r.lo, r.ctx), 0);
  r.hi = dec_hi(p, r.ctx, p.nq - 1, append);
  return r;
}

// How a call's keys are shared out when the caller sets no split count (p.nsplit 0). The lengths
// stay on the device, so every workgroup works out the shares by itself, from units of UNIT keys (a
// sequence has one at least):
//  * even: `parts` workgroups per (K/V head, row group); each sequence is cut into runs of `per`
//    units, `per` the least for which the runs fit the parts, so every workgroup has one run at
//    most. Taken where that is at most a quarter above an even share (few or alike sequences), or
//    kSegUnits units: a stream's workgroup pays a second segment, which costs about as much.
//  * stream: otherwise (many sequences of unequal lengths) the sequences' units follow one another
//    and each workgroup (two per part when there are more sequences than parts) takes as many, whatever sequences they belong to.
// A sequence that lies in one workgroup is finished there; of the others each writes a partial record
// (a stream's workgroup one for a sequence it goes on with, slot 0, and one for a sequence that goes
// on after it, slot 1). Two equal splits per sequence, the host's choice before, left 48 requests of 64
// to 8192 keys (Hq 64 / Hk 8, D 128) waiting for the longest: 142 us, 125 as a stream.
template <int UNIT>
__device__ __forceinline__ int dec_units(const DecSpan& r) { return max((r.hi - r.lo + UNIT - 1) / UNIT, 1); }
// inclusive prefix sum over the wave (row shifts within 16 lanes, then two broadcasts)
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
// Every wave for itself: lane l holds the span of sequence base + l, read from memory once for
// batches of up to 64 sequences (a chain of dependent loads ahead of the first row load is what a
// short segment takes longest for).
// (ALIGN: the first key of a sequence is taken down to a multiple of it)
template <int UNIT, int ALIGN = 1>
struct DecShare {
  DecSpan mine;
  int units;        // of sequence base + lane; 0 past the batch
  int base;
  int total, per;   // units of the call, units per run (even) or workgroup (stream)
  bool even;
  __device__ __forceinline__ void load(const FableDecParams& p, int append, int b0, int lane) {
    base = b0;
    mine = DecSpan{0, 0, 0};
    units = 0;
    if (b0 + lane < p.batch) {
      mine = dec_span(p, b0 + lane, append);
      mine.lo &= -ALIGN;
      units = dec_units<UNIT>(mine);
    }
  }
  // sum over the batch of f(units); sequence 0's lanes are loaded afterwards
  template <typename F>
  __device__ __forceinline__ int sum(const FableDecParams& p, int append, int lane, F&& f) {
    int t = 0;
#pragma nounroll
    for (int b0 = (p.batch - 1) & ~63; b0 >= 0; b0 -= 64) {
      if (b0 != base) load(p, append, b0, lane);
      t += wave_sum(f(units));
    }
    return t;
  }
  __device__ __forceinline__ void init(const FableDecParams& p, int append, int parts, int lane) {
    load(p, append, 0, lane);
    total = sum(p, append, lane, [](int u) { return u; });
    const int least = max((int)((unsigned)(total + parts - 1) / (unsigned)parts), 1);
    even = false;
    if (p.batch <= parts) {
#pragma nounroll
      for (per = least; 4 * per <= 5 * least || per <= least + kSegUnits; per += max(per >> 4, 1)) {
        if (sum(p, append, lane, [=](int u) { return (int)((unsigned)(u + per - 1) / (unsigned)per); }) <= parts) {
          even = true;
          break;
        }
      }
    }
    if (!even) per = p.batch <= parts ? least : (least + 1) / 2;
  }
  // items: runs (even) or units (stream) of a sequence
  __device__ __forceinline__ int items(int u) const { return even ? (int)((unsigned)(u + per - 1) / (unsigned)per) : u; }
  __device__ __forceinline__ DecSpan span(int b) const {
    const int l = b - base;
    return DecSpan{__builtin_amdgcn_readlane(mine.ctx, l), __builtin_amdgcn_readlane(mine.lo, l), __builtin_amdgcn_readlane(mine.hi, l)};
  }
  // the sequence that holds item `at`, and its first item (p.batch: no such item); after init
  __device__ __forceinline__ int seek(const FableDecParams& p, int append, int at, int lane, int& first) {
    first = 0;
#pragma nounroll
    for (;;) {
      const int inc = wave_scan(items(units)), sum = __builtin_amdgcn_readlane(inc, 63);
      if (at >= first + sum) {
        first += sum;
        if (base + 64 >= p.batch) return p.batch;
        load(p, append, base + 64, lane);
        continue;
      }
      const int n = __popcll(__builtin_amdgcn_ballot_w64(first + inc <= at));   // sequences that end before `at`
      if (n > 0) first += __builtin_amdgcn_readlane(inc, n - 1);
      return base + n;
    }
  }
  // (at least 4 units per run and streams from a quarter above the even share on: 24 sequences of 500 keys, Hq 32 /
  // Hk 8, D 128, 21.3 us, 19.0 now; 3 of 500 13.7 and 11.6; 5 of 300 14.1 and 11.2)
  static constexpr int kSegUnits = 6;
};

// the kernel's argument (of type A, whole) read again from the kernel argument segment
template <class A>
__device__ __forceinline__ A dec_reload() {
  auto k = (const __attribute__((address_space(4))) uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  struct {
    uint64_t w[sizeof(A) / 8];
  } raw;
  static_assert(sizeof(raw) == sizeof(A), "whole words");
#pragma unroll
  for (int i = 0; i < (int)(sizeof(A) / 8); i++) raw.w[i] = k[i];
  return __builtin_bit_cast(A, raw);
}

// floats ahead of the records: two ints per sequence, for the combine
__host__ __device__ inline long long dec_meta_floats(const FableDecParams& p) { return (2ll * p.batch + 63) / 64 * 64; }

// row groups of 16 per (sequence, K/V head)
inline int dec_groups(const FableDecParams& p) { return (int)(((long long)p.nq * p.gqa + 15) / 16); }

// Parts of a call (DecShare): one workgroup per CU (more in flight per CU read a batch of alike
// sequences slower: C4 0.96x with two, 0.86x with three), or two where the (K/V head, row group) count
// leaves more than an eighth of the CUs out of a round of one.
inline int dec_parts(const FableDecParams& p, int unit, int wh = 1) {   // (wh: K/V heads of a workgroup)
  const long long X = (long long)(p.NH / p.gqa / wh) * dec_groups(p);
  long long parts = 256 / X;
  if (parts * X < 224) parts = (512 + X - 1) / X;
  const long long units = (long long)p.batch * (((long long)p.max_blocks * p.page + unit - 1) / unit + 1);
  parts = parts < units ? parts : units;
  return parts > 1 ? (int)parts : 1;
}
// workgroups per (K/V head, row group) (DecShare::init)
inline int dec_share_wgs(const FableDecParams& p, int unit, int wh = 1) {
  const int parts = dec_parts(p, unit, wh);
  return p.batch <= parts ? parts : 2 * parts;
}
// scratch: two records of 16 rows per workgroup
inline long long dec_share_bytes(const FableDecParams& p, int unit, int wh = 1) {
  return (dec_meta_floats(p) + (long long)dec_share_wgs(p, unit, wh) * 2 * (p.NH / p.gqa) * dec_groups(p) * 16 * (p.HD + 2)) * 4;
}

// merge of the partials in p.scratch into p.o and p.lse_out (fp16/bf16; decode.hip): of p.nsplit splits per
// row, or with `share` of a call whose shares were worked out on the device
int dec_combine(const FableDecParams& p, int dtype, hipStream_t st, bool share);

}  // namespace fa
