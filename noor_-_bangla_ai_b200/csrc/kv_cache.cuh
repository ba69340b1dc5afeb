// kv_cache.cuh -- the paged 8-bit cache: writing new tokens and reading back.
//
// A block (the `block` tokens of one page and one kv head) of k or of v has
// one scale s, a power of two; a value x is held as code = round(x / s), ties
// to even, int8 (|code| <= 127) or e4m3 (<= 448).  s is the smallest power of
// two (>= 2^-126) with max|x| <= Q s.  A power of two makes x / s exact, so a
// code depends on x alone and not on how a quotient rounds, and when a later
// token needs a larger scale the old codes are rounded again from
// code * (s_old / s), exact too.  It costs int8 up to one of its bits against
// max|x| / 127; e4m3 loses nothing.
#pragma once

#include <cuda_fp8.h>
#include "common.cuh"
#include "noor_moe.h"
#include "rope.cuh"

#include <type_traits>

namespace noor {
namespace kv {

enum Format : int { INT8 = 0, E4M3 = 1 };

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int32_t* status;
  int64_t P;
  int32_t H, D, blk;
};

struct Batch {
  const int32_t* table;
  int64_t tstride;
  const int32_t* lens;
  const int32_t* cu;
  int64_t N;
  int32_t B, maxb;
};

__device__ __forceinline__ void flag(int32_t* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

struct Seq {
  int32_t row0, n, len;  // first row, rows, tokens
};

// Sequence b's rows and length (no lengths given: all that its pages hold),
// checked: a sequence whose metadata is wrong has no rows (and sets the
// status word).
__device__ __forceinline__ Seq sequence(const Batch& b, const int32_t* cu, const int32_t* lens, int blk, int i,
                                        int32_t* status) {
  Seq s;
  s.row0 = __ldg(cu + i);
  const int32_t end = __ldg(cu + i + 1);
  s.len = lens != nullptr ? __ldg(lens + i) : b.maxb * blk;
  s.n = end - s.row0;
  if (s.row0 < 0 || end < s.row0 || (int64_t)end > b.N) {
    flag(status, NOOR_KV_BAD_ROWS);
    s.n = 0;
    s.row0 = 0;
  }
  if (s.len < 0 || (int64_t)s.len > (int64_t)b.maxb * blk) {
    flag(status, NOOR_KV_BAD_LENGTH);
    s.n = 0;
    s.len = 0;
  }
  return s;
}

// One block of a sequence that a call touches.
struct Task {
  int32_t b;          // sequence, -1: none
  int32_t j;          // block of the sequence
  int32_t row0;       // row of the first token in [first, first + n)
  int32_t first, n;   // tokens of the call in this block: slots first .. first + n - 1
  int64_t page;
};

// The t-th touched block in batch order, found by the whole block of THREADS
// threads, a sequence for each at a time: each sequence touches the blocks of
// its tokens [pos0, pos0 + n).  starts: pos0 of each sequence (reading), or
// NULL for the last n tokens (writing).  All threads call it and get it.
template <int THREADS>
__device__ __forceinline__ Task find_task(const Cache& c, const Batch& b, const int32_t* starts, bool write, int32_t t) {
  __shared__ Task s_task;
  __shared__ int32_t s_warp[THREADS / 32];
  const int blk = c.blk, lblk = 31 - __clz(blk), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s_task.b = -1;
  int32_t before = 0;  // touched blocks of earlier sequences
  for (int base = 0; base < b.B; base += THREADS) {
    const int i = base + threadIdx.x;
    int32_t pos0 = 0, touched = 0;
    Seq s{0, 0, 0};
    if (i < b.B) {
      s = sequence(b, b.cu, b.lens, blk, i, c.status);
      pos0 = write ? s.len - s.n : (starts ? __ldg(starts + i) : 0);
      if (s.n > 0 && (pos0 < 0 || pos0 > s.len - s.n)) {
        flag(c.status, NOOR_KV_BAD_LENGTH);
        s.n = 0;
      }
      if (s.n > 0) touched = ((pos0 + s.n - 1) >> lblk) - (pos0 >> lblk) + 1;
    }
    int32_t incl = touched;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int32_t mine = before, total = before;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) mine += s_warp[w];
      total += s_warp[w];
    }
    const int32_t local = t - (mine + incl - touched);  // which of this sequence's blocks
    if (local >= 0 && local < touched) {
      Task k;
      k.b = i;
      k.j = (pos0 >> lblk) + local;
      const int32_t lo = max(pos0, k.j << lblk), hi = min(pos0 + s.n, (k.j + 1) << lblk);
      k.first = lo - (k.j << lblk);
      k.n = hi - lo;
      k.row0 = s.row0 + (lo - pos0);
      const int32_t page = __ldg(b.table + (int64_t)k.b * b.tstride + k.j);
      k.page = page;
      if (page < 0 || (int64_t)page >= c.P) {
        flag(c.status, NOOR_KV_BAD_PAGE);
        k.page = -1;
      }
      s_task = k;
    }
    before = total;
    __syncthreads();
    if (t < before) break;
  }
  return s_task;
}

// ------------------------------------------------------------- codes

template <int FMT>
struct Code;
template <>
struct Code<INT8> {
  // exponent of the smallest power of two that holds amax (a finite f32, as bits)
  static constexpr int kExp = 6;                  // 127 = 1.984375 * 2^6
  static constexpr uint32_t kMant = 0x7E0000u;    // mantissa bits of 1.984375
  __device__ static float value(uint8_t c) { return (float)(int8_t)c; }
};
template <>
struct Code<E4M3> {
  static constexpr int kExp = 8;                  // 448 = 1.75 * 2^8
  static constexpr uint32_t kMant = 0x600000u;
  __device__ static float value(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
  }
};

// Smallest power of two s >= 2^-126 with amax <= Q s, from amax's bits; NaN
// if amax is not finite.
template <int FMT>
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  int e = (int)(amax_bits >> 23) - 127 - Code<FMT>::kExp;
  if ((amax_bits & 0x7FFFFFu) > Code<FMT>::kMant) ++e;
  e = max(e, -126);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// A scale as readers take it: one that the write cannot have left (negative,
// not finite, or above 2^126, beyond which its reciprocal is no normal float)
// reads as NaN, so that it reaches the rows that see its block and no others.
constexpr float kMostScale = 8.5070592e37f;
__device__ __forceinline__ float read_scale(float s) {
  return s >= 0.f && s <= kMostScale ? s : __uint_as_float(0x7FC00000u);
}

// A readable scale (or the largest of some) up to a power of two, and a power
// of two's reciprocal; zero counts as 2^-126 or, reciprocally, 2^127.
__device__ __forceinline__ float power_up(float s) {
  return __uint_as_float(max((__float_as_uint(s) + 0x7FFFFFu) & 0x7F800000u, 0x800000u));
}
__device__ __forceinline__ float power_inverse(float p) { return __uint_as_float(0x7F000000u - __float_as_uint(p)); }

// The scale of a block that held tokens at s_old and now needs s_new: the
// larger, as a power of two; NaN stays.  (A poisoned block's codes are stored
// as zeros: a reader's zero weight times any stored code is zero.)
__device__ __forceinline__ float grown_scale(float s_old, float s_new) {
  if (s_old == 0.f) return s_new;
  if (!(s_old > 0.f && s_old <= kMostScale) || s_new != s_new) return __uint_as_float(0x7FC00000u);
  uint32_t b = __float_as_uint(s_old);
  if (b & 0x7FFFFFu) b = (b & 0x7F800000u) + 0x800000u;  // a scale not written here: up to a power of two
  return fmaxf(__uint_as_float(b), s_new);
}

constexpr int kAppendThreads = 256;

struct AppendArgs {
  Cache c;
  Batch b;
  rope::View k, v;
  rope::Args r;       // k's rotation; q and q_out for the q part
  int32_t heads;      // kv heads of one grid block
  int32_t kv_blocks;  // grid blocks that write the cache: task major, then k or v, then head group (the rest rotate q)
  int32_t q_tok;      // rows of q per block
  bool kvec, vvec;    // k / v can be read four elements at a time
  bool qvec;          // q can be rotated 16 bytes at a time
};

constexpr int kHeadsAtOnce = 64;  // 256 threads over the 4 that a head of 16 dims takes

// Largest magnitudes (as bits) of the heads that a grid block works on at
// once, in three alternating rows: while one is read, the next is cleared.
struct Maxima {
  uint32_t m[3][kHeadsAtOnce];
};

// Every thread's v joins its head's maximum; returns the head's.  `pass`
// counts the calls.  All threads of the block call it.
__device__ __forceinline__ uint32_t head_max(uint32_t v, int hl, Maxima& s, int pass) {
  uint32_t* m = s.m[pass % 3];
  const int first = __shfl_sync(0xffffffffu, hl, 0);
  if (__all_sync(0xffffffffu, hl == first)) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0 && hl < kHeadsAtOnce) atomicMax(m + hl, v);
  } else if (hl < kHeadsAtOnce) {
    atomicMax(m + hl, v);
  }
  if (threadIdx.x < kHeadsAtOnce) s.m[(pass + 1) % 3][threadIdx.x] = 0;
  __syncthreads();
  return hl < kHeadsAtOnce ? m[hl] : 0;
}

// Four elements as they are stored.
template <typename T>
using Raw4 = typename std::conditional<sizeof(T) == 2, uint2, float4>::type;
__device__ __forceinline__ float4 two_runs(const float* p, const float* q) {
  const float2 u = *reinterpret_cast<const float2*>(p), v = *reinterpret_cast<const float2*>(q);
  return make_float4(u.x, u.y, v.x, v.y);
}
__device__ __forceinline__ uint2 two_runs(const bf16* p, const bf16* q) {
  return make_uint2(*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(q));
}
__device__ __forceinline__ float4 four(float a, float b, float c, float d) { return make_float4(a, b, c, d); }
__device__ __forceinline__ uint2 four(bf16 a, bf16 b, bf16 c, bf16 d) {
  return make_uint2(__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16,
                    __bfloat16_as_ushort(c) | (uint32_t)__bfloat16_as_ushort(d) << 16);
}
// As floats; `turned`: runs (0, 2) and (1, 3) were loaded and the pairs are (0, 1), (2, 3).
__device__ __forceinline__ float4 widen4(float4 r, bool turned) { return turned ? make_float4(r.x, r.z, r.y, r.w) : r; }
__device__ __forceinline__ float4 widen4(uint2 r, bool turned) {
  return widen4(make_float4(bf16_lo(r.x), bf16_hi(r.x), bf16_lo(r.y), bf16_hi(r.y)), turned);
}

// Codes of two values in steps, x in the low byte.
template <int FMT>
__device__ __forceinline__ uint32_t codes2(float x, float y) {
  if constexpr (FMT == INT8) {
    // 1.5 2^23 + x rounds x to an integer, ties to even; |x| <= 127 by the
    // scale's choice
    return (__float_as_uint(x + 12582912.f) & 0xFFu) | ((__float_as_uint(y + 12582912.f) & 0xFFu) << 8);
  } else {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
    return r;
  }
}
// A block's old codes, four of a word, rounded again under a grown scale.
template <int FMT>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  const float a = Code<FMT>::value(w & 0xFF), b = Code<FMT>::value((w >> 8) & 0xFF), c = Code<FMT>::value((w >> 16) & 0xFF),
              d = Code<FMT>::value(w >> 24);
  return codes2<FMT>(a * ratio, b * ratio) | (codes2<FMT>(c * ratio, d * ratio) << 16);
}

// Larger magnitude, NaN if either is.
__device__ __forceinline__ float max_abs(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}

// f64 values rounded to f32 such that rounding those to codes gives what
// rounding the values would: where the nearest f32 could be a border of a code
// or of a scale (they have at most 9 significant bits) and the value is not it,
// the neighbour on the value's side.  Powers of two scale both alike, so this
// can come before the scale is known.
__device__ __forceinline__ float toward(double x, float h) {
  const double r = x - (double)h;
  if ((__float_as_uint(h) & 0x7FFFu) != 0 || r == 0.0 || !(fabsf(h) <= 3.4028235e38f)) return h;
  if (h == 0.f) return r > 0.0 ? 1e-45f : -1e-45f;
  return __uint_as_float(__float_as_uint(h) + ((r > 0.0) == (h > 0.0) ? 1 : -1));
}
__device__ __forceinline__ float4 toward4(const double (&x)[4]) {
  float4 h = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
  const uint32_t low = min(min(__float_as_uint(h.x) & 0x7FFFu, __float_as_uint(h.y) & 0x7FFFu),
                           min(__float_as_uint(h.z) & 0x7FFFu, __float_as_uint(h.w) & 0x7FFFu));
  if (low == 0) {  // one in thousands, but for values that the rotation leaves as they are
    h.x = toward(x[0], h.x);
    h.y = toward(x[1], h.y);
    h.z = toward(x[2], h.z);
    h.w = toward(x[3], h.w);
  }
  return h;
}

// Keys of one touched block, kv heads h0 .. h1 - 1.  A thread owns two pairs of
// a head and every G-th token; a decode step's single token leaves room for
// several heads at once.  Its angle is made once in f64 and advanced from
// token to token by the angle of G positions (a complex product; 16 of them
// lose a few units of 2^-53), so a sine and cosine pair is paid for once per
// thread and not per element.  The rotation is done in f64 and kept as the f32
// that rounds alike, so the codes are those of the exact rotation.
// Bound by memory once enough blocks run: the elements are read once into
// registers.  Measured with the values' and q's launches: 8 ragged prompts of up
// to 4096 tokens, 32 + 8 heads of 128 dims, BF16 to e4m3, 111 us = 3.7 TB/s (half
// of it is q at 6.7 TB/s; the rest waits on f64 products and the block's
// maximum); a decode step of 128 streams 8.6 us, the time of one block's chain
// of loads: its place, its page, the old scale.
template <typename T, int FMT, int TPT>
__device__ void append_keys(const AppendArgs& a, const Task& k, int h0, int h1, Maxima& s_max) {
  const Cache& c = a.c;
  const int D = c.D, blk = c.blk, tid = threadIdx.x, rot = a.r.rot;
  const int quads = D >> 2, G = min(kAppendThreads / quads, k.n), slots = quads * G, at_once = kAppendThreads / slots;
  const int hl = tid / slots, qd = tid % quads, g = tid / quads - hl * G;
  const bool thread_live = hl < at_once;
  // the thread's pairs (x0, x1), (x2, x3) as dims
  const bool half = a.r.layout == rope::HALF;
  auto dim0 = [&](int p) { return half && 2 * p < rot ? p : 2 * p; };
  auto dim1 = [&](int p) { return half && 2 * p < rot ? p + (rot >> 1) : 2 * p + 1; };
  const int d0 = dim0(2 * qd), d1 = dim1(2 * qd), d2 = dim0(2 * qd + 1), d3 = dim1(2 * qd + 1);
  // two runs of two, each on an even element: a half layout with an odd rot / 2
  // starts the second on an odd one, which a two-element access must not touch
  const bool split = d2 == d0 + 1 && d3 == d1 + 1 && (d1 & 1) == 0;
  const bool run = d1 == d0 + 1 && d2 == d0 + 2 && d3 == d0 + 3;    // one run of four
  // first angle and step of both pairs
  double c0[2] = {1.0, 1.0}, s0[2] = {0.0, 0.0}, cg[2] = {1.0, 1.0}, sg[2] = {0.0, 0.0};
  const int32_t pos0 = k.j * blk + k.first;
  bool turned[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int p = 2 * qd + x;
    turned[x] = thread_live && 2 * p < rot;
    if (turned[x]) {
      const float f = __ldg(a.r.inv_freq + p);
      sincospi(2.0 * rope::turn_fraction(pos0 + g, f), &s0[x], &c0[x]);
      c0[x] *= a.r.factor;
      s0[x] *= a.r.factor;
      if (g + G < k.n) sincospi(2.0 * rope::turn_fraction(G, f), &sg[x], &cg[x]);
    }
  }
  Raw4<T> raw[TPT];
  auto load = [&](int hb) {
    const bool live = thread_live && hb + hl < h1;
    const T* p = static_cast<const T*>(a.k.p) + (int64_t)(k.row0 + g) * a.k.st + (hb + hl) * a.k.sh;
    const int64_t step = G * a.k.st;
#pragma unroll
    for (int j = 0; j < TPT; ++j, p += step) {
      if (G * j >= k.n) break;
      const int s = g + G * j;
      raw[j] = Raw4<T>{};
      if (live && s < k.n) {
        if (a.kvec && run)
          raw[j] = *reinterpret_cast<const Raw4<T>*>(p + d0);
        else if (a.kvec && split)
          raw[j] = two_runs(p + d0, p + d1);
        else
          raw[j] = four(p[d0], p[d1], p[d2], p[d3]);
      }
    }
  };
  load(h0);
  for (int hb = h0, pass = 0; hb < h1; hb += at_once, ++pass) {
    const int h = hb + hl;
    const bool live = thread_live && h < h1;
    const int64_t ph = k.page * c.H + (live ? h : hb);
    const float s_old = k.first > 0 ? c.ks[ph] : 0.f;  // (rewritten below: not a read-only load)
    float4 x[TPT];
#pragma unroll
    for (int j = 0; j < TPT; ++j) {
      if (G * j >= k.n) break;
      x[j] = widen4(raw[j], a.kvec && !run && split);
    }
    if (hb + at_once < h1) load(hb + at_once);  // the next heads', while these are worked on
    // ---- rotate; the largest magnitude chooses the scale
    float fmx = 0.f;
    double c1[2] = {c0[0], c0[1]}, s1[2] = {s0[0], s0[1]};
#pragma unroll
    for (int j = 0; j < TPT; ++j) {
      if (G * j >= k.n) break;
      if (turned[0]) {  // (both pairs or, where rot / 2 is odd, the first)
        double y[4];
        const double x0 = x[j].x, x1 = x[j].y, x2 = x[j].z, x3 = x[j].w;
        y[0] = x0 * c1[0] - x1 * s1[0];
        y[1] = x0 * s1[0] + x1 * c1[0];
        y[2] = x2 * c1[1] - x3 * s1[1];
        y[3] = x2 * s1[1] + x3 * c1[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const double cn = c1[e] * cg[e] - s1[e] * sg[e];
          s1[e] = s1[e] * cg[e] + c1[e] * sg[e];
          c1[e] = cn;
        }
        x[j] = toward4(y);
      }
      fmx = max_abs(max_abs(max_abs(max_abs(fmx, x[j].x), x[j].y), x[j].z), x[j].w);
    }
    const uint32_t amax = head_max(__float_as_uint(fmx), live ? hl : kHeadsAtOnce, s_max, pass);
    if (!live) continue;
    const float scale = k.first > 0 ? grown_scale(s_old, scale_for<FMT>(amax)) : scale_for<FMT>(amax);
    const bool poisoned = scale != scale;
    const float inv = 1.f / scale;
    uint8_t* kc = c.k + ph * blk * D;
    // ---- the old codes under a grown scale
    if (k.first > 0 && scale != s_old) {
      const float ratio = poisoned ? 0.f : s_old / scale;
      for (int i = tid - hl * slots; i < k.first * quads; i += slots) {
        uint32_t* w = reinterpret_cast<uint32_t*>(kc) + i;
        *w = poisoned ? 0 : recode4<FMT>(*w, ratio);
      }
    }
    // ---- codes of the new tokens
#pragma unroll
    for (int j = 0; j < TPT; ++j) {
      const int s = g + G * j;
      if (s >= k.n) break;
      uint32_t e = codes2<FMT>(x[j].x * inv, x[j].y * inv), f = codes2<FMT>(x[j].z * inv, x[j].w * inv);
      if (poisoned) e = f = 0;
      uint8_t* o = kc + (k.first + s) * D;
      if (run) {
        *reinterpret_cast<uint32_t*>(o + d0) = e | (f << 16);
      } else if (split) {
        *reinterpret_cast<uint16_t*>(o + d0) = (uint16_t)((e & 0xFF) | ((f & 0xFF) << 8));
        *reinterpret_cast<uint16_t*>(o + d1) = (uint16_t)((e >> 8) | (f & 0xFF00));
      } else {
        o[d0] = (uint8_t)e;
        o[d1] = (uint8_t)(e >> 8);
        o[d2] = (uint8_t)f;
        o[d3] = (uint8_t)(f >> 8);
      }
    }
    if (tid == hl * slots) c.ks[ph] = scale;
  }
}

// Values of one touched block: a thread takes DPT dims of 16 tokens in
// registers, turns the codes over and writes 16 tokens of each dim, the
// cache's order.  Where a 16-token run is not all new it is read, merged and
// written back (this block alone owns the page).  Only runs with new tokens
// take threads; where they leave room, several heads are done at once.
template <typename T, int FMT, int DPT>
__device__ void append_values(const AppendArgs& a, const Task& k, int h0, int h1, Maxima& s_max) {
  const Cache& c = a.c;
  const int D = c.D, blk = c.blk, tid = threadIdx.x, parts = D / DPT;
  const int r0 = k.first >> 4, runs = ((k.first + k.n - 1) >> 4) - r0 + 1;
  const int slots = parts * runs, at_once = kAppendThreads / slots;   // at most 4 x 64
  const int hl = tid / slots, run = (tid - hl * slots) / parts, d = (tid % parts) * DPT, lo = 16 * (r0 + run);
  const bool all_new = lo >= k.first && lo + 16 <= k.first + k.n;
  // 16 tokens of DPT dims as they are stored, in 32-bit words
  constexpr int W = DPT * (int)sizeof(T) / 4;
  uint32_t next[16][W];
  auto load = [&](int hb) {
    const bool live = hl < at_once && hb + hl < h1;
    const int s0 = lo - k.first;
    const T* p = static_cast<const T*>(a.v.p) + ((int64_t)k.row0 + s0) * a.v.st + (hb + hl) * a.v.sh + d;
    if (live && all_new && a.vvec) {
#pragma unroll
      for (int i = 0; i < 16; ++i, p += a.v.st) {
        if constexpr (W == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(p);
          next[i][0] = u.x; next[i][1] = u.y; next[i][2] = u.z; next[i][3] = u.w;
        } else if constexpr (W == 2) {
          const uint2 u = *reinterpret_cast<const uint2*>(p);
          next[i][0] = u.x; next[i][1] = u.y;
        } else {
          next[i][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i, p += a.v.st) {
      const int s = s0 + i;
#pragma unroll
      for (int x = 0; x < W; ++x) next[i][x] = 0;
      if (live && s >= 0 && s < k.n) {
        if constexpr (W == 4) {
          if (a.vvec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            next[i][0] = u.x; next[i][1] = u.y; next[i][2] = u.z; next[i][3] = u.w;
            continue;
          }
        } else if constexpr (W == 2) {
          if (a.vvec) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            next[i][0] = u.x; next[i][1] = u.y;
            continue;
          }
        } else {
          if (a.vvec) {
            next[i][0] = *reinterpret_cast<const uint32_t*>(p);
            continue;
          }
        }
#pragma unroll
        for (int x = 0; x < W; ++x) {
          if constexpr (sizeof(T) == 2) {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(p) + 2 * x;
            next[i][x] = e[0] | (uint32_t)e[1] << 16;
          } else {
            next[i][x] = __float_as_uint(p[x]);
          }
        }
      }
    }
  };
  load(h0);
  for (int hb = h0, pass = 0; hb < h1; hb += at_once, ++pass) {
    const int h = hb + hl;
    const bool live = hl < at_once && h < h1;
    const int64_t ph = k.page * c.H + (live ? h : hb);
    const float s_old = k.first > 0 ? c.vs[ph] : 0.f;  // (rewritten below: not a read-only load)
    uint8_t* vc = c.v + ph * blk * D + (int64_t)d * blk + lo;
    uint32_t x[16][W], amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int y = 0; y < W; ++y) {
        x[i][y] = next[i][y];
        amax = sizeof(T) == 2 ? __vmaxu2(amax, x[i][y] & 0x7FFF7FFFu) : max(amax, x[i][y] & 0x7FFFFFFFu);
      }
    if constexpr (sizeof(T) == 2) amax = max(amax & 0x7FFF0000u, amax << 16);
    if (hb + at_once < h1) load(hb + at_once);  // the next heads', while these are worked on
    amax = head_max(amax, live ? hl : kHeadsAtOnce, s_max, pass);
    if (!live) continue;
    const float scale = k.first > 0 ? grown_scale(s_old, scale_for<FMT>(amax)) : scale_for<FMT>(amax);
    const bool poisoned = scale != scale, grow = k.first > 0 && scale != s_old;
    const float inv = 1.f / scale, ratio = s_old / scale;
    if (tid == hl * slots) c.vs[ph] = scale;
    if (grow && r0 > 0) {  // whole runs of old codes under a grown scale
      for (int i = tid - hl * slots; i < D * r0; i += slots) {
        uint4* p = reinterpret_cast<uint4*>(c.v + ph * blk * D + (int64_t)(i / r0) * blk) + i % r0;
        uint4 o = make_uint4(0, 0, 0, 0);
        if (!poisoned) {
          o = *p;
          o = make_uint4(recode4<FMT>(o.x, ratio), recode4<FMT>(o.y, ratio), recode4<FMT>(o.z, ratio), recode4<FMT>(o.w, ratio));
        }
        *p = o;
      }
    }
    auto value = [&](int i, int y) -> float {  // dim y of token i
      if constexpr (sizeof(T) == 2)
        return (y & 1) ? bf16_hi(x[i][y >> 1]) : bf16_lo(x[i][y >> 1]);
      else
        return __uint_as_float(x[i][y]);
    };
#pragma unroll
    for (int y = 0; y < DPT; y += 2) {
      uint32_t w[2][4];  // [dim y, y + 1][word of 4 tokens]
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        uint32_t t[4];  // a token's 2 codes
#pragma unroll
        for (int i = 0; i < 4; ++i)
          t[i] = codes2<FMT>(value(4 * z + i, y) * inv, value(4 * z + i, y + 1) * inv);
        const uint32_t lo2 = __byte_perm(t[0], t[1], 0x5410), hi2 = __byte_perm(t[2], t[3], 0x5410);
        w[0][z] = __byte_perm(lo2, hi2, 0x6420);
        w[1][z] = __byte_perm(lo2, hi2, 0x7531);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (poisoned) w[e][0] = w[e][1] = w[e][2] = w[e][3] = 0;
        uint4* dst = reinterpret_cast<uint4*>(vc + (int64_t)(y + e) * blk);
        if (!all_new) {
          const uint4 was = *dst;
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            // bytes of new tokens and of old ones in this word
            const int s = lo + 4 * z, n_old = min(max(k.first - s, 0), 4), n_end = min(max(k.first + k.n - s, 0), 4);
            const uint32_t mo = n_old == 4 ? 0xFFFFFFFFu : (1u << (8 * n_old)) - 1u;
            const uint32_t mn = (n_end == 4 ? 0xFFFFFFFFu : (1u << (8 * n_end)) - 1u) & ~mo;
            const uint32_t o = z == 0 ? was.x : z == 1 ? was.y : z == 2 ? was.z : was.w;
            uint32_t kept = o;
            if (grow && mo) kept = (o & ~mo) | ((poisoned ? 0 : recode4<FMT>(o, ratio)) & mo);
            w[e][z] = (w[e][z] & mn) | (kept & ~mn);
          }
        }
        *dst = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
      }
    }
  }
}

// Rotate q_tok rows of q to their sequences' positions.
template <typename T, bool VEC>
__device__ void append_rotate_q(const AppendArgs& a, uint8_t* smem) {
  float2* tab = reinterpret_cast<float2*>(smem);
  __shared__ int32_t s_pos[8];
  const int64_t t0 = (int64_t)(blockIdx.x - a.kv_blocks) * a.q_tok;
  const int nt = (int)min((int64_t)a.q_tok, a.b.N - t0);
  const int tid = threadIdx.x;
  if (tid < nt) {  // last b with cu[b] <= row: the row's sequence, if it lies below cu[b + 1]
    const int32_t row = (int32_t)t0 + tid;
    int lo = 0, hi = a.b.B;
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (__ldg(a.b.cu + m) <= row) lo = m; else hi = m;
    }
    const Seq s = sequence(a.b, a.b.cu, a.b.lens, a.c.blk, lo, a.c.status);
    const int32_t pos = s.len - s.n + (row - s.row0);
    s_pos[tid] = row >= s.row0 && row < s.row0 + s.n && s.len >= s.n ? pos : -1;
  }
  __syncthreads();
  const int half = a.r.rot >> 1;
  for (int i = tid; i < nt * half; i += blockDim.x) {
    const int t = i / half, p = i - t * half;
    tab[i] = rope::angle_f32(s_pos[t], __ldg(a.r.inv_freq + p), a.r.factor, 1.f);
  }
  __syncthreads();
  const int units = rope::head_units<T, VEC>(a.r.D, a.r.rot, a.r.layout), per_tok = a.r.hq * units;
  for (int i = tid; i < nt * per_tok; i += blockDim.x) {
    const int t = i / per_tok, r = i - t * per_tok, h = r / units, u = r - h * units;
    if (s_pos[t] < 0) continue;
    rope::rotate_head<T, VEC>(static_cast<const T*>(a.r.q.p) + (t0 + t) * a.r.q.st + h * a.r.q.sh,
                              static_cast<T*>(const_cast<void*>(a.r.q_out.p)) + (t0 + t) * a.r.q_out.st +
                                  h * a.r.q_out.sh,
                              a.r.D, a.r.rot, a.r.layout, tab + t * half, u);
  }
}

// Keys and values in one launch: blocks alternate between them.
template <typename T, int FMT, int TPT>
__global__ void __launch_bounds__(kAppendThreads, TPT == 16 ? 1 : 2) append_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) uint8_t s_append[];
  __shared__ Maxima s_max;
  if ((int)blockIdx.x >= a.kv_blocks) {
    if (a.qvec)
      append_rotate_q<T, true>(a, s_append);
    else
      append_rotate_q<T, false>(a, s_append);
    return;
  }
  if (threadIdx.x < kHeadsAtOnce) s_max.m[0][threadIdx.x] = 0;
  const int groups = (a.c.H + a.heads - 1) / a.heads;
  const int t = blockIdx.x / (2 * groups), r = blockIdx.x - t * 2 * groups;
  const Task k = find_task<kAppendThreads>(a.c, a.b, nullptr, true, t);
  if (k.b < 0 || k.page < 0) return;
  const int h0 = (r >> 1) * a.heads, h1 = min(h0 + a.heads, a.c.H);
  if (r & 1)
    append_values<T, FMT, TPT == 16 ? 4 : 2>(a, k, h0, h1, s_max);
  else
    append_keys<T, FMT, TPT>(a, k, h0, h1, s_max);
}

// The same as two launches of half the grid, for batches with enough blocks to
// fill the GPU: apart, keys and values need fewer registers each, so that more
// blocks run at once.
template <typename T, int FMT, int TPT>
__global__ void __launch_bounds__(kAppendThreads, TPT == 16 ? 1 : TPT == 8 || sizeof(T) == 4 ? 2 : 3) keys_kernel(const AppendArgs a) {
  __shared__ Maxima s_max;
  if (threadIdx.x < kHeadsAtOnce) s_max.m[0][threadIdx.x] = 0;
  const int groups = (a.c.H + a.heads - 1) / a.heads, t = blockIdx.x / groups, h0 = (blockIdx.x - t * groups) * a.heads;
  const Task k = find_task<kAppendThreads>(a.c, a.b, nullptr, true, t);
  if (k.b < 0 || k.page < 0) return;
  append_keys<T, FMT, TPT>(a, k, h0, min(h0 + a.heads, a.c.H), s_max);
}
template <typename T, int FMT, int DPT>
__global__ void __launch_bounds__(kAppendThreads, DPT * sizeof(T) == 4 ? 3 : DPT * sizeof(T) == 8 ? 2 : 1) values_kernel(const AppendArgs a) {
  __shared__ Maxima s_max;
  if (threadIdx.x < kHeadsAtOnce) s_max.m[0][threadIdx.x] = 0;
  const int groups = (a.c.H + a.heads - 1) / a.heads, t = blockIdx.x / groups, h0 = (blockIdx.x - t * groups) * a.heads;
  const Task k = find_task<kAppendThreads>(a.c, a.b, nullptr, true, t);
  if (k.b < 0 || k.page < 0) return;
  append_values<T, FMT, DPT>(a, k, h0, min(h0 + a.heads, a.c.H), s_max);
}

// The rotation of q by itself, for batches whose q would wait for the few
// blocks that the registers of append_kernel let run at once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) rotate_q_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) uint8_t s_rotate[];
  append_rotate_q<T, VEC>(a, s_rotate);
}

// ------------------------------------------------------------- read back

struct ReadArgs {
  Cache c;
  Batch b;
  const int32_t* starts;
  void* k_out;
  void* v_out;
  int32_t heads;  // kv heads of one grid block
};

// Four codes of one 32-bit word times a scale.
template <int FMT>
__device__ __forceinline__ float4 values4(uint32_t w, float s) {
  if constexpr (FMT == INT8) {
    // code + 128 in the low byte of 2^23 is the float 2^23 + 128 + code
    w ^= 0x80808080u;
    const float bias = 8388736.f;
    return make_float4((__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540)) - bias) * s,
                       (__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7541)) - bias) * s,
                       (__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7542)) - bias) * s,
                       (__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7543)) - bias) * s);
  } else {
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)w, __NV_E4M3)));
    const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((uint16_t)(w >> 16), __NV_E4M3)));
    return make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
  }
}
__device__ __forceinline__ void store16(float* p, const float4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[i] = v[i];
}
__device__ __forceinline__ void store16(bf16* p, const float4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<uint4*>(p)[i] =
        make_uint4(pack_bf16(v[2 * i].x, v[2 * i].y), pack_bf16(v[2 * i].z, v[2 * i].w),
                   pack_bf16(v[2 * i + 1].x, v[2 * i + 1].y), pack_bf16(v[2 * i + 1].z, v[2 * i + 1].w));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

constexpr int kReadThreads = 256;

// One grid block per touched block, group of heads, and k or v.  Keys go
// straight across, 16 codes a thread.  Values lie token minor: a thread takes
// 16 tokens of 4 dims (four 16-byte loads), turns each 4 x 4 bytes over in
// registers and writes 4 dims of each token, so a warp's stores are whole
// rows.  Bound by memory: codes in, 2 or 4 bytes a code out.  32 ragged prefixes
// of up to 4096 tokens, 8 heads of 128 dims, to BF16: 91 us, 5.2 TB/s.
template <typename T, int FMT>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadArgs a) {
  const Cache& c = a.c;
  const int D = c.D, blk = c.blk, tid = threadIdx.x;
  const int groups = (c.H + a.heads - 1) / a.heads, t = blockIdx.x / (2 * groups), r = blockIdx.x - t * 2 * groups;
  const int h0 = (r >> 1) * a.heads, nh = min(a.heads, c.H - h0);
  const Task k = find_task<kReadThreads>(c, a.b, a.starts, false, t);
  if (k.b < 0) return;
  const bool bad = k.page < 0;
  const float nan = __uint_as_float(0x7FC00000u);
  const int64_t ph0 = bad ? 0 : k.page * c.H + h0, row = (int64_t)c.H * D, head = (int64_t)blk * D;
  if ((r & 1) == 0) {
    const int pieces = D >> 4, per = k.n * pieces;
    const uint8_t* kc = c.k + ph0 * head + (int64_t)k.first * D;
    T* ko = static_cast<T*>(a.k_out) + (int64_t)k.row0 * row + h0 * D;
#pragma unroll 4
    for (int i = tid; i < nh * per; i += kReadThreads) {
      const int hl = i / per, j = i - hl * per, s = j / pieces, d = (j - s * pieces) * 16;
      const uint4 w = bad ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(kc + hl * head + s * D + d));
      const float ks = bad ? nan : read_scale(__ldg(c.ks + ph0 + hl));
      const float4 v[4] = {values4<FMT>(w.x, ks), values4<FMT>(w.y, ks), values4<FMT>(w.z, ks), values4<FMT>(w.w, ks)};
      store16(ko + s * row + hl * D + d, v);
    }
  } else {
    // 16-token runs that the call's tokens touch
    const int quads = D >> 2, r0 = k.first >> 4, runs = ((k.first + k.n - 1) >> 4) - r0 + 1, per = runs * quads;
    const uint8_t* vc = c.v + ph0 * head;
    T* vo = static_cast<T*>(a.v_out) + (int64_t)k.row0 * row + h0 * D;
    for (int i = tid; i < nh * per; i += kReadThreads) {
      const int hl = i / per, j = i - hl * per, g = j / quads, d = (j - g * quads) * 4, lo = 16 * (r0 + g);
      uint4 w[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        w[x] = bad ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(vc + hl * head + (int64_t)(d + x) * blk + lo));
      const float vs = bad ? nan : read_scale(__ldg(c.vs + ph0 + hl));
      T* o = vo + hl * D + d;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t w0 = y == 0 ? w[0].x : y == 1 ? w[0].y : y == 2 ? w[0].z : w[0].w;
        const uint32_t w1 = y == 0 ? w[1].x : y == 1 ? w[1].y : y == 2 ? w[1].z : w[1].w;
        const uint32_t w2 = y == 0 ? w[2].x : y == 1 ? w[2].y : y == 2 ? w[2].z : w[2].w;
        const uint32_t w3 = y == 0 ? w[3].x : y == 1 ? w[3].y : y == 2 ? w[3].z : w[3].w;
        // 4 x 4 bytes turned over
        const uint32_t a0 = __byte_perm(w0, w1, 0x5140), a1 = __byte_perm(w0, w1, 0x7362);
        const uint32_t b0 = __byte_perm(w2, w3, 0x5140), b1 = __byte_perm(w2, w3, 0x7362);
        const uint32_t q[4] = {__byte_perm(a0, b0, 0x5410), __byte_perm(a0, b0, 0x7632), __byte_perm(a1, b1, 0x5410),
                               __byte_perm(a1, b1, 0x7632)};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int s = lo + 4 * y + x - k.first;
          if (s >= 0 && s < k.n) store4(o + s * row, values4<FMT>(q[x], vs));
        }
      }
    }
  }
}

}  // namespace kv
}  // namespace noor
