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

// The t-th touched block in batch order, found by one warp: each sequence
// touches the blocks of its tokens [pos0, pos0 + n).  starts: pos0 of each
// sequence (reading), or NULL for the last n tokens (writing).  Returned in
// every lane.
__device__ __forceinline__ Task find_task(const Cache& c, const Batch& b, const int32_t* starts, bool write, int32_t t,
                                          int lane) {
  Task k;
  k.b = -1;
  const int blk = c.blk;
  int32_t before = 0;
  for (int base = 0; base < b.B; base += 32) {
    const int i = base + lane;
    int32_t pos0 = 0, touched = 0;
    Seq s{0, 0, 0};
    if (i < b.B) {
      s = sequence(b, b.cu, b.lens, blk, i, c.status);
      pos0 = write ? s.len - s.n : (starts ? __ldg(starts + i) : 0);
      if (s.n > 0 && (pos0 < 0 || pos0 > s.len - s.n)) {
        flag(c.status, NOOR_KV_BAD_LENGTH);
        s.n = 0;
      }
      if (s.n > 0) touched = (pos0 + s.n - 1) / blk - pos0 / blk + 1;
    }
    int32_t incl = touched;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int32_t local = t - before;
    const unsigned hit = __ballot_sync(0xffffffffu, local >= incl - touched && local < incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int32_t e0 = __shfl_sync(0xffffffffu, incl - touched, src);
      const int32_t p0 = __shfl_sync(0xffffffffu, pos0, src);
      const int32_t n = __shfl_sync(0xffffffffu, s.n, src);
      const int32_t r0 = __shfl_sync(0xffffffffu, s.row0, src);
      k.b = base + src;
      k.j = p0 / blk + (local - e0);
      const int32_t lo = max(p0, k.j * blk), hi = min(p0 + n, (k.j + 1) * blk);
      k.first = lo - k.j * blk;
      k.n = hi - lo;
      k.row0 = r0 + (lo - p0);
      const int32_t page = __ldg(b.table + (int64_t)k.b * b.tstride + k.j);
      k.page = page;
      if (page < 0 || (int64_t)page >= c.P) {
        if (lane == 0) flag(c.status, NOOR_KV_BAD_PAGE);
        k.page = -1;
      }
      return k;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return k;
}

// ------------------------------------------------------------- codes

template <int FMT>
struct Code;
template <>
struct Code<INT8> {
  // exponent of the smallest power of two that holds amax (a finite f32, as bits)
  static constexpr int kExp = 6;                  // 127 = 1.984375 * 2^6
  static constexpr uint32_t kMant = 0x7E0000u;    // mantissa bits of 1.984375
  __device__ static uint8_t make(double x) {
    const int v = __double2int_rn(fmin(fmax(x, -127.0), 127.0));
    return (uint8_t)(int8_t)v;
  }
  __device__ static uint8_t make(float x) {
    const int v = __float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f));
    return (uint8_t)(int8_t)v;
  }
  __device__ static float value(uint8_t c) { return (float)(int8_t)c; }
};
template <>
struct Code<E4M3> {
  static constexpr int kExp = 8;                  // 448 = 1.75 * 2^8
  static constexpr uint32_t kMant = 0x600000u;
  // A NaN code is never stored (the block's scale says NaN): a reader's zero
  // weight times any stored code is zero.
  __device__ static uint8_t finite(uint8_t c) { return (c & 0x7F) == 0x7F ? 0 : c; }
  __device__ static uint8_t make(double x) { return finite(__nv_cvt_double_to_fp8(x, __NV_SATFINITE, __NV_E4M3)); }
  __device__ static uint8_t make(float x) { return finite(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3)); }
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

// The scale of a block that held tokens at s_old and now needs s_new: the
// larger, as a power of two; NaN stays.
__device__ __forceinline__ float grown_scale(float s_old, float s_new) {
  if (!(s_old > 0.f)) return s_old == 0.f ? s_new : __uint_as_float(0x7FC00000u);
  uint32_t b = __float_as_uint(s_old);
  if (b >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  if (b & 0x7FFFFFu) b = (b & 0x7F800000u) + 0x800000u;  // a scale not written here: up to a power of two
  if (b >= 0x7F800000u || s_new != s_new) return __uint_as_float(0x7FC00000u);
  return fmaxf(__uint_as_float(b), s_new);
}

constexpr int kAppendThreads = 256;

struct AppendArgs {
  Cache c;
  Batch b;
  rope::View k, v;
  rope::Args r;       // k's rotation; q and q_out for the q part
  int32_t kv_blocks;  // blocks of the grid that write the cache (the rest rotate q)
  int32_t q_tok;      // rows of q per block
};

// Magnitude bits of the largest |x| over the block's threads.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s_red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) s_red[warp] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) m = max(m, s_red[i]);
  __syncthreads();
  return m;
}

// Write the new tokens of one (touched block, head): grid.x counts them head
// minor.
template <typename T, int FMT>
__device__ void append_block(const AppendArgs& a, uint8_t* smem) {
  const Cache& c = a.c;
  const int D = c.D, blk = c.blk;
  __shared__ Task s_task;
  __shared__ uint32_t s_red[kAppendThreads / 32];
  const int tid = threadIdx.x;
  const int t = blockIdx.x / c.H, h = blockIdx.x - t * c.H;
  if (tid < 32) {
    const Task k = find_task(c, a.b, nullptr, true, t, tid);
    if (tid == 0) s_task = k;
  }
  __syncthreads();
  const Task k = s_task;
  if (k.b < 0 || k.page < 0) return;
  const int64_t ph = k.page * c.H + h;
  T* s_x = reinterpret_cast<T*>(smem);               // [n][D] keys, then values
  uint8_t* s_c = smem + (size_t)blk * D * sizeof(T);  // codes, [n][D]
  const float s_old_k = k.first > 0 ? c.ks[ph] : 0.f, s_old_v = k.first > 0 ? c.vs[ph] : 0.f;

  // ---- keys: rotate in f64 (twice, once for the largest, once for the codes)
  const T* kp = static_cast<const T*>(a.k.p) + (int64_t)k.row0 * a.k.st + h * a.k.sh;
  for (int i = tid; i < k.n * D; i += kAppendThreads) {
    const int s = i / D, d = i - s * D;
    s_x[i] = kp[s * a.k.st + d];
  }
  __syncthreads();
  const int pairs = D >> 1, rot = a.r.rot;
  const int32_t pos0 = k.j * blk + k.first;
  uint32_t amax = 0;
  float scale = 1.f;
  double inv = 1.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = tid; i < k.n * pairs; i += kAppendThreads) {
      const int s = i / pairs, p = i - s * pairs;
      const bool r = 2 * p < rot;
      const int d0 = r && a.r.layout == rope::HALF ? p : 2 * p;
      const int d1 = r && a.r.layout == rope::HALF ? p + (rot >> 1) : d0 + 1;
      double x0 = (double)rope::to_f32(s_x[s * D + d0]), x1 = (double)rope::to_f32(s_x[s * D + d1]);
      if (r) {
        double sn, cs;
        sincospi(2.0 * rope::turn_fraction(pos0 + s, __ldg(a.r.inv_freq + p)), &sn, &cs);
        const double y0 = (x0 * cs - x1 * sn) * a.r.factor, y1 = (x0 * sn + x1 * cs) * a.r.factor;
        x0 = y0;
        x1 = y1;
      }
      if (pass == 0) {
        amax = max(amax, max(__float_as_uint((float)fabs(x0)), __float_as_uint((float)fabs(x1))));
      } else {
        s_c[s * D + d0] = Code<FMT>::make(x0 * inv);
        s_c[s * D + d1] = Code<FMT>::make(x1 * inv);
      }
    }
    if (pass == 0) {
      amax = block_max(amax, s_red);
      scale = k.first > 0 ? grown_scale(s_old_k, scale_for<FMT>(amax)) : scale_for<FMT>(amax);
      inv = 1.0 / (double)scale;
    }
  }
  uint8_t* kc = c.k + ph * blk * D;
  if (k.first > 0 && scale != s_old_k) {  // (NaN too: harmless)
    const float ratio = s_old_k / scale;
    for (int i = tid; i < k.first * D; i += kAppendThreads) kc[i] = Code<FMT>::make(Code<FMT>::value(kc[i]) * ratio);
  }
  __syncthreads();
  for (int i = tid; i < k.n * D; i += kAppendThreads) kc[(int64_t)k.first * D + i] = s_c[i];
  if (tid == 0) c.ks[ph] = scale;
  __syncthreads();

  // ---- values
  const T* vp = static_cast<const T*>(a.v.p) + (int64_t)k.row0 * a.v.st + h * a.v.sh;
  amax = 0;
  for (int i = tid; i < k.n * D; i += kAppendThreads) {
    const int s = i / D, d = i - s * D;
    const T x = vp[s * a.v.st + d];
    s_x[i] = x;
    amax = max(amax, __float_as_uint(fabsf(rope::to_f32(x))));
  }
  amax = block_max(amax, s_red);
  scale = k.first > 0 ? grown_scale(s_old_v, scale_for<FMT>(amax)) : scale_for<FMT>(amax);
  const float finv = 1.0f / scale;
  uint8_t* vc = c.v + ph * blk * D;
  const bool grow = k.first > 0 && scale != s_old_v;
  const float ratio = grow ? s_old_v / scale : 1.f;
  for (int i = tid; i < D * blk; i += kAppendThreads) {
    const int d = i / blk, s = i - d * blk;
    if (s >= k.first && s < k.first + k.n)
      vc[i] = Code<FMT>::make(rope::to_f32(s_x[(s - k.first) * D + d]) * finv);
    else if (grow && s < k.first)
      vc[i] = Code<FMT>::make(Code<FMT>::value(vc[i]) * ratio);
  }
  if (tid == 0) c.vs[ph] = scale;
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

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  extern __shared__ __align__(16) uint8_t s_append[];
  if ((int)blockIdx.x < a.kv_blocks)
    append_block<T, FMT>(a, s_append);
  else
    append_rotate_q<T, VEC>(a, s_append);
}

// ------------------------------------------------------------- read back

struct ReadArgs {
  Cache c;
  Batch b;
  const int32_t* starts;
  void* k_out;
  void* v_out;
};

// Four codes of one 32-bit word times a scale.
template <int FMT>
__device__ __forceinline__ float4 values4(uint32_t w, float s) {
  return make_float4(Code<FMT>::value(w & 0xFF) * s, Code<FMT>::value((w >> 8) & 0xFF) * s,
                     Code<FMT>::value((w >> 16) & 0xFF) * s, Code<FMT>::value(w >> 24) * s);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

constexpr int kReadThreads = 256;

// One block per (touched block, head).  Keys go straight across, 4 codes a
// thread.  Values lie token minor: a thread takes 16 tokens of 4 dims (four
// 16-byte loads), turns each 4 x 4 bytes over in registers and writes 4 dims
// of each token, so a warp's stores are whole rows.  Bound by memory: codes in,
// 2 or 4 bytes a code out.
template <typename T, int FMT>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadArgs a) {
  const Cache& c = a.c;
  const int D = c.D, blk = c.blk, tid = threadIdx.x;
  const int t = blockIdx.x / c.H, h = blockIdx.x - t * c.H;
  const Task k = find_task(c, a.b, a.starts, false, t, tid & 31);
  if (k.b < 0) return;
  const bool bad = k.page < 0;
  const int64_t ph = bad ? 0 : k.page * c.H + h;
  const float nan = __uint_as_float(0x7FC00000u);
  const float ks = bad ? nan : c.ks[ph], vs = bad ? nan : c.vs[ph];
  const uint8_t* kc = c.k + ph * blk * D + (int64_t)k.first * D;
  const uint8_t* vc = c.v + ph * blk * D;
  const int64_t row = (int64_t)c.H * D;
  T* ko = static_cast<T*>(a.k_out) + (int64_t)k.row0 * row + h * D;
  T* vo = static_cast<T*>(a.v_out) + (int64_t)k.row0 * row + h * D;
  const int quads = D >> 2;
#pragma unroll 4
  for (int i = tid; i < k.n * quads; i += kReadThreads) {
    const int s = i / quads, d = (i - s * quads) * 4;
    const uint32_t w = bad ? 0 : __ldg(reinterpret_cast<const uint32_t*>(kc + s * D + d));
    float4 v = values4<FMT>(w, ks);
    if (bad) v = make_float4(nan, nan, nan, nan);
    store4(ko + s * row + d, v);
  }
  for (int i = tid; i < (blk >> 4) * quads; i += kReadThreads) {
    const int g = i / quads, d = (i - g * quads) * 4;
    if (16 * g + 16 <= k.first || 16 * g >= k.first + k.n) continue;
    uint4 r[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
      r[x] = bad ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(vc + (int64_t)(d + x) * blk + 16 * g));
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const uint32_t w0 = y == 0 ? r[0].x : y == 1 ? r[0].y : y == 2 ? r[0].z : r[0].w;
      const uint32_t w1 = y == 0 ? r[1].x : y == 1 ? r[1].y : y == 2 ? r[1].z : r[1].w;
      const uint32_t w2 = y == 0 ? r[2].x : y == 1 ? r[2].y : y == 2 ? r[2].z : r[2].w;
      const uint32_t w3 = y == 0 ? r[3].x : y == 1 ? r[3].y : y == 2 ? r[3].z : r[3].w;
      // 4 x 4 bytes turned over
      const uint32_t a0 = __byte_perm(w0, w1, 0x5140), a1 = __byte_perm(w0, w1, 0x7362);
      const uint32_t b0 = __byte_perm(w2, w3, 0x5140), b1 = __byte_perm(w2, w3, 0x7362);
      const uint32_t o[4] = {__byte_perm(a0, b0, 0x5410), __byte_perm(a0, b0, 0x7632), __byte_perm(a1, b1, 0x5410),
                             __byte_perm(a1, b1, 0x7632)};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int s = 16 * g + 4 * y + x - k.first;
        if (s < 0 || s >= k.n) continue;
        store4(vo + s * row + d, bad ? make_float4(nan, nan, nan, nan) : values4<FMT>(o[x], vs));
      }
    }
  }
}

}  // namespace kv
}  // namespace noor
