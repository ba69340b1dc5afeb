// rope.cuh -- rotary positions.
//
// Pair i of a head (dims 2i, 2i+1, or i, i + rot/2 in the half layout) at
// position p turns by a = p * inv_freq[i]:
//   y0 = f (x0 cos a - x1 sin a),  y1 = f (x0 sin a + x1 cos a)
// and back by -a, which with the same f is the transpose: the gradient.
//
// The product p * inv_freq is formed in f64 (31 + 24 bits: off by less than
// 2^-22 of a turn at the farthest position) and reduced to a fraction of a
// turn before the cosine is taken in f32; an f32 product would be off by
// whole radians at p = 2^24.
#pragma once

#include "common.cuh"

namespace noor {
namespace rope {

enum Layout : int { INTERLEAVED = 0, HALF = 1 };

struct View {
  const void* p;
  int64_t st, sh;  // element strides of a token and of a head
};

struct Args {
  const float* inv_freq;
  int32_t rot;     // rotated dims
  int32_t layout;
  float factor;
  float sign;      // -1: the inverse rotation
  View q, q_out, k, k_out;
  int32_t hq, hk;  // hk 0: no k
  int32_t D;
  const int32_t* positions;
  int64_t T;
};

// The angle of one pair as a fraction of a turn in [-1/2, 1/2], in f64.
__device__ __forceinline__ double turn_fraction(int32_t pos, float inv_freq) {
  const double t = (double)pos * (double)inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  return t - rint(t);
}

// (cos, sin) of one pair, to f32.
__device__ __forceinline__ float2 angle_f32(int32_t pos, float inv_freq, float factor, float sign) {
  float s, c;
  sincospif(2.0f * (float)turn_fraction(pos, inv_freq), &s, &c);
  return make_float2(c * factor, s * factor * sign);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// The plain products and sums of the formula, each rounded: what the
// unfused 32-bit form gives.
__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
  const float y0 = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
  const float y1 = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
  a = y0;
  b = y1;
}

// 16 bytes of a head as floats.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void load(const float* p, float (&v)[4]) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
  }
  __device__ static void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec<bf16> {
  static constexpr int N = 8;
  __device__ static void load(const bf16* p, float (&v)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16_lo(r.x); v[1] = bf16_hi(r.x); v[2] = bf16_lo(r.y); v[3] = bf16_hi(r.y);
    v[4] = bf16_lo(r.z); v[5] = bf16_hi(r.z); v[6] = bf16_lo(r.w); v[7] = bf16_hi(r.w);
  }
  __device__ static void store(bf16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};

// Rotate one head with the token's (cos, sin) table in shared memory: `lane`
// of `lanes` threads.  VEC moves 16 bytes at a time (rows 16-byte aligned; in
// the half layout rot / 2 a multiple of the vector); the other form moves a
// pair of elements.  A pair is read and written by one thread, so out may be x.
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_head(const T* x, T* out, int D, int rot, int layout, const float2* tab,
                                            int unit) {
  constexpr int N = VEC ? Vec<T>::N : 1;
  if constexpr (VEC) {
    const int nrot = rot / N;  // units that lie whole in the rotated part
    if (layout == INTERLEAVED || rot == 0) {
      const int d = unit * N;
      float v[N];
      Vec<T>::load(x + d, v);
#pragma unroll
      for (int j = 0; j < N; j += 2)
        if (d + j < rot) turn(v[j], v[j + 1], tab[(d + j) >> 1]);
      Vec<T>::store(out + d, v);
    } else if (unit < nrot / 2) {
      const int d = unit * N, h = rot >> 1;
      float a[N], b[N];
      Vec<T>::load(x + d, a);
      Vec<T>::load(x + d + h, b);
#pragma unroll
      for (int j = 0; j < N; ++j) turn(a[j], b[j], tab[d + j]);
      Vec<T>::store(out + d, a);
      Vec<T>::store(out + d + h, b);
    } else {
      const int d = rot + (unit - nrot / 2) * N;
      float v[N];
      Vec<T>::load(x + d, v);
      Vec<T>::store(out + d, v);
    }
  } else {
    const bool r = 2 * unit < rot;
    const int d0 = r && layout == HALF ? unit : 2 * unit;
    const int d1 = r && layout == HALF ? unit + (rot >> 1) : d0 + 1;
    float a = to_f32(x[d0]), b = to_f32(x[d1]);
    if (r) turn(a, b, tab[unit]);
    out[d0] = from_f32<T>(a);
    out[d1] = from_f32<T>(b);
  }
}

// Work units of one head.
template <typename T, bool VEC>
__host__ __device__ __forceinline__ int head_units(int D, int rot, int layout) {
  constexpr int N = VEC ? Vec<T>::N : 2;
  if (!VEC || layout == INTERLEAVED || rot == 0) return D / N;
  return rot / N / 2 + (D - rot) / N;
}

// One block per `tok` tokens: the table of each token's angles is made once
// in shared memory and used by every head of q and k.  Bound by memory: each
// element is read and written once.  32768 tokens of 32 + 8 heads of 128 dims,
// BF16, forward and gradient: 230-240 us, 5.6-5.8 TB/s; a decode step's 64 tokens 3.1 us, a launch's time.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) rope_kernel(const Args a, int tok) {
  extern __shared__ float2 s_tab[];
  const int64_t t0 = (int64_t)blockIdx.x * tok;
  const int nt = (int)min((int64_t)tok, a.T - t0);
  const int half = a.rot >> 1;
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int t = i / half, p = i - t * half;
    s_tab[i] = angle_f32(__ldg(a.positions + t0 + t), __ldg(a.inv_freq + p), a.factor, a.sign);
  }
  __syncthreads();
  const int units = head_units<T, VEC>(a.D, a.rot, a.layout);
  const int heads = a.hq + a.hk, per_tok = heads * units;
#pragma unroll 2
  for (int i = threadIdx.x; i < nt * per_tok; i += blockDim.x) {
    const int t = i / per_tok, r = i - t * per_tok;
    int h = r / units;
    const int u = r - h * units;
    const bool isk = h >= a.hq;
    if (isk) h -= a.hq;
    const View& x = isk ? a.k : a.q;
    const View& y = isk ? a.k_out : a.q_out;
    rotate_head<T, VEC>(static_cast<const T*>(x.p) + (t0 + t) * x.st + h * x.sh,
                        static_cast<T*>(const_cast<void*>(y.p)) + (t0 + t) * y.st + h * y.sh, a.D, a.rot, a.layout,
                        s_tab + t * half, u);
  }
}

}  // namespace rope
}  // namespace noor
