// kv_prompt.cuh -- attention over the 8-bit cache for many query rows, on
// tcgen05 tensor cores (BF16 activations, head_dim up to 128).
//
// A block takes one unit: 256 rows (query row, query head of the group) of one
// kv head, as two row tiles of 128, and their visible tokens in tiles of 128:
// all of them, or one of several equal runs where there are fewer units than
// SMs; combine_kernel then joins a unit's parts.  The same sums as the streamed kernel (kv_attention.cuh):
//   s = q.k (f16 codes and f16 queries, f32 sums), p = 2^(s f - m + shift) in
//   f16, o += p v, with f = scale log2(e) 2^e(row) k scale(block).
// Roles:
//   warps 0-3, 4-7  softmax of row tile 0 / 1, a thread for each row
//   warps 8-11      widen: codes in shared memory -> f16 operand tiles
//   warp 12         one thread issues the mma's; the warp owns TMEM
//   warp 13         loader: page table, scales, bulk copies of raw pages
// TMEM (512 columns): S of both row tiles (2 x 128; p overwrites its own s as
// f16 and is read from there as the second product's first operand), o of both.
// While one row tile's softmax runs, the tensor core does the other's p v and
// next q k.  Both operand layouts are the cache's own (k rows and v columns
// contiguous along the contraction), so widening copies straight across into
// the 128-byte-swizzled tiles.
//
// m is a reference that follows the row's maximum lazily: o is rescaled only
// when the maximum has grown by more than 2^8, so most tiles never touch o.
// p <= 2^15 then fits f16; shift 7 keeps p down to 2^-31 of the largest.
//
// Measured: 2 sequences of 2048 rows on 8192 tokens, 32 / 8 heads of 128 dims,
// 549-558 us = 860-880 TFLOP/s of visible products.  Bound by the softmax warps: an
// exponential, its scaling and the sums for each score, beside TMEM reads; the
// tensor core waits for p.
// V scales.  o of a row is held relative to the largest v scale (up to a power
// of two) among the tokens that the row has seen so far, and follows when that
// grows; what a row does not see leaves its bits alone.
//   A tile that every row of the unit sees whole is widened relative to its own
//   largest scale (exact for powers of two down to 2^-24 of it for int8 and
//   2^-15 for e4m3; below, to 2^-25 of the largest scale), and its ratio to the row's, a power of two, goes into the
//   exponential: p comes out scaled, and its sum is scaled back.
//   In the other tiles (the context's end, a window's start) values are codes
//   alone, and each p is multiplied by its block's scale over the row's.
#pragma once

#include "kv_attention.cuh"

namespace noor {
namespace prompt {

using attn::Args;

constexpr int kThreads = 512;  // warps 14 and 15 only fill their register group
constexpr int kTok = 128;    // tokens of a tile
constexpr float kShift = 7.0f, kLazy = 8.0f;
constexpr int kMeta = 4;     // tiles of block factors in flight

template <int DP>
struct Smem {
  static constexpr int kQ = 128 * DP * 2;      // one row tile, f16
  static constexpr int kK = kTok * DP * 2;     // one token tile, f16
  static constexpr int kRaw = kTok * DP;       // one token tile of codes
  static constexpr int kBytes = 2 * kQ + 4 * kK + 2 * kRaw + 1024;  // + alignment
};

struct Bars {
  uint64_t raw_full[2], raw_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], q_full[2], s_full[2], p_full[2],
      o_full[2], drain;
};

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One thread of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// 16-byte piece `chunk` of row `row` in a 128-byte-swizzled block.
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

// PARTS: whether units may be cut (compiled apart: the tests cost registers, 8% of the time)
template <int DP, int FMT, bool PARTS>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const Args a) {
  using S = Smem<DP>;
  extern __shared__ uint8_t s_raw_base[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw_base) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;                    // [2][DP / 64][128 rows][128 B]
  uint8_t* s_k = s_q + 2 * S::kQ;         // [2 slots][DP / 64][128 tokens][128 B]
  uint8_t* s_v = s_k + 2 * S::kK;         // [2 slots][2][DP dims][128 B]
  uint8_t* s_rk = s_v + 2 * S::kK;        // raw pages
  uint8_t* s_rv = s_rk + S::kRaw;
  __shared__ __align__(8) Bars bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  // of each 16 tokens: scores' factor, widened values' factor, v scale; and the tile's largest, a power of two
  __shared__ float s_kf[kMeta][8], s_vf[kMeta][8], s_vs[kMeta][8], s_vc[kMeta];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.c.D, blk = a.c.blk;

  // ---- the block's unit: last row tiles first, they see the most tokens
  // ---- parts of each unit, from the units that the batch has
  int parts = 1;
  if constexpr (PARTS) {
    __shared__ int32_t s_units, s_tiles;
    if (threadIdx.x == 0) s_units = s_tiles = 0;
    __syncthreads();
    int32_t n = 0, longest = 0;  // units of a kv head; most tiles of their sequences
    for (int i = threadIdx.x; i < a.b.B; i += kThreads) {
      const attn::SeqWork w = attn::seq_work(a, i);
      n += w.rtiles;
      if (w.rtiles > 0) longest = max(longest, (w.s.len + kTok - 1) / kTok);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0 && n > 0) {
      atomicAdd(&s_units, n);
      atomicMax(&s_tiles, longest);
    }
    __syncthreads();
    // (the host knows the page table's width and the window, not the lengths)
    const int32_t units = s_units * a.c.H, seen = min(a.seen, s_tiles);
    if (units < a.sms) {
      const int most = attn::most_parts(units, seen, a.sms, a.pairs);
      uint32_t best = 0xFFFFFFFFu;  // cost, then parts
      for (int s = 2 + lane; s <= most; s += 32) {
        const uint32_t cost = attn::part_cost(units, seen, s, a.sms);
        best = min(best, min(cost, (1u << 22) - 1) << 10 | (uint32_t)s);
      }
      best = __reduce_min_sync(0xffffffffu, best);
      if (best != 0xFFFFFFFFu && 20 * (best >> 10) < 19 * (uint32_t)attn::part_cost(units, seen, 1, a.sms)) parts = best & 1023;
    }
  }
  const bool cut = PARTS && parts > 1;
  const int part = blockIdx.x % parts, unit = blockIdx.x / parts, h = unit % a.c.H;
  int sb = -1, rt = 0;
  {
    int32_t before = 0;
    const int32_t t = unit / a.c.H;
    for (int base = 0; base < a.b.B && sb < 0; base += 32) {
      int32_t n = 0;
      if (base + lane < a.b.B) n = attn::seq_work(a, base + lane).rtiles;
      int32_t incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > t);
      if (hit) {
        const int src = __ffs(hit) - 1;
        sb = base + src;
        rt = before + __shfl_sync(0xffffffffu, incl, src) - 1 - t;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  // (row offsets that overlap may count more units than there are slots)
  if (cut && (int64_t)unit * parts + parts > a.pairs) sb = -1;
  if (PARTS && threadIdx.x == 0 && blockIdx.x < a.pairs)
    a.desc[blockIdx.x] = make_int4(cut && part == 0 ? sb : -1, h, rt, (int)(blockIdx.x + parts - 1) << 1);
  if (sb < 0) return;
  const attn::SeqWork w = attn::seq_work(a, sb);
  const int e0 = 256 * rt, nrows = min(256, w.s.n * a.g - e0), nw = nrows > 128 ? 2 : 1;
  const int pos0 = w.s.len - w.s.n;
  const int p_first = pos0 + e0 / a.g, p_last = pos0 + (e0 + nrows - 1) / a.g;
  const int lo_tok = a.window > 0 ? max(p_first - a.window, 0) : 0, hi_tok = p_last + 1;
  const int first = lo_tok / kTok, count = (hi_tok + kTok - 1) / kTok - first;
  const int tb = first + (int)((int64_t)count * part / parts);
  const int T = first + (int)((int64_t)count * (part + 1) / parts) - tb;
  const int32_t* table = a.b.table + (int64_t)sb * a.b.tstride;
  // whether every row of the unit sees all of the tile of tokens tok0 ..
  auto sees_whole = [&](int tok0) { return tok0 + kTok - 1 <= p_first && (a.window <= 0 || p_last - tok0 <= a.window); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bar.raw_full[i], 1);
      tc::mbar_init(&bar.raw_empty[i], 4);
      tc::mbar_init(&bar.k_full[i], 4);
      tc::mbar_init(&bar.k_empty[i], 1);
      tc::mbar_init(&bar.v_full[i], 4);
      tc::mbar_init(&bar.v_empty[i], 1);
      tc::mbar_init(&bar.q_full[i], 4);
      tc::mbar_init(&bar.s_full[i], 1);
      tc::mbar_init(&bar.p_full[i], 4);
      tc::mbar_init(&bar.o_full[i], 1);
    }
    tc::mbar_init(&bar.drain, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    async_fence();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(&tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // Bounded wait: false once a wait anywhere in the block gave up.
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
    if (tc::mbar_try_wait(b, parity)) return true;
    const long long start = clock64();
    while (true) {
      if (tc::mbar_try_wait_sleep(b, parity)) return true;
      if (abort_flag) return false;
      if (clock64() - start > kWaitLimitCycles) {
        abort_flag = 1;
        kv::flag(a.c.status, NOOR_KV_TIMEOUT);
        return false;
      }
    }
  };

  // Registers: 128 a thread at launch (512 x 128, the whole file); the eight
  // softmax warps take 160, the other eight keep 96 (256 x 160 + 256 x 96 =
  // 65536).  Nothing spills with whole contexts at 128 dims; their cut form spills 12
  // bytes (stores), the forms for 64 dims 64-76.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    // ------------------------------------------------------- softmax
    const int wg = warp >> 2, r = (warp & 3) * 32 + lane;  // row of this row tile
    const int e = e0 + 128 * wg + r;
    const bool live = 128 * wg + r < nrows;
    const int row = w.s.row0 + e / a.g, head = h * a.g + e % a.g;
    const int pos = live ? pos0 + e / a.g : -1;
    const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 128u * wg, t_o = t_s + 256u;
    if (wg < nw) {
      // the row's queries, scaled by a power of two (negative if the scale is)
      // so that the largest is in 2^14 .. 2^15
      const bf16* qp = static_cast<const bf16*>(a.q.p) + (int64_t)row * a.q.st + (int64_t)head * a.q.sh;
      const bool qvec = (reinterpret_cast<uintptr_t>(a.q.p) | (uintptr_t)(a.q.st * 2) | (uintptr_t)(a.q.sh * 2)) % 16 == 0;
      uint4 qr[DP / 8];  // all loads in flight together
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        qr[d] = make_uint4(0, 0, 0, 0);
        if (live && 8 * d < D) {
          if (qvec) {
            qr[d] = *reinterpret_cast<const uint4*>(qp + 8 * d);
          } else {
            const uint16_t* e16 = reinterpret_cast<const uint16_t*>(qp + 8 * d);
            qr[d] = make_uint4(e16[0] | (uint32_t)e16[1] << 16, e16[2] | (uint32_t)e16[3] << 16,
                               e16[4] | (uint32_t)e16[5] << 16, e16[6] | (uint32_t)e16[7] << 16);
          }
        }
      }
      uint32_t mb = 0;  // magnitudes, two at a time
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        mb = __vmaxu2(mb, __vmaxu2(__vmaxu2(qr[d].x & 0x7FFF7FFFu, qr[d].y & 0x7FFF7FFFu),
                                   __vmaxu2(qr[d].z & 0x7FFF7FFFu, qr[d].w & 0x7FFF7FFFu)));
      const uint32_t mx = max(mb & 0x7FFF0000u, mb << 16);
      const int ex = max(min((int)(mx >> 23) - 127, 127), -112);
      float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
      // (NaN where an element is not finite, as in the streamed kernel)
      const float fac = mx < 0x7F800000u ? fabsf(a.scale2) * __uint_as_float((uint32_t)(ex - 14 + 127) << 23)
                                         : __uint_as_float(0x7FC00000u);
      if (a.scale2 < 0.f) up = -up;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        if (8 * d >= D) break;
        uint4 u;
        u.x = attn::pack_half(bf16_lo(qr[d].x) * up, bf16_hi(qr[d].x) * up);
        u.y = attn::pack_half(bf16_lo(qr[d].y) * up, bf16_hi(qr[d].y) * up);
        u.z = attn::pack_half(bf16_lo(qr[d].z) * up, bf16_hi(qr[d].z) * up);
        u.w = attn::pack_half(bf16_lo(qr[d].w) * up, bf16_hi(qr[d].w) * up);
        *reinterpret_cast<uint4*>(s_q + wg * S::kQ + (d >> 3) * (128 * 128) + swizzled(r, d & 7)) = u;
      }
      async_fence();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.q_full[wg]);

      float m = -INFINITY, l = 0.f, ref = 1.17549435e-38f;  // ref: the largest v scale so far, a power of two
      bool ok = true;
      // One tile's scores to probabilities, compiled apart for tiles that every
      // row sees whole: a test for each score costs more than its exponential.
      auto tile = [&](auto all, int i, int clo, int chi) {
        constexpr bool whole = decltype(all)::value;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = s_kf[i % kMeta][j] * fac;
        float mx2 = -INFINITY;
        uint32_t sb2[2][32];  // the next 32 columns load while these are worked on
        tc::tmem_ld32(t_s, sb2[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tc::tmem_ld_wait();
          tc::tmem_ld32(t_s + 32 * ((c + 1) & 3), sb2[(c + 1) & 1]);  // (the last: the second pass's first)
          const uint32_t* s = sb2[c & 1];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float g = -INFINITY;
            if constexpr (whole) {
#pragma unroll
              for (int x = 0; x < 16; x += 2)
                g = max3(g, __uint_as_float(s[16 * y + x]), __uint_as_float(s[16 * y + x + 1]));
            } else {
#pragma unroll
              for (int x = 0; x < 16; ++x) {
                const int col = 32 * c + 16 * y + x;
                g = fmaxf(g, col >= clo && col <= chi ? __uint_as_float(s[16 * y + x]) : -INFINITY);
              }
            }
            // (nothing visible: -inf, whatever the factor)
            mx2 = fmaxf(mx2, g == -INFINITY ? -INFINITY : g * f[2 * c + y]);
          }
        }
        const bool grow = mx2 > m + kLazy || (m == -INFINITY && mx2 > -INFINITY);
        float vseen = 0.f;  // the largest v scale that the row sees here
        if constexpr (whole) {
          vseen = s_vc[i % kMeta];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (16 * j <= chi && 16 * j + 15 >= clo) vseen = fmaxf(vseen, s_vs[i % kMeta][j]);
          vseen = kv::power_up(vseen);
        }
        const float vnew = fmaxf(ref, vseen);
        if (i == 0) {
          m = mx2;
          ref = vnew;
        } else if (__any_sync(0xffffffffu, grow || vnew != ref)) {
          // (o holds all earlier tiles: its last product ran before this s)
          float alpha = grow ? attn::exp2_approx(m - mx2) : 1.f;
          if (grow) m = mx2;
          l *= alpha;
          alpha *= ref * kv::power_inverse(vnew);
          ref = vnew;
          for (int c = 0; c < D; c += 16) {
            uint32_t v[16];
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                  "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                : "r"(t_o + c));
            tc::tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * alpha);
            tmem_st16(t_o + c, v);
          }
        }
        const float mref = m == -INFINITY ? 0.f : m - kShift;
        // the tile's scale over the row's, 2^-down: in the exponent of p (below
        // 2^-42 no p reaches f16, and the sum keeps its bits)
        const int down = whole ? min((int)(__float_as_uint(ref) - __float_as_uint(vseen)) >> 23, 42) : 0;
        const float vi = kv::power_inverse(ref), neg1 = -mref - (float)down;
        const uint64_t neg = pair2(neg1, neg1);
        uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
          tc::tmem_ld_wait();
          if (c < 3) tc::tmem_ld32(t_s + 32 * (c + 1), sb2[(c + 1) & 1]);
          const uint32_t* s = sb2[c & 1];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            const float fj = f[2 * c + (x >> 4)];
            float2 z = split2(fma2(pair2(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), pair2(fj, fj), neg));
            z.x = attn::exp2_approx(z.x);
            z.y = attn::exp2_approx(z.y);
            if constexpr (!whole) {
              const int col = 32 * c + x;
              z.x = col >= clo && col <= chi ? z.x : 0.f;
              z.y = col + 1 >= clo && col + 1 <= chi ? z.y : 0.f;
            }
            sum[(x >> 1) & 3] = add2(sum[(x >> 1) & 3], pair2(z.x, z.y));
            if constexpr (!whole) {
              const float vr = fminf(s_vs[i % kMeta][2 * c + (x >> 4)] * vi, 1.f);  // (above 1: a block it does not see)
              z.x *= vr;
              z.y *= vr;
            }
            p[x >> 1] = attn::pack_half(z.x, z.y);
          }
          // columns 16 c .. of p lie over scores that were read already
          tmem_st16(t_s + 16 * c, p);
        }
        const float2 t2 = split2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
        l = fmaf(t2.x + t2.y, __uint_as_float((uint32_t)(127 + down) << 23), l);
        tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bar.p_full[wg]);
      };
      for (int i = 0; i < T && ok; ++i) {
        const int tok0 = (tb + i) * kTok;
        const bool whole = sees_whole(tok0);
        // visible columns of this row
        const int chi = min(pos - tok0, kTok - 1), clo = a.window > 0 ? pos - a.window - tok0 : 0;
        ok = __all_sync(0xffffffffu, wait(&bar.s_full[wg], i & 1));
        if (!ok) break;
        tc::tc_fence_after();
        if (whole)
          tile(std::true_type{}, i, clo, chi);
        else
          tile(std::false_type{}, i, clo, chi);
      }
      if (ok && T > 0) {
        ok = __all_sync(0xffffffffu, wait(&bar.o_full[wg], 0));
        tc::tc_fence_after();
      }
      if (ok) {
        // a part leaves its sums as they are, with the reference of the join's shift
        const float inv = cut ? ref : l == 0.f ? 0.f : 1.f / l * ref;
        const int64_t slot = (int64_t)blockIdx.x * 256 + 128 * wg + r;
        bf16* op = static_cast<bf16*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.st + (int64_t)head * a.out.sh;
        const bool ovec = (reinterpret_cast<uintptr_t>(a.out.p) | (uintptr_t)(a.out.st * 2) | (uintptr_t)(a.out.sh * 2)) % 16 == 0;
        for (int c = 0; c < D; c += 16) {
          uint32_t v[16];
          if (T > 0) {
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                  "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                : "r"(t_o + c));
            tc::tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = 0;
          }
          float z[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) z[x] = __uint_as_float(v[x]) * inv;
          if (cut) {
            if (live)
#pragma unroll
              for (int x = 0; x < 16; x += 4) *reinterpret_cast<float4*>(a.part_o + slot * D + c + x) = make_float4(z[x], z[x + 1], z[x + 2], z[x + 3]);
          } else if (live && ovec) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
              *reinterpret_cast<uint4*>(op + c + 8 * y) =
                  make_uint4(pack_bf16(z[8 * y], z[8 * y + 1]), pack_bf16(z[8 * y + 2], z[8 * y + 3]),
                             pack_bf16(z[8 * y + 4], z[8 * y + 5]), pack_bf16(z[8 * y + 6], z[8 * y + 7]));
          } else if (live) {
#pragma unroll
            for (int x = 0; x < 16; ++x) op[c + x] = __float2bfloat16_rn(z[x]);
          }
          __syncwarp();
        }
        if (cut && live)
          *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(m + (attn::kPShift - kShift), l);
        else if (live && a.lse != nullptr)
          a.lse[(int64_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m - kShift + log2f(l)) * 0.69314718055994531f;
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ------------------------------------------------------- widen
    // Each thread keeps its 16-byte piece and walks down the rows, so that
    // addresses (and the swizzle, rows 16 or 32 apart) only advance; four
    // pieces are in flight.
    const int th = threadIdx.x - 256;  // 0 .. 127
    constexpr int kPieces = DP / 16, kRowStep = 128 / kPieces;
    const int kp = th % kPieces, kr = th / kPieces;
    const bool kin = 16 * kp < D;
    const int kch = 2 * (kp & 3), kfirst = (kp >> 2) & 1;  // the order in which banks do not meet
    const uint32_t ksw0 = (kp >> 2) * (kTok * 128) + swizzled(kr, kch + kfirst);
    const uint32_t ksw1 = (kp >> 2) * (kTok * 128) + swizzled(kr, kch + (kfirst ^ 1));
    const int vq = th & 7, vd = th >> 3;
    const int vch = 2 * (vq & 3), vfirst = (vq >> 2) & 1;
    const uint32_t vsw0 = (vq >> 2) * (DP * 128) + swizzled(vd, vch + vfirst);
    const uint32_t vsw1 = (vq >> 2) * (DP * 128) + swizzled(vd, vch + (vfirst ^ 1));
    const uint8_t* vsrc = s_rv + (16 * vq / blk) * (blk * D) + vd * blk + 16 * vq % blk;
    bool ok = true;
    for (int i = 0; i < T && ok; ++i) {
      const int slot = i & 1;
      const uint32_t ph = (i >> 1) & 1;
      // keys: piece p of a row becomes chunks 2 p, 2 p + 1 of its 64-dim blocks
      ok = __all_sync(0xffffffffu, wait(&bar.raw_full[0], i & 1) && wait(&bar.k_empty[slot], ph ^ 1));
      if (!ok) break;
      uint8_t* dk = s_k + slot * S::kK;
      if (kin) {
#pragma unroll 1
        for (int it = 0; it < kTok / kRowStep; it += 4) {
          uint4 c[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            c[y] = *reinterpret_cast<const uint4*>(s_rk + (kr + (it + y) * kRowStep) * D + 16 * kp);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint4 u, v;
            attn::widen<FMT>(c[y].x, u.x, u.y);
            attn::widen<FMT>(c[y].y, u.z, u.w);
            attn::widen<FMT>(c[y].z, v.x, v.y);
            attn::widen<FMT>(c[y].w, v.z, v.w);
            const uint32_t down = (it + y) * kRowStep * 128;
            *reinterpret_cast<uint4*>(dk + ksw0 + down) = kfirst ? v : u;
            *reinterpret_cast<uint4*>(dk + ksw1 + down) = kfirst ? u : v;
          }
        }
      }
      async_fence();
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(&bar.k_full[slot]);
        tc::mbar_arrive(&bar.raw_empty[0]);
      }
      // values: 16 tokens of a dim become chunks 2 q, 2 q + 1 of its 64-token block
      ok = __all_sync(0xffffffffu, wait(&bar.raw_full[1], i & 1) && wait(&bar.v_empty[slot], ph ^ 1));
      if (!ok) break;
      uint8_t* dv = s_v + slot * S::kK;
      const float vf = s_vf[i % kMeta][vq];
      // (a factor below f16's normal range is taken in two steps: as one it would
      // lose the bits that its products still have, and be zero below 2^-24)
      const bool low = vf < 6.1035156e-05f;  // 2^-14
      const __half2 hf = __float2half2_rn(low ? vf * 16384.f : vf), h14 = __float2half2_rn(6.1035156e-05f);
      // codes past the last visible token, or of a page that cannot be read, count as zero
      const int nv = vf != 0.f ? min(max(hi_tok - ((tb + i) * kTok + 16 * vq), 0), 16) : 0;
      uint32_t keep[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int n = min(max(nv - 4 * y, 0), 4);
        keep[y] = n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
      }
#pragma unroll 1
      for (int it = 0; it < DP / 16; it += 4) {
        uint4 c[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (16 * (it + y) < D) c[y] = *reinterpret_cast<const uint4*>(vsrc + 16 * (it + y) * blk);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if (16 * (it + y) >= D) break;
          uint4 u, v;
          attn::widen<FMT>(c[y].x & keep[0], u.x, u.y);
          attn::widen<FMT>(c[y].y & keep[1], u.z, u.w);
          attn::widen<FMT>(c[y].z & keep[2], v.x, v.y);
          attn::widen<FMT>(c[y].w & keep[3], v.z, v.w);
          if (vf != 1.f && nv > 0) {
            uint32_t* w8[8] = {&u.x, &u.y, &u.z, &u.w, &v.x, &v.y, &v.z, &v.w};
#pragma unroll
            for (int z = 0; z < 8; ++z) {
              __half2 m2 = __hmul2(*reinterpret_cast<__half2*>(w8[z]), hf);
              if (low) m2 = __hmul2(m2, h14);
              *w8[z] = *reinterpret_cast<const uint32_t*>(&m2);
            }
          }
          const uint32_t down = 16 * (it + y) * 128;
          *reinterpret_cast<uint4*>(dv + vsw0 + down) = vfirst ? v : u;
          *reinterpret_cast<uint4*>(dv + vsw1 + down) = vfirst ? u : v;
        }
      }
      async_fence();
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(&bar.v_full[slot]);
        tc::mbar_arrive(&bar.raw_empty[1]);
      }
    }
  } else if (warp == 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ------------------------------------------------------- mma
    // The whole warp runs the loop, so that descriptors and TMEM addresses stay
    // in uniform registers; one elected thread issues.
    if (T > 0) {
      // f16 operands, f32 sums, both K-major, M 128, N 128 tokens or D dims
      const uint32_t id_s = (1u << 4) | ((uint32_t)(kTok >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      // Descriptors are made once; a step along the contraction adds to the
      // address field (16-byte units).
      const uint64_t dq = tc::sdesc_sw128(tc::smem_addr(s_q)), dk = tc::sdesc_sw128(tc::smem_addr(s_k)),
                     dv = tc::sdesc_sw128(tc::smem_addr(s_v));
      bool issued = false;
      auto scores = [&](int wg, int slot, bool free_k) {
        const uint64_t q0 = dq + (uint32_t)(wg * (S::kQ >> 4)), k0 = dk + (uint32_t)(slot * (S::kK >> 4));
        const uint32_t d = tmem + 128u * wg;
        issued = true;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks) {
            if (16 * ks >= D) break;
            const uint32_t off = (ks >> 2) * (128 * 128 >> 4) + (ks & 3) * 2;
            tc::umma_bf16(d, q0 + off, k0 + off, id_s, ks != 0);
          }
          tc::umma_commit(&bar.s_full[wg]);
          if (free_k) tc::umma_commit(&bar.k_empty[slot]);
        }
        __syncwarp();
      };
      bool ok = true;
      for (int wg = 0; wg < nw && ok; ++wg) ok = __all_sync(0xffffffffu, wait(&bar.q_full[wg], 0));
      if (ok) ok = __all_sync(0xffffffffu, wait(&bar.k_full[0], 0));
      if (ok) {
        tc::tc_fence_after();
        for (int wg = 0; wg < nw; ++wg) scores(wg, 0, wg == nw - 1);
      }
      for (int i = 0; i < T && ok; ++i) {
        const int slot = i & 1, next = slot ^ 1;
        const uint64_t v0 = dv + (uint32_t)(slot * (S::kK >> 4));
        for (int wg = 0; wg < nw && ok; ++wg) {
          ok = __all_sync(0xffffffffu, wait(&bar.p_full[wg], i & 1) && (wg > 0 || wait(&bar.v_full[slot], (i >> 1) & 1)));
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t d = tmem + 256u + 128u * wg, p = tmem + 128u * wg;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < kTok / 16; ++ks)
              umma_ts(d, p + 8u * ks, v0 + (uint32_t)((ks >> 2) * (DP * 128 >> 4) + (ks & 3) * 2), id_o, ks != 0 || i != 0);
            if (wg == nw - 1) tc::umma_commit(&bar.v_empty[slot]);
            if (i + 1 == T) tc::umma_commit(&bar.o_full[wg]);
          }
          __syncwarp();
          if (i + 1 < T) {
            if (wg == 0) {
              ok = __all_sync(0xffffffffu, wait(&bar.k_full[next], ((i + 1) >> 1) & 1));
              if (!ok) break;
              tc::tc_fence_after();
            }
            scores(wg, next, wg == nw - 1);
          }
        }
      }
      if (issued) {  // every mma retires before TMEM is released
        if (elect_one()) tc::umma_commit(&bar.drain);
        __syncwarp();
        const long long start = clock64();
        while (!tc::mbar_try_wait(&bar.drain, 0) && clock64() - start < kWaitLimitCycles) {
        }
      }
    }
    __syncwarp();
  } else if (warp > 13) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ------------------------------------------------------- loader
    const int pages = kTok / blk;
    const uint32_t bytes = (uint32_t)blk * D;
    const float nan = __uint_as_float(0x7FC00000u);
    int issued = 0;  // tiles whose copies were issued (k, and v one step later)
    bool ok = true, vpending = false;
    for (int i = 0; i < T && ok; ++i) {
      const int tok0 = (tb + i) * kTok;
      int32_t page = -1;
      if (lane < pages && tok0 + lane * blk < hi_tok) {
        page = __ldg(table + tok0 / blk + lane);
        if (page < 0 || (int64_t)page >= a.c.P) {
          kv::flag(a.c.status, NOOR_KV_BAD_PAGE);
          page = -1;
        }
      }
      const int64_t ph = (int64_t)page * a.c.H + h;
      // factors of each 16 tokens: NaN where the page or its values cannot be
      // read (the rows that see them come out NaN), values then zero
      float ks = page >= 0 ? kv::read_scale(__ldg(a.c.ks + ph)) : nan, vs = page >= 0 ? kv::read_scale(__ldg(a.c.vs + ph)) : nan;
      const int src = (16 * (lane & 7)) / blk;
      ks = __shfl_sync(0xffffffffu, ks, src);
      vs = __shfl_sync(0xffffffffu, vs, src);
      const bool fin = vs == vs;
      const float vc = kv::power_up(__uint_as_float(__reduce_max_sync(0xffffffffu, fin ? __float_as_uint(vs) & 0x7FFFFFFFu : 0u)));
      ok = wait(&bar.raw_empty[0], (i & 1) ^ 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane < 8) {
        s_kf[i % kMeta][lane] = fin ? ks : nan;
        s_vf[i % kMeta][lane] = !fin ? 0.f : sees_whole(tok0) ? vs * kv::power_inverse(vc) : 1.f;
        s_vs[i % kMeta][lane] = fin ? vs : 0.f;
        s_vc[i % kMeta] = vc;
      }
      const unsigned who = __ballot_sync(0xffffffffu, page >= 0);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_expect_tx(&bar.raw_full[0], __popc(who) * bytes);
      __syncwarp();
      if (page >= 0) attn::bulk_load(s_rk + lane * bytes, a.c.k + ph * bytes, bytes, &bar.raw_full[0]);
      issued = i + 1;
      vpending = true;
      ok = wait(&bar.raw_empty[1], (i & 1) ^ 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) tc::mbar_arrive_expect_tx(&bar.raw_full[1], __popc(who) * bytes);
      __syncwarp();
      if (page >= 0) attn::bulk_load(s_rv + lane * bytes, a.c.v + ph * bytes, bytes, &bar.raw_full[1]);
      vpending = false;
    }
    if (!ok && lane == 0 && issued > 0) {  // gave up: the copies in flight land before the block ends
      const long long start = clock64();
      while (!tc::mbar_try_wait(&bar.raw_full[0], (issued - 1) & 1) && clock64() - start < kWaitLimitCycles) {
      }
      const int v = vpending ? issued - 1 : issued;
      while (v > 0 && !tc::mbar_try_wait(&bar.raw_full[1], (v - 1) & 1) && clock64() - start < kWaitLimitCycles) {
      }
    }
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

}  // namespace prompt
}  // namespace noor
