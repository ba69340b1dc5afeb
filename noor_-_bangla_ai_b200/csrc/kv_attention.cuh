// kv_attention.cuh -- attention over the 8-bit cache, streamed.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),
// with the running maximum m and sum l of the softmax carried over one pass
// through the visible tokens.
//
// For few query rows the time is that of reading the codes once, so the work
// is cut by bytes: the batch's visible 64-token tiles of every (sequence, kv
// head, 16-row tile of queries) form one list, and every warp of the grid
// takes an equal contiguous share of it, whatever the sequences' lengths.  A
// warp works alone, with no barrier to the others: it streams its tiles through its own ring
// in shared memory with bulk copies and keeps o, m and l in registers.  A unit
// (sequence, head, row tile) cut between warps leaves partial (m, l, o), which
// combine_kernel joins in a fixed order.
//
// The products run on mma.sync m16n8k16 in f16 with f32 sums: the query rows
// of a kv head's group fill the 16 rows, which tcgen05's 128-row tiles would
// leave empty, and at one pass per byte the tensor work is far below the
// memory time.  Codes (|int8| <= 127, e4m3) are exact in f16.  Queries are
// scaled by a power of two for each row so that f16 holds them: exactly for BF16
// (elements under 2^-38 of the row's largest aside), and for F32 as a sum of
// two f16 parts (22 bits).  Probabilities p are f16 as well, off by 2^-12
// relative, an eighth of the BF16 output's half step (F32: two parts again),
// scaled by 2^14 so that p down to 2^-38 counts in a long context.  A block's
// v scale multiplies its p, relative to the largest scale so far.
//
// The contraction index of an mma may be permuted at will if both operands
// agree: thread c of a quad takes 16 consecutive bytes of a key row and of a
// value row and feeds them to four mma steps, so both operands come straight
// from the stored layouts with 16-byte shared loads; a score tile's column n
// is token 16 (n / 2) + 2 t + n % 2, which makes the thread that holds a
// score the one that needs it for p v.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "kv_cache.cuh"
#include "rope.cuh"
#include "tc_gemm.cuh"

namespace noor {
namespace attn {

using kv::Batch;
using kv::Cache;

constexpr int kTile = 64;  // tokens of a tile
constexpr float kPShift = 14.0f;

struct Args {
  Cache c;
  Batch b;
  rope::View q, out;
  float* lse;
  int32_t Hq, g;   // query heads, query heads per kv head
  float scale2;    // scale * log2(e)
  int32_t window;
  // partial results: [2 * warps] slots of 16 rows of (D o's), and [2 * warps][32] (m, l)
  float* part_o;
  float* part_ml;
  int4* desc;      // [warps] of the split units: (sequence, head | row tile << 12.., first warp, last warp)
  int32_t warps;   // warps of the grid that share the work
};

// ------------------------------------------------------------ mma pieces

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four codes to two f16 pairs, exactly.
template <int FMT>
__device__ __forceinline__ void widen(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kv::INT8) {
    // code + 128 in the low byte of 0x6400 is the f16 1024 + 128 + code
    const uint32_t u = x ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&l), bias), b = __hsub2(*reinterpret_cast<__half2*>(&h), bias);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
  }
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The part of (a, b) that the f16 pair leaves.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_half(a - f.x, b - f.y);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   tc::smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_addr(bar))
               : "memory");
}

// ------------------------------------------------------------ the work list

struct SeqWork {
  kv::Seq s;
  int32_t rtiles;    // 16-row tiles of (row, query head of the group)
  int32_t t0, tiles; // first visible 64-token tile and their number, over all rows
};

__device__ __forceinline__ SeqWork seq_work(const Args& a, int i) {
  SeqWork w;
  w.s = kv::sequence(a.b, a.b.cu, a.b.lens, a.c.blk, i, a.c.status);
  if (w.s.n > 0 && w.s.len < w.s.n) kv::flag(a.c.status, NOOR_KV_BAD_LENGTH);
  w.rtiles = (int)(((int64_t)w.s.n * a.g + 15) >> 4);
  // rows at negative positions see nothing; at least one tile, so that rows
  // which see nothing are written too
  const int32_t p0 = max(w.s.len - w.s.n, 0);
  const int32_t lo = a.window > 0 ? max(p0 - a.window, 0) : 0;
  w.t0 = lo / kTile;
  w.tiles = max((w.s.len + kTile - 1) / kTile - w.t0, 1);
  return w;
}

// Warps per block and shared memory: a ring of two tiles (k and v) and the
// query fragments for each warp.
template <int DP, int PARTS>
struct Shape {
  static constexpr int kWarps = DP == 64 ? 8 : DP == 128 ? (PARTS == 1 ? 6 : 5) : (PARTS == 1 ? 3 : 2);
  static constexpr int kStages = 2;
  static constexpr int kQBytes = DP / 16 * 32 * 16 * PARTS;
  // v pages of 16 or 32 tokens lie 32 or 64 bytes apart, so that the quads'
  // reads of different pages fall into different banks
  static constexpr int kVPad = 128;
  static __host__ __device__ int warp_bytes(int D) { return kStages * (2 * kTile * D + kVPad) + kQBytes; }
  static __host__ __device__ int smem_bytes(int D) { return kWarps * (warp_bytes(D) + 2 * kStages * 8) + 128; }
};

template <int DP, int FMT, int PARTS>
__global__ void __launch_bounds__(Shape<DP, PARTS>::kWarps * 32, 1) stream_kernel(const Args a) {
  using Sh = Shape<DP, PARTS>;
  using T = typename std::conditional<PARTS == 1, bf16, float>::type;
  constexpr int NST = Sh::kStages;
  extern __shared__ __align__(128) uint8_t s_attn[];
  const int D = a.c.D, blk = a.c.blk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, qc = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_attn) + warp * 2 * NST;  // k barriers, then v
  uint8_t* mine = s_attn + (Sh::kWarps * 2 * NST * 8 + 127) / 128 * 128 + warp * Sh::warp_bytes(D);
  const int kbytes = kTile * D, vbytes = kTile * D + Sh::kVPad;
  uint8_t* s_k = mine;
  uint8_t* s_v = mine + NST * kbytes;
  uint4* s_q = reinterpret_cast<uint4*>(mine + NST * (kbytes + vbytes));  // [part][k step][lane]
  if (lane < 2 * NST) tc::mbar_init(bars + lane, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();

  // ---- this warp's share of the list
  const int wid = warp * gridDim.x + blockIdx.x;
  int64_t total = 0;
  for (int base = 0; base < a.b.B; base += 32) {
    int64_t n = 0;
    if (base + lane < a.b.B) {
      const SeqWork w = seq_work(a, base + lane);
      n = (int64_t)w.rtiles * w.tiles * a.c.H;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  if (lane == 0) a.desc[wid] = make_int4(-1, 0, 0, 0);
  // no more warps than tiles: every share has one, so a cut unit's parts lie
  // in consecutive warps
  const int64_t warps = min((int64_t)a.warps, total);
  if (wid >= warps) return;
  const int64_t beg = total * wid / warps, end = total * (wid + 1) / warps;
  // ---- find the sequence of `beg`
  int sb = 0;
  int64_t seq0 = 0;  // list position of sequence sb
  {
    bool found = false;
    for (int base = 0; base < a.b.B && !found; base += 32) {
      int64_t n = 0;
      if (base + lane < a.b.B) {
        const SeqWork w = seq_work(a, base + lane);
        n = (int64_t)w.rtiles * w.tiles * a.c.H;
      }
      int64_t incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, seq0 + incl > beg);
      if (hit) {
        const int src = __ffs(hit) - 1;
        sb = base + src;
        seq0 += __shfl_sync(0xffffffffu, incl - n, src);
        found = true;
      } else {
        seq0 += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
  }

  uint32_t kphase = 0, vphase = 0;  // bit s: parity that stage s waits for
  bool dead = false;                // a wait gave up: nothing more is issued or waited for
  int64_t at = beg;
  SeqWork w = seq_work(a, sb);
  int piece = 0;  // pieces of units left as partials by this warp
  while (at < end) {
    const int64_t unit_tiles = w.tiles, seq_units = (int64_t)w.rtiles * a.c.H;
    if (at - seq0 >= unit_tiles * seq_units) {  // next sequence (those without rows are passed over)
      seq0 += unit_tiles * seq_units;
      ++sb;
      w = seq_work(a, sb);
      continue;
    }
    const int64_t u = (at - seq0) / unit_tiles;
    const int64_t u0 = seq0 + u * unit_tiles, u1 = u0 + unit_tiles;
    const int h = (int)(u / w.rtiles), rt = (int)(u % w.rtiles);
    const int64_t stop = min(end, u1);

    // rows of the unit: index e = 16 rt + i is query row e / g, head h g + e % g
    const int nrows = min(16, w.s.n * a.g - 16 * rt);
    const int p_first = w.s.len - w.s.n + (16 * rt) / a.g;
    const int p_last = w.s.len - w.s.n + (16 * rt + nrows - 1) / a.g;
    int qpos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = gr + 8 * i;
      qpos[i] = r < nrows ? w.s.len - w.s.n + (16 * rt + r) / a.g : -1;
    }
    // the unit's own visible tiles, within this warp's share
    const int lo_tok = a.window > 0 ? max(p_first - a.window, 0) : 0;
    const int hi_tok = p_last + 1;  // one past the last visible token
    const int tb = max(w.t0 + (int)(at - u0), lo_tok / kTile);
    const int te = min(w.t0 + (int)(stop - u0), (hi_tok + kTile - 1) / kTile);

    // ---- query fragments
    float qfac[2] = {0.f, 0.f};
    {
      const T* qp[2] = {nullptr, nullptr};
      float mx[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = gr + 8 * i;
        if (r < nrows) {
          const int e = 16 * rt + r;
          qp[i] = static_cast<const T*>(a.q.p) + (int64_t)(w.s.row0 + e / a.g) * a.q.st + (int64_t)(h * a.g + e % a.g) * a.q.sh;
          for (int d = qc; d < D; d += 4) mx[i] = fmaxf(mx[i], fabsf(rope::to_f32(qp[i][d])));
        }
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      }
      float up[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // 2^e <= mx < 2^(e + 1) becomes 2^14: up = 2^(14 - e), within f32's exponents
        int ex = (int)(__float_as_uint(mx[i]) >> 23) - 127;
        ex = max(min(ex, 127), -112);
        up[i] = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
        qfac[i] = a.scale2 * __uint_as_float((uint32_t)(ex - 14 + 127) << 23);
      }
      __syncwarp();
      for (int ks = 0; ks < DP / 16; ++ks) {
        // step ks = 4 j + s takes bytes 4 s .. 4 s + 3 of chunk 4 j + c
        const int d0 = 16 * (4 * (ks >> 2) + qc) + 4 * (ks & 3);
        float v[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) v[i][x] = qp[i] != nullptr && d0 < D ? rope::to_f32(qp[i][d0 + x]) * up[i] : 0.f;
        const uint4 hi = make_uint4(pack_half(v[0][0], v[0][1]), pack_half(v[1][0], v[1][1]), pack_half(v[0][2], v[0][3]),
                                    pack_half(v[1][2], v[1][3]));
        s_q[ks * 32 + lane] = hi;
        if constexpr (PARTS == 2)
          s_q[(DP / 16 + ks) * 32 + lane] =
              make_uint4(pack_rest(v[0][0], v[0][1], hi.x), pack_rest(v[1][0], v[1][1], hi.y),
                         pack_rest(v[0][2], v[0][3], hi.z), pack_rest(v[1][2], v[1][3], hi.w));
      }
      __syncwarp();
    }

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float vref = 1.17549435e-38f;

    // Issue tile t into a stage: every quad lane knows its own page (16-token
    // quarter qc of the tile) and the first quad's lanes issue one copy per
    // page.  Returns the page's scales and whether it can be read.
    const int32_t* table = a.b.table + (int64_t)sb * a.b.tstride;
    const int per_page = blk / 16;  // quarters of a page
    auto issue = [&](int t, int stage, float& ks, float& vs, bool& have) {
      const int tok = t * kTile + 16 * qc;
      have = false;
      ks = vs = 0.f;
      int32_t page = -1;
      if (tok / blk * blk < hi_tok) {
        page = __ldg(table + tok / blk);
        have = page >= 0 && (int64_t)page < a.c.P;
        if (!have) {
          kv::flag(a.c.status, NOOR_KV_BAD_PAGE);
          ks = vs = __uint_as_float(0x7FC00000u);
        }
      }
      const int64_t ph = have ? (int64_t)page * a.c.H + h : 0;
      const bool first = gr == 0 && qc % per_page == 0 && have && !dead;
      const unsigned who = __ballot_sync(0xffffffffu, first);
      const uint32_t bytes = (uint32_t)blk * D;
      if (!dead) {
        if (lane == 0) {
          tc::mbar_arrive_expect_tx(bars + stage, __popc(who) * bytes);
          tc::mbar_arrive_expect_tx(bars + NST + stage, __popc(who) * bytes);
        }
        __syncwarp();
        if (first) {
          const int pg = qc / per_page;
          bulk_load(s_k + stage * kbytes + pg * bytes, a.c.k + ph * bytes, bytes, bars + stage);
          bulk_load(s_v + stage * vbytes + pg * (bytes + 2 * blk), a.c.v + ph * bytes, bytes, bars + NST + stage);
        }
      }
      if (have) {
        ks = __ldg(a.c.ks + ph);
        vs = __ldg(a.c.vs + ph);
      }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (dead || tc::mbar_try_wait(bar, parity)) return;
      const long long start = clock64();
      while (!tc::mbar_try_wait(bar, parity))
        if (clock64() - start > kWaitLimitCycles) {
          dead = true;
          kv::flag(a.c.status, NOOR_KV_TIMEOUT);
          break;
        }
      dead = __any_sync(0xffffffffu, dead);
    };

    float ks_s[NST], vs_s[NST];
    bool have_s[NST];
#pragma unroll
    for (int i = 0; i < NST; ++i)
      if (tb + i < te) issue(tb + i, i, ks_s[i], vs_s[i], have_s[i]);

    for (int t = tb; t < te; ++t) {
      const int stage = (t - tb) % NST;
      const float ks = ks_s[0], vs = vs_s[0];
      const bool have = have_s[0];
      // ---- scores
      wait(bars + stage, (kphase >> stage) & 1);
      kphase ^= 1u << stage;
      float sc[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[i][x] = 0.f;
      const uint8_t* kt = s_k + stage * kbytes + (16 * (gr >> 1) + (gr & 1)) * D + 16 * qc;
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) {
        if (64 * j >= D) break;
        const bool in = 64 * j + 16 * qc < D;
        uint4 qf[4 * PARTS];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          qf[s] = s_q[(4 * j + s) * 32 + lane];
          if constexpr (PARTS == 2) qf[4 + s] = s_q[(DP / 16 + 4 * j + s) * 32 + lane];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint4 kb = make_uint4(0, 0, 0, 0);
          if (in) kb = *reinterpret_cast<const uint4*>(kt + 2 * i * D + 64 * j);
          const uint32_t w4[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            uint32_t b0, b1;
            widen<FMT>(w4[s], b0, b1);
            mma_f16(sc[i], qf[s].x, qf[s].y, qf[s].z, qf[s].w, b0, b1);
            if constexpr (PARTS == 2) mma_f16(sc[i], qf[4 + s].x, qf[4 + s].y, qf[4 + s].z, qf[4 + s].w, b0, b1);
          }
        }
      }
      // ---- scale, mask, running maximum
      const float f0 = qfac[0] * ks, f1 = qfac[1] * ks;
      const int tok0 = t * kTile + 16 * qc;
      const bool whole = t * kTile + kTile - 1 <= p_first && (a.window <= 0 || p_last - t * kTile <= a.window);
      float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v = sc[i][x] * (x < 2 ? f0 : f1);
          if (!whole) {
            const int tok = tok0 + 2 * i + (x & 1), p = qpos[x >> 1];
            if (tok > p || (a.window > 0 && p - tok > a.window)) v = -INFINITY;
          }
          sc[i][x] = v;
          tm[x >> 1] = fmaxf(tm[x >> 1], v);
        }
      float alpha[2], mref[2];
      const float vmax = fmaxf(fabsf(vs), __shfl_xor_sync(0xffffffffu, fabsf(vs), 1));
      const float vnew = fmaxf(vref, fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2)));
      const float vstep = vref / vnew, vrel = vs / vnew;
      vref = vnew;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tm[i] = fmaxf(tm[i], __shfl_xor_sync(0xffffffffu, tm[i], 1));
        tm[i] = fmaxf(tm[i], __shfl_xor_sync(0xffffffffu, tm[i], 2));
        const float mn = fmaxf(m[i], tm[i]);
        mref[i] = mn == -INFINITY ? 0.f : mn - kPShift;
        alpha[i] = mn == -INFINITY ? 1.f : exp2_approx(m[i] - mn);
        m[i] = mn;
      }
      // ---- probabilities (f16 pairs are mma's first operand)
      uint32_t pf[8][2 * PARTS];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float p = exp2_approx(sc[i][x] - mref[x >> 1]);
          sum[x >> 1] += p;
          // a masked token's p is zero whatever its block's scale
          sc[i][x] = sc[i][x] == -INFINITY ? 0.f : p * vrel;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          pf[i][r] = pack_half(sc[i][2 * r], sc[i][2 * r + 1]);
          if constexpr (PARTS == 2) pf[i][2 + r] = pack_rest(sc[i][2 * r], sc[i][2 * r + 1], pf[i][r]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] = l[i] * alpha[i] + sum[i];
        alpha[i] *= vstep;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][x] *= alpha[x >> 1];
      }
      // ---- values; codes past the last visible token (or of a page that
      // could not be read) are whatever the memory holds, and count as zero
      wait(bars + NST + stage, (vphase >> stage) & 1);
      vphase ^= 1u << stage;
      const int nv = have ? min(max(hi_tok - tok0, 0), 16) : 0;
      const bool clip = __any_sync(0xffffffffu, nv < 16);
      uint32_t vm[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = min(max(nv - 4 * s, 0), 4);
        vm[s] = n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
      }
      const uint8_t* vt = s_v + stage * vbytes + (qc / per_page) * (blk * D + 2 * blk) + gr * blk + 16 * (qc % per_page);
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        if (8 * i >= D) break;
        const uint4 vb = *reinterpret_cast<const uint4*>(vt + 8 * i * blk);
        uint32_t w4[4] = {vb.x, vb.y, vb.z, vb.w};
        if (clip)
#pragma unroll
          for (int s = 0; s < 4; ++s) w4[s] &= vm[s];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint32_t b0, b1;
          widen<FMT>(w4[s], b0, b1);
          mma_f16(o[i], pf[2 * s][0], pf[2 * s][1], pf[2 * s + 1][0], pf[2 * s + 1][1], b0, b1);
          if constexpr (PARTS == 2)
            mma_f16(o[i], pf[2 * s][2], pf[2 * s][3], pf[2 * s + 1][2], pf[2 * s + 1][3], b0, b1);
        }
      }
      __syncwarp();  // every lane has read the stage
#pragma unroll
      for (int i = 0; i + 1 < NST; ++i) {
        ks_s[i] = ks_s[i + 1];
        vs_s[i] = vs_s[i + 1];
        have_s[i] = have_s[i + 1];
      }
      if (t + NST < te) issue(t + NST, stage, ks_s[NST - 1], vs_s[NST - 1], have_s[NST - 1]);
    }

    // ---- the unit's result, or this warp's part of it
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (at == u0 && stop == u1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = gr + 8 * i;
        if (r >= nrows) continue;
        const int e = 16 * rt + r, row = w.s.row0 + e / a.g, head = h * a.g + e % a.g;
        const float f = l[i] == 0.f ? 0.f : vref / l[i];
        T* op = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.st + (int64_t)head * a.out.sh;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          if (8 * d >= D) break;
          op[8 * d + 2 * qc] = rope::from_f32<T>(o[d][2 * i] * f);
          op[8 * d + 2 * qc + 1] = rope::from_f32<T>(o[d][2 * i + 1] * f);
        }
        if (a.lse != nullptr && qc == 0)
          a.lse[(int64_t)row * a.Hq + head] =
              l[i] == 0.f ? -INFINITY : (m[i] - kPShift + log2f(l[i])) * 0.69314718055994531f;
      }
    } else {
      const int64_t slot = 2 * (int64_t)wid + (piece > 0 ? 1 : 0);
      float* po = a.part_o + slot * 16 * D;
      float* pm = a.part_ml + slot * 32;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = gr + 8 * i;
        if (r >= nrows) continue;
        if (qc == 0) {
          pm[2 * r] = l[i] == 0.f ? -INFINITY : m[i];
          pm[2 * r + 1] = l[i];
        }
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          if (8 * d >= D) break;
          po[r * D + 8 * d + 2 * qc] = o[d][2 * i] * vref;
          po[r * D + 8 * d + 2 * qc + 1] = o[d][2 * i + 1] * vref;
        }
      }
      if (at == u0 && lane == 0) {
        // the unit goes on past this warp: warps wid .. last hold its parts
        // (the first warp whose share ends at or past u1)
        const int lw = (int)((u1 * warps + total - 1) / total) - 1;
        a.desc[wid] = make_int4(sb, h, rt, (lw << 1) | (piece > 0 ? 1 : 0));
      }
    }
    ++piece;
    at = stop;
  }
}

// Join the parts of one cut unit's row: block (warp that holds the first
// part, row).  The first warp's part may be its last piece (slot 1); every
// later warp's is its first (slot 0).
template <typename T>
__global__ void __launch_bounds__(128) combine_kernel(const Args a) {
  const int wid = blockIdx.x, r = blockIdx.y;
  const int4 d = a.desc[wid];
  if (d.x < 0) return;
  const kv::Seq s = kv::sequence(a.b, a.b.cu, a.b.lens, a.c.blk, d.x, nullptr);
  const int e = 16 * d.z + r;
  if (e >= s.n * a.g) return;
  const int D = a.c.D, last = d.w >> 1;
  const int64_t slot0 = 2 * (int64_t)wid + (d.w & 1);
  float m = -INFINITY;
  for (int i = wid + threadIdx.x; i <= last; i += blockDim.x)
    m = fmaxf(m, a.part_ml[(i == wid ? slot0 : 2 * (int64_t)i) * 32 + 2 * r]);
  __shared__ float s_m[4];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const int row = s.row0 + e / a.g, head = d.y * a.g + e % a.g;
  T* op = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.st + (int64_t)head * a.out.sh;
  for (int c = threadIdx.x; c < D; c += blockDim.x) {
    float acc = 0.f, l = 0.f;
    for (int i = wid; i <= last; ++i) {
      const int64_t slot = i == wid ? slot0 : 2 * (int64_t)i;
      const float mi = a.part_ml[slot * 32 + 2 * r], li = a.part_ml[slot * 32 + 2 * r + 1];
      if (li == 0.f) continue;
      const float f = exp2_approx(mi - m);
      l += li * f;
      acc += a.part_o[(slot * 16 + r) * D + c] * f;
    }
    op[c] = rope::from_f32<T>(l == 0.f ? 0.f : acc / l);
    if (a.lse != nullptr && c == 0)
      a.lse[(int64_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m - kPShift + log2f(l)) * 0.69314718055994531f;
  }
}

}  // namespace attn
}  // namespace noor
