// kv_attention.cuh -- attention over the 8-bit cache, streamed.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),
// with the running maximum m and sum l of the softmax carried over one pass
// through the visible tokens.
//
// For few query rows the time is that of reading the codes once, so the work
// is cut by bytes: the batch's visible 64-token tiles of every (sequence, kv
// head, tile of query rows) form one list, and every warp pair of the grid takes an
// equal contiguous share of it, whatever the sequences' lengths.  A pair works
// alone: its first warp streams the tiles into the pair's own ring in
// shared memory with bulk copies, each warp takes 32 of a tile's 64 tokens and
// keeps its o, m and l in registers, and the two are joined when a unit
// (sequence, head, row tile) ends.  A unit cut between pairs leaves partial
// (m, l, o), which combine_kernel joins in a fixed order.
//
// The products run on mma.sync m16n8k16 in f16 with f32 sums, with tokens (and
// for p v, head dims) as the 16 rows and 8 query rows as the columns: a decode
// step has 1 to 8 query rows for a kv head, which tcgen05's 128-row tiles would
// leave nearly empty, and at one pass per byte the tensor work is far below
// the memory time.  F32 with many rows (NB = 4: 32) shares each widened code.
// Codes (|int8| <= 127, e4m3) are exact in f16.  Queries are
// scaled by a power of two for each row so that f16 holds them: exactly for BF16
// (elements under 2^-38 of the row's largest aside), and for F32 as a sum of
// two f16 parts (22 bits).  Probabilities p are f16 as well, off by 2^-11
// relative, an eighth of the BF16 output's half step (F32: two parts again),
// scaled by 2^14 so that p down to 2^-38 counts in a long context.  A block's
// v scale multiplies its p, relative to the largest scale (up to a power of two)
// among the tokens that the row has seen so far: what a row does not see leaves
// its bits alone.
//
// Measured at 32 / 8 heads of 128 dims: 64 ragged sequences of up to 8192
// tokens, a row each, e4m3, 122-124 us = 5.5 TB/s of codes; 4 x 131072 tokens,
// int8, 215-220 us = 4.9 TB/s.  int8 takes five instructions to widen a word, e4m3
// two: e4m3 is bound by memory, int8 by its pairs' chains (0.50 instructions a
// cycle and scheduler, between waits on shared loads and fixed latencies).  One stream of 1000 tokens
// takes 13 us, the chain of its loads (lengths, page table, codes) and the join.
//
// The contraction index of an mma may be permuted at will if both operands
// agree: thread c of a quad takes 16 consecutive bytes of a key row and feeds
// them to four mma steps, so keys come straight from the stored layout with
// 16-byte shared loads; token 8 (r / 2) + 2 G + r % 2 is row r of score group
// G, which leaves thread c with 8 consecutive tokens of each value row.
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
  bool qvec;       // q can be read four elements at a time
  float scale2;    // scale * log2(e)
  int32_t window;
  // partial results: [slots * pairs] slots of `rows` rows of D o's, and of `rows` (m, l)
  float* part_o;
  float* part_ml;
  int4* desc;      // [pairs] the cut unit that starts in a pair's share: (sequence or -1, head, row tile,
                   // last pair << 1 | slot of its part)
  int32_t slots;   // 2: a pair's first and last piece; tensor-core kernel 1: a block's part of a unit
  int32_t pairs;   // warp pairs of the grid that share the work; tensor-core kernel: blocks with a slot (0: none)
  int32_t sms, seen;  // tensor-core kernel: SMs, and most tiles of 128 tokens that a unit sees
  int32_t rows;    // query rows of a row tile
  int64_t min_e, max_e;  // sequences with min_e <= rows * g < max_e are this launch's
};

// Time of the tensor-core kernel's last SM with each unit cut in s parts, in
// sixteenths of a tile of 128 tokens (2.2 us): a block's start and end cost some
// six tiles, the join four.  BF16 over int8, 512 rows of 16 / 4 heads of
// 128 dims: 8192 tokens 162 us whole, 81 us in four parts; 1024 tokens (1024
// rows) 43 us whole, 49 us in two.
__host__ __device__ inline int part_cost(int units, int tiles, int s, int sms) {
  return (s * units + sms - 1) / sms * (16 * tiles / s + 96) + (s > 1 ? 64 : 0);
}
// Most parts: at least four tiles each, two blocks for an SM, a slot for each.
__host__ __device__ inline int most_parts(int units, int tiles, int sms, int slots) {
  const int blocks = 2 * sms < slots ? 2 * sms : slots, by_blocks = units > 0 ? blocks / units : 0;
  return by_blocks < tiles / 4 ? by_blocks : tiles / 4;
}

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
  int32_t rtiles;    // row tiles of (row, query head of the group)
  int32_t t0, tiles; // first visible 64-token tile and their number, over all rows
};

__device__ __forceinline__ SeqWork seq_work(const Args& a, int i) {
  SeqWork w;
  w.s = kv::sequence(a.b, a.b.cu, a.b.lens, a.c.blk, i, a.c.status);
  if (w.s.len < w.s.n) {  // skipped, as the write does
    kv::flag(a.c.status, NOOR_KV_BAD_LENGTH);
    w.s.n = 0;
  }
  const int64_t e = (int64_t)w.s.n * a.g;
  if (e < a.min_e || e >= a.max_e) w.s.n = 0;
  w.rtiles = (int)(((int64_t)w.s.n * a.g + a.rows - 1) / a.rows);
  const int32_t lo = a.window > 0 ? max(w.s.len - w.s.n - a.window, 0) : 0;
  w.t0 = lo / kTile;
  w.tiles = (w.s.len + kTile - 1) / kTile - w.t0;  // at least one if it has rows: a row sees itself
  return w;
}

// Transpose the 8x8 f16 matrix whose row r, columns 2c, 2c + 1 thread (r, c) holds.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void pair_sync(int pair) {
  asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory");
}

// After a wait gave up: the copies still in flight land before the block can
// end (a stage without any only waits the limit out).
static __device__ __noinline__ void drain(uint64_t* bars, int stages, uint32_t kphase, uint32_t vphase) {
  const long long start = clock64();
  for (int i = 0; i < 2 * stages; ++i) {
    const uint32_t parity = ((i < stages ? kphase : vphase) >> (i % stages)) & 1;
    while (!tc::mbar_try_wait(bars + i, parity) && clock64() - start < kWaitLimitCycles) {
    }
  }
}

// Pairs per block and shared memory: a ring of two tiles (k and v) for each
// pair, and the query fragments where they do not fit into registers.
template <int DP, int PARTS, int NB>
struct Shape {
  static constexpr int kRows = 8 * NB;
  static constexpr bool kQShared = DP / 8 * NB * PARTS > 32;
  static constexpr int kPairs = DP == 64 ? (NB == 1 ? 8 : 4)
                                : DP == 128 ? (NB == 1 ? 6 : 4)
                                            : (NB == 1 ? 3 : 2);
  static constexpr int kStages = 2;
  static constexpr int kQBytes = kQShared ? DP / 16 * NB * PARTS * 32 * 8 : 0;
  // with four column groups, each lane's rows' v references
  static constexpr int kRefBytes = NB > 2 ? 64 * NB * 8 : 0;
  // v pages of 16 or 32 tokens lie 32 or 64 bytes apart, so that the quads'
  // reads of different pages fall into different banks
  static constexpr int kVPad = 128;
  // bytes of the second warp's part when the pair joins (it reuses the ring)
  static constexpr int kJoin = (DP / 16 * NB * 4 + 6 * NB) * 32 * 4;
  static __host__ __device__ int pair_bytes(int D) {
    const int ring = kStages * (2 * kTile * D + kVPad);
    return (ring > kJoin ? ring : kJoin) + kQBytes + kRefBytes;
  }
  static constexpr int kBarBytes = (kPairs * 2 * kStages * 8 + 127) / 128 * 128;
  static __host__ __device__ int smem_bytes(int D) { return kBarBytes + kPairs * pair_bytes(D); }
};

template <int DP, int FMT, int PARTS, int NB>
__global__ void __launch_bounds__(Shape<DP, PARTS, NB>::kPairs * 64, 1) stream_kernel(const Args a) {
  using Sh = Shape<DP, PARTS, NB>;
  using T = typename std::conditional<PARTS == 1, bf16, float>::type;
  constexpr int NST = Sh::kStages, R = Sh::kRows;
  extern __shared__ __align__(128) uint8_t s_attn[];
  const int D = a.c.D, blk = a.c.blk, lblk = 31 - __clz(blk);  // (16, 32 or 64)
  const int pair = threadIdx.x >> 6, half = (threadIdx.x >> 5) & 1, lane = threadIdx.x & 31, gr = lane >> 2, qc = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_attn) + pair * 2 * NST;  // k barriers, then v
  uint8_t* mine = s_attn + Sh::kBarBytes + pair * Sh::pair_bytes(D);
  const int kbytes = kTile * D, vbytes = kTile * D + Sh::kVPad;
  uint8_t* s_k = mine;
  uint8_t* s_v = mine + NST * kbytes;
  float* s_join = reinterpret_cast<float*>(mine);
  uint2* s_q = reinterpret_cast<uint2*>(mine + Sh::pair_bytes(D) - Sh::kQBytes - Sh::kRefBytes);  // [part][k step][nb][lane]
  float* s_ref = reinterpret_cast<float*>(mine + Sh::pair_bytes(D) - Sh::kRefBytes) + 64 * half * NB + 2 * lane;  // [half][nb][lane][2]
  if (half == 0 && lane < 2 * NST) tc::mbar_init(bars + lane, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  pair_sync(pair);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be launched; it waits for this grid's end
  // ---- this pair's share of the list
  const int wid = pair * gridDim.x + blockIdx.x;
  int64_t total = 0, n0 = 0;  // n0: tiles of this lane's sequence among the first 32
  for (int base = 0; base < a.b.B; base += 32) {
    int64_t n = 0;
    if (base + lane < a.b.B) {
      const SeqWork w = seq_work(a, base + lane);
      n = (int64_t)w.rtiles * w.tiles * a.c.H;
    }
    if (base == 0) n0 = n;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  if (wid >= a.pairs) return;
  if (half == 0 && lane == 0) a.desc[wid] = make_int4(-1, 0, 0, 0);
  // no more shares than tiles: every share has one, so a cut unit's parts lie
  // in consecutive pairs
  const int64_t pairs = min((int64_t)a.pairs, total);
  if (wid >= pairs) return;
  const int64_t beg = total * wid / pairs, end = total * (wid + 1) / pairs;
  // ---- find the sequence of `beg`
  int sb = 0;
  int64_t seq0 = 0;  // list position of sequence sb
  {
    bool found = false;
    for (int base = 0; base < a.b.B && !found; base += 32) {
      int64_t n = n0;
      if (base > 0) {
        n = 0;
        if (base + lane < a.b.B) {
          const SeqWork w = seq_work(a, base + lane);
          n = (int64_t)w.rtiles * w.tiles * a.c.H;
        }
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
  int piece = 0;  // pieces of units so far
  const int my_tok = 8 * (gr >> 1) + (gr & 1);  // this lane's token of score group 0, within its warp's 32
  const float nan = __uint_as_float(0x7FC00000u);
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

    // rows of the unit: index e = R rt + i is query row e / g, head h g + e % g
    const int e0 = R * rt;
    const int nrows = min(R, w.s.n * a.g - e0);
    const int pos0 = w.s.len - w.s.n;
    const int p_first = pos0 + e0 / a.g;
    const int p_last = pos0 + (e0 + nrows - 1) / a.g;
    // the unit's own visible tiles, within this pair's share
    const int lo_tok = a.window > 0 ? max(p_first - a.window, 0) : 0;
    const int hi_tok = p_last + 1;  // one past the last visible token
    const int tb = max(w.t0 + (int)(at - u0), lo_tok / kTile);
    const int te = min(w.t0 + (int)(stop - u0), (hi_tok + kTile - 1) / kTile);

    // Query rows: lane (row gr of each group of 8, c) loads dims d0 .. d0 + 3 of
    // step ks = 4 j + s, d0 = 16 (4 j + c) + 4 s, so that the quad's four lanes
    // hold the whole row between them; the loads are in flight together and
    // with those of the page table.
    kv::Raw4<T> raw[NB][DP / 16];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = 8 * nb + gr, e = e0 + r;
      const T* qp = nullptr;
      if (r < nrows)
        qp = static_cast<const T*>(a.q.p) + (int64_t)(w.s.row0 + e / a.g) * a.q.st + (int64_t)(h * a.g + e % a.g) * a.q.sh;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const int d0 = 16 * (4 * (ks >> 2) + qc) + 4 * (ks & 3);
        raw[nb][ks] = kv::Raw4<T>{};
        if (qp != nullptr && d0 < D)
          raw[nb][ks] = a.qvec ? *reinterpret_cast<const kv::Raw4<T>*>(qp + d0)
                               : kv::four(qp[d0], qp[d0 + 1], qp[d0 + 2], qp[d0 + 3]);
      }
    }
    // Page numbers and scales of 32 pages at a time, a page for each lane: the
    // list in use and the one after it, loaded a list ahead, so that no tile
    // waits for the page table.  -1: past the visible tokens; -2: unreadable
    // (its scales are NaN).
    const int32_t* table = a.b.table + (int64_t)sb * a.b.tstride;
    const int tile_pages = kTile >> lblk, page0 = tb * tile_pages, page_end = (hi_tok + blk - 1) >> lblk;
    auto list_pages = [&](int first) -> int32_t {
      const int i = first + lane;
      return i < page_end ? __ldg(table + i) : -1;
    };
    auto list_scales = [&](int first, int32_t& pg, float& ks, float& vs) {
      ks = vs = 0.f;
      if (first + lane < page_end) {
        if (pg < 0 || (int64_t)pg >= a.c.P) {
          kv::flag(a.c.status, NOOR_KV_BAD_PAGE);
          pg = -2;
          ks = vs = nan;
        } else {
          const int64_t ph = (int64_t)pg * a.c.H + h;
          ks = kv::read_scale(__ldg(a.c.ks + ph));
          vs = kv::read_scale(__ldg(a.c.vs + ph));
        }
      }
    };
    int32_t pg = list_pages(page0), pg_next = list_pages(page0 + 32);
    float pks, pvs, pks_next = 0.f, pvs_next = 0.f;
    list_scales(page0, pg, pks, pvs);
    // The first warp issues tile t into a stage: lane p one copy for page p of
    // the tile, at place `at` of the list.
    auto issue = [&](int32_t list, int at, int stage) {
      const int32_t page = __shfl_sync(0xffffffffu, list, (at + lane) & 31);
      const bool mine = lane < tile_pages && page >= 0;
      if (dead) return;
      const unsigned who = __ballot_sync(0xffffffffu, mine);
      const uint32_t bytes = (uint32_t)blk * D;
      if (lane == 0) {
        tc::mbar_arrive_expect_tx(bars + stage, __popc(who) * bytes);
        tc::mbar_arrive_expect_tx(bars + NST + stage, __popc(who) * bytes);
      }
      __syncwarp();
      if (mine) {
        const int64_t ph = ((int64_t)page * a.c.H + h) * bytes;
        bulk_load(s_k + stage * kbytes + lane * bytes, a.c.k + ph, bytes, bars + stage);
        bulk_load(s_v + stage * vbytes + lane * (bytes + 2 * blk), a.c.v + ph, bytes, bars + NST + stage);
      }
    };
    // Each lane waits for itself; the warp votes once all its lanes are back (a
    // barrier's test may answer them differently).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      bool gave_up = false;
      if (!dead && !tc::mbar_try_wait(bar, parity)) {
        const long long start = clock64();
        while (!gave_up && !tc::mbar_try_wait(bar, parity))
          if (clock64() - start > kWaitLimitCycles) {
            gave_up = true;
            kv::flag(a.c.status, NOOR_KV_TIMEOUT);
            drain(bars, NST, kphase, vphase);
          }
      }
      if (__any_sync(0xffffffffu, gave_up)) dead = true;
    };

    if (half == 0) {
#pragma unroll
      for (int i = 0; i < NST; ++i)
        if (tb + i < te) issue(pg, i * tile_pages, i);
    }

    // ---- query fragments
    uint2 qreg[Sh::kQShared ? 1 : PARTS * DP / 16 * NB];
    float qfac[NB][2];  // score factors of rows 2c, 2c + 1 of each group
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const float4 v = kv::widen4(raw[nb][ks], false);
        mx = fmaxf(fmaxf(fmaxf(mx, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^e <= mx < 2^(e + 1) becomes 2^14: up = 2^(14 - e), within f32's exponents
      const int ex = max(min((int)(__float_as_uint(mx) >> 23) - 127, 127), -112);
      const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
      // (an infinite element's scores would be infinities, and a row with none above
      // -inf would look like one that sees nothing: they are NaN)
      const float down = mx <= 3.4028235e38f ? a.scale2 * __uint_as_float((uint32_t)(ex - 14 + 127) << 23) : nan;
      qfac[nb][0] = __shfl_sync(0xffffffffu, down, 8 * qc);
      qfac[nb][1] = __shfl_sync(0xffffffffu, down, 8 * qc + 4);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        const float4 v = kv::widen4(raw[nb][ks], false);
        const uint2 hi = make_uint2(pack_half(v.x * up, v.y * up), pack_half(v.z * up, v.w * up));
        const uint2 lo = make_uint2(pack_rest(v.x * up, v.y * up, hi.x), pack_rest(v.z * up, v.w * up, hi.y));
        if constexpr (Sh::kQShared) {
          if (half == 0) {  // both warps use it
            s_q[(ks * NB + nb) * 32 + lane] = hi;
            if constexpr (PARTS == 2) s_q[((DP / 16 + ks) * NB + nb) * 32 + lane] = lo;
          }
        } else {
          qreg[ks * NB + nb] = hi;
          if constexpr (PARTS == 2) qreg[(DP / 16 + ks) * NB + nb] = lo;
        }
      }
    }
    if constexpr (Sh::kQShared) pair_sync(pair);
    int qpos[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < 2; ++x) qpos[nb][x] = pos0 + (e0 + 8 * nb + 2 * qc + x) / a.g;

    float o[DP / 16][NB][4];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][nb][x] = 0.f;
    float m[NB][2], l[NB][2];
    // One over each row's largest v scale so far, up to a power of two: in
    // registers, or with four column groups (whose sums leave none) in shared
    // memory, a place of its own for each lane (one for the eight lanes of a row
    // would need the warp to meet between its reads and writes: 6% of the time).
    float vreg[NB][2];
    auto vinv = [&](int nb, int x) -> float& {
      if constexpr (NB <= 2)
        return vreg[nb][x];
      else
        return s_ref[64 * nb + x];
    };
    float vlow = 1.17549435e-38f;  // the smallest of the rows' references, or less
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[nb][x] = -INFINITY;
        l[nb][x] = 0.f;
        vinv(nb, x) = kv::kMostScale;  // (2^126)
      }

    // Fixed parts of this lane's addresses: its score tokens' page and rows, its
    // value tokens' page and bytes.
    const int k_page = (32 * half + 8 * (gr >> 1)) >> lblk, v_page = (32 * half + 8 * qc) >> lblk;
    const uint8_t* k_lane = s_k + (32 * half + my_tok) * D + 16 * qc;
    const uint8_t* v_lane = s_v + v_page * (blk * D + 2 * blk) + gr * blk + ((32 * half + 8 * qc) & (blk - 1));
    bool list_bad = __any_sync(0xffffffffu, pg == -2);
    // One tile, compiled apart for tiles that every row sees whole and whose
    // pages can be read: those need no mask.
    auto tile = [&](auto all, int t, int stage, int place) {
      constexpr bool whole = decltype(all)::value;
      const float ks = __shfl_sync(0xffffffffu, pks, place + k_page), vs = __shfl_sync(0xffffffffu, pvs, place + k_page);
      const int tok0 = t * kTile + 32 * half;
      // ---- scores of this warp's 32 tokens
      wait(bars + stage, (kphase >> stage) & 1);
      kphase ^= 1u << stage;
      float sc[2][NB][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[i][nb][x] = 0.f;
      const uint8_t* kt = k_lane + stage * kbytes;
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) {
        if (64 * j >= D) break;
        const bool in = 64 * j + 16 * qc < D;
        uint4 kb[4];
#pragma unroll
        for (int G = 0; G < 4; ++G) {
          kb[G] = make_uint4(0, 0, 0, 0);
          if (in) kb[G] = *reinterpret_cast<const uint4*>(kt + 2 * G * D + 64 * j);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint2 qf[PARTS][NB];
#pragma unroll
          for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const int qi = (pt * DP / 16 + 4 * j + s) * NB + nb;
              qf[pt][nb] = Sh::kQShared ? s_q[qi * 32 + lane] : qreg[Sh::kQShared ? 0 : qi];
            }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 x0 = kb[2 * i], x1 = kb[2 * i + 1];
            const uint32_t w0 = s == 0 ? x0.x : s == 1 ? x0.y : s == 2 ? x0.z : x0.w;
            const uint32_t w1 = s == 0 ? x1.x : s == 1 ? x1.y : s == 2 ? x1.z : x1.w;
            uint32_t a0, a1, a2, a3;
            widen<FMT>(w0, a0, a2);
            widen<FMT>(w1, a1, a3);
#pragma unroll
            for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) mma_f16(sc[i][nb], a0, a1, a2, a3, qf[pt][nb].x, qf[pt][nb].y);
          }
        }
      }
      // ---- scale, mask, running maximum
      float alpha[NB][2], mref[NB][2];
      const float vmax = fmaxf(fmaxf(vs, 0.f), __shfl_xor_sync(0xffffffffu, vs, 16));
      const float vup = kv::power_up(vmax);
      const bool vgrow = vup > vlow;
      bool moved = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float tm[2] = {-INFINITY, -INFINITY}, vseen[2] = {0.f, 0.f};  // (masked) largest scale that the row sees here
        const float f0 = qfac[nb][0] * ks, f1 = qfac[nb][1] * ks;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float v = sc[i][nb][x] * ((x & 1) ? f1 : f0);
            if constexpr (!whole) {
              const int tok = tok0 + my_tok + 2 * (2 * i + (x >> 1)), p = qpos[nb][x & 1];
              if (tok > p || (a.window > 0 && p - tok > a.window))
                v = -INFINITY;
              else
                vseen[x & 1] = fmaxf(vs, 0.f);
            }
            sc[i][nb][x] = v;
            tm[x & 1] = fmaxf(tm[x & 1], v);
          }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          tm[x] = fmaxf(tm[x], __shfl_xor_sync(0xffffffffu, tm[x], 4));
          tm[x] = fmaxf(tm[x], __shfl_xor_sync(0xffffffffu, tm[x], 8));
          tm[x] = fmaxf(tm[x], __shfl_xor_sync(0xffffffffu, tm[x], 16));
          const float mn = fmaxf(m[nb][x], tm[x]);
          mref[nb][x] = mn == -INFINITY ? 0.f : mn - kPShift;
          alpha[nb][x] = mn == -INFINITY ? 1.f : exp2_approx(m[nb][x] - mn);
          m[nb][x] = mn;
          l[nb][x] *= alpha[nb][x];
          if constexpr (!whole) {
            vseen[x] = fmaxf(vseen[x], __shfl_xor_sync(0xffffffffu, vseen[x], 4));
            vseen[x] = fmaxf(vseen[x], __shfl_xor_sync(0xffffffffu, vseen[x], 8));
            vseen[x] = fmaxf(vseen[x], __shfl_xor_sync(0xffffffffu, vseen[x], 16));
          }
          if (!whole || vgrow) {
            const float was = vinv(nb, x), now = fminf(was, kv::power_inverse(whole ? vup : kv::power_up(vseen[x])));
            alpha[nb][x] *= now * kv::power_inverse(was);
            vinv(nb, x) = now;
          }
          moved |= alpha[nb][x] != 1.f;
        }
      }
      if (whole && vgrow) vlow = vup;
      // ---- probabilities, transposed into the second operand's layout
      uint32_t pf[PARTS][NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float sum[2] = {0.f, 0.f};
        const float vrel[2] = {vs * vinv(nb, 0), vs * vinv(nb, 1)};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float p = exp2_approx(sc[i][nb][x] - mref[nb][x & 1]);
            sum[x & 1] += p;
            // a masked token's p is zero whatever its block's scale
            sc[i][nb][x] = !whole && sc[i][nb][x] == -INFINITY ? 0.f : p * vrel[x & 1];
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t hi = pack_half(sc[i][nb][2 * y], sc[i][nb][2 * y + 1]);
            pf[0][nb][2 * i + y] = transpose8(hi);
            if constexpr (PARTS == 2) pf[1][nb][2 * i + y] = transpose8(pack_rest(sc[i][nb][2 * y], sc[i][nb][2 * y + 1], hi));
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) l[nb][x] += sum[x];
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][nb][x] *= alpha[nb][x & 1];
      }
      // ---- values; codes past the last visible token (or of a page that
      // could not be read) are whatever the memory holds, and count as zero
      wait(bars + NST + stage, (vphase >> stage) & 1);
      vphase ^= 1u << stage;
      uint32_t vm0 = 0xFFFFFFFFu, vm1 = 0xFFFFFFFFu;
      if constexpr (!whole) {
        const bool vhave = __shfl_sync(0xffffffffu, pg, place + v_page) >= 0;  // of tokens 8c .. 8c + 7
        const int nv = vhave ? min(max(hi_tok - (tok0 + 8 * qc), 0), 8) : 0;
        vm0 = nv >= 4 ? 0xFFFFFFFFu : (1u << (8 * nv)) - 1u;
        vm1 = nv >= 8 ? 0xFFFFFFFFu : nv <= 4 ? 0u : (1u << (8 * (nv - 4))) - 1u;
      }
      const uint8_t* vt = v_lane + stage * vbytes;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        if (16 * i >= D) break;
        uint2 v0 = *reinterpret_cast<const uint2*>(vt + 16 * i * blk);
        uint2 v1 = *reinterpret_cast<const uint2*>(vt + (16 * i + 8) * blk);
        if constexpr (!whole) {
          v0.x &= vm0; v0.y &= vm1; v1.x &= vm0; v1.y &= vm1;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t a0, a1, a2, a3;
          widen<FMT>(y ? v0.y : v0.x, a0, a2);
          widen<FMT>(y ? v1.y : v1.x, a1, a3);
#pragma unroll
          for (int pt = 0; pt < PARTS; ++pt)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_f16(o[i][nb], a0, a1, a2, a3, pf[pt][nb][2 * y], pf[pt][nb][2 * y + 1]);
        }
      }
    };
    for (int t = tb; t < te; ++t) {
      const int stage = (t - tb) % NST, place = (t - tb) * tile_pages & 31;  // of the tile's first page in the list
      const int tok0 = t * kTile + 32 * half;
      if (tok0 + 31 <= p_first && (a.window <= 0 || p_last - tok0 <= a.window) && !list_bad)
        tile(std::true_type{}, t, stage, place);
      else
        tile(std::false_type{}, t, stage, place);
      pair_sync(pair);  // both warps have read the stage
      if (t + NST < te && half == 0) {
        const int at = place + NST * tile_pages;
        if (at < 32)
          issue(pg, at, stage);
        else
          issue(pg_next, at - 32, stage);
      }
      // halfway through a list the next one's pages are there: load its scales
      if (place == 16) list_scales(page0 + ((t - tb) * tile_pages & ~31) + 32, pg_next, pks_next, pvs_next);
      if (place + tile_pages == 32) {  // to the next list
        pg = pg_next;
        pks = pks_next;
        pvs = pvs_next;
        list_bad = __any_sync(0xffffffffu, pg == -2);
        pg_next = list_pages(page0 + (t + 1 - tb) * tile_pages + 32);
      }
    }

    // ---- join the pair: the second warp hands its part to the first through
    // the ring, which no copy is filling now
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[nb][x] += __shfl_xor_sync(0xffffffffu, l[nb][x], s);
    if (tb >= te) pair_sync(pair);  // no tile parted this piece from the last one's join
    if (half == 1) {
      float* j = s_join + lane;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          j[(4 * nb + 2 * x) * 32] = m[nb][x];
          j[(4 * nb + 2 * x + 1) * 32] = l[nb][x];
          j[(4 * NB + 2 * nb + x) * 32] = kv::power_inverse(vinv(nb, x));
        }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int x = 0; x < 4; ++x) j[(6 * NB + (i * NB + nb) * 4 + x) * 32] = o[i][nb][x];
    }
    pair_sync(pair);
    if (half == 0) {
      const float* j = s_join + lane;
      const bool done = at == u0 && stop == u1;
      const int64_t slot = 2 * (int64_t)wid + (piece > 0 ? 1 : 0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float m1 = j[(4 * nb + 2 * x) * 32], l1 = j[(4 * nb + 2 * x + 1) * 32];
          const float mm = fmaxf(m[nb][x], m1);
          // a side without visible tokens has m = -inf, l = 0 and o = 0
          const float f0 = l[nb][x] == 0.f ? 0.f : exp2_approx(m[nb][x] - mm), f1 = l1 == 0.f ? 0.f : exp2_approx(m1 - mm);
          const float ll = l[nb][x] * f0 + l1 * f1;
          const int r = 8 * nb + 2 * qc + x;
          if (r >= nrows) continue;
          const int e = e0 + r, row = w.s.row0 + e / a.g, head = h * a.g + e % a.g;
          const float inv = !done ? 1.f : ll == 0.f ? 0.f : 1.f / ll;
          const float g0 = f0 * kv::power_inverse(vinv(nb, x)) * inv, g1 = f1 * j[(4 * NB + 2 * nb + x) * 32] * inv;
          if (gr == 0) {
            if (!done) {
              a.part_ml[(slot * R + r) * 2] = ll == 0.f ? -INFINITY : mm;
              a.part_ml[(slot * R + r) * 2 + 1] = ll;
            } else if (a.lse != nullptr) {
              a.lse[(int64_t)row * a.Hq + head] =
                  ll == 0.f ? -INFINITY : (mm - kPShift + log2f(ll)) * 0.69314718055994531f;
            }
          }
          T* op = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.st + (int64_t)head * a.out.sh;
          float* po = a.part_o + (slot * R + r) * D;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            if (16 * i >= D) break;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int d = 16 * i + 8 * y + gr;
              const float v = o[i][nb][2 * y + x] * g0 + j[(6 * NB + (i * NB + nb) * 4 + 2 * y + x) * 32] * g1;
              if (done)
                op[d] = rope::from_f32<T>(v);
              else
                po[d] = v;
            }
          }
        }
      if (!done && at == u0 && lane == 0) {
        // the unit goes on past this pair: pairs wid .. lw hold its parts
        // (the first pair whose share ends at or past u1)
        const int lw = (int)((u1 * pairs + total - 1) / total) - 1;
        a.desc[wid] = make_int4(sb, h, rt, (lw << 1) | (piece > 0 ? 1 : 0));
      }
      // the next piece's copies overwrite what ordinary stores wrote
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    ++piece;
    at = stop;
  }
}

// Join the parts of one cut unit: a block for the pair that holds the first
// part and 8 of its rows, a warp for each row.  The first pair's part may be
// its last piece (slot 1); every later pair's is its first (slot 0).  A lane
// weighs one part (32 at a time), then all lanes sum 4 dims each over the
// parts, in the parts' order.  Bound by latency: it adds some 4 us.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32, 4) combine_kernel(const Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched while the streamed kernel still runs)
  const int wid = blockIdx.x, lane = threadIdx.x & 31;
  const int4 d = a.desc[wid];  // (written while this grid waits: not a read-only load)
  if (d.x < 0) return;
  const int r = min(blockIdx.y * kJoinWarps + (threadIdx.x >> 5), (unsigned)a.rows - 1u);
  const int D = a.c.D, parts = (d.w >> 1) - wid + 1;
  auto slot = [&](int i) -> int64_t {  // row r of part i
    return (a.slots * ((int64_t)wid + i) + (i == 0 ? (d.w & 1) : 0)) * a.rows + r;
  };
  // (rows past the unit's read their slots and write nothing: the loads need not
  // wait for the sequence's)
  const float2 none = make_float2(-INFINITY, 0.f);
  auto part = [&](int i) { return i < parts ? *reinterpret_cast<const float2*>(a.part_ml + slot(i) * 2) : none; };
  const float2 ml0 = part(lane);
  const kv::Seq s = kv::sequence(a.b, a.b.cu, a.b.lens, a.c.blk, d.x, nullptr);
  float m = ml0.x;
  for (int i = lane + 32; i < parts; i += 32) m = fmaxf(m, part(i).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int base = 0; base < parts; base += 32) {
    const int n = min(32, parts - base);
    const float2 ml = base == 0 ? ml0 : part(base + lane);
    const float w = ml.y == 0.f ? 0.f : exp2_approx(ml.x - m), wl = ml.y * w;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float f = __shfl_sync(0xffffffffu, w, i);
      l += __shfl_sync(0xffffffffu, wl, i);
      const float* po = a.part_o + slot(base + i) * D;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int c = 4 * lane + 128 * y;
        if (c < D) {
          const float4 v = *reinterpret_cast<const float4*>(po + c);
          acc[4 * y] = fmaf(v.x, f, acc[4 * y]);
          acc[4 * y + 1] = fmaf(v.y, f, acc[4 * y + 1]);
          acc[4 * y + 2] = fmaf(v.z, f, acc[4 * y + 2]);
          acc[4 * y + 3] = fmaf(v.w, f, acc[4 * y + 3]);
        }
      }
    }
  }
  const int64_t e = (int64_t)a.rows * d.z + r;
  if (blockIdx.y * kJoinWarps + (threadIdx.x >> 5) >= (unsigned)a.rows || e >= (int64_t)s.n * a.g) return;
  const int row = s.row0 + (int)(e / a.g), head = d.y * a.g + (int)(e % a.g);
  T* op = static_cast<T*>(const_cast<void*>(a.out.p)) + (int64_t)row * a.out.st + (int64_t)head * a.out.sh;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int y = 0; y < 2; ++y)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = 4 * lane + 128 * y + x;
      if (c < D) op[c] = rope::from_f32<T>(acc[4 * y + x] * inv);
    }
  if (a.lse != nullptr && lane == 0)
    a.lse[(int64_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m - kPShift + log2f(l)) * 0.69314718055994531f;
}

}  // namespace attn
}  // namespace noor
