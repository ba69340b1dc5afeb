// noor_attention.cu -- C ABI of the attention half of a block: rotary
// positions, the paged 8-bit cache (write, read back) and attention over it.
// Every entry point checks its host arguments, sets the device for the call,
// enqueues on the caller's stream and allocates nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <exception>
#include <initializer_list>
#include <type_traits>

#include "noor_moe.h"

#include "common.cuh"
#include "host.h"
#include "kv_attention.cuh"
#include "kv_cache.cuh"
#include "kv_stream.h"
#include "rope.cuh"

using namespace noor;

namespace {

// C callers never see an exception.
template <typename F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return NOOR_MOE_ERR_OOM;
  } catch (...) {
    return NOOR_MOE_ERR_OOM;
  }
}

int check_device(int dev) {
  int n = 0;
  CK(cudaGetDeviceCount(&n));
  if (dev < 0 || dev >= n) return fail(NOOR_MOE_ERR_INVALID, "device %d not in 0 .. %d", dev, n - 1);
  return NOOR_MOE_OK;
}

// Streaming multiprocessors of a device (looked up once).
int sm_count(int dev, int* out) {
  static std::mutex mu;
  static int known[64] = {0};
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && known[dev]) {
    *out = known[dev];
    return NOOR_MOE_OK;
  }
  CK(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) known[dev] = *out;
  return NOOR_MOE_OK;
}

int check_dtype(int dtype) {
  if (dtype != NOOR_DTYPE_F32 && dtype != NOOR_DTYPE_BF16) return fail(NOOR_MOE_ERR_INVALID, "unknown dtype %d", dtype);
  return NOOR_MOE_OK;
}

size_t esize(int dtype) { return dtype == NOOR_DTYPE_BF16 ? 2 : 4; }

int check_rotary(const noor_rotary* r, int D) {
  if (r->rotate_dim < 0 || r->rotate_dim % 2 != 0 || r->rotate_dim > D)
    return fail(NOOR_MOE_ERR_INVALID, "rotate_dim %d is not an even number in 0 .. %d", r->rotate_dim, D);
  if (r->layout != NOOR_ROPE_INTERLEAVED && r->layout != NOOR_ROPE_HALF)
    return fail(NOOR_MOE_ERR_INVALID, "unknown rotary layout %d", r->layout);
  if (r->rotate_dim > 0 && !r->inv_freq) return fail(NOOR_MOE_ERR_INVALID, "null inv_freq");
  return NOOR_MOE_OK;
}

int check_view(const noor_heads* v, int dtype, const char* what) {
  if (!v || !v->data) return fail(NOOR_MOE_ERR_INVALID, "null %s", what);
  if (reinterpret_cast<uintptr_t>(v->data) % esize(dtype) != 0)
    return fail(NOOR_MOE_ERR_INVALID, "%s is not aligned to its elements", what);
  return NOOR_MOE_OK;
}

// An output's heads lie apart: two of them that share elements would be written
// by two threads at once.  (Strides that overlap in other ways are the caller's.)
int check_out(const noor_heads* v, int64_t tokens, int heads, int D, int dtype, const char* what) {
  CKR(check_view(v, dtype, what));
  if ((tokens > 1 && std::abs(v->token_stride) < D) || (heads > 1 && std::abs(v->head_stride) < D))
    return fail(NOOR_MOE_ERR_INVALID, "%s: heads of %d elements overlap (strides %lld and %lld)", what, D,
                (long long)v->token_stride, (long long)v->head_stride);
  return NOOR_MOE_OK;
}

rope::View view(const noor_heads* v) {
  return v ? rope::View{v->data, v->token_stride, v->head_stride} : rope::View{nullptr, 0, 0};
}

bool vector_rows(const rope::View& v, int dtype) {
  const size_t e = esize(dtype);
  return reinterpret_cast<uintptr_t>(v.p) % 16 == 0 && v.st * (int64_t)e % 16 == 0 && v.sh * (int64_t)e % 16 == 0;
}

// 16-byte vectors fit the heads of `views` and the rotary layout.
bool vector_heads(const rope::Args& a, int dtype, std::initializer_list<rope::View> views) {
  const int n = 16 / (int)esize(dtype);
  if (a.D % n != 0 || (a.layout == rope::HALF && a.rot / 2 % n != 0)) return false;
  for (const auto& v : views)
    if (v.p && !vector_rows(v, dtype)) return false;
  return true;
}

template <typename F>
int by_dtype(int dtype, F&& f) {
  return dtype == NOOR_DTYPE_BF16 ? f(bf16{}) : f(float{});
}

int check_cache(const noor_kv_cache* c) {
  if (!c) return fail(NOOR_MOE_ERR_INVALID, "null cache");
  if (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale) return fail(NOOR_MOE_ERR_INVALID, "null cache array");
  for (const void* p : {(const void*)c->k_codes, (const void*)c->v_codes, (const void*)c->k_scale, (const void*)c->v_scale})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return fail(NOOR_MOE_ERR_INVALID, "cache arrays must be 16-byte aligned");
  if (c->block != 16 && c->block != 32 && c->block != 64)
    return fail(NOOR_MOE_ERR_UNSUPPORTED, "block %d is not 16, 32 or 64", c->block);
  if (c->head_dim <= 0 || c->head_dim % 16 != 0 || c->head_dim > 256)
    return fail(NOOR_MOE_ERR_UNSUPPORTED, "head_dim %d is not a multiple of 16 up to 256", c->head_dim);
  if (c->format != NOOR_KV_INT8 && c->format != NOOR_KV_E4M3)
    return fail(NOOR_MOE_ERR_INVALID, "unknown cache format %d", c->format);
  if (c->num_blocks <= 0 || c->num_blocks > INT32_MAX || c->n_kv_heads <= 0 || c->n_kv_heads > 4096)
    return fail(NOOR_MOE_ERR_INVALID, "num_blocks or n_kv_heads out of range");
  if (c->device < 0) return fail(NOOR_MOE_ERR_INVALID, "device %d", c->device);
  return NOOR_MOE_OK;
}

int check_batch(const noor_kv_cache* c, const noor_kv_batch* b, bool need_lens = true) {
  if (!b || !b->block_table || (need_lens && !b->kv_lens) || !b->cu_rows) return fail(NOOR_MOE_ERR_INVALID, "null batch argument");
  if (b->batch <= 0 || b->batch > (1 << 20)) return fail(NOOR_MOE_ERR_INVALID, "batch %d out of range", b->batch);
  if (b->n_rows < 0 || b->n_rows > (1 << 28)) return fail(NOOR_MOE_ERR_INVALID, "n_rows out of range");
  if (b->max_blocks <= 0 || (int64_t)b->max_blocks * c->block > (1 << 30) || b->table_stride < 0)
    return fail(NOOR_MOE_ERR_INVALID, "max_blocks or table_stride out of range");
  return NOOR_MOE_OK;
}

// The write and the read back number the blocks that 256 sequences touch in 32
// bits; row offsets that overlap may give each of them all the rows.
int check_touched(const noor_kv_cache* c, const noor_kv_batch* b) {
  if (b->n_rows / c->block + 2 > INT32_MAX / 256) return fail(NOOR_MOE_ERR_INVALID, "n_rows out of range");
  return NOOR_MOE_OK;
}

kv::Cache cache_of(const noor_kv_cache* c) {
  return kv::Cache{static_cast<uint8_t*>(c->k_codes), static_cast<uint8_t*>(c->v_codes), c->k_scale, c->v_scale,
                   c->status, c->num_blocks, c->n_kv_heads, c->head_dim, c->block};
}

kv::Batch batch_of(const noor_kv_batch* b) {
  return kv::Batch{b->block_table, b->table_stride, b->kv_lens, b->cu_rows, b->n_rows, b->batch, b->max_blocks};
}

// The most blocks that a batch's rows can touch: each sequence with n rows
// touches at most (n - 1) / block + 2 of them and at most n.
int64_t most_tasks(const noor_kv_cache* c, const noor_kv_batch* b) {
  return std::min<int64_t>(b->n_rows, b->n_rows / c->block + 2 * std::min<int64_t>(b->batch, b->n_rows));
}

// kv heads that one grid block takes in turn, so that finding its place and
// (for keys) the angles is paid for once: as many as leave eight blocks for
// every SM, at most 8.  Against one head, at 8 kv heads of 128
// dims: 8 ragged prompts of up to 4096 tokens written and read back in 145 us
// instead of 201, 32 ragged prefixes of up to 4096 read back in 94 instead of 115.
int heads_per_block(const noor_kv_cache* c, int64_t tasks, int32_t* heads) {
  int sms = 0;
  CKR(sm_count(c->device, &sms));
  *heads = 1;
  while (*heads < 8 && *heads < c->n_kv_heads && tasks * c->n_kv_heads / (2 * *heads) >= 8 * (int64_t)sms) *heads *= 2;
  return NOOR_MOE_OK;
}

// Elements of k from which q, k and v get a launch each: below, launches cost
// more than the registers that they free.  4 / 8 kv heads of 128 dims, BF16:
// 2048 rows 16.4 / 25.9 us in one launch, 17.5 / 22.6 in three; 4096 rows
// 26.0 / 53.2 and 22.6 / 40.4 (F32 alike).
constexpr int64_t kApartElements = 3 << 19;

// Four elements of a head can be loaded at once from any multiple of four.
bool four_elements(const rope::View& v, int dtype) {
  const size_t e = esize(dtype);
  return reinterpret_cast<uintptr_t>(v.p) % (4 * e) == 0 && v.st % 4 == 0 && v.sh % 4 == 0;
}

}  // namespace

extern "C" {

int noor_rope_apply(const noor_rotary* r, const noor_heads* q, const noor_heads* q_out, int32_t q_heads,
                    const noor_heads* k, const noor_heads* k_out, int32_t k_heads, const int32_t* positions,
                    int64_t tokens, int32_t head_dim, int32_t dtype, int32_t inverse, int32_t device, void* stream) {
  return guarded([&]() -> int {
    if (!r) return fail(NOOR_MOE_ERR_INVALID, "null rotary");
    CKR(check_dtype(dtype));
    if (head_dim <= 0 || head_dim % 2 != 0 || head_dim > 1024)
      return fail(NOOR_MOE_ERR_UNSUPPORTED, "head_dim %d is not an even number up to 1024", head_dim);
    CKR(check_rotary(r, head_dim));
    if (tokens < 0 || tokens > (1 << 28) || q_heads <= 0 || q_heads > 4096 || (k && (k_heads <= 0 || k_heads > 4096)))
      return fail(NOOR_MOE_ERR_INVALID, "tokens or heads out of range");
    if (tokens == 0) return NOOR_MOE_OK;
    CKR(check_view(q, dtype, "q"));
    CKR(check_out(q_out, tokens, q_heads, head_dim, dtype, "q_out"));
    if (k) CKR(check_view(k, dtype, "k"));
    if (k) CKR(check_out(k_out, tokens, k_heads, head_dim, dtype, "k_out"));
    if (!positions) return fail(NOOR_MOE_ERR_INVALID, "null positions");
    CKR(check_device(device));
    DeviceGuard g(device);
    rope::Args a{r->inv_freq, r->rotate_dim, r->layout, r->factor, inverse ? -1.f : 1.f, view(q), view(q_out),
                 view(k), view(k ? k_out : nullptr), q_heads, k ? k_heads : 0, head_dim, positions, tokens};
    // tokens of a block: one for a decode step, whose time is latency, up to 4
    // while eight blocks for every SM remain
    int sms = 0;
    CKR(sm_count(device, &sms));
    int tok = 4;
    while (tok > 1 && tokens / tok < 8 * sms) tok /= 2;
    const unsigned grid = (unsigned)((tokens + tok - 1) / tok);
    const size_t smem = (size_t)tok * (r->rotate_dim / 2) * sizeof(float2);
    const bool vec = vector_heads(a, dtype, {a.q, a.q_out, a.k, a.k_out});
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      if (vec)
        rope::rope_kernel<T, true><<<grid, 256, smem, s>>>(a, tok);
      else
        rope::rope_kernel<T, false><<<grid, 256, smem, s>>>(a, tok);
      CK(cudaGetLastError());
      return NOOR_MOE_OK;
    });
  });
}

int noor_kv_append(const noor_kv_cache* c, const noor_kv_batch* b, const noor_heads* k, const noor_heads* v,
                   const noor_rotary* r, const noor_heads* q, const noor_heads* q_out, int32_t q_heads, int32_t dtype,
                   void* stream) {
  return guarded([&]() -> int {
    CKR(check_cache(c));
    CKR(check_batch(c, b));
    CKR(check_touched(c, b));
    CKR(check_dtype(dtype));
    if (r) CKR(check_rotary(r, c->head_dim));
    if (!r) q = nullptr;
    if (b->n_rows == 0) return NOOR_MOE_OK;
    CKR(check_view(k, dtype, "k"));
    CKR(check_view(v, dtype, "v"));
    if (q) {
      CKR(check_view(q, dtype, "q"));
      if (q_heads <= 0 || q_heads > 4096) return fail(NOOR_MOE_ERR_INVALID, "q_heads %d out of range", q_heads);
      CKR(check_out(q_out, b->n_rows, q_heads, c->head_dim, dtype, "q_out"));
    }
    CKR(check_device(c->device));
    DeviceGuard g(c->device);
    kv::AppendArgs a{};
    a.c = cache_of(c);
    a.b = batch_of(b);
    a.k = view(k);
    a.v = view(v);
    a.r.D = c->head_dim;
    a.r.factor = 1.f;
    if (r) {
      a.r.inv_freq = r->inv_freq;
      a.r.rot = r->rotate_dim;
      a.r.layout = r->layout;
      a.r.factor = r->factor;
    }
    a.r.q = view(q);
    a.r.q_out = view(q ? q_out : nullptr);
    a.r.hq = q ? q_heads : 0;
    int sms = 0;
    CKR(sm_count(c->device, &sms));
    a.q_tok = 4;
    while (a.q_tok > 1 && b->n_rows / a.q_tok < 8 * sms) a.q_tok /= 2;
    const int64_t tasks = most_tasks(c, b), qb = q ? (b->n_rows + a.q_tok - 1) / a.q_tok : 0;
    CKR(heads_per_block(c, 2 * tasks, &a.heads));
    // few tokens a block leave its threads room for more heads
    const int64_t per_head = std::min<int64_t>(b->n_rows / tasks, 64) * (c->head_dim / 4);
    a.heads = (int32_t)std::max<int64_t>(a.heads, std::min<int64_t>(c->n_kv_heads, kv::kAppendThreads / std::max<int64_t>(per_head, 1)));
    const int64_t kvb = tasks * 2 * ((c->n_kv_heads + a.heads - 1) / a.heads);
    if (kvb + qb > INT32_MAX) return fail(NOOR_MOE_ERR_INVALID, "too many rows");
    a.kv_blocks = (int32_t)kvb;
    a.kvec = four_elements(a.k, dtype);
    a.vvec = four_elements(a.v, dtype);
    a.qvec = q && vector_heads(a.r, dtype, {a.r.q, a.r.q_out});
    const size_t smem = q ? (size_t)a.q_tok * (a.r.rot / 2) * sizeof(float2) : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // one launch, or for many rows one each for q, k and v
    const bool apart = b->n_rows * c->n_kv_heads * c->head_dim >= kApartElements;
    return by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      if (apart && q) {
        kv::AppendArgs alone = a;
        alone.kv_blocks = 0;
        if (a.qvec)
          kv::rotate_q_kernel<T, true><<<(unsigned)qb, kv::kAppendThreads, smem, s>>>(alone);
        else
          kv::rotate_q_kernel<T, false><<<(unsigned)qb, kv::kAppendThreads, smem, s>>>(alone);
        CK(cudaGetLastError());
      }
      // tokens a thread can own: a block's over the 256 / (head_dim / 4) that share a pair
      const int share = kv::kAppendThreads / (c->head_dim / 4), own = (c->block + share - 1) / share;
      auto go = [&](auto fmt, auto tpt) -> int {
        if (apart) {
          kv::keys_kernel<T, fmt(), tpt()><<<(unsigned)(kvb / 2), kv::kAppendThreads, 0, s>>>(a);
          kv::values_kernel<T, fmt(), tpt() == 16 ? 4 : 2><<<(unsigned)(kvb / 2), kv::kAppendThreads, 0, s>>>(a);
        } else {
          kv::append_kernel<T, fmt(), tpt()><<<(unsigned)(kvb + qb), kv::kAppendThreads, smem, s>>>(a);
        }
        CK(cudaGetLastError());
        return NOOR_MOE_OK;
      };
      auto by_own = [&](auto fmt) -> int {
        if (own <= 4 && c->head_dim <= 128) return go(fmt, std::integral_constant<int, 4>{});
        if (c->head_dim <= 128) return go(fmt, std::integral_constant<int, 8>{});
        return go(fmt, std::integral_constant<int, 16>{});
      };
      return c->format == NOOR_KV_INT8 ? by_own(std::integral_constant<int, kv::INT8>{})
                                       : by_own(std::integral_constant<int, kv::E4M3>{});
    });
  });
}

int noor_kv_read(const noor_kv_cache* c, const noor_kv_batch* b, const int32_t* starts, void* k_out, void* v_out,
                 int32_t dtype, void* stream) {
  return guarded([&]() -> int {
    CKR(check_cache(c));
    CKR(check_batch(c, b, false));
    CKR(check_touched(c, b));
    CKR(check_dtype(dtype));
    if (b->n_rows == 0) return NOOR_MOE_OK;
    if (!k_out || !v_out) return fail(NOOR_MOE_ERR_INVALID, "null output");
    if (reinterpret_cast<uintptr_t>(k_out) % 16 != 0 || reinterpret_cast<uintptr_t>(v_out) % 16 != 0)
      return fail(NOOR_MOE_ERR_INVALID, "outputs must be 16-byte aligned");
    CKR(check_device(c->device));
    DeviceGuard g(c->device);
    kv::ReadArgs a{cache_of(c), batch_of(b), starts, k_out, v_out, 1};
    const int64_t tasks = most_tasks(c, b);
    CKR(heads_per_block(c, 2 * tasks, &a.heads));
    const int64_t grid = tasks * 2 * ((c->n_kv_heads + a.heads - 1) / a.heads);
    if (grid > INT32_MAX) return fail(NOOR_MOE_ERR_INVALID, "too many rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      if (c->format == NOOR_KV_INT8)
        kv::read_kernel<T, kv::INT8><<<(unsigned)grid, kv::kReadThreads, 0, s>>>(a);
      else
        kv::read_kernel<T, kv::E4M3><<<(unsigned)grid, kv::kReadThreads, 0, s>>>(a);
      CK(cudaGetLastError());
      return NOOR_MOE_OK;
    });
  });
}

}  // extern "C"

// ------------------------------------------------------------- attention

namespace {

struct StreamPlan {
  int grid = 0, pairs = 0, nb = 1;
  int prompt = 0, slots = 0, seen = 0, sms = 0;  // tensor-core kernel: most units (0: not launched), slots of parts, Args
  int64_t off_ml = 0, off_desc = 0, off_prompt = 0, off_prompt_ml = 0, off_prompt_desc = 0, bytes = 0;
};

// Rows (times query heads of a group) from which a sequence runs on the
// tensor-core kernel.  4 kv heads of 128 dims, int8, groups of 4, for 1 / 16 / 64
// sequences of 4096 / 4096 / 2048 tokens: 4 new rows 25 / 62 / 97 us there and
// 22 / 40 / 65 us on the streamed kernel, 7 rows 26 / 64 / 96 and 24 / 63 / 114.
constexpr int64_t kPromptRows = 32;

bool prompt_fits(const noor_kv_cache* c, const noor_kv_batch* b, int g, int max_rows, int dtype) {
  return dtype == NOOR_DTYPE_BF16 && c->head_dim <= 128 && (int64_t)max_rows * g >= kPromptRows &&
         b->n_rows * g >= kPromptRows;
}

// Whether that many of the tensor-core kernel's units are better cut (the
// kernel counts the units that there are, and chooses the parts).
bool cut_pays(int units, int tiles, int sms) {
  const int64_t whole = attn::part_cost(units, tiles, 1, sms);
  for (int s = 2; s <= attn::most_parts(units, tiles, sms, INT32_MAX); ++s)
    if (20 * (int64_t)attn::part_cost(units, tiles, s, sms) < 19 * whole) return true;
  return false;
}

// Grid of the streamed kernel: one block per SM, fewer where the batch cannot
// have that many tiles.  With one column group of the mma a row tile is 8 query
// rows, and more rows read a tile's codes again (from L2); with as many as the
// registers hold, codes are widened once for 32 rows (16 at more than 128 dims),
// but a tile's chain is longer and less runs beside it.  16 sequences of 4096
// tokens, 4 kv heads, one group / many: F32 at 128 dims 12 rows 41 / 69 us,
// 48 rows 91 / 108, 64 rows 113 / 114; at 256 dims 12 rows 101 / 101, 32 rows
// 177 / 154 (BF16 154 / 133).  BF16 up to 128 dims has the other kernel for
// more rows.
int stream_plan(const noor_kv_cache* c, const noor_kv_batch* b, int Hq, int max_rows, int window, int dtype, StreamPlan* p) {
  int sms = 0;
  CKR(sm_count(c->device, &sms));
  const int64_t g = Hq / c->n_kv_heads;
  if (c->head_dim > 128)
    p->nb = max_rows * g <= 8 ? 1 : 2;
  else
    p->nb = dtype == NOOR_DTYPE_BF16 || max_rows * g <= 48 ? 1 : 4;
  const int64_t R = 8 * p->nb;
  int per = 0;
  auto pairs_of = [&](auto parts) {
    return attn::by_shape<parts()>(c->head_dim, p->nb, [&](auto dp, auto nb) -> int {
      per = attn::Shape<dp(), parts(), nb()>::kPairs;
      return NOOR_MOE_OK;
    });
  };
  CKR(dtype == NOOR_DTYPE_F32 ? pairs_of(std::integral_constant<int, 2>{}) : pairs_of(std::integral_constant<int, 1>{}));
  const int64_t rtiles = std::min(b->n_rows * g, b->n_rows * g / R + b->batch);
  const int64_t tiles = ((int64_t)b->max_blocks * c->block + attn::kTile - 1) / attn::kTile;
  const double most = (double)rtiles * c->n_kv_heads * tiles;
  p->grid = (int)std::min<double>(sms, std::max(1.0, most));
  p->pairs = (int)std::min<double>((double)p->grid * per, std::max(1.0, most));  // no share without a tile
  p->off_ml = (int64_t)p->pairs * 2 * R * c->head_dim * 4;
  p->off_desc = p->off_ml + (int64_t)p->pairs * 2 * R * 2 * 4;
  p->bytes = p->off_desc + (int64_t)p->pairs * 16;
  if (prompt_fits(c, b, (int)g, max_rows, dtype)) {
    const int64_t units = std::min(b->n_rows * g, b->n_rows * g / 256 + b->batch) * c->n_kv_heads;
    if (units > INT32_MAX) return fail(NOOR_MOE_ERR_INVALID, "too many rows");
    p->prompt = (int)units;
    // a unit's rows see at most that many tiles
    int64_t seen = (tiles + 1) / 2;
    if (window > 0) seen = std::min(seen, ((int64_t)window + 256 / g) / 128 + 2);
    // The fewest units, were all rows prompts' but those of sequences just below
    // the limit: where they would not be cut, none is.
    const int64_t least = std::max<int64_t>((b->n_rows * g - (kPromptRows - 1) * b->batch) / 256, 1) * c->n_kv_heads;
    p->sms = sms;
    p->seen = (int)seen;
    if (least < sms && cut_pays((int)least, (int)seen, sms)) p->slots = (int)std::min<int64_t>(2 * sms, units * (seen / 4));
    const int64_t n = p->slots;
    p->off_prompt = (p->bytes + 15) / 16 * 16;
    p->off_prompt_ml = p->off_prompt + n * 256 * c->head_dim * 4;
    p->off_prompt_desc = p->off_prompt_ml + n * 256 * 2 * 4;
    p->bytes = p->off_prompt_desc + n * 16;
  }
  return NOOR_MOE_OK;
}

// The join of the `n` slots' cut units, launched behind the kernel that leaves
// the parts without waiting for its end.  rows: the most rows a unit can have.
template <typename T>
int launch_join(const attn::Args& a, int n, int rows, cudaStream_t s) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)n, (unsigned)((rows + attn::kJoinWarps - 1) / attn::kJoinWarps));
  cfg.blockDim = dim3(attn::kJoinWarps * 32);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  CK(cudaLaunchKernelEx(&cfg, attn::combine_kernel<T>, a));
  return NOOR_MOE_OK;
}

int check_heads(const noor_kv_cache* c, const noor_kv_batch* b, int Hq) {
  if (Hq <= 0 || Hq > 65536 || Hq % c->n_kv_heads != 0)
    return fail(NOOR_MOE_ERR_INVALID, "%d query heads over %d kv heads", Hq, c->n_kv_heads);
  // the kernels number a kv head's (row, query head) pairs in 32 bits, and round up to a tile of 256
  if (b->n_rows * (Hq / c->n_kv_heads) > INT32_MAX - 256)
    return fail(NOOR_MOE_ERR_INVALID, "n_rows %lld times %d query heads of a kv head is past 32 bits", (long long)b->n_rows,
                Hq / c->n_kv_heads);
  return NOOR_MOE_OK;
}

}  // namespace

extern "C" {

int noor_kv_attention_workspace(const noor_kv_cache* c, const noor_kv_batch* b, int32_t q_heads, int32_t max_rows,
                                int32_t dtype, int64_t* bytes) {
  return guarded([&]() -> int {
    CKR(check_cache(c));
    CKR(check_batch(c, b));
    CKR(check_dtype(dtype));
    CKR(check_heads(c, b, q_heads));
    if (!bytes || max_rows < 0) return fail(NOOR_MOE_ERR_INVALID, "null bytes or negative max_rows");
    StreamPlan p;
    CKR(stream_plan(c, b, q_heads, max_rows, 0, dtype, &p));  // (a window never needs more)
    *bytes = p.bytes;
    return NOOR_MOE_OK;
  });
}

int noor_kv_attention(const noor_kv_cache* c, const noor_kv_batch* b, const noor_heads* q, const noor_heads* out,
                      float* lse, int32_t q_heads, int32_t max_rows, float scale, int32_t window, int32_t dtype,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    CKR(check_cache(c));
    CKR(check_batch(c, b));
    CKR(check_dtype(dtype));
    CKR(check_heads(c, b, q_heads));
    if (max_rows < 0 || window < 0) return fail(NOOR_MOE_ERR_INVALID, "negative max_rows or window");
    if (window >= (int64_t)b->max_blocks * c->block) window = 0;  // longer than any sequence (positions less it stay in 32 bits)
    if (!std::isfinite(scale)) return fail(NOOR_MOE_ERR_INVALID, "scale is not finite");
    if (b->n_rows == 0) return NOOR_MOE_OK;
    CKR(check_view(q, dtype, "q"));
    CKR(check_out(out, b->n_rows, q_heads, c->head_dim, dtype, "out"));
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(NOOR_MOE_ERR_INVALID, "workspace is null or not 16-byte aligned");
    StreamPlan p;
    CKR(stream_plan(c, b, q_heads, max_rows, window, dtype, &p));
    if (workspace_bytes < p.bytes)
      return fail(NOOR_MOE_ERR_INVALID, "workspace of %lld bytes, needs %lld", (long long)workspace_bytes,
                  (long long)p.bytes);
    CKR(check_device(c->device));
    DeviceGuard g(c->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    attn::Args a{};
    a.c = cache_of(c);
    a.b = batch_of(b);
    a.q = view(q);
    a.out = view(out);
    a.lse = lse;
    a.Hq = q_heads;
    a.g = q_heads / c->n_kv_heads;
    a.qvec = four_elements(a.q, dtype);
    a.scale2 = scale * 1.4426950408889634f;
    a.window = window;
    a.pairs = p.pairs;
    a.slots = 2;
    a.rows = 8 * p.nb;
    a.min_e = 0;
    a.max_e = INT64_MAX;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + p.off_ml);
    a.desc = reinterpret_cast<int4*>(ws + p.off_desc);
    // Sequences with many rows go to the tensor-core kernel, the others to the
    // streamed one (only the device knows which a batch has).
    if (p.prompt) {
      attn::Args t = a;
      t.rows = 256;
      t.min_e = kPromptRows;
      t.slots = 1;
      t.pairs = p.slots;
      t.sms = p.sms;
      t.seen = p.seen;
      const int blocks = std::max(p.prompt, p.slots);
      t.part_o = reinterpret_cast<float*>(ws + p.off_prompt);
      t.part_ml = reinterpret_cast<float*>(ws + p.off_prompt_ml);
      t.desc = reinterpret_cast<int4*>(ws + p.off_prompt_desc);
      CKR(c->format == NOOR_KV_INT8 ? attn::prompt_int8(t, blocks, s) : attn::prompt_e4m3(t, blocks, s));
      if (p.slots) CKR(launch_join<bf16>(t, p.slots, 256, s));
      a.max_e = kPromptRows;
    }
    if (dtype == NOOR_DTYPE_BF16)
      CKR(c->format == NOOR_KV_INT8 ? attn::stream_bf16_int8(a, p.nb, p.grid, s) : attn::stream_bf16_e4m3(a, p.nb, p.grid, s));
    else
      CKR(c->format == NOOR_KV_INT8 ? attn::stream_f32_int8(a, p.nb, p.grid, s) : attn::stream_f32_e4m3(a, p.nb, p.grid, s));
    return by_dtype(dtype, [&](auto t) -> int {
      return launch_join<decltype(t)>(a, a.pairs, (int)std::min<int64_t>(a.rows, b->n_rows * a.g), s);
    });
  });
}

}  // extern "C"
