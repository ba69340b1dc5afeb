// kv_stream.h -- launches of the streamed attention kernel, one source file
// for each activation type and cache format (they compile side by side).
#pragma once

#include <type_traits>

#include "host.h"
#include "kv_attention.cuh"

namespace noor {
namespace attn {

// Calls f(bound of head_dim, column groups) as integral constants.  BF16 (one
// f16 part) up to 128 dims always has one group.
template <int PARTS, typename F>
int by_shape(int D, int nb, F&& f) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using More = integral_constant<int, PARTS == 1 ? 1 : 4>;
  if (D <= 64) return nb == 1 ? f(integral_constant<int, 64>{}, One{}) : f(integral_constant<int, 64>{}, More{});
  if (D <= 128) return nb == 1 ? f(integral_constant<int, 128>{}, One{}) : f(integral_constant<int, 128>{}, More{});
  return nb == 1 ? f(integral_constant<int, 256>{}, One{}) : f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
}

template <int FMT, int PARTS>
int stream_launch(const Args& a, int nb, int grid, cudaStream_t s) {
  return by_shape<PARTS>(a.c.D, nb, [&](auto dp, auto n) -> int {
    using Sh = Shape<dp(), PARTS, n()>;
    auto kern = stream_kernel<dp(), FMT, PARTS, n()>;
    const int smem = Sh::smem_bytes(a.c.D);
    CKR(ensure_smem_limit(kern, smem));
    kern<<<grid, Sh::kPairs * 64, smem, s>>>(a);
    CK(cudaGetLastError());
    return NOOR_MOE_OK;
  });
}

// The tensor-core kernel for many rows (kv_prompt.cuh).
int prompt_int8(const Args& a, int blocks, cudaStream_t s);
int prompt_e4m3(const Args& a, int blocks, cudaStream_t s);

int stream_bf16_int8(const Args& a, int nb, int grid, cudaStream_t s);
int stream_bf16_e4m3(const Args& a, int nb, int grid, cudaStream_t s);
int stream_f32_int8(const Args& a, int nb, int grid, cudaStream_t s);
int stream_f32_e4m3(const Args& a, int nb, int grid, cudaStream_t s);

}  // namespace attn
}  // namespace noor
