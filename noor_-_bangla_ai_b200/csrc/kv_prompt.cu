// The tensor-core attention kernel over int8 and e4m3 codes.
#include "kv_prompt.cuh"
#include "kv_stream.h"

namespace noor {
namespace attn {
namespace {

template <int DP, int FMT, bool PARTS>
int launch(const Args& a, int blocks, cudaStream_t s) {
  auto kern = prompt::prompt_kernel<DP, FMT, PARTS>;
  constexpr int smem = prompt::Smem<DP>::kBytes;
  CKR(ensure_smem_limit(kern, smem));
  kern<<<blocks, prompt::kThreads, smem, s>>>(a);
  CK(cudaGetLastError());
  return NOOR_MOE_OK;
}

template <int FMT>
int by_dim(const Args& a, int blocks, cudaStream_t s) {
  if (a.c.D <= 64) return a.pairs > 0 ? launch<64, FMT, true>(a, blocks, s) : launch<64, FMT, false>(a, blocks, s);
  return a.pairs > 0 ? launch<128, FMT, true>(a, blocks, s) : launch<128, FMT, false>(a, blocks, s);
}

}  // namespace

int prompt_int8(const Args& a, int blocks, cudaStream_t s) { return by_dim<kv::INT8>(a, blocks, s); }
int prompt_e4m3(const Args& a, int blocks, cudaStream_t s) { return by_dim<kv::E4M3>(a, blocks, s); }

}  // namespace attn
}  // namespace noor
