// The tensor-core attention kernel over int8 and e4m3 codes.
#include "kv_prompt.cuh"
#include "kv_stream.h"

namespace noor {
namespace attn {
namespace {

template <int DP, int FMT>
int launch(const Args& a, int units, cudaStream_t s) {
  auto kern = prompt::prompt_kernel<DP, FMT>;
  constexpr int smem = prompt::Smem<DP>::kBytes;
  CKR(ensure_smem_limit(kern, smem));
  kern<<<units, prompt::kThreads, smem, s>>>(a);
  CK(cudaGetLastError());
  return NOOR_MOE_OK;
}

}  // namespace

int prompt_int8(const Args& a, int units, cudaStream_t s) {
  return a.c.D <= 64 ? launch<64, kv::INT8>(a, units, s) : launch<128, kv::INT8>(a, units, s);
}
int prompt_e4m3(const Args& a, int units, cudaStream_t s) {
  return a.c.D <= 64 ? launch<64, kv::E4M3>(a, units, s) : launch<128, kv::E4M3>(a, units, s);
}

}  // namespace attn
}  // namespace noor
