// The streamed attention kernel for BF16 activations over e4m3 codes.
#include "kv_stream.h"

int noor::attn::stream_bf16_e4m3(const Args& a, int nb, int grid, cudaStream_t s) {
  return stream_launch<kv::E4M3, 1>(a, nb, grid, s);
}
