// The streamed attention kernel for BF16 activations over int8 codes.
#include "kv_stream.h"

int noor::attn::stream_bf16_int8(const Args& a, int nb, int grid, cudaStream_t s) {
  return stream_launch<kv::INT8, 1>(a, nb, grid, s);
}
