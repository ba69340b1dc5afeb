// The streamed attention kernel for F32 activations over int8 codes.
#include "kv_stream.h"

int noor::attn::stream_f32_int8(const Args& a, int nb, int grid, cudaStream_t s) {
  return stream_launch<kv::INT8, 2>(a, nb, grid, s);
}
