// The streamed attention kernel for F32 activations over e4m3 codes.
#include "kv_stream.h"

int noor::attn::stream_f32_e4m3(const Args& a, int nb, int grid, cudaStream_t s) {
  return stream_launch<kv::E4M3, 2>(a, nb, grid, s);
}
