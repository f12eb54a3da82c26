// The paged decode attention over int8 pages (a file of its own, so that the two kinds compile side by side).
#include "paged_attn8.cuh"

int dkv::pattn::launch8_int8(int q_dtype, const Params &p, const Shape &s, cudaStream_t st) {
  return launch8<DKV_I8>(q_dtype, p, s, st);
}
