// Cross attention, fp16 inputs (a translation unit of its own: the variants compile in parallel).
#include "cross_attn.cuh"

extern "C" int dfl_cross_attention_f16(const CrossArgs* a, cudaStream_t stream) { return cross_entry<true>(a, stream); }
