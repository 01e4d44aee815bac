// Attention within packed documents, forward, of 16-bit heads wider than 128: compiled with the sums in accumulation registers
// (build.py), which leaves the others to operands read ahead (8192 tokens, 8/4 heads of 256: 438 to 382 us).
#include "doc_attention_forward.h"

namespace dllm_hip {

template void launch_forward<__bf16, 256>(const DocAttention&, __bf16*, hipStream_t);
template void launch_forward<_Float16, 256>(const DocAttention&, _Float16*, hipStream_t);

}  // namespace dllm_hip
