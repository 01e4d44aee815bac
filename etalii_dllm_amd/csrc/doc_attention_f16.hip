// Attention within packed documents in float16.
#include "doc_attention_backward.h"
#include "doc_attention_forward.h"

namespace dllm_hip {

template int launch_document_attention<_Float16>(DocAttention, void*, char*, hipStream_t);
template int launch_document_attention_backward<_Float16>(DocAttention, char*, hipStream_t);

}  // namespace dllm_hip
