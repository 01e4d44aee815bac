// Attention within packed documents in float32.
#include "doc_attention_backward.h"
#include "doc_attention_forward.h"

namespace dllm_hip {

template int launch_document_attention<float>(DocAttention, void*, char*, hipStream_t);
template int launch_document_attention_backward<float>(DocAttention, char*, hipStream_t);

}  // namespace dllm_hip
