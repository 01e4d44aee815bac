// Attention within packed documents in float32.
#include "doc_attention_backward.h"
#include "doc_attention_forward.h"

namespace dllm_hip {

template int launch_document_attention<float>(const DocAttention&, void*, hipStream_t);
template int launch_document_attention_backward<float>(const DocAttention&, hipStream_t);

}  // namespace dllm_hip
