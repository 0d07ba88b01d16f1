// dms_amd/csrc/linear_attention_bf16.hip -- the chunk kernels of linear_attention.inl for __bf16 tensors.
#include "linear_attention.inl"

namespace dmn {
namespace la {
template int launch_chunks<__bf16>(const Args &, int, int, int, hipStream_t);
}
}
