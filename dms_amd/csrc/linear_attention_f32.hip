// dms_amd/csrc/linear_attention_f32.hip -- the chunk kernels of linear_attention.inl for float tensors.
#include "linear_attention.inl"

namespace dmn {
namespace la {
template int launch_chunks<float>(const Args &, int, int, int, hipStream_t);
}
}
