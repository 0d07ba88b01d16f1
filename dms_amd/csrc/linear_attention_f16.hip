// dms_amd/csrc/linear_attention_f16.hip -- the chunk kernels of linear_attention.inl for _Float16 tensors.
#include "linear_attention.inl"

namespace dmn {
namespace la {
template int launch_chunks<_Float16>(const Args &, int, int, int, hipStream_t);
}
}
