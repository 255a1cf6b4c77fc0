// The decode kernels over 8-bit codes (see quantized_decode.cuh).
#include "quantized_decode.cuh"

namespace tdist {
namespace qdecode {
template int launch_bits<8>(const Params&, int, int, bool, bool, bool, int, cudaStream_t);
}  // namespace qdecode
}  // namespace tdist
