// The decode kernels over 4-bit codes (see quantized_decode.cuh).
#include "quantized_decode.cuh"

namespace tdist {
namespace qdecode {
template int launch_bits<4>(const Params&, int, int, bool, bool, bool, int, cudaStream_t);
}  // namespace qdecode
}  // namespace tdist
