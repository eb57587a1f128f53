// The decode kernels of fsa_quant_dec.cuh for one format, in a source of their own: they take minutes to compile.
#include "fsa_quant_dec.cuh"

namespace fsa {
template QuantDecShape quant_decode_shape<FSA_QC_E4M3>(const FsaQuantCache&, int, int);
template cudaError_t launch_quant_decode<FSA_QC_E4M3>(const QuantDecParams&, int, cudaStream_t);
}  // namespace fsa
