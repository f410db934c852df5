// The tensor-core decode for the block-scaled fp8 formats (every block size;
// these formats have no CUDA-core decode).
#include "decode_tc.cuh"

namespace mj {
template cudaError_t launch_tc_fmt<MJ_KV_FP8_B16>(const mj_decode_args&, int, bool, const CUtensorMap&, const CUtensorMap&,
                                              cudaStream_t, bool);
}  // namespace mj
