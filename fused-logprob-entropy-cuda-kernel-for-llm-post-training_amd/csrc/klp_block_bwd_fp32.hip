// klp_block_bwd_fp32.hip — klp_block_bwd.h's __global__ functions for fp32 rows.
#include "klp_block_bwd.h"

namespace klp {

template <>
hipError_t launch_block_rows<kFP32>(const BlockBwdParams& p, hipStream_t stream) {
    return launch_rows_dt<kFP32>(p, stream);
}

}  // namespace klp
