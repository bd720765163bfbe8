// klp_block_bwd_fp16.hip — klp_block_bwd.h's __global__ functions for fp16 rows.
#include "klp_block_bwd.h"

namespace klp {

template <>
hipError_t launch_block_rows<kFP16>(const BlockBwdParams& p, hipStream_t stream) {
    return launch_rows_dt<kFP16>(p, stream);
}

}  // namespace klp
