// klp_block_bwd_bf16.hip — klp_block_bwd.h's __global__ functions for bf16 rows.
#include "klp_block_bwd.h"

namespace klp {

template <>
hipError_t launch_block_rows<kBF16>(const BlockBwdParams& p, hipStream_t stream) {
    return launch_rows_dt<kBF16>(p, stream);
}

}  // namespace klp
