// klp_block.h — what the kernels of the norms around a block share: the shapes
// that hold a row, loads of weights and gates, the rows' backward.
#pragma once

#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

// Threads of a workgroup: several groups where a group has fewer.
template <int T> constexpr int kForwardThreads = T < 256 ? 256 : T;
template <int T> constexpr int kBackwardThreads = T < 512 ? 512 : T;

template <int V> using Int = std::integral_constant<int, V>;

// f(threads, chunks) of the shape that holds rows of `dim` elements.
template <typename F>
auto with_shape(int64_t dim, F f) {
    if (dim <= 512) return f(Int<64>{}, Int<1>{});
    if (dim <= 1024) return f(Int<64>{}, Int<2>{});
    if (dim <= 2048) return f(Int<128>{}, Int<2>{});
    if (dim <= 4096) return f(Int<256>{}, Int<2>{});
    if (dim <= 8192) return f(Int<512>{}, Int<2>{});
    return f(Int<1024>{}, Int<2>{});
}

// 8 elements of a weight or gate, float32 or of the rows' dtype.
template <int DT>
__device__ __forceinline__ void load_either(const void* w, bool f32, int64_t at, int64_t left,
                                            float (&x)[kChunk]) {
    if (DT == kFP32 || f32)
        load_chunk<kFP32>(static_cast<const uint32_t*>(w) + at, left, x);
    else
        load_chunk<DT>(static_cast<const typename Traits<DT>::elem*>(w) + at, left, x);
}

// The backward's pass over the rows (klp_block_bwd_*.hip: one dtype each).
template <int DT>
hipError_t launch_block_rows(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kBF16>(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kFP16>(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kFP32>(const BlockBwdParams& p, hipStream_t stream);

}  // namespace klp
