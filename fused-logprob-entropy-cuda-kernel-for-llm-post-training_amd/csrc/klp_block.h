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

// group_sum of one barrier: calls alternate between two slots of `lds`, so that
// a slot's readers have met once more before it is written again.
template <int T>
__device__ __forceinline__ float group_sum_alternate(float v, float (&lds)[2][T / 64], int& slot) {
    v = xrow_sum(row_sum16(v));
    if constexpr (T > 64) {
        float (&part)[T / 64] = lds[slot];
        slot ^= 1;
        if ((threadIdx.x & 63) == 0) part[(threadIdx.x % T) >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v += part[i];
    }
    return v;
}

// How a kernel's rows and weights lie.  Whole rows (every one at a multiple of
// 16 bytes, dim of 8) are read by buffer loads whose range ends with the row:
// they need no branch and stay on their way until their values are used, where
// the loads of any other rows wait for their tails.
enum : int {
    kWhole = 0,     // weights of the rows' dtype
    kWholeF32 = 1,  // float32 weights
    kAny = 2        // any rows, weights of either dtype
};
template <int DT, int kMode>
constexpr int kWeight = kMode == kWhole ? DT : kFP32;  // what weights are held as

// Columns c .. c + 7 of a row of `dim` elements that starts `at` elements behind
// `base` (the same for the wave); 0 behind it, and where base is null.
template <int DT, bool kWholeRow>
__device__ __forceinline__ RawChunk<DT> fetch(const void* base, int64_t at, int c, int dim) {
    typedef typename Traits<DT>::elem elem;
    const elem* row = static_cast<const elem*>(base) + at;
    if constexpr (!kWholeRow) {
        return load_raw<DT>(row + c, base != nullptr ? dim - c : 0);
    } else {
        constexpr int kSize = sizeof(elem);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<elem*>(row), 0, base != nullptr ? dim * kSize : 0, 0x00020000);
        RawChunk<DT> r;
#pragma unroll
        for (int k = 0; k < RawChunk<DT>::kVecs; ++k)
            r.v[k] = __builtin_amdgcn_raw_buffer_load_b128(rs, c * kSize + 16 * k, 0, 0);
        return r;
    }
}
// The same of a weight or gate, float32 or of the rows' dtype, as values.
template <int DT, bool kWholeRow>
__device__ __forceinline__ void fetch_either(const void* w, bool f32, int64_t at, int c, int dim,
                                             float (&x)[kChunk]) {
    if constexpr (DT == kFP32) {
        fetch<kFP32, kWholeRow>(w, at, c, dim).values(x);
    } else {
        // Both, one of them empty: the two sides of a branch would leave registers
        // that neither is sure to write.
        float wide[kChunk];
        fetch<kFP32, kWholeRow>(f32 ? w : nullptr, at, c, dim).values(wide);
        fetch<DT, kWholeRow>(f32 ? nullptr : w, at, c, dim).values(x);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) x[j] = f32 ? wide[j] : x[j];
    }
}
// Element c of a row that starts `at` elements behind `base`: a base that the wave
// shares and an offset of 32 bits.
template <typename E>
__device__ __forceinline__ E* column(void* base, int64_t at, int c) {
    return reinterpret_cast<E*>(reinterpret_cast<char*>(static_cast<E*>(base) + at) +
                                static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(E)));
}
// A weight's chunk, held as kWeight.
template <int DT, int kMode>
__device__ __forceinline__ RawChunk<kWeight<DT, kMode>> fetch_weight(const void* w, bool f32,
                                                                     int c, int dim) {
    if constexpr (kMode == kAny) {
        float x[kChunk];
        fetch_either<DT, false>(w, f32, 0, c, dim, x);
        RawChunk<kFP32> r;
        r.v[0] = pack<kFP32>(x);
        r.v[1] = pack<kFP32>(x + 4);
        return r;
    } else {
        return fetch<kWeight<DT, kMode>, true>(w, 0, c, dim);
    }
}
// 8 codes of a row of e4m3 codes, as fetch.
template <bool kWholeRow>
__device__ __forceinline__ uint2 fetch_codes(const uint8_t* base, int64_t at, int c, int dim) {
    if constexpr (!kWholeRow) return load_codes(base + at + c, dim - c);
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(base + at), 0, dim, 0x00020000);
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, c, 0, 0);
    return make_uint2(v[0], v[1]);
}

// f(mode) of a launch.
template <int DT, typename P, typename F>
hipError_t with_mode(const P& p, F f) {
    if (!p.whole) return f(Int<kAny>{});
    return DT == kFP32 || p.weight_f32 ? f(Int<kWholeF32>{})
                                       : f(Int<DT == kFP32 ? kWholeF32 : kWhole>{});
}

// The backward's pass over the rows (klp_block_bwd_*.hip: one dtype each).
template <int DT>
hipError_t launch_block_rows(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kBF16>(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kFP16>(const BlockBwdParams& p, hipStream_t stream);
template <> hipError_t launch_block_rows<kFP32>(const BlockBwdParams& p, hipStream_t stream);

}  // namespace klp
