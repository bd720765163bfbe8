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
// they need no branch and stay on their way until their values are used.  So do
// the loads of other rows (kOdd): a chunk that the row ends in is read 8 elements
// from its end and moved into place when it is used (settle).  Short rows of that
// kind (kAny, up to 512 elements, fewer than 8 among them) wait for their tails.
// bf16, forward + backward, us, as kAny and so: 8192 x 4090 94 + 199, 58 + 91; 16384 x
// 1601 85 + 185, 64 + 82; 2048 x 13001 82 + 152, 84 + 125; float32 8192 x 1601 53 +
// 104, 48 + 66, 4096 x 4097 69 + 123, 76 + 94.
enum : int {
    kWhole = 0,     // weights of the rows' dtype
    kWholeF32 = 1,  // float32 weights
    kAny = 2,       // any rows, weights of either dtype
    kOdd = 3        // the same, of at least 8 elements
};
template <int DT, int kMode>
constexpr int kWeight = kMode == kWhole ? DT : kFP32;  // what weights are held as

// Element c of a row that starts `at` elements behind `base`: a base that the wave
// shares and an offset of 32 bits.
template <typename E>
__device__ __forceinline__ E* column(void* base, int64_t at, int c) {
    return reinterpret_cast<E*>(reinterpret_cast<char*>(static_cast<E*>(base) + at) +
                                static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(E)));
}
// How far a chunk of column c is read before its place, 8 where none of it exists.
__device__ __forceinline__ int shift_of(int c, int dim) {
    const int s = c - (dim - kChunk);
    return s < 0 ? 0 : s < kChunk ? s : kChunk;
}
// A chunk read `s` elements early into place, zeros behind it.
__device__ __forceinline__ void settle16(u32x4& v, int s) {
    if (!__any(s != 0)) return;
    const uint32_t bits = static_cast<uint32_t>(s & 1) * 16;
#pragma unroll
    for (int d = 0; d < 4; ++d) v[d] = s & 8 ? 0 : v[d];
    v = u32x4{s & 4 ? v[2] : v[0], s & 4 ? v[3] : v[1], s & 4 ? 0 : v[2], s & 4 ? 0 : v[3]};
    v = u32x4{s & 2 ? v[1] : v[0], s & 2 ? v[2] : v[1], s & 2 ? v[3] : v[2], s & 2 ? 0 : v[3]};
    v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], bits),
              __builtin_amdgcn_alignbit(v[2], v[1], bits),
              __builtin_amdgcn_alignbit(v[3], v[2], bits),
              __builtin_amdgcn_alignbit(0, v[3], bits)};
}
__device__ __forceinline__ void settle32(u32x4 (&v)[2], int s) {
    if (!__any(s != 0)) return;
    uint32_t d[kChunk];
#pragma unroll
    for (int j = 0; j < kChunk; ++j) d[j] = s & 8 ? 0 : v[j / 4][j % 4];
#pragma unroll
    for (int by = 4; by > 0; by /= 2)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const uint32_t further = j + by < kChunk ? d[j + by] : 0;
            d[j] = s & by ? further : d[j];
        }
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j / 4][j % 4] = d[j];
}
template <int DT, int kMode>
__device__ __forceinline__ void settle(RawChunk<DT>& r, int c, int dim) {
    if constexpr (kMode == kOdd) {
        if constexpr (DT == kFP32) settle32(r.v, shift_of(c, dim));
        else settle16(r.v[0], shift_of(c, dim));
    }
}

// Columns c .. c + 7 of a row of `dim` elements that starts `at` elements behind
// `base` (the same for the wave); 0 behind it, and where base is null.  (kOdd: to
// be settled, and base is not null.)
template <int DT, int kMode>
__device__ __forceinline__ RawChunk<DT> fetch(const void* base, int64_t at, int c, int dim) {
    typedef typename Traits<DT>::elem elem;
    const elem* row = static_cast<const elem*>(base) + at;
    if constexpr (kMode == kAny) {
        return load_raw<DT>(row + c, base != nullptr ? dim - c : 0);
    } else if constexpr (kMode == kOdd) {
        RawChunk<DT> r;
        const auto* v = reinterpret_cast<const Unaligned16<elem>*>(
            column<elem>(const_cast<void*>(base), at, c < dim - kChunk ? c : dim - kChunk));
#pragma unroll
        for (int k = 0; k < RawChunk<DT>::kVecs; ++k) r.v[k] = v[k].v;
        return r;
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
// kOdd's chunk of a weight or gate of either dtype as it lies in memory, and its
// values: a 16-bit one is read twice.
template <int DT>
__device__ __forceinline__ RawChunk<kFP32> fetch_two(const void* w, bool f32, int64_t at, int c,
                                                     int dim) {
    const int start = c < dim - kChunk ? c : dim - kChunk;
    const int shift = f32 ? 2 : 1;
    const auto* v = reinterpret_cast<const Unaligned16<uint16_t>*>(
        static_cast<const char*>(w) + (at << shift) + (static_cast<uint32_t>(start) << shift));
    RawChunk<kFP32> r;
    r.v[0] = v[0].v;
    r.v[1] = v[f32 ? 1 : 0].v;
    return r;
}
template <int DT>
__device__ __forceinline__ void settle_two(RawChunk<kFP32>& r, bool f32, int c, int dim) {
    // Both, one of them chosen: the two sides of a branch would leave registers
    // that neither is sure to write.
    const int s = shift_of(c, dim);
    u32x4 narrow = r.v[0];
    float x[kChunk];
    settle16(narrow, s);
    unpack<DT>(narrow, x);
    settle32(r.v, s);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
        const uint32_t wide = r.v[j / 4][j % 4];
        r.v[j / 4][j % 4] = f32 ? wide : __float_as_uint(x[j]);
    }
}
// A weight or gate, float32 or of the rows' dtype, as values.
template <int DT, int kMode>
__device__ __forceinline__ void fetch_either(const void* w, bool f32, int64_t at, int c, int dim,
                                             float (&x)[kChunk]) {
    if constexpr (DT == kFP32) {
        RawChunk<kFP32> r = fetch<kFP32, kMode>(w, at, c, dim);
        settle<kFP32, kMode>(r, c, dim);
        r.values(x);
    } else if constexpr (kMode == kOdd) {
        RawChunk<kFP32> r = fetch_two<DT>(w, f32, at, c, dim);
        settle_two<DT>(r, f32, c, dim);
        r.values(x);
    } else {
        // Both, one of them empty, as there.
        float wide[kChunk];
        fetch<kFP32, kMode>(f32 ? w : nullptr, at, c, dim).values(wide);
        fetch<DT, kMode>(f32 ? nullptr : w, at, c, dim).values(x);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) x[j] = f32 ? wide[j] : x[j];
    }
}
// A weight's chunk, held as kWeight (kOdd: to be settled).
template <int DT, int kMode>
__device__ __forceinline__ RawChunk<kWeight<DT, kMode>> fetch_weight(const void* w, bool f32,
                                                                     int c, int dim) {
    if constexpr (kMode == kAny) {
        float x[kChunk];
        fetch_either<DT, kAny>(w, f32, 0, c, dim, x);
        RawChunk<kFP32> r;
        r.v[0] = pack<kFP32>(x);
        r.v[1] = pack<kFP32>(x + 4);
        return r;
    } else if constexpr (kMode == kOdd && DT != kFP32) {
        return fetch_two<DT>(w, f32, 0, c, dim);
    } else {
        return fetch<kWeight<DT, kMode>, kMode>(w, 0, c, dim);
    }
}
template <int DT, int kMode>
__device__ __forceinline__ void settle_weight(RawChunk<kWeight<DT, kMode>>& w, bool f32, int c,
                                              int dim) {
    if constexpr (kMode == kOdd) {
        if constexpr (DT == kFP32) settle32(w.v, shift_of(c, dim));
        else settle_two<DT>(w, f32, c, dim);
    }
}
// 8 codes of a row of e4m3 codes, as fetch.
template <int kMode>
__device__ __forceinline__ uint2 fetch_codes(const uint8_t* base, int64_t at, int c, int dim) {
    if constexpr (kMode == kAny) return load_codes(base + at + c, dim - c);
    if constexpr (kMode == kOdd) {
        const Unaligned8 v = *reinterpret_cast<const Unaligned8*>(
            base + at + static_cast<uint32_t>(c < dim - kChunk ? c : dim - kChunk));
        return make_uint2(v.lo, v.hi);
    }
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(base + at), 0, dim, 0x00020000);
    const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, c, 0, 0);
    return make_uint2(v[0], v[1]);
}

template <int kMode>
__device__ __forceinline__ void settle_codes(uint2& w, int c, int dim) {
    if constexpr (kMode == kOdd) {
        const int s = shift_of(c, dim);
        if (!__any(s != 0)) return;
        const uint32_t bits = static_cast<uint32_t>(s & 3) * 8;
        w = make_uint2(s & 8 ? 0 : w.x, s & 8 ? 0 : w.y);
        w = make_uint2(s & 4 ? w.y : w.x, s & 4 ? 0 : w.y);
        w = make_uint2(__builtin_amdgcn_alignbit(w.y, w.x, bits),
                       __builtin_amdgcn_alignbit(0, w.y, bits));
    }
}

// f(mode) of a launch of T threads and N chunks a row.
template <int DT, int T, int N, typename P, typename F>
hipError_t with_mode(const P& p, F f) {
    if (!p.whole) return f(Int<T == 64 && N == 1 ? kAny : kOdd>{});
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
