// klp_rows.h — rows read and written 8 consecutive elements a lane (a chunk),
// at any element alignment: the norm, quantization and sampling kernels'.
#pragma once

#include "klp_device.h"

namespace klp {

constexpr int kChunk = 8;

// Elements at any element-aligned address in one or two 16-byte accesses:
// global memory takes dword accesses at any byte address, at the price of the
// lines that a misaligned one touches.
template <typename E>
struct __attribute__((packed, aligned(alignof(E)))) Unaligned16 {
    u32x4 v;
};

// x[j] = p[j] for j < left, 0 (or with kNegInf -inf) behind; all 8 when left
// >= 8.  Two branches of one side each, on conditions that the compiler cannot
// join to an if and else: its registers are then written before either, and on
// no path hold what another wave left.
template <int DT, bool kNegInf = false>
__device__ __forceinline__ void load_chunk(const typename Traits<DT>::elem* p, int64_t left,
                                           float (&x)[kChunk]) {
    typedef typename Traits<DT>::elem elem;
    constexpr int kVecs = DT == kFP32 ? 2 : 1;
    constexpr uint32_t kFill = kNegInf ? Traits<DT>::kNegInfWord : 0;
    u32x4 raw[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) raw[k] = u32x4{kFill, kFill, kFill, kFill};
    if (left >= kChunk) {
        const auto* v = reinterpret_cast<const Unaligned16<elem>*>(p);
#pragma unroll
        for (int k = 0; k < kVecs; ++k) raw[k] = v[k].v;
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) asm("" : "+v"(raw[k]));
    int some = left > 0 && left < kChunk ? static_cast<int>(left) : 0;
    asm("" : "+v"(some));
    if (some > 0) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const uint32_t e = p[j < some ? j : some - 1];
            const uint32_t fill = DT == kFP32 ? kFill : kFill & 0xFFFFu;
            const uint32_t w = j < some ? e : fill;
            if constexpr (DT == kFP32) raw[j / 4][j % 4] = w;
            else if (j & 1) raw[0][j / 2] |= w << 16;
            else raw[0][j / 2] = w;
        }
    }
    unpack<DT>(raw[0], x);
    if constexpr (DT == kFP32) unpack<DT>(raw[1], x + 4);
}

// p[j] = round(x[j]) for j < left.
template <int DT>
__device__ __forceinline__ void store_chunk(typename Traits<DT>::elem* p, int64_t left,
                                            const float (&x)[kChunk]) {
    typedef typename Traits<DT>::elem elem;
    if (left >= kChunk) {
        auto* v = reinterpret_cast<Unaligned16<elem>*>(p);
        v[0].v = pack<DT>(x);
        if constexpr (DT == kFP32) v[1].v = pack<DT>(x + 4);
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (j < left) p[j] = from_f32<DT>(x[j]);
    }
}

// ---------------------------------------------------------------------------
// e4m3 with a scale per block.  With a the block's largest magnitude:
//   scale = a / 448 (1 for a block of zeros), q = round(x * (448 / a)),
// 448 being e4m3's largest value.  a below 2^-100 counts as 2^-100, so that
// neither quotient leaves float32's normal range.  A NaN or an infinity makes
// the scale NaN or infinite: every value of its block then stands for NaN.
// ---------------------------------------------------------------------------
constexpr float kE4m3Max = 448.0f;
constexpr float kE4m3MinAmax = 7.88860905221011805e-31f;  // 2^-100

struct E4m3Scale {
    float scale;
    float inv;
};
__device__ __forceinline__ E4m3Scale e4m3_scale(float amax) {
    if (amax == 0.0f) return E4m3Scale{1.0f, 1.0f};
    // A NaN goes through: the comparison is false.
    const float a = amax < kE4m3MinAmax ? kE4m3MinAmax : amax;
    return E4m3Scale{a / kE4m3Max, kE4m3Max / a};
}

// 8 values times inv, rounded to nearest even, packed in memory order.  The
// quotient's rounding can leave a block's largest value one float32 step above
// 448: it rounds to 448 as its neighbours do.
__device__ __forceinline__ uint2 e4m3_pack8(const float (&x)[kChunk], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * inv, x[4 * h + 1] * inv, 0, false);
        v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv, v, true);
        w[h] = static_cast<uint32_t>(v);
    }
    return make_uint2(w[0], w[1]);
}

struct __attribute__((packed, aligned(1))) Unaligned8 {
    uint32_t lo, hi;
};
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t left, uint2 w) {
    if (left >= kChunk) {
        *reinterpret_cast<Unaligned8*>(p) = Unaligned8{w.x, w.y};
    } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (j < left) p[j] = static_cast<uint8_t>((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

// Largest magnitude of a chunk; a NaN among them is the result.
__device__ __forceinline__ float chunk_amax(const float (&x)[kChunk]) {
    float a = fabsf(x[0]);
#pragma unroll
    for (int j = 1; j < kChunk; ++j) a = fmax_nan(a, fabsf(x[j]));
    return a;
}

}  // namespace klp
