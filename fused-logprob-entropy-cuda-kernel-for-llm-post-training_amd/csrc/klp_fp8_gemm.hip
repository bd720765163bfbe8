// klp_fp8_gemm.hip — product of e4m3 matrices with float32 scales for each
// 128 of K, for gfx950:
//
//   out[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k]
//
// One v_mfma_f32_16x16x128_f8f6f4 is one scale block of K: it starts from
// zero, and its four sums a lane are then multiplied by the two scales and
// added to float32 accumulators.  The weight is the M side, so that a lane
// holds 4 consecutive n of one token: its token's scale is one register, its
// weight's scale one scalar, and its 4 outputs lie side by side.  Lane l
// holds row l % 16 of an operand block and 32 of its 128 k; which 32 is free,
// as long as both operands agree: two 16-byte pieces, at 16 (l / 16) and 64 +
// 16 (l / 16), so that 4 lanes read 64 consecutive bytes.
#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kK = kScaleBlock;

// Sums of one scale block, from zero; both block scales of the instruction
// are 1 (2^(127 - 127)).
__device__ __forceinline__ f32x4 mul_block(i32x8 a, i32x8 b) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, 0, 0, 0, 0, 0,
                                                            0);
}

// 32 bytes of k of an operand row: pieces at k0 and k0 + 64.
__device__ __forceinline__ i32x8 load_operand(const uint8_t* row, int64_t k0) {
    union {
        u32x4 h[2];
        i32x8 v;
    } u;
    u.h[0] = *reinterpret_cast<const u32x4*>(row + k0);
    u.h[1] = *reinterpret_cast<const u32x4*>(row + k0 + 64);
    return u.v;
}
// The same where K ends inside the block: zeros behind it (K % 16 == 0).
__device__ __forceinline__ i32x8 load_operand_tail(const uint8_t* row, int64_t k0, int64_t k) {
    union {
        u32x4 h[2];
        i32x8 v;
    } u;
    const u32x4 zero = {0, 0, 0, 0};
    u.h[0] = k0 < k ? *reinterpret_cast<const u32x4*>(row + k0) : zero;
    u.h[1] = k0 + 64 < k ? *reinterpret_cast<const u32x4*>(row + k0 + 64) : zero;
    return u.v;
}

// 4 outputs of one token, n .. n + 3 (`left` of them).
template <int DT>
__device__ __forceinline__ void store4(typename Traits<DT>::elem* p, int64_t left, f32x4 v) {
    typedef typename Traits<DT>::elem elem;
    elem e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = from_f32<DT>(v[j]);
    if (left >= 4) {
        __builtin_memcpy(p, e, sizeof e);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) p[j] = e[j];
    }
}

// Few tokens: a wave streams 16 VB rows of the weight against 16 MB tokens,
// both straight from memory to registers (the tokens' rows stay in the
// caches).  kSplit waves of a workgroup share those rows' K; their sums meet
// in LDS and are added in order.
template <int DT, int MB, int VB, int kSplit>
__global__ __launch_bounds__(256, 2) void klp_fp8_stream_kernel(Fp8LinearParams p) {
    __shared__ f32x4 part[kSplit > 1 ? (kSplit - 1) * MB * VB * 64 : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tile = kSplit > 1 ? static_cast<int64_t>(blockIdx.x)
                                    : static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int64_t v0 = tile * 16 * VB;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * 16 * MB;
    if (v0 >= p.n) return;  // a whole wave; with kSplit > 1 a whole workgroup
    const int lrow = lane & 15, lq = lane >> 4;

    // Rows past the end repeat the last one; their outputs are not stored.
    const uint8_t* w[VB];
    const uint8_t* x[MB];
    const float* xs[MB];
#pragma unroll
    for (int i = 0; i < VB; ++i) {
        const int64_t r = v0 + 16 * i + lrow;
        w[i] = p.w + (r < p.n ? r : p.n - 1) * p.ld_w + 16 * lq;
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t r = t0 + 16 * j + lrow;
        const int64_t m = r < p.m ? r : p.m - 1;
        x[j] = p.x + m * p.ld_x + 16 * lq;
        xs[j] = p.xs + m * p.n_blocks;
    }
    const float* ws = p.ws + v0 / kScaleBlock * p.n_blocks;

    const int nb = static_cast<int>(p.n_blocks);
    const int first = kSplit > 1 ? nb * wave / kSplit : 0;
    const int end = kSplit > 1 ? nb * (wave + 1) / kSplit : nb;
    f32x4 acc[VB][MB];
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto fold = [&](const i32x8 (&a)[VB], const i32x8 (&b)[MB], const float (&s)[MB], float g) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const float f = s[j] * g;
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                const f32x4 c = mul_block(a[i], b[j]);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(c[r], f, acc[i][j][r]);
            }
        }
    };
    auto load = [&](int b, i32x8 (&a)[VB], i32x8 (&c)[MB], float (&s)[MB], float& g) {
        const int64_t k0 = static_cast<int64_t>(b) * kK;
#pragma unroll
        for (int i = 0; i < VB; ++i) a[i] = load_operand(w[i], k0);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            c[j] = load_operand(x[j], k0);
            s[j] = xs[j][b];
        }
        g = ws[b];
    };

    // Whole blocks, the next one's loads in flight; then K's last part.
    const int whole = static_cast<int>(p.k / kK);
    const int stop = end < whole ? end : whole;
    i32x8 a[2][VB], c[2][MB];
    float s[2][MB], g[2];
    int b = first;
    if (b < stop) {
        load(b, a[0], c[0], s[0], g[0]);
        for (; b + 2 < stop; b += 2) {
            load(b + 1, a[1], c[1], s[1], g[1]);
            fold(a[0], c[0], s[0], g[0]);
            load(b + 2, a[0], c[0], s[0], g[0]);
            fold(a[1], c[1], s[1], g[1]);
        }
        if (b + 1 < stop) {
            load(b + 1, a[1], c[1], s[1], g[1]);
            fold(a[0], c[0], s[0], g[0]);
            fold(a[1], c[1], s[1], g[1]);
        } else {
            fold(a[0], c[0], s[0], g[0]);
        }
    }
    if (end > whole) {
        const int64_t k0 = static_cast<int64_t>(whole) * kK;
        const int64_t left = p.k - 16 * lq;  // the rows' pointers start at 16 lq
#pragma unroll
        for (int i = 0; i < VB; ++i) a[0][i] = load_operand_tail(w[i], k0, left);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            c[0][j] = load_operand_tail(x[j], k0, left);
            s[0][j] = xs[j][whole];
        }
        fold(a[0], c[0], s[0], ws[whole]);
    }

    if constexpr (kSplit > 1) {
        if (wave > 0) {
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j)
                    part[((wave - 1) * VB * MB + i * MB + j) * 64 + lane] = acc[i][j];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int z = 0; z < kSplit - 1; ++z)
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    const f32x4 o = part[(z * VB * MB + i * MB + j) * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] += o[r];
                }
    }

    typedef typename Traits<DT>::elem elem;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t m = t0 + 16 * j + lrow;
        if (m >= p.m) continue;
        elem* out = static_cast<elem*>(p.out) + m * p.ld_out;
#pragma unroll
        for (int i = 0; i < VB; ++i) {
            const int64_t n = v0 + 16 * i + 4 * lq;
            store4<DT>(out + n, p.n - n, acc[i][j]);
        }
    }
}

template <int DT, int MB, int VB, int kSplit>
hipError_t launch_stream(const Fp8LinearParams& p, hipStream_t stream) {
    const int64_t tiles = (p.n + 16 * VB - 1) / (16 * VB);
    const dim3 grid(static_cast<unsigned>(kSplit > 1 ? tiles : (tiles + 3) / 4),
                    static_cast<unsigned>((p.m + 16 * MB - 1) / (16 * MB)));
    return launch_kernel(klp_fp8_stream_kernel<DT, MB, VB, kSplit>, grid, dim3(256), stream, p);
}

template <int DT, int VB, int kSplit>
hipError_t launch_stream_tokens(const Fp8LinearParams& p, hipStream_t stream) {
    if (p.m <= 16) return launch_stream<DT, 1, VB, kSplit>(p, stream);
    if (p.m <= 32) return launch_stream<DT, 2, VB, kSplit>(p, stream);
    return launch_stream<DT, 4, VB, kSplit>(p, stream);
}

template <int DT>
hipError_t launch_fp8_linear_dt(const Fp8LinearParams& p, hipStream_t stream) {
    // Too few waves of 64 rows to fill the chip: 16 rows, K split four ways.
    if (p.n < 64 * 1024) return launch_stream_tokens<DT, 1, 4>(p, stream);
    return launch_stream_tokens<DT, 4, 1>(p, stream);
}

}  // namespace

hipError_t launch_fp8_linear(int out_dtype, const Fp8LinearParams& p, hipStream_t stream) {
    switch (out_dtype) {
        case kBF16: return launch_fp8_linear_dt<kBF16>(p, stream);
        case kFP16: return launch_fp8_linear_dt<kFP16>(p, stream);
        case kFP32: return launch_fp8_linear_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
