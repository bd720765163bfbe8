// klp_norm.hip — root-mean-square norm with the residual's addition, its
// backward, and the same norm with an e4m3 output, for gfx950.
//
//   h = round(x + residual)          (h = x without one)
//   s = (mean(h^2) + eps)^-1/2       per row
//   y = round(h s w), or per 128 columns e4m3 codes of h s w and their scale
//   dx = gh + s (gy w - h s^2 mean(gy w h)),   dw = sum over rows of gy h s
//
// The statistics are those of the stored (rounded) h, so that the backward,
// which reads h, differentiates what the forward computed.  All sums are
// float32; y, dx and dw are rounded once.
//
// Bound by memory: the forward reads x (and the residual) once and writes y
// (and h) once, holding the row in registers between its two uses; the
// backward reads h and the gradients once.  A row is held by a group of 64 to
// 1024 threads, 8 elements (a chunk) a thread and pass, 1 to 8 chunks a
// thread: rows of up to 65536 elements.
//
// Measured: 8192 rows of 4096 bf16 with a residual 48 us forward (5.55 TB/s),
// 55.6 backward (h and two gradients in, one out: 4.8 TB/s, 5.1 with the
// shares) and 4.8 for the sum of the shares; 16384 rows of 3584 to e4m3 74 us
// (5.56 TB/s); a copy of this size runs at 5.9.  64 rows: 4 us, the launch's.
// 4096 rows of 32768 bf16: 113 us forward, 363 backward, whose shares of dw go
// through memory for every row (below); 4096 of 16384: 48 and 90.
//
// dw: a group walks rows with a fixed stride and keeps its share of the sum
// in registers; the shares, [groups, dim] float32 in a workspace, are added
// in group order by a second kernel, so that the result depends on nothing
// but the sizes.
#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

namespace {

constexpr int kBlockThreads = 256;

// Sum over a group of T threads (T = 64: one wave of the workgroup).
template <int T>
__device__ __forceinline__ float group_sum(float v, float* lds) {
    v = xrow_sum(row_sum16(v));
    if constexpr (T > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();  // the last sum's readers
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v += lds[i];
    }
    return v;
}

template <bool kF32, int DT>
__device__ __forceinline__ void load_weight(const void* w, int64_t at, int64_t left,
                                            float (&x)[kChunk]) {
    if constexpr (kF32)
        load_chunk<kFP32>(static_cast<const uint32_t*>(w) + at, left, x);
    else
        load_chunk<DT>(static_cast<const typename Traits<DT>::elem*>(w) + at, left, x);
}

// T threads a row, N chunks a thread; kFp8: codes and scales instead of y.
// kWF32: a float32 weight.
template <int DT, int T, int N, bool kWF32, bool kResidual, bool kFp8>
__global__ __launch_bounds__(T < kBlockThreads ? kBlockThreads : T) void klp_norm_kernel(
    NormParams p) {
    typedef typename Traits<DT>::elem elem;
    __shared__ float lds[16];
    constexpr int kGroups = T < kBlockThreads ? kBlockThreads / T : 1;
    const int t = threadIdx.x % T;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / T;
    if (row >= p.rows) return;  // whole groups; T < 256 has no barrier
    const int dim = static_cast<int>(p.dim);
    const elem* x = static_cast<const elem*>(p.x) + row * p.ld_x;
    const elem* r = static_cast<const elem*>(p.residual) + row * p.ld_r;

    float h[N][kChunk];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * T + t) * kChunk;
        load_chunk<DT>(x + c, dim - c, h[i]);
    }
    if constexpr (kResidual) {
        elem* out = static_cast<elem*>(p.h) + row * p.dim;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * T + t) * kChunk;
            float b[kChunk];
            load_chunk<DT>(r + c, dim - c, b);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) h[i][j] = to_f32<DT>(from_f32<DT>(h[i][j] + b[j]));
            store_chunk<DT>(out + c, dim - c, h[i]);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    sum = group_sum<T>(sum, lds);
    const float s = 1.0f / sqrtf(sum / static_cast<float>(dim) + p.eps);
    if (p.rstd != nullptr && t == 0) p.rstd[row] = s;

#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * T + t) * kChunk;
        float w[kChunk], y[kChunk];
        load_weight<kWF32, DT>(p.weight, c, dim - c, w);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) y[j] = h[i][j] * s * w[j];
        if constexpr (kFp8) {
            // 16 lanes hold the 128 columns of a scale.
            const E4m3Scale e = e4m3_scale(row_max16(chunk_amax(y)));
            if (c < dim) {
                store_codes(p.q + row * p.dim + c, dim - c, e4m3_pack8(y, e.inv));
                if ((t & 15) == 0) p.scales[row * p.n_blocks + c / kScaleBlock] = e.scale;
            }
        } else {
            store_chunk<DT>(static_cast<elem*>(p.y) + row * p.dim + c, dim - c, y);
        }
    }
}

// The backward: group g of the grid takes rows g, g + groups, ...
template <int DT, int T, int N, bool kWF32, bool kWithH>
__global__ __launch_bounds__(T < kBlockThreads ? kBlockThreads : T) void klp_norm_bwd_kernel(
    NormBwdParams p) {
    typedef typename Traits<DT>::elem elem;
    __shared__ float lds[16];
    constexpr int kGroups = T < kBlockThreads ? kBlockThreads / T : 1;
    const int t = threadIdx.x % T;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / T;
    const int64_t groups = static_cast<int64_t>(gridDim.x) * kGroups;
    const int dim = static_cast<int>(p.dim);
    const float inv_dim = 1.0f / static_cast<float>(dim);
    uint32_t* share = reinterpret_cast<uint32_t*>(p.partials) + group * p.dim;

    // dx of a chunk, from its h and gy w.
    auto put = [&](int64_t row, int c, float s, float a, const float (&h)[kChunk],
                   const float (&gw)[kChunk]) {
        float d[kChunk];
        if constexpr (kWithH)
            load_chunk<DT>(static_cast<const elem*>(p.g_h) + row * p.dim + c, dim - c, d);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const float v = fmaf(-a, h[j], gw[j]);
            d[j] = kWithH ? fmaf(s, v, d[j]) : s * v;
        }
        store_chunk<DT>(static_cast<elem*>(p.d_x) + row * p.dim + c, dim - c, d);
    };

    if constexpr (N <= 2 || T < 1024) {
        float dw[N][kChunk];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < kChunk; ++j) dw[i][j] = 0.0f;
        for (int64_t row = group; row < p.rows; row += groups) {
            const elem* hp = static_cast<const elem*>(p.h) + row * p.ld_h;
            const elem* gp = static_cast<const elem*>(p.g_y) + row * p.dim;
            const float s = p.rstd[row];
            float h[N][kChunk], g[N][kChunk];
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (i * T + t) * kChunk;
                load_chunk<DT>(hp + c, dim - c, h[i]);
                load_chunk<DT>(gp + c, dim - c, g[i]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (i * T + t) * kChunk;
                float w[kChunk];
                load_weight<kWF32, DT>(p.weight, c, dim - c, w);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    dw[i][j] = fmaf(g[i][j] * s, h[i][j], dw[i][j]);
                    g[i][j] *= w[j];
                    dot = fmaf(g[i][j], h[i][j], dot);
                }
            }
            dot = group_sum<T>(dot, lds);
            const float a = s * s * dot * inv_dim;
#pragma unroll
            for (int i = 0; i < N; ++i) put(row, (i * T + t) * kChunk, s, a, h[i], g[i]);
        }
        if (p.partials != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (i * T + t) * kChunk;
                store_chunk<kFP32>(share + c, dim - c, dw[i]);
            }
        }
    } else {
        // Rows beyond 16384 columns: h, gy w and the sums of dw do not fit the
        // 128 registers that a thread of 1024 has.  h and gy are read twice,
        // the second time from L2, and the sums are kept where they end up, in
        // the group's share of the workspace, each column by one thread.
        for (int64_t row = group; row < p.rows; row += groups) {
            const elem* hp = static_cast<const elem*>(p.h) + row * p.ld_h;
            const elem* gp = static_cast<const elem*>(p.g_y) + row * p.dim;
            const float s = p.rstd[row];
            float dot = 0.0f, h[kChunk], g[kChunk], w[kChunk];
#pragma unroll 1
            for (int c = t * kChunk; c < dim; c += T * kChunk) {
                load_chunk<DT>(hp + c, dim - c, h);
                load_chunk<DT>(gp + c, dim - c, g);
                load_weight<kWF32, DT>(p.weight, c, dim - c, w);
                if (p.partials != nullptr) {
                    float dw[kChunk];
                    load_chunk<kFP32>(share + c, row == group ? 0 : dim - c, dw);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) dw[j] = fmaf(g[j] * s, h[j], dw[j]);
                    store_chunk<kFP32>(share + c, dim - c, dw);
                }
#pragma unroll
                for (int j = 0; j < kChunk; ++j) dot = fmaf(g[j] * w[j], h[j], dot);
            }
            dot = group_sum<T>(dot, lds);
            const float a = s * s * dot * inv_dim;
#pragma unroll 1
            for (int c = t * kChunk; c < dim; c += T * kChunk) {
                load_chunk<DT>(hp + c, dim - c, h);
                load_chunk<DT>(gp + c, dim - c, g);
                load_weight<kWF32, DT>(p.weight, c, dim - c, w);
#pragma unroll
                for (int j = 0; j < kChunk; ++j) g[j] *= w[j];
                put(row, c, s, a, h, g);
            }
        }
    }
}

// dw[c] = the groups' shares of column c: 64 columns a workgroup, its 16
// waves take every 16th share and are added in order.
constexpr int kSumWaves = 16;
template <int DT>
__global__ __launch_bounds__(kSumWaves * 64) void klp_norm_dw_kernel(NormBwdParams p) {
    typedef typename Traits<DT>::elem elem;
    __shared__ float part[kSumWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (c < p.dim) {
#pragma unroll 8
        for (int64_t g = wave; g < p.groups; g += kSumWaves) s += p.partials[g * p.dim + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.dim) {
#pragma unroll
        for (int i = 1; i < kSumWaves; ++i) s += part[i][lane];
        static_cast<elem*>(p.d_weight)[c] = from_f32<DT>(s);
    }
}

template <int DT, int T, int N, bool kWF32>
hipError_t launch_norm_shape(const NormParams& p, hipStream_t stream) {
    constexpr int kGroups = T < kBlockThreads ? kBlockThreads / T : 1;
    const dim3 grid(static_cast<unsigned>((p.rows + kGroups - 1) / kGroups));
    const dim3 block(T < kBlockThreads ? kBlockThreads : T);
    const auto launch = [&](auto kernel) {
        return launch_kernel(kernel, grid, block, stream, p);
    };
    if (p.q != nullptr)
        return p.residual != nullptr ? launch(klp_norm_kernel<DT, T, N, kWF32, true, true>)
                                     : launch(klp_norm_kernel<DT, T, N, kWF32, false, true>);
    return p.residual != nullptr ? launch(klp_norm_kernel<DT, T, N, kWF32, true, false>)
                                 : launch(klp_norm_kernel<DT, T, N, kWF32, false, false>);
}

template <int DT, int T, int N, bool kWF32>
hipError_t launch_norm_bwd_shape(const NormBwdParams& p, hipStream_t stream) {
    constexpr int kGroups = T < kBlockThreads ? kBlockThreads / T : 1;
    const dim3 grid(static_cast<unsigned>(p.groups / kGroups));
    const dim3 block(T < kBlockThreads ? kBlockThreads : T);
    return p.g_h != nullptr
               ? launch_kernel(klp_norm_bwd_kernel<DT, T, N, kWF32, true>, grid, block, stream, p)
               : launch_kernel(klp_norm_bwd_kernel<DT, T, N, kWF32, false>, grid, block, stream,
                               p);
}

template <int V> using Int = std::integral_constant<int, V>;

// f(threads, chunks) for the shape that holds rows of `dim` elements.
template <typename F>
hipError_t with_shape(int64_t dim, F f) {
    if (dim <= 512) return f(Int<64>{}, Int<1>{});
    if (dim <= 1024) return f(Int<64>{}, Int<2>{});
    if (dim <= 2048) return f(Int<64>{}, Int<4>{});
    if (dim <= 4096) return f(Int<256>{}, Int<2>{});
    if (dim <= 8192) return f(Int<512>{}, Int<2>{});
    if (dim <= 16384) return f(Int<1024>{}, Int<2>{});
    if (dim <= 32768) return f(Int<1024>{}, Int<4>{});
    return f(Int<1024>{}, Int<8>{});
}

template <int DT>
hipError_t launch_norm_dt(const NormParams& p, hipStream_t stream) {
    return with_shape(p.dim, [&](auto t, auto n) {
        constexpr int T = decltype(t)::value, N = decltype(n)::value;
        return DT == kFP32 || p.weight_f32 ? launch_norm_shape<DT, T, N, true>(p, stream)
                                           : launch_norm_shape<DT, T, N, DT == kFP32>(p, stream);
    });
}
template <int DT>
hipError_t launch_norm_bwd_dt(const NormBwdParams& p, hipStream_t stream) {
    return with_shape(p.dim, [&](auto t, auto n) {
        constexpr int T = decltype(t)::value, N = decltype(n)::value;
        return DT == kFP32 || p.weight_f32
                   ? launch_norm_bwd_shape<DT, T, N, true>(p, stream)
                   : launch_norm_bwd_shape<DT, T, N, DT == kFP32>(p, stream);
    });
}

}  // namespace

hipError_t launch_norm(int dtype, const NormParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_norm_dt<kBF16>(p, stream);
        case kFP16: return launch_norm_dt<kFP16>(p, stream);
        case kFP32: return launch_norm_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

int64_t norm_threads(int64_t dim) {
    int64_t threads = 0;
    with_shape(dim, [&](auto t, auto) {
        threads = decltype(t)::value;
        return hipSuccess;
    });
    return threads;
}

// Groups of the backward: enough workgroups to fill the chip, a multiple of
// the groups of one, and no more shares of dw than rows.
int64_t norm_bwd_groups(int64_t rows, int64_t dim) {
    const int64_t threads = norm_threads(dim);
    const int64_t per = threads < kBlockThreads ? kBlockThreads / threads : 1;
    int64_t groups = kNormBwdThreads / threads;
    if (groups > rows) groups = rows;
    return (groups + per - 1) / per * per;
}

hipError_t launch_norm_bwd(int dtype, const NormBwdParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_norm_bwd_dt<kBF16>(p, stream);
        case kFP16: return launch_norm_bwd_dt<kFP16>(p, stream);
        case kFP32: return launch_norm_bwd_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_norm_dw(int dtype, const NormBwdParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((p.dim + 63) / 64));
    const dim3 block(kSumWaves * 64);
    switch (dtype) {
        case kBF16: return launch_kernel(klp_norm_dw_kernel<kBF16>, grid, block, stream, p);
        case kFP16: return launch_kernel(klp_norm_dw_kernel<kFP16>, grid, block, stream, p);
        case kFP32: return launch_kernel(klp_norm_dw_kernel<kFP32>, grid, block, stream, p);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
