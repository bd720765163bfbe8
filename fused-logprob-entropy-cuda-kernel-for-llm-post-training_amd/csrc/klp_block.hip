// klp_block.hip — the norms around a block: its output through a norm, a gate
// and a residual scale into the residual stream, and the next block's norm;
// their backward; for gfx950.
//
//   s_x = (mean(x^2) + eps)^-1/2,   z = x s_x wp        (z = x without wp)
//   h = round(r + c g z)
//   s_h = (mean(h^2) + eps)^-1/2,   y = round(h s_h w), or e4m3 codes of it
//
//   dh = gh + s_h (gy w - h s_h^2 mean(gy w h)),        dr = dh
//   dz = c g dh,   dx = s_x (dz wp - x s_x^2 mean(dz wp x))   (dx = dz without)
//   dw = sum gy h s_h,   dwp = sum dz x s_x,   dg = sum c z dh
//
// the sums over all rows, dg's over the rows that share a gate.  Statistics are
// those of the stored h; all sums are float32, every output is rounded once.
//
// Checkpoints: the forward also leaves e4m3 codes of x and h with a float32
// scale for each 128 columns, and the backward takes the values that they stand
// for in place of x and h; s_x and s_h are the exact ones.  An element then
// keeps 2.06 bytes of the block alive instead of 4.
//
// Bound by memory: the forward reads x and r once and writes h and y once, the
// backward reads x, h and two gradients once and writes two, a row in the
// registers of a group of 64 to 1024 threads, 8 elements (a chunk) a thread and
// pass.  bf16, us (TB/s), post norm and a gate of all rows:
//   rows x dim     forward     backward                its sums
//   32768 x 1024   49 (5.5)    84 (4.8)                4
//   8192 x 4096    51 (5.3)    87 (4.6)                6
//     no gate      51          82
//     bare         42 (6.4)    50 (6.7: 5 arrays)
//     gate of 128 rows         87                      5 + 7 (the gate's)
//     of a row     60 (5.6)    111 (4.8: 8 arrays)     5
//     checkpoints  65 (5.2)    78 (4.3)                5
//   4096 x 8192    54          90                      11
//   2048 x 16384   55          118                     9
//   4096 x 4096    61          84 (float32)            5
// Widths between a shape's, 8192 rows, us (TB/s); lanes behind the row hold nothing:
//   2304           35 (4.3)    58 (3.9)                4
//   3584           46 (5.2)    72 (4.9)                6
//   4097 (odd)     123 (2.2)   136 (3.0)               7
//   4608           71 (4.3)    101 (4.5)               7
//   5120           74 (4.5)    110 (4.6)               7
//   6144           82 (4.9)    140 (4.3)               11
//   7168           92 (5.1)    158 (4.5)               12
//   2048 x 12288   48 (4.2)    93 (3.3)                7
//   2048 x 13001   86 (2.5)    128 (2.5)               10
// e4m3 output, no gate: 64 x 3584 4.4 (the launch); 8192 x 3584 36 (5.7), x 4096 39
// (6.0), x 5120 59 (5.0); 2048 x 16384 46 (5.1).
// The forward prefetches nothing beyond its row: many workgroups a CU do that.
// The backward's groups are few and long, and with each load waiting for the one
// before (143 us at 8192 x 4096) it was bound by latency, so 16-bit rows have the
// next row's under this row's sums.
//
// Sums over rows: a group takes consecutive rows and keeps its sums in
// registers; the groups of a workgroup are added in LDS, the workgroups' shares
// by a second kernel in order, so that nothing depends on timing.  A gate of
// fewer rows ends inside a group or goes on past it: whole ones are written as
// they end, the parts of others go to the group's two shares.
#include "klp_block.h"

namespace klp {

namespace {

// Codes and scale of a chunk; 16 lanes hold the 128 columns of a scale.
__device__ __forceinline__ void put_codes(const float (&v)[kChunk], uint8_t* q, float* scales,
                                          int64_t row, int64_t dim, int64_t n_blocks, int c) {
    const E4m3Scale e = e4m3_scale(row_max16(chunk_amax(v)));
    if (c < dim) {
        store_codes(column<uint8_t>(q, row * dim, c), dim - c, e4m3_pack8(v, e.inv));
        if ((threadIdx.x & 15) == 0) scales[row * n_blocks + c / kScaleBlock] = e.scale;
    }
}

template <int DT, int T, int N, int kMode, bool kPost, bool kFp8>
__global__ __launch_bounds__(kForwardThreads<T>) void klp_block_kernel(BlockParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int kGroups = kForwardThreads<T> / T;
    __shared__ float lds[kGroups][2][T / 64];
    int slot = 0;
    const int t = threadIdx.x % T;
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
    // Groups past the last row repeat it, with the same results, and meet the
    // others at every barrier.
    if (row >= p.rows) row = p.rows - 1;
    const int dim = static_cast<int>(p.dim);

    // What the first sum does not need is on its way while it is made.
    RawChunk<DT> in[N], res[N];
    RawChunk<kWeight<DT, kMode>> wp[N], w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * T + t) * kChunk;
        in[i] = fetch<DT, kMode>(p.x, row * p.ld_x, c, dim);
        res[i] = fetch<DT, kMode>(p.residual, row * p.ld_r, c, dim);
        if constexpr (kPost) wp[i] = fetch_weight<DT, kMode>(p.post, p.weight_f32, c, dim);
        w[i] = fetch_weight<DT, kMode>(p.weight, p.weight_f32, c, dim);
    }

    float h[N][kChunk];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        settle<DT, kMode>(in[i], (i * T + t) * kChunk, dim);
        in[i].values(h[i]);
    }
    if (p.x_codes != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            put_codes(h[i], p.x_codes, p.x_scales, row, p.dim, p.n_blocks,
                      (i * T + t) * kChunk);
    }
    if constexpr (kPost) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < kChunk; ++j) sum = fmaf(h[i][j], h[i][j], sum);
        sum = group_sum_alternate<T>(sum, lds[group], slot);
        const float s = 1.0f / sqrtf(sum / static_cast<float>(dim) + p.eps);
        if (p.rstd_x != nullptr && t == 0) p.rstd_x[row] = s;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[kChunk];
            settle_weight<DT, kMode>(wp[i], p.weight_f32, (i * T + t) * kChunk, dim);
            wp[i].values(v);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) h[i][j] = h[i][j] * s * v[j];
        }
    }
    if (p.gate != nullptr) {
        const int64_t at = static_cast<uint32_t>(row) / static_cast<uint32_t>(p.per_gate) * p.dim;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[kChunk];
            fetch_either<DT, kMode>(p.gate, p.gate_f32, at, (i * T + t) * kChunk, dim, v);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) h[i][j] *= v[j];
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * T + t) * kChunk;
        float b[kChunk];
        settle<DT, kMode>(res[i], c, dim);
        res[i].values(b);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            h[i][j] = to_f32<DT>(from_f32<DT>(fmaf(h[i][j], p.scale, b[j])));
            sum = fmaf(h[i][j], h[i][j], sum);
        }
        store_chunk<DT>(column<elem>(p.h, row * p.dim, c), dim - c, h[i]);
    }
    if (p.h_codes != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            put_codes(h[i], p.h_codes, p.h_scales, row, p.dim, p.n_blocks,
                      (i * T + t) * kChunk);
    }
    sum = group_sum_alternate<T>(sum, lds[group], slot);
    const float s = 1.0f / sqrtf(sum / static_cast<float>(dim) + p.eps);
    if (p.rstd_h != nullptr && t == 0) p.rstd_h[row] = s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * T + t) * kChunk;
        float y[kChunk], v[kChunk];
        settle_weight<DT, kMode>(w[i], p.weight_f32, c, dim);
        w[i].values(v);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) y[j] = h[i][j] * s * v[j];
        if constexpr (kFp8) put_codes(y, p.q, p.scales, row, p.dim, p.n_blocks, c);
        else store_chunk<DT>(column<elem>(p.y, row * p.dim, c), dim - c, y);
    }
}

// out[c] = the shares of column c added in order: 64 columns a workgroup, its
// 16 waves take every 16th share and are added in order.
struct BlockSumParams {
    const float* shares;
    int64_t n;
    int64_t dim;
    void* out;
    int dtype;
};
constexpr int kSumWaves = 16;
__device__ __forceinline__ void put_either(void* out, int dtype, int64_t at, float v) {
    switch (dtype) {
        case kBF16: static_cast<uint16_t*>(out)[at] = from_f32<kBF16>(v); break;
        case kFP16: static_cast<uint16_t*>(out)[at] = from_f32<kFP16>(v); break;
        default: static_cast<float*>(out)[at] = v;
    }
}
struct BlockSums {
    BlockSumParams of[3];
};
__global__ __launch_bounds__(kSumWaves * 64) void klp_block_sum_kernel(BlockSums all) {
    const BlockSumParams& p = all.of[blockIdx.y];
    __shared__ float part[kSumWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (c < p.dim) {
#pragma unroll 8
        for (int64_t g = wave; g < p.n; g += kSumWaves) s += p.shares[g * p.dim + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.dim) {
#pragma unroll
        for (int i = 1; i < kSumWaves; ++i) s += part[i][lane];
        put_either(p.out, p.dtype, c, s);
    }
}

// A gate whose rows several groups took: from the last share of the group that
// it begins in and the first ones of the others, added as above.  blockIdx.y is
// the gate, or with by_group the group in which one begins that goes on.
// A lane takes 4 columns, the workgroup's 4 waves every 4th share.
constexpr int kGateWaves = 4;
__global__ __launch_bounds__(kGateWaves * 64) void klp_block_gate_kernel(BlockBwdParams p,
                                                                        int dtype,
                                                                        bool by_group) {
    __shared__ float part[kGateWaves][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t y = blockIdx.y;
    const int64_t group_end = (y + 1) * p.per_group < p.rows ? (y + 1) * p.per_group : p.rows;
    const int64_t gate = by_group ? (group_end - 1) / p.per_gate : y;
    const int64_t begin = gate * p.per_gate;
    const int64_t end = begin + p.per_gate < p.rows ? begin + p.per_gate : p.rows;
    const int64_t from = begin / p.per_group, to = (end - 1) / p.per_group;
    if (from == to || (by_group && from != y)) return;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 64 + lane) * 4;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int64_t g = from + wave; g <= to; g += kGateWaves) {
        const float* share = p.gate_shares + (2 * g + (g == from ? 1 : 0)) * p.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += share[c + j < p.dim ? c + j : 0];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][j][lane] = s[j];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 1; i < kGateWaves; ++i) s[j] += part[i][j][lane];
        if (c + j < p.dim) put_either(p.d_gate, dtype, gate * p.dim + c + j, s[j]);
    }
}

template <int DT, int T, int N, int kMode>
hipError_t launch_block_shape(const BlockParams& p, hipStream_t stream) {
    constexpr int kThreads = kForwardThreads<T>, kGroups = kThreads / T;
    const dim3 grid(static_cast<unsigned>((p.rows + kGroups - 1) / kGroups)), block(kThreads);
    const auto launch = [&](auto kernel) {
        return launch_kernel(kernel, grid, block, stream, p);
    };
    if (p.q != nullptr)
        return p.post != nullptr ? launch(klp_block_kernel<DT, T, N, kMode, true, true>)
                                 : launch(klp_block_kernel<DT, T, N, kMode, false, true>);
    return p.post != nullptr ? launch(klp_block_kernel<DT, T, N, kMode, true, false>)
                             : launch(klp_block_kernel<DT, T, N, kMode, false, false>);
}

template <int DT>
hipError_t launch_block_dt(const BlockParams& p, hipStream_t stream) {
    return with_shape(p.dim, [&](auto t, auto n) {
        constexpr int T = decltype(t)::value, N = decltype(n)::value;
        return with_mode<DT, T, N>(p, [&](auto mode) {
            return launch_block_shape<DT, T, N, decltype(mode)::value>(p, stream);
        });
    });
}
}  // namespace

hipError_t launch_block(int dtype, const BlockParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_block_dt<kBF16>(p, stream);
        case kFP16: return launch_block_dt<kFP16>(p, stream);
        case kFP32: return launch_block_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

// Groups of the backward: 1024 threads a CU, and no more than rows.
BlockShape block_shape(int64_t rows, int64_t dim) {
    return with_shape(dim, [&](auto t, auto) {
        constexpr int T = decltype(t)::value;
        constexpr int kGroups = kBackwardThreads<T> / T;
        BlockShape s;
        s.groups = kNormBwdThreads / T < rows ? kNormBwdThreads / T : rows;
        s.per_group = (rows + s.groups - 1) / s.groups;
        s.groups = (rows + s.per_group - 1) / s.per_group;
        s.shares = (s.groups + kGroups - 1) / kGroups;
        return s;
    });
}

hipError_t launch_block_bwd(int dtype, const BlockBwdParams& p, hipStream_t stream) {
    hipError_t e = hipErrorInvalidValue;
    switch (dtype) {
        case kBF16: e = launch_block_rows<kBF16>(p, stream); break;
        case kFP16: e = launch_block_rows<kFP16>(p, stream); break;
        case kFP32: e = launch_block_rows<kFP32>(p, stream); break;
        default: break;
    }
    if (e != hipSuccess) return e;
    const int weight_dtype = p.weight_f32 ? kFP32 : dtype;
    const int gate_dtype = p.gate_f32 ? kFP32 : dtype;
    const int64_t shares = block_shape(p.rows, p.dim).shares;
    const bool one_gate = p.gate != nullptr && p.per_gate >= p.rows;
    BlockSums sums{};
    int n = 0;
    if (p.d_weight != nullptr)
        sums.of[n++] = BlockSumParams{p.weight_shares, shares, p.dim, p.d_weight, weight_dtype};
    if (p.d_post != nullptr)
        sums.of[n++] = BlockSumParams{p.post_shares, shares, p.dim, p.d_post, weight_dtype};
    if (one_gate && p.d_gate != nullptr)
        sums.of[n++] = BlockSumParams{p.gate_shares, shares, p.dim, p.d_gate, gate_dtype};
    if (n > 0) {
        const dim3 grid(static_cast<unsigned>((p.dim + 63) / 64), static_cast<unsigned>(n));
        e = launch_kernel(klp_block_sum_kernel, grid, dim3(kSumWaves * 64), stream, sums);
        if (e != hipSuccess) return e;
    }
    // A gate of one row lies in one group.
    if (p.gate != nullptr && !one_gate && p.d_gate != nullptr && p.per_gate > 1) {
        const int64_t gates = (p.rows + p.per_gate - 1) / p.per_gate;
        const bool by_group = gates > p.groups;
        const dim3 grid(static_cast<unsigned>((p.dim + 255) / 256),
                        static_cast<unsigned>(by_group ? p.groups : gates));
        e = launch_kernel(klp_block_gate_kernel, grid, dim3(kGateWaves * 64), stream, p, gate_dtype,
                          by_group);
    }
    return e;
}

}  // namespace klp
