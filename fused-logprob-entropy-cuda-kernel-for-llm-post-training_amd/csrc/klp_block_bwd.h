// klp_block_bwd.h — the rows' pass of the backward of the norms around a block
// (the formulas: klp_block.hip); each dtype's instances are a file of their own.
#pragma once

#include "klp_block.h"

namespace klp {

namespace {

// A row's x or h: as stored, or the values of its checkpoint.
template <int DT, bool kKept, int kMode>
struct Stored {
    RawChunk<DT> raw;
    __device__ __forceinline__ void load(const void* rows, int64_t ld, const uint8_t*,
                                         const float*, int64_t row, int64_t, int c, int dim) {
        raw = fetch<DT, kMode>(rows, row * ld, c, dim);
    }
    __device__ __forceinline__ void in_place(int c, int dim) { settle<DT, kMode>(raw, c, dim); }
    __device__ __forceinline__ void values(float (&x)[kChunk]) const { raw.values(x); }
};
template <int DT, int kMode>
struct Stored<DT, true, kMode> {
    uint2 codes;
    float scale;
    __device__ __forceinline__ void load(const void*, int64_t, const uint8_t* q,
                                         const float* scales, int64_t row, int64_t n_blocks,
                                         int c, int dim) {
        codes = fetch_codes<kMode>(q, row * dim, c, dim);
        const float* of_row = scales + row * n_blocks;
        scale = of_row[static_cast<uint32_t>(c < dim ? c : 0) / kScaleBlock];
    }
    __device__ __forceinline__ void in_place(int c, int dim) { settle_codes<kMode>(codes, c, dim); }
    __device__ __forceinline__ void values(float (&x)[kChunk]) const {
        code_values(codes, scale, x);
    }
};

// kGate: 0 none, 1 one for all rows, 2 one for every per_gate rows.
template <int DT, int T, int N, int kMode, bool kPost, int kGate, bool kKept>
__global__ __launch_bounds__(kBackwardThreads<T>) void klp_block_bwd_kernel(BlockBwdParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int kGroups = kBackwardThreads<T> / T;
    constexpr int kCols = T * N * kChunk;
    constexpr bool kX = kPost || kGate != 0;  // x enters a gradient
    __shared__ float lds[kGroups][2][T / 64];
    // The sums of the workgroup's other groups, of one kind at a time.
    __shared__ float meet[kGroups > 1 ? (kGroups - 1) * kCols : 1];
    const int t = threadIdx.x % T;
    const int in_block = __builtin_amdgcn_readfirstlane(threadIdx.x / T);
    const int64_t group = static_cast<int64_t>(blockIdx.x) * kGroups + in_block;
    const int dim = static_cast<int>(p.dim);
    const float inv_dim = 1.0f / static_cast<float>(dim);
    const int64_t first = group * p.per_group;
    const int64_t end = first + p.per_group < p.rows ? first + p.per_group : p.rows;

    // A thread's sums.  A thread of 1024 has 128 registers: there the gate's and
    // the post weight's are kept in LDS, each by its own thread.  Even so, with a
    // post norm and a gate of all rows, 5 to 24 registers are spilled there, and 11
    // to 20 of 256 in 16-bit rows off 16-byte boundaries with a gate of some rows.
    constexpr bool kInLds = T == 1024;
    constexpr int kLdsSums = kInLds ? (kPost ? 1 : 0) + (kGate != 0 ? 1 : 0) : 0;
    __shared__ float held[kLdsSums > 0 ? kLdsSums * kCols : 1];
    float dw[N][kChunk], dp[kPost && !kInLds ? N : 1][kChunk],
        dg[kGate != 0 && !kInLds ? N : 1][kChunk];
    auto in_lds = [&](int which, int i, int j) -> float& {
        return held[(which * N * kChunk + i * kChunk + j) * T + t];
    };
    constexpr int kGateAt = kPost ? 1 : 0;
    auto sum_p = [&](int i, int j) -> float& {
        if constexpr (kInLds) return in_lds(0, i, j);
        else return dp[i][j];
    };
    auto sum_g = [&](int i, int j) -> float& {
        if constexpr (kInLds) return in_lds(kGateAt, i, j);
        else return dg[i][j];
    };
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            dw[i][j] = 0.0f;
            if constexpr (kPost) sum_p(i, j) = 0.0f;
            if constexpr (kGate != 0) sum_g(i, j) = 0.0f;
        }

    // A row's operands; 16-bit rows (and codes) have the next one's on their way
    // while one is worked on.  Two float32 rows do not fit the registers.
    constexpr bool kAhead = DT != kFP32 && T < 1024 && kMode != kAny;
    struct Row {
        Stored<DT, kKept, kMode> hs[N], xs[kX ? N : 1];
        RawChunk<DT> gys[N], ghs[N];
        float s_h, s_x;
    };
    // Keeps the chunks' work apart where registers are few.
    auto apart = [] {
        if constexpr (T == 1024 || kMode == kAny) __builtin_amdgcn_sched_barrier(0);
    };
    // A lane's column; hidden there, so that no address made of it is kept.
    auto column_of = [&](int i) {
        int c = (i * T + t) * kChunk;
        if constexpr (T == 1024) asm volatile("" : "+v"(c));
        return c;
    };
    // (kOdd reads the other gradient in the place of one that is not there.)
    const void* g_y = kMode == kOdd && p.g_y == nullptr ? p.g_h : p.g_y;
    const void* g_h = kMode == kOdd && p.g_h == nullptr ? p.g_y : p.g_h;
    auto load_row = [&](Row& r, int64_t step) {
        // The groups of a workgroup take the same number of steps, for their
        // barriers: those past a group's rows repeat the last and store nothing.
        const int64_t row = first + step < end ? first + step : p.rows - 1;
        r.s_h = p.rstd_h[row];
        r.s_x = kPost ? p.rstd_x[row] : 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            apart();
            const int c = column_of(i);
            r.hs[i].load(p.h, p.dim, p.h_codes, p.h_scales, row, p.n_blocks, c, dim);
            if constexpr (kX)
                r.xs[i].load(p.x, p.ld_x, p.x_codes, p.x_scales, row, p.n_blocks, c, dim);
            r.gys[i] = fetch<DT, kMode>(g_y, row * p.dim, c, dim);
            r.ghs[i] = fetch<DT, kMode>(g_h, row * p.dim, c, dim);
        }
    };
    // Before a row's first use.
    auto in_place = [&](Row& r) {
        if constexpr (kMode == kOdd) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                apart();
                const int c = column_of(i);
                r.hs[i].in_place(c, dim);
                if constexpr (kX) r.xs[i].in_place(c, dim);
                settle<DT, kMode>(r.gys[i], c, dim);
                settle<DT, kMode>(r.ghs[i], c, dim);
#pragma unroll
                for (int k = 0; k < RawChunk<DT>::kVecs; ++k) {
                    r.gys[i].v[k] &= p.g_y != nullptr ? ~0u : 0u;
                    r.ghs[i].v[k] &= p.g_h != nullptr ? ~0u : 0u;
                }
            }
        }
    };
    // Weights, and the gate while it lasts, in registers where they fit.
    constexpr bool kHold = T < 1024 && kMode != kAny;
    RawChunk<kWeight<DT, kMode>> w_held[kHold ? N : 1], wp_held[kHold && kPost ? N : 1];
    float by_held[kHold && kGate != 0 ? N : 1][kChunk];
    auto loaded_weight = [&](const void* of, int i) {
        const int c = column_of(i);
        auto w = fetch_weight<DT, kMode>(of, p.weight_f32, c, dim);
        settle_weight<DT, kMode>(w, p.weight_f32, c, dim);
        return w;
    };
    auto weight = [&](int i, float (&v)[kChunk]) {
        if constexpr (kHold) w_held[i].values(v);
        else loaded_weight(p.weight, i).values(v);
    };
    auto post = [&](int i, float (&v)[kChunk]) {
        if constexpr (kHold) wp_held[kPost ? i : 0].values(v);
        else loaded_weight(p.post, i).values(v);
    };
    auto load_gate = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            fetch_either<DT, kMode>(p.gate, p.gate_f32, row * p.dim, column_of(i), dim,
                                        by_held[kHold && kGate != 0 ? i : 0]);
    };
    if constexpr (kHold) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w_held[i] = loaded_weight(p.weight, i);
            if constexpr (kPost) wp_held[i] = loaded_weight(p.post, i);
        }
    }
    // Rows of the gate before `first`, and the gate's.
    const uint32_t per_gate = static_cast<uint32_t>(p.per_gate);
    uint32_t gate_row = 0, of_gate = 0;
    if constexpr (kGate == 2) {
        gate_row = static_cast<uint32_t>(first < p.rows ? first : p.rows - 1) / per_gate;
        of_gate = static_cast<uint32_t>(first < p.rows ? first : p.rows - 1) - gate_row * per_gate;
    }
    bool begun_here = of_gate == 0;
    if constexpr (kHold && kGate != 0) load_gate(gate_row);
    int slot = 0;
    Row r;
    if constexpr (kAhead) load_row(r, 0);
    for (int64_t step = 0; step < p.per_group; ++step) {
        const int64_t row = first + step;
        const bool live = row < end;
        Row next;
        if constexpr (kAhead) load_row(next, step + 1);
        else load_row(r, step);
        in_place(r);
        const float s_h = r.s_h, s_x = r.s_x;

        float dh[N][kChunk], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            apart();
            float w[kChunk], h[kChunk], g[kChunk];
            weight(i, w);
            r.hs[i].values(h);
            r.gys[i].values(g);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                if (live) dw[i][j] = fmaf(g[j] * s_h, h[j], dw[i][j]);
                dh[i][j] = g[j] * w[j];
                dot = fmaf(dh[i][j], h[j], dot);
            }
        }
        dot = group_sum_alternate<T>(dot, lds[in_block], slot);
        const float a_h = s_h * s_h * dot * inv_dim;
        float dot_x = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            apart();
            const int c = column_of(i);
            float h[kChunk], gh[kChunk], x[kChunk], by[kChunk], wp[kChunk];
            r.hs[i].values(h);
            r.ghs[i].values(gh);
#pragma unroll
            for (int j = 0; j < kChunk; ++j)
                dh[i][j] = fmaf(s_h, fmaf(-a_h, h[j], dh[i][j]), gh[j]);
            if (live && p.d_r != nullptr)
                store_chunk<DT>(column<elem>(p.d_r, row * p.dim, c), dim - c, dh[i]);
            if constexpr (kX) r.xs[i].values(x);
            if constexpr (kPost) post(i, wp);
            if constexpr (kGate != 0 && kHold) {
#pragma unroll
                for (int j = 0; j < kChunk; ++j) by[j] = by_held[i][j];
            } else if constexpr (kGate != 0) {
                fetch_either<DT, kMode>(p.gate, p.gate_f32,
                                            static_cast<int64_t>(gate_row) * p.dim, c, dim, by);
            }
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                const float d = dh[i][j] * p.scale;  // c dh
                if constexpr (kGate != 0) {
                    const float z = kPost ? x[j] * s_x * wp[j] : x[j];
                    if (live) sum_g(i, j) = fmaf(d, z, sum_g(i, j));
                }
                float dz = kGate != 0 ? d * by[j] : d;
                if constexpr (kPost) {
                    if (live) sum_p(i, j) = fmaf(dz * s_x, x[j], sum_p(i, j));
                    dz *= wp[j];
                    dot_x = fmaf(dz, x[j], dot_x);
                }
                dh[i][j] = dz;
            }
        }
        float a_x = 0.0f;
        if constexpr (kPost) {
            dot_x = group_sum_alternate<T>(dot_x, lds[in_block], slot);
            a_x = s_x * s_x * dot_x * inv_dim;
        }
        if (live && p.d_x != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                apart();
                const int c = column_of(i);
                if constexpr (kPost) {
                    float x[kChunk];
                    r.xs[i].values(x);
#pragma unroll
                    for (int j = 0; j < kChunk; ++j)
                        dh[i][j] = s_x * fmaf(-a_x, x[j], dh[i][j]);
                }
                store_chunk<DT>(column<elem>(p.d_x, row * p.dim, c), dim - c, dh[i]);
            }
        }
        if constexpr (kGate == 2) {
            // The gate's rows end here, or the group's do.
            const bool gate_ends = row + 1 == p.rows || of_gate + 1 == per_gate;
            if (live && p.d_gate != nullptr && (gate_ends || row + 1 == end)) {
                const int64_t from = static_cast<int64_t>(gate_row) * p.dim;
                float* share = p.gate_shares + (2 * group + (begun_here ? 1 : 0)) * p.dim;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int c = column_of(i);
                    float v[kChunk];
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) {
                        v[j] = sum_g(i, j);
                        sum_g(i, j) = 0.0f;
                    }
                    if (!(gate_ends && begun_here))
                        store_chunk<kFP32>(column<uint32_t>(share, 0, c), dim - c, v);
                    else if (DT == kFP32 || p.gate_f32)
                        store_chunk<kFP32>(column<uint32_t>(p.d_gate, from, c), dim - c, v);
                    else
                        store_chunk<DT>(column<elem>(p.d_gate, from, c), dim - c, v);
                }
            }
            if (live) {
                if (gate_ends && row + 1 < p.rows) {
                    ++gate_row;
                    if constexpr (kHold) load_gate(gate_row);
                }
                of_gate = gate_ends ? 0 : of_gate + 1;
                begun_here |= gate_ends;
            }
        }
        if constexpr (kAhead) r = next;
    }

    // The workgroup's sums: its groups' in order, into its share.
    auto share = [&](auto of, float* shares) {
        if (shares == nullptr) return;
        float sum[N][kChunk];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < kChunk; ++j) sum[i][j] = of(i, j);
        if constexpr (kGroups > 1) {
            __syncthreads();
            if (in_block > 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < kChunk; ++j)
                        meet[(in_block - 1) * kCols + (i * kChunk + j) * T + t] = sum[i][j];
            }
            __syncthreads();
            if (in_block > 0) return;
#pragma unroll
            for (int q = 0; q < kGroups - 1; ++q)
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < kChunk; ++j)
                        sum[i][j] += meet[q * kCols + (i * kChunk + j) * T + t];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * T + t) * kChunk;
            store_chunk<kFP32>(column<uint32_t>(shares, blockIdx.x * p.dim, c), dim - c, sum[i]);
        }
    };
    share([&](int i, int j) { return dw[i][j]; }, p.weight_shares);
    if constexpr (kPost) share(sum_p, p.post_shares);
    if constexpr (kGate == 1) share(sum_g, p.gate_shares);
}

template <int DT, int T, int N, int kMode, bool kPost, int kGate>
hipError_t launch_bwd_kept(const BlockBwdParams& p, hipStream_t stream) {
    constexpr int kThreads = kBackwardThreads<T>, kGroups = kThreads / T;
    const dim3 grid(static_cast<unsigned>((p.groups + kGroups - 1) / kGroups)), block(kThreads);
    return p.h_codes != nullptr
               ? launch_kernel(klp_block_bwd_kernel<DT, T, N, kMode, kPost, kGate, true>, grid,
                               block, stream, p)
               : launch_kernel(klp_block_bwd_kernel<DT, T, N, kMode, kPost, kGate, false>, grid,
                               block, stream, p);
}
template <int DT, int T, int N, int kMode, bool kPost>
hipError_t launch_bwd_gate(const BlockBwdParams& p, hipStream_t stream) {
    if (p.gate == nullptr) return launch_bwd_kept<DT, T, N, kMode, kPost, 0>(p, stream);
    return p.per_gate >= p.rows ? launch_bwd_kept<DT, T, N, kMode, kPost, 1>(p, stream)
                                : launch_bwd_kept<DT, T, N, kMode, kPost, 2>(p, stream);
}
template <int DT, int T, int N, int kMode>
hipError_t launch_bwd_shape(const BlockBwdParams& p, hipStream_t stream) {
    return p.post != nullptr ? launch_bwd_gate<DT, T, N, kMode, true>(p, stream)
                             : launch_bwd_gate<DT, T, N, kMode, false>(p, stream);
}

template <int DT>
hipError_t launch_rows_dt(const BlockBwdParams& p, hipStream_t stream) {
    return with_shape(p.dim, [&](auto t, auto n) {
        constexpr int T = decltype(t)::value, N = decltype(n)::value;
        return with_mode<DT, T, N>(p, [&](auto mode) {
            return launch_bwd_shape<DT, T, N, decltype(mode)::value>(p, stream);
        });
    });
}

}  // namespace

}  // namespace klp
