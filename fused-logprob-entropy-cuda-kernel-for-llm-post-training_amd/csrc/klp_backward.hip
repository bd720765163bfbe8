// klp_backward.hip — backward kernel for gfx950 (replaces the reference's
// fused_logprob_entropy_v1_backward_kernel, csrc/fused_logprob.cu:243-282).
//
// For every element of a row:
//   lp = x - lse,  p = exp(lp),
//   d  = p * (c0 - g_ent * lp) + (v == t ? g_logp : 0),
//   c0 = g_lse - g_logp - g_ent * H          (hoisted per row, as at :271)
// One 16-byte load and one 16-byte store per 16 bytes of logits; nothing else
// touches memory except eight per-row scalars.
//
// p is computed as 2^(x*log2e - lse*log2e) with lse*log2e split into a
// rounded head and its exact fma remainder, so the exponent carries one
// rounding.  A -inf logit gets a gradient of exactly 0 (p = 0), where the
// reference's 0 * inf gives NaN; lp is clamped for that.
//
// With a temperature T (BwdParams::scale = 1/T != 1) the logits are scaled by
// 1/T on load, as in the forward, and the gradient is multiplied by 1/T.
//
// With alternatives (kTop: klp_bwd_top) each of their log-probabilities adds
//   g_top[j] ((v == id_j) - p)
// so that c0 loses the sum of g_top, and the few id_j that lie in a
// workgroup's piece are listed in LDS while its first vectors are on their
// way; every vector looks the list through before it is rounded.  1024 rows of
// 152064 bf16: 98 to 106 us without, 118 to 126 with 1 to 128 alternatives, 132
// with 256.
#include "klp_device.h"
#include "klp_launch.h"

namespace klp {

// The alternatives of a workgroup's piece: their vector of the piece (-1: an
// element of the row's edges), their element of it (of the row), and their
// gradient.
struct TopHits {
    int n;
    int vec[kTopMax];
    int elem[kTopMax];
    float grad[kTopMax];
    float sum[16];  // of the waves' g_top
};
template <bool kTop> struct TopOf {};
template <> struct TopOf<true> { TopHits h; };

// A 16-byte vector at the alignment of the shortest element.
typedef u32x4 u32x4_elem_aligned __attribute__((aligned(2)));

// The piece's 16-byte vectors [vb, ve) (the body of klp_bwd_kernel).  `vout`
// is 16-byte aligned; `vin` is too, or, with kInAligned false, only as an
// element is.
template <int DT, int WAVES, int U, bool kNtStore, bool kScaled, bool kInAligned, bool kLseNonNeg,
          bool kTop>
__device__ __forceinline__ void bwd_vectors(const BwdParams& p, const u32x4* vin, u32x4* vout,
                                            int64_t vb, int64_t ve, int64_t t_vec,
                                            int t_lane_elem, const RowGrad& g,
                                            const TopOf<kTop>& top) {
    constexpr int NTHREADS = WAVES * 64;
    constexpr int EPV = Traits<DT>::kPerVec;
    const int tid = threadIdx.x;
    // Buffer loads through a descriptor over the piece, with 32-bit offsets
    // (the caller keeps pieces under 2 GiB): C4 3113-3132 us against
    // 3166-3195 us for global loads of the same policy, C2 equal.  Temporal
    // loads here (non-temporal in the forward): measured best for a forward
    // followed by a backward over the same logits.
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<u32x4*>(vin + vb), 0, static_cast<int>((ve - vb) * 16), 0x00020000);
    for (int64_t i0 = vb; i0 < ve; i0 += static_cast<int64_t>(NTHREADS) * U) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t idx = i0 + tid + u * NTHREADS;
            if (idx < ve) {
                if constexpr (kInAligned)
                    v[u] = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, static_cast<int>((idx - vb) * 16), 0, 0);
                else
                    v[u] = reinterpret_cast<const u32x4_elem_aligned*>(vin)[idx];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t idx = i0 + tid + u * NTHREADS;
            if (idx < ve) {
                float x[EPV];
                unpack<DT>(v[u], x);
#pragma unroll
                for (int j = 0; j < EPV; ++j)
                    x[j] = grad_elem<DT, kLseNonNeg>(kScaled ? x[j] * p.scale : x[j], g);
                if (idx == t_vec) {
#pragma unroll
                    for (int j = 0; j < EPV; ++j)
                        if (j == t_lane_elem) x[j] += g.g_logp;
                }
                if constexpr (kTop) {
                    for (int h = 0; h < top.h.n; ++h) {
                        if (top.h.vec[h] != static_cast<int>(idx - vb)) continue;
                        const int e = top.h.elem[h];
#pragma unroll
                        for (int j = 0; j < EPV; ++j)
                            if (j == e) x[j] += top.h.grad[h];
                    }
                }
                if (kScaled) {
#pragma unroll
                    for (int j = 0; j < EPV; ++j) x[j] *= p.scale;
                }
                if constexpr (kNtStore) __builtin_nontemporal_store(pack<DT>(x), vout + idx);
                else vout[idx] = pack<DT>(x);
            }
        }
    }
}

// fp32 rows take their Fast2Sum operand order from the sign of lse
// (grad_one_fp32): one branch per row, outside the element loop.
template <int DT, int WAVES, int U, bool kNtStore, bool kScaled, bool kInAligned, bool kTop>
__device__ __forceinline__ void bwd_piece(const BwdParams& p, const u32x4* vin, u32x4* vout,
                                          int64_t vb, int64_t ve, int64_t t_vec, int t_lane_elem,
                                          const RowGrad& g, const TopOf<kTop>& top) {
    if (DT != kFP32 || g.lse >= 0.0f)
        bwd_vectors<DT, WAVES, U, kNtStore, kScaled, kInAligned, true, kTop>(
            p, vin, vout, vb, ve, t_vec, t_lane_elem, g, top);
    else
        bwd_vectors<DT, WAVES, U, kNtStore, kScaled, kInAligned, false, kTop>(
            p, vin, vout, vb, ve, t_vec, t_lane_elem, g, top);
}

// Rows of up to this many elements whose input and output sit at different
// offsets go one element a lane: a few loads a lane in flight at once, where
// the edges come before the vectors.  GPU time, us, bf16, elements / vectors:
// 4096 x 100 5.4 / 8.7, 4096 x 1001 7.5 / 9.2, 512 x 1501 3.7 / 3.4, 4096 x
// 2001 11.7 / 10.0; fp32 4096 x 1001 9.0 / 9.4, 4096 x 1501 11.2 / 10.5.
constexpr int64_t kBwdElementRow = 1024;

// The alternatives that place(id, &vec, &elem) finds in the workgroup's part,
// into `h`; returns the sum of the gradients of all that exist.  The ids of a
// row differ, so that the list's order is of no consequence.
template <int WAVES, typename F>
__device__ __forceinline__ float list_top(const BwdParams& p, int64_t row, TopHits& h, F place) {
    static_assert(WAVES <= 16, "the waves' sums");
    const int64_t* ids = p.top_ids + row * p.k;
    const float* grads = p.g_top + row * p.k;
    if (threadIdx.x == 0) h.n = 0;
    __syncthreads();
    float s = 0.0f;
    for (int j = threadIdx.x; j < p.k; j += WAVES * 64) {
        const int64_t id = ids[j];
        const float g = grads[j];
        if (id < 0 || id >= p.vocab) continue;
        s += g;
        int vec, elem;
        if (!place(id, &vec, &elem)) continue;
        const int at = atomicAdd(&h.n, 1);
        h.vec[at] = vec;
        h.elem[at] = elem;
        h.grad[at] = g;
    }
    s = xrow_sum(row_sum16(s));
    if ((threadIdx.x & 63) == 0) h.sum[threadIdx.x >> 6] = s;
    __syncthreads();
    s = h.sum[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += h.sum[w];
    return s;
}
// What an element of the edges (or of a row taken element by element) gets.
__device__ __forceinline__ float top_at(const TopHits& h, int64_t v) {
    float g = 0.0f;
    for (int i = 0; i < h.n; ++i)
        if (h.vec[i] < 0 && h.elem[i] == static_cast<int>(v)) g = h.grad[i];
    return g;
}

// A workgroup's part of a row.
struct BwdPart {
    int64_t head, tail_begin;  // elements before the first vector, and from here on
    int64_t vb, ve;            // its vectors
};
template <int EPV>
__device__ __forceinline__ BwdPart bwd_part(uintptr_t out_addr, int64_t vocab, int splits,
                                            int split) {
    constexpr int ESZ = 16 / EPV;
    int64_t head = static_cast<int64_t>(((16u - (out_addr & 15u)) & 15u) / ESZ);
    if (head > vocab) head = vocab;
    const int64_t nvec = (vocab - head) / EPV;
    // Pieces are whole multiples of 8 vectors (128 bytes, one cache line
    // when the row is line-aligned), so that no line is written, or read,
    // by two workgroups (C4's 18992-vector rows in 8 pieces would otherwise
    // split a line at every boundary: +1.2% HBM writes).
    int64_t per = (nvec + splits - 1) / splits;
    per = (per + 7) & ~int64_t{7};
    int64_t vb = static_cast<int64_t>(split) * per;
    int64_t ve = vb + per;
    if (vb > nvec) vb = nvec;
    if (ve > nvec) ve = nvec;
    return BwdPart{head, head + nvec * EPV, vb, ve};
}

// A far row's part (far_row) once more, over what was put there, element by
// element.  It reads the kernel's arguments again: kept for it, they would take the
// usual way's SGPRs beyond what lets 8 waves of it run (4096 x 151936 bf16 386 to
// 417 us), and a branch before that would keep its loads waiting for lse (397).
template <int DT, int WAVES, bool kScaled, bool kTop>
__device__ __forceinline__ void redo_far(TopOf<kTop>& top) {
    typedef typename Traits<DT>::elem elem;
    constexpr int EPV = Traits<DT>::kPerVec;
    uintptr_t args = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+v"(args));
    BwdParams p;
    __builtin_memcpy(&p, reinterpret_cast<const void*>(args), sizeof p);
    const int64_t row = blockIdx.x / p.splits;
    const int split = static_cast<int>(blockIdx.x - row * p.splits);
    const elem* rp = static_cast<const elem*>(p.logits) + row_offset(p.rm, row);
    elem* dp = static_cast<elem*>(p.d_logits) + row * p.vocab;
    const float ent = p.entropy[row];
    const float maximum = far_maximum(p.lse[row], ent);
    const int64_t tgt = p.targets[row];
    const BwdPart part =
        bwd_part<EPV>(reinterpret_cast<uintptr_t>(dp), p.vocab, p.splits, split);
    RowGrad g = row_grad(ent, ent, p.g_logp ? p.g_logp[row] : 0.0f, p.g_ent ? p.g_ent[row] : 0.0f,
                         p.g_lse ? p.g_lse[row] : 0.0f);
    // Its vectors' elements [b, e), with split 0 those before and behind all vectors.
    const int64_t b = part.head + part.vb * EPV, e = part.head + part.ve * EPV;
    const int64_t e0 = split == 0 ? part.head : 0, b1 = split == 0 ? part.tail_begin : p.vocab;
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    __syncthreads();
    if constexpr (kTop)
        g.c0 -= list_top<WAVES>(p, row, top.h, [&](int64_t id, int* vec, int* elem) {
            *vec = -1;
            *elem = static_cast<int>(id);
            return (id >= b && id < e) || id < e0 || id >= b1;
        });
    const int64_t n = e - b + e0 + (p.vocab - b1);
    for (int64_t i = threadIdx.x; i < n; i += WAVES * 64) {
        const int64_t edge = i - (e - b);
        const int64_t v = edge < 0 ? b + i : edge < e0 ? edge : b1 + (edge - e0);
        float x = to_f32<DT>(rp[v]);
        if (kScaled) x *= p.scale;
        x = near_logit(x, maximum);
        float d = grad_elem<DT, true>(x, g);
        if (v == tgt) d += g.g_logp;
        if constexpr (kTop) d += top_at(top.h, v);
        if (kScaled) d *= p.scale;
        dp[v] = from_f32<DT>(d);
    }
}

template <int DT, int WAVES, int U, bool kNtStore, bool kScaled, bool kTop>
__global__ __launch_bounds__(WAVES * 64) void klp_bwd_kernel(BwdParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int EPV = Traits<DT>::kPerVec;

    const int tid = threadIdx.x;
    const int64_t row = static_cast<int64_t>(blockIdx.x) / p.splits;
    const int split = static_cast<int>(static_cast<int64_t>(blockIdx.x) - row * p.splits);

    const int64_t vocab = p.vocab;
    const elem* rp = static_cast<const elem*>(p.logits) + row_offset(p.rm, row);
    elem* dp = static_cast<elem*>(p.d_logits) + row * vocab;
    const int64_t tgt = p.targets[row];

    RowGrad g = row_grad(p.lse[row], p.entropy[row], p.g_logp ? p.g_logp[row] : 0.0f,
                         p.g_ent ? p.g_ent[row] : 0.0f, p.g_lse ? p.g_lse[row] : 0.0f);
    __shared__ TopOf<kTop> top;

    const uintptr_t in_addr = reinterpret_cast<uintptr_t>(rp);
    const uintptr_t out_addr = reinterpret_cast<uintptr_t>(dp);
    if (((in_addr ^ out_addr) & 15u) != 0 && vocab <= kBwdElementRow && !far_row(g.lse)) {
        const int64_t per = (vocab + p.splits - 1) / p.splits;
        const int64_t b = static_cast<int64_t>(split) * per;
        const int64_t e = b + per < vocab ? b + per : vocab;
        if constexpr (kTop)
            g.c0 -= list_top<WAVES>(p, row, top.h, [&](int64_t id, int* vec, int* elem) {
                *vec = -1;
                *elem = static_cast<int>(id);
                return id >= b && id < e;
            });
        for (int64_t v = b + tid; v < e; v += WAVES * 64) {
            float x = to_f32<DT>(rp[v]);
            if (kScaled) x *= p.scale;
            float d = g.lse >= 0.0f ? grad_elem<DT, true>(x, g) : grad_elem<DT, false>(x, g);
            if (v == tgt) d += g.g_logp;
            if constexpr (kTop) d += top_at(top.h, v);
            if (kScaled) d *= p.scale;
            dp[v] = from_f32<DT>(d);
        }
        return;
    }

    const BwdPart part = bwd_part<EPV>(out_addr, vocab, p.splits, split);
    const int64_t head = part.head, tail_begin = part.tail_begin, vb = part.vb, ve = part.ve;
    const u32x4* vin = reinterpret_cast<const u32x4*>(rp + head);
    u32x4* vout = reinterpret_cast<u32x4*>(dp + head);

    if constexpr (kTop)
        g.c0 -= list_top<WAVES>(p, row, top.h, [&](int64_t id, int* vec, int* elem) {
            if (id < head || id >= tail_begin) {
                *vec = -1;
                *elem = static_cast<int>(id);
                return split == 0;
            }
            const int64_t v = (id - head) / EPV;
            *vec = static_cast<int>(v - vb);
            *elem = static_cast<int>(id - head - v * EPV);
            return v >= vb && v < ve;
        });

    if (split == 0) {
        const int64_t n_edge = head + (vocab - tail_begin);
        if (tid < n_edge) {
            const int64_t v = (tid < head) ? tid : tail_begin + (tid - head);
            float x = to_f32<DT>(rp[v]);
            if (kScaled) x *= p.scale;
            float d = g.lse >= 0.0f ? grad_elem<DT, true>(x, g) : grad_elem<DT, false>(x, g);
            if (v == tgt) d += g.g_logp;
            if constexpr (kTop) d += top_at(top.h, v);
            if (kScaled) d *= p.scale;
            dp[v] = from_f32<DT>(d);
        }
    }

    // Vector index holding the target's one-hot term (or -1).
    const int64_t t_rel = tgt - head;
    const int64_t t_vec = (tgt >= head && tgt < tail_begin) ? t_rel / EPV : -1;
    const int t_lane_elem = (t_vec >= 0) ? static_cast<int>(t_rel - t_vec * EPV) : 0;

    // Longer rows whose input and output sit at different offsets within 16
    // bytes (a sliced window of an odd vocabulary: seven rows of eight) keep whole
    // aligned 16-byte stores and read the same elements with 16-byte loads at
    // the elements' own alignment, which global memory serves.  Like the
    // aligned rows they are then bound by memory: bf16 [8, 512 of 513, 50257]
    // at T = 0.9 146 us (5.6 TB/s), where one element per lane and load took
    // 299 us (2.8 TB/s).
    if (((in_addr ^ out_addr) & 15u) != 0)
        bwd_piece<DT, WAVES, U, kNtStore, kScaled, false>(p, vin, vout, vb, ve, t_vec,
                                                          t_lane_elem, g, top);
    else
        bwd_piece<DT, WAVES, U, kNtStore, kScaled, true>(p, vin, vout, vb, ve, t_vec,
                                                         t_lane_elem, g, top);
    if (far_row(g.lse)) redo_far<DT, WAVES, kScaled, kTop>(top);
}

template <int DT, int WAVES, int U, bool kNtStore, bool kTop>
static hipError_t launch_bwd_t(const BwdParams& p, hipStream_t stream) {
    if (p.scale != 1.0f)
        return launch_kernel(klp_bwd_kernel<DT, WAVES, U, kNtStore, true, kTop>,
                             dim3(static_cast<unsigned>(p.n_rows * p.splits)),
                             dim3(WAVES * 64), stream, p);
    return launch_kernel(klp_bwd_kernel<DT, WAVES, U, kNtStore, false, kTop>,
                         dim3(static_cast<unsigned>(p.n_rows * p.splits)), dim3(WAVES * 64),
                         stream, p);
}

template <int DT>
static hipError_t launch_bwd_dt(const BwdParams& p, const BwdConfig& c, hipStream_t stream) {
    const bool nt = (c.flags & kFlagNtStore) != 0;
    // Alternatives come with the default shapes only.
    if (p.top_ids != nullptr) {
#define KLP_BWD_TOP_CASE(W)                                                    \
    if (c.waves == W && c.unroll == 2 && nt)                                   \
        return launch_bwd_t<DT, W, 2, true, true>(p, stream);
        KLP_BWD_TOP_CASE(4)
        KLP_BWD_TOP_CASE(8)
        KLP_BWD_TOP_CASE(16)
#undef KLP_BWD_TOP_CASE
        return hipErrorInvalidValue;
    }
#define KLP_BWD_CASE(W, U)                                                     \
    if (c.waves == W && c.unroll == U)                                         \
        return nt ? launch_bwd_t<DT, W, U, true, false>(p, stream)         \
                  : launch_bwd_t<DT, W, U, false, false>(p, stream);
    KLP_BWD_CASE(4, 2)
    KLP_BWD_CASE(4, 4)
    KLP_BWD_CASE(8, 2)
    KLP_BWD_CASE(8, 4)
    KLP_BWD_CASE(16, 2)
    KLP_BWD_CASE(16, 4)
#undef KLP_BWD_CASE
    return hipErrorInvalidValue;
}

hipError_t launch_bwd(int dtype, const BwdParams& p, const BwdConfig& c, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_bwd_dt<kBF16>(p, c, stream);
        case kFP16: return launch_bwd_dt<kFP16>(p, c, stream);
        case kFP32: return launch_bwd_dt<kFP32>(p, c, stream);
        default: return hipErrorInvalidValue;
    }
}

bool bwd_config_supported(const BwdConfig& c) {
    const bool w = (c.waves == 4 || c.waves == 8 || c.waves == 16);
    const bool u = (c.unroll == 2 || c.unroll == 4);
    return w && u && (c.flags & ~kFlagNtStore) == 0;
}

}  // namespace klp
