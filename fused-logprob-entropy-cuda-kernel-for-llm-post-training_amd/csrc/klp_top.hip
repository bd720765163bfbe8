// klp_top.hip — log-probabilities of given tokens with the entropy, the given
// token's rank and the k most likely tokens, in one pass over the logits, for
// gfx950.
//
// Per row, with y = x / T and the order by falling x (equal ones by index):
//   lse = ln sum e^y,   logp = y_target - lse,   entropy = lse - sum p y,
//   rank = tokens before the target in the order,
//   top j = the order's token j, with y - lse.
//
// The sums run online in base 2, as the forward's do: with m the largest x so
// far, S = log2(e) / T and o = RN(m S), z = sum 2^(x S - o) and t = sum (x S -
// o) 2^(x S - o).  x S - o is one fma, so that a temperature costs no rounding
// of its own and the differences that log-probabilities are, (x - m) / T - ln
// z, keep their precision next to 0.
//
// The k largest come from maxima, without a sort and without a second pass:
// while a thread streams, it leaves the maximum of every few vectors (a
// record) in LDS.  The k-th largest of the threads' own maxima is a lower
// bound tau of the row's k-th largest element, and only records that reach it
// are read again, some k of them, 32 to 64 bytes each.  Their elements from tau
// up, about k (1 + k / (2 threads)) of them where large ones lie anywhere, are
// ranked against each other as whole numbers: the value's bits above, the
// index below.  Rows whose list overflows (many equal logits, or large ones
// that all fall to few threads) find the k-th value by a radix search and
// break its ties in index order, with the same result.
//
// Few rows are cut into pieces of a workgroup each; a piece leaves its state
// and its own k largest in the workspace, and the last to arrive merges them.
#include "klp_launch.h"

namespace klp {

namespace {

constexpr int kRecords = 16;           // a thread's records at most
constexpr int kWork = 1024;            // records read again at most
constexpr int kTopList = 1024;         // elements ranked at most (unsplit)
constexpr unsigned long long kNoKey = 0;

// A rising whole number of a float; -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kOrderedNegInf = 0x007FFFFFu;

// The order's key of element `index` with value x: larger comes first.
__device__ __forceinline__ unsigned long long order_key(float x, uint32_t index) {
    return static_cast<unsigned long long>(ordered(x)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    return from_ordered(static_cast<uint32_t>(k >> 32));
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) {
    return 0xFFFFFFFFu - static_cast<uint32_t>(k);
}

// absorb() of klp_device.h with a base-2 factor: K values into the state, and
// their maximum.  -inf values add nothing (their exponent is clamped).
template <int K>
__device__ __forceinline__ float absorb_scaled(Stat& s, const float* x, float factor) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < K; ++j) top = fmax_nan(top, x[j]);
    const float c = fmax_nan(s.m, top);
    const float o_raw = c * factor;
    const float o = (c == -INFINITY) ? 0.0f : o_raw;
    const float d = (s.m == -INFINITY) ? kNegBig : fmax_nan(s.m * factor - o_raw, kNegBig);
    const float sc = exp2_hw(d);
    float z0 = sc * s.z, z1 = 0.0f;
    float t0 = sc * fmaf(d, s.z, s.t), t1 = 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float u = fmax_nan(fmaf(x[j], factor, -o), kNegBig);
        const float e = exp2_hw(u);
        if (j & 1) {
            z1 += e;
            t1 = fmaf(u, e, t1);
        } else {
            z0 += e;
            t0 = fmaf(u, e, t0);
        }
    }
    s.m = c;
    s.z = z0 + z1;
    s.t = t0 + t1;
    return top;
}

__device__ __forceinline__ void rescale_scaled(const Stat& s, float m, float factor, float& z,
                                               float& t) {
    const bool live = s.m != -INFINITY;
    const float d = live ? s.m * factor - m * factor : 0.0f;
    const float sc = live ? exp2_hw(d) : 0.0f;
    z = live ? sc * s.z : 0.0f;
    t = live ? sc * fmaf(d, s.z, s.t) : 0.0f;
}
__device__ __forceinline__ Stat wave_reduce_scaled(const Stat& s, float factor) {
    const float m = xrow_max(row_max16(s.m));
    float z, t;
    rescale_scaled(s, m, factor, z, t);
    return Stat{m, xrow_sum(row_sum16(z)), xrow_sum(row_sum16(t))};
}

// What a row's log-probabilities are made of: y - lse = (x - m) / T - l.
struct RowEnd {
    float m, l, ent;
    bool bad;  // a NaN or +inf logit: no distribution
};
__device__ __forceinline__ RowEnd row_end(const Stat& s, float factor) {
    const float lnz = logf(s.z);
    float rho = 0.0f;
    if (s.m != -INFINITY) rho = -fmaf(s.m, factor, -s.m * factor);
    return RowEnd{s.m, fmaf(rho, kLn2, lnz), fmaf(-kLn2, s.t / s.z, lnz),
                  !(s.m < INFINITY)};
}

__device__ __forceinline__ unsigned long long shfl_xor_u64(unsigned long long v, int off) {
    return static_cast<unsigned long long>(__shfl_xor(static_cast<long long>(v), off, 64));
}

// A workgroup's part of a row: elements [begin, end), its 16-byte vectors
// [vb, ve) of those from element `head` on.
struct Piece {
    int64_t head, begin, end;
    int64_t vb, ve;
};

template <int WAVES, bool kSplit>
struct TopShared {
    static constexpr int NT = WAVES * 64;
    // Pieces' lists together, of which the merge keeps at most all.
    static constexpr int kList = kSplit ? kTopMergeKeys : kTopList;
    float record[kRecords][NT];  // histograms of the radix search later
    union {
        unsigned long long list[kList];
        float thread_max[NT];
    };
    uint32_t work[kWork];
    Stat wave_stat[WAVES];
    uint32_t wave_count[WAVES];
    uint32_t n_list, n_work, arrived;
    float tau;
    Stat total;
    uint32_t count;
};

template <int DT>
__device__ __forceinline__ float element(const typename Traits<DT>::elem* rp, int64_t i) {
    return to_f32<DT>(rp[i]);
}

// The piece's k first elements in the order into sh.list (sh.n_list of them,
// not in order): digits of the k-th value from the top by histograms, then its
// ties in index order.  All threads call it; elements are read as they come.
template <int DT, int WAVES, bool kSplit>
__device__ void select_exact(TopShared<WAVES, kSplit>& sh, const typename Traits<DT>::elem* rp,
                             const Piece& pc, int k) {
    constexpr int NT = WAVES * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t* hist = reinterpret_cast<uint32_t*>(&sh.record[0][0]);  // 256 bins
    uint32_t* found = hist + 256;                                    // digit, count above, total
    uint32_t prefix = 0, left = static_cast<uint32_t>(k);
    bool all = false;  // fewer than k elements have a probability
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += NT) hist[b] = 0;
        __syncthreads();
        for (int64_t i = pc.begin + tid; i < pc.end; i += NT) {
            const uint32_t key = ordered(element<DT>(rp, i));
            if (key <= kOrderedNegInf) continue;
            if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8))
                atomicAdd(&hist[key >> shift & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // Lane l holds bins 255 - 4 l down to 252 - 4 l: running sums from
            // the top.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = hist[255 - 4 * lane - j];
                sum += c[j];
            }
            uint32_t run = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_up(run, off, 64);
                if (lane >= off) run += o;
            }
            const uint32_t total = __shfl(run, 63, 64);
            uint32_t above = run - sum;
            if (lane == 63) found[2] = total;
            if (above < left && run >= left) {
                int digit = 255 - 4 * lane;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above + c[j] >= left) break;
                    above += c[j];
                    --digit;
                }
                found[0] = static_cast<uint32_t>(digit);
                found[1] = above;
            }
        }
        __syncthreads();
        if (found[2] < left) {  // the first digit only
            all = true;
            break;
        }
        prefix |= found[0] << shift;
        left -= found[1];
        __syncthreads();
    }
    __syncthreads();
    // Elements above the k-th value; with `all`, every one there is.
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    const uint32_t bound = all ? kOrderedNegInf : prefix;
    for (int64_t i = pc.begin + tid; i < pc.end; i += NT) {
        const float x = element<DT>(rp, i);
        if (ordered(x) > bound)
            sh.list[atomicAdd(&sh.n_list, 1u)] = order_key(x, static_cast<uint32_t>(i));
    }
    __syncthreads();
    if (all) return;
    // The first `left` of the elements equal to it.
    for (int64_t base = pc.begin; base < pc.end && left > 0; base += NT) {
        const int64_t i = base + tid;
        float x = 0.0f;
        bool tie = false;
        if (i < pc.end) {
            x = element<DT>(rp, i);
            tie = ordered(x) == prefix;
        }
        const unsigned long long ties = __ballot(tie);
        if (lane == 0) found[3 + wave] = static_cast<uint32_t>(__popcll(ties));
        __syncthreads();
        uint32_t before = static_cast<uint32_t>(
            __popcll(ties & ((1ull << lane) - 1ull)));
        uint32_t here = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += found[3 + w];
            here += found[3 + w];
        }
        if (tie && before < left)
            sh.list[atomicAdd(&sh.n_list, 1u)] = order_key(x, static_cast<uint32_t>(i));
        left -= here < left ? here : left;
        __syncthreads();
    }
}

// Places in the order of the list's n keys: f(place, key) for each of the
// first k.
template <int NT, typename F>
__device__ __forceinline__ void ranked(const unsigned long long* list, int n, int k, F f) {
    for (int i = threadIdx.x; i < n; i += NT) {
        const unsigned long long mine = list[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += list[j] > mine ? 1 : 0;
        if (place < k) f(place, mine);
    }
}

template <int DT, int WAVES, int U, bool kSplit>
__global__ __launch_bounds__(WAVES * 64) void klp_top_kernel(TopParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int NT = WAVES * 64;
    constexpr int EPV = Traits<DT>::kPerVec;
    constexpr int ESZ = 16 / EPV;
    __shared__ TopShared<WAVES, kSplit> sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = kSplit ? static_cast<int64_t>(blockIdx.x) / p.splits : blockIdx.x;
    const int split = kSplit ? static_cast<int>(blockIdx.x - row * p.splits) : 0;
    const int splits = kSplit ? p.splits : 1;
    const int64_t vocab = p.vocab;
    const int k = p.k;
    const elem* rp = static_cast<const elem*>(p.logits) + row_offset(p.rm, row);

    Piece pc;
    pc.head = static_cast<int64_t>(((16u - (reinterpret_cast<uintptr_t>(rp) & 15u)) & 15u) / ESZ);
    if (pc.head > vocab) pc.head = vocab;
    const int64_t nvec = (vocab - pc.head) / EPV;
    const int64_t tail_begin = pc.head + nvec * EPV;
    const int64_t per = (nvec + splits - 1) / splits;
    pc.vb = split * per < nvec ? split * per : nvec;
    pc.ve = pc.vb + per < nvec ? pc.vb + per : nvec;
    pc.begin = split == 0 ? 0 : pc.head + pc.vb * EPV;
    pc.end = split == splits - 1 ? vocab : pc.head + pc.ve * EPV;
    const u32x4* vp = reinterpret_cast<const u32x4*>(rp + pc.head) + pc.vb;
    const int nv = static_cast<int>(pc.ve - pc.vb);

    constexpr int kStep = NT * U;  // vectors of a chunk
    const int n_full = nv / kStep;
    const int n_chunks = (nv + kStep - 1) / kStep;
    int shift = 0;  // chunks of a record, as a power of two
    while (((n_chunks - 1) >> shift) >= kRecords) ++shift;

    // Whole chunks, kFwdRing - 1 in flight; loads past them are out of the
    // buffer's range and are not used.
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<u32x4*>(vp), 0, n_full * kStep * 16, 0x00020000);
    u32x4 set[kFwdRing][U];
    auto load = [&](u32x4 (&dst)[U], int c) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            dst[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, ((c * U + u) * NT + tid) * 16, 0,
                                                           kBufNonTemporal);
    };
#pragma unroll
    for (int r = 0; r < kFwdRing - 1; ++r) load(set[r], r);
    __builtin_amdgcn_sched_barrier(0);

    // The target, and what counts as before it in the order: from its value up
    // in vectors before its own, above its value elsewhere.
    const int64_t target = p.targets[row];
    const bool has_target = target >= 0 && target < vocab;
    const float x_t = has_target ? element<DT>(rp, target) : 0.0f;
    const float above_t = has_target ? from_ordered(ordered(x_t) + 1u) : INFINITY;
    // (vectors of the piece)
    int t_vec = 0;
    if (has_target && target >= pc.head) {
        const int64_t v = (target - pc.head) / EPV - pc.vb;
        t_vec = static_cast<int>(v < 0 ? 0 : v < nv ? v : nv);
    }
    uint32_t count = 0;  // of the wave

    Stat s = stat_empty();
    float best = -INFINITY, current = -INFINITY;
    auto take = [&](const u32x4 (&v)[U], int c) {
        float x[U * EPV];
#pragma unroll
        for (int u = 0; u < U; ++u) unpack<DT>(v[u], x + u * EPV);
        const float top = absorb_scaled<U * EPV>(s, x, p.factor);
        current = (c & ((1 << shift) - 1)) == 0 ? top : fmax_nan(current, top);
        best = fmax_nan(best, top);
        sh.record[c >> shift][tid] = current;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float from = (c * U + u) * NT + tid < t_vec ? x_t : above_t;
#pragma unroll
            for (int j = 0; j < EPV; ++j)
                count += static_cast<uint32_t>(__popcll(__ballot(x[u * EPV + j] >= from)));
        }
    };
    int c = 0;
    for (; c + kFwdRing <= n_full; c += kFwdRing) {
#pragma unroll
        for (int r = 0; r < kFwdRing; ++r) {
            load(set[(r + kFwdRing - 1) % kFwdRing], c + r + kFwdRing - 1);
            __builtin_amdgcn_sched_barrier(0);
            take(set[r], c + r);
        }
    }
#pragma unroll
    for (int r = 0; r < kFwdRing - 1; ++r)
        if (c + r < n_full) take(set[r], c + r);
    if (n_full < n_chunks) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (n_full * U + u) * NT + tid;
            const uint32_t w = Traits<DT>::kNegInfWord;
            v[u] = u32x4{w, w, w, w};
            if (i < nv) v[u] = load16<true>(vp + i);
        }
        take(v, n_full);
    }
    // The elements before the first vector and behind the last.
    const int n_head = split == 0 ? static_cast<int>(pc.head) : 0;
    const int n_edge = n_head + (split == splits - 1 ? static_cast<int>(vocab - tail_begin) : 0);
    float x_edge = -INFINITY;
    uint32_t i_edge = 0;
    bool edge_before = false, tie_before = false;
    if (tid < n_edge) {
        i_edge = static_cast<uint32_t>(tid < n_head ? tid : tail_begin + (tid - n_head));
        x_edge = element<DT>(rp, i_edge);
        absorb_scaled<1>(s, &x_edge, p.factor);
        best = fmax_nan(best, x_edge);
        edge_before = x_edge >= (i_edge < target ? x_t : above_t);
    }
    // Ties before the target in its own vector.
    if (has_target && target >= pc.head && target < tail_begin && tid < EPV) {
        const int64_t v = (target - pc.head) / EPV;
        const int64_t i = pc.head + v * EPV + tid;
        if (v >= pc.vb && v < pc.ve && i < target) tie_before = element<DT>(rp, i) == x_t;
    }
    count += static_cast<uint32_t>(__popcll(__ballot(edge_before)) +
                                   __popcll(__ballot(tie_before)));

    s = wave_reduce_scaled(s, p.factor);
    sh.thread_max[tid] = best;
    if (lane == 0) {
        sh.wave_stat[wave] = s;
        sh.wave_count[wave] = count;
    }
    if (tid == 0) {
        sh.n_list = 0;
        sh.n_work = 0;
    }
    __syncthreads();
    if (wave == 0) {
        const Stat total =
            wave_reduce_scaled(lane < WAVES ? sh.wave_stat[lane] : stat_empty(), p.factor);
        uint32_t mine[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mine[w] = ordered(sh.thread_max[w * 64 + lane]);
        // The largest number that k of the maxima reach, bit by bit; one that
        // exactly k reach will do.
        uint32_t bound = 0;
        for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
            const uint32_t b = bound | bit;
            int n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(mine[w] >= b));
            if (n >= k) {
                bound = b;
                if (n == k) break;
            }
        }
        if (lane == 0) {
            sh.total = total;
            sh.tau = bound <= kOrderedNegInf ? -INFINITY : from_ordered(bound);
            uint32_t n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += sh.wave_count[w];
            sh.count = n;
        }
    }
    __syncthreads();
    const float tau = sh.tau;
    const bool bad_piece = !(sh.total.m < INFINITY);
    if (!bad_piece) {
        auto keep = [&](float x, uint32_t i) {
            if (x >= tau && x > -INFINITY) {
                const uint32_t at = atomicAdd(&sh.n_list, 1u);
                if (at < static_cast<uint32_t>(TopShared<WAVES, kSplit>::kList))
                    sh.list[at] = order_key(x, i);
            }
        };
        if (tid < n_edge) keep(x_edge, i_edge);
        if (best >= tau && best > -INFINITY) {
            const int records = n_chunks > 0 ? ((n_chunks - 1) >> shift) + 1 : 0;
            for (int r = 0; r < records; ++r) {
                const float x = sh.record[r][tid];
                if (x >= tau && x > -INFINITY) {
                    const uint32_t at = atomicAdd(&sh.n_work, 1u);
                    if (at < kWork) sh.work[at] = static_cast<uint32_t>(r * NT + tid);
                }
            }
        }
        __syncthreads();
        const uint32_t n_work = sh.n_work;
        if (n_work <= kWork) {
            const uint32_t of_record = static_cast<uint32_t>(U) << shift;
            for (uint32_t w = tid; w < n_work * of_record; w += NT) {
                const uint32_t item = sh.work[w / of_record];
                const int r = static_cast<int>(item / NT), t = static_cast<int>(item % NT);
                const int i = ((r << shift) * U + static_cast<int>(w % of_record)) * NT + t;
                if (i < nv) {
                    float x[EPV];
                    unpack<DT>(vp[i], x);
                    const uint32_t at =
                        static_cast<uint32_t>(pc.head + (pc.vb + i) * EPV);
#pragma unroll
                    for (int j = 0; j < EPV; ++j) keep(x[j], at + j);
                }
            }
        }
        __syncthreads();
        if (n_work > kWork ||
            sh.n_list > static_cast<uint32_t>(TopShared<WAVES, kSplit>::kList)) {
            __syncthreads();
            select_exact<DT, WAVES, kSplit>(sh, rp, pc, k);
        }
    }
    int n = bad_piece ? 0 : static_cast<int>(sh.n_list);
    Stat total = sh.total;
    uint32_t before = sh.count;

    if constexpr (kSplit) {
        // This piece's state and keys in order, then its arrival: agent-scope
        // stores, which write through to the device's coherence point, and a
        // wait for them before the count.
        unsigned long long* keys = p.keys + row * splits * k;
        float* states = p.states + row * splits * 4;
        ranked<NT>(sh.list, n, k, [&](int place, unsigned long long key) {
            __hip_atomic_store(keys + split * k + place, key, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        });
        for (int j = n + tid; j < k; j += NT)
            __hip_atomic_store(keys + split * k + j, kNoKey, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        if (tid == 0) {
            float* slot = states + split * 4;
            __hip_atomic_store(slot + 0, total.m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(slot + 1, total.z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(slot + 2, total.t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(slot + 3, __uint_as_float(before), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        if (tid == 0)
            sh.arrived = __hip_atomic_fetch_add(p.counters + row, 1u, __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (sh.arrived != static_cast<uint32_t>(splits - 1)) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        if (tid == 0) {
            __hip_atomic_store(p.counters + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.n_list = 0;
        }
        // Lane l merges pieces l (at most 64).  Of the pieces' keys, those from
        // the least of their ceil(k / splits)-th up hold the row's k first, and
        // so do those from the largest k-th up.
        if (wave == 0) {
            Stat a = stat_empty();
            uint32_t cnt = 0;
            unsigned long long least = ~0ull, most = 0;
            if (lane < splits) {
                const float4 q = reinterpret_cast<const float4*>(states)[lane];
                a = Stat{q.x, q.y, q.z};
                cnt = __float_as_uint(q.w);
                least = keys[lane * k + (k + splits - 1) / splits - 1];
                most = keys[lane * k + k - 1];
            }
            a = wave_reduce_scaled(a, p.factor);
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                cnt += __shfl_xor(cnt, off, 64);
                const unsigned long long l = shfl_xor_u64(least, off), h = shfl_xor_u64(most, off);
                least = l < least ? l : least;
                most = h > most ? h : most;
            }
            if (lane == 0) {
                sh.total = a;
                sh.count = cnt;
                *reinterpret_cast<unsigned long long*>(sh.work) = least > most ? least : most;
            }
        }
        __syncthreads();
        total = sh.total;
        before = sh.count;
        const unsigned long long from = *reinterpret_cast<unsigned long long*>(sh.work);
        if (total.m < INFINITY) {
            for (int j = tid; j < splits * k; j += NT) {
                const unsigned long long key = keys[j];
                if (key != kNoKey && key >= from) sh.list[atomicAdd(&sh.n_list, 1u)] = key;
            }
        }
        __syncthreads();
        n = total.m < INFINITY ? static_cast<int>(sh.n_list) : 0;
    }

    const RowEnd e = row_end(total, p.factor);
    if (tid == 0) {
        p.lse[row] = fmaf(e.m, p.inv_t, e.l);
        p.entropy[row] = e.ent;
        // A target outside the row counts as a logit of 0.
        p.logprob[row] = fmaf(x_t - e.m, p.inv_t, -e.l);
        p.rank[row] = has_target && !e.bad ? static_cast<int64_t>(before) : -1;
    }
    int64_t* ids = p.top_ids + row * k;
    float* logps = p.top_logprob + row * k;
    ranked<NT>(sh.list, n, k, [&](int place, unsigned long long key) {
        ids[place] = key_index(key);
        logps[place] = fmaf(key_value(key) - e.m, p.inv_t, -e.l);
    });
    for (int j = n + tid; j < k; j += NT) {
        ids[j] = -1;
        logps[j] = e.bad ? NAN : -INFINITY;
    }
}

template <int DT, int WAVES, int U>
hipError_t launch_top_t(const TopParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.n_rows * p.splits)), block(WAVES * 64);
    return p.splits > 1 ? launch_kernel(klp_top_kernel<DT, WAVES, U, true>, grid, block, stream, p)
                        : launch_kernel(klp_top_kernel<DT, WAVES, U, false>, grid, block, stream,
                                        p);
}

template <int DT>
hipError_t launch_top_dt(const TopParams& p, hipStream_t stream) {
    return p.waves == 8 ? launch_top_t<DT, 8, 2>(p, stream) : launch_top_t<DT, 4, 2>(p, stream);
}

}  // namespace

hipError_t launch_top(int dtype, const TopParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_top_dt<kBF16>(p, stream);
        case kFP16: return launch_top_dt<kFP16>(p, stream);
        case kFP32: return launch_top_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
