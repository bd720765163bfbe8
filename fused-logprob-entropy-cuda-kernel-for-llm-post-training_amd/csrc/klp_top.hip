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
// z, keep their precision next to 0.  o's rounding stays in z as an exponent and
// is taken out at the end; where it could be more than 64, from |o| = 2^31 on,
// sums are relative to m S itself, with (x - m) S for x S - o.
//
// The k largest come from maxima, without a sort and without a second pass:
// while a thread streams, it leaves the maximum of every few vectors (a
// record) in LDS: 32 bytes of a thread's logits, or as many times that, in powers
// of two, as leave it 16 records of its part (32 bytes up to 256 KB of a row, 64
// for 152064 bf16, 128 for 152064 float32, 32 KB for 2^26).  The k-th largest of
// the threads' own maxima is a lower bound tau of the row's k-th largest element,
// and only records that reach it are read again, some k of them.  Their elements
// from tau
// up, about k (1 + k / (2 threads)) of them where large ones lie anywhere, are
// ranked against each other as whole numbers: the value's bits above, the
// index below.  Rows whose list overflows (many equal logits, or large ones
// that all fall to few threads) find the k-th value by a radix search and
// break its ties in index order, with the same result.
//
// Few rows are cut into pieces of a workgroup each; a piece leaves its state
// and its own k largest in the workspace, and the last to arrive merges them.
//
// One pass over the bytes bounds many long rows: 4096 rows of 128256 fp16 take
// 180 us, 5.8 TB/s (154 for klp_fwd_kernel's three numbers), 1024 of 152064 bf16
// 56 (k = 20; 61 with k = 64; 47).  Few long rows are bound by their steps: 64 of
// 152064 take 14 us, of which the bytes are 4.
//
// Masks cost (152064 bf16, k = 20, us for 64 / 1024 rows; the last 128, half, all
// but 100 logits of a row masked):
//   none           14 / 56
//   -inf           14 / 56, 14 / 114, 19 / 111   (a thread's part read again)
//   -1e9           14 / 57, 183 / 56, 149 / 56   (a piece of equal logits: its
//   lowest value   14 / 55, 187 / 114, 154 / 114  list overflows)
//
// Short rows (klp_top_short_kernel) stay in the registers of as many waves as
// they need, and the bound comes from maxima of a few elements or from the
// elements themselves.
#include "klp_launch.h"

namespace klp {

namespace {

constexpr int kRecords = 16;           // a thread's records at most
// Elements ranked at most (unsplit; fewer where more workgroups then fit a CU).
constexpr int kTopList = 1024, kTopListSmall = 512;
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

// A record: the upper half of a float that is its maximum (bf16 logits) or the
// next one up.
template <int DT>
__device__ __forceinline__ uint16_t record_of(float x) {
    uint32_t b = __float_as_uint(x);
    if constexpr (DT != kBF16) b += ~(static_cast<int32_t>(b) >> 31) & 0xFFFF;
    return static_cast<uint16_t>(b >> 16);
}
__device__ __forceinline__ float record_value(uint16_t r) {
    return __uint_as_float(static_cast<uint32_t>(r) << 16);
}

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

// A thread's sums: klp_device.h's Stat with its offset o = RN(m S).
struct Sums {
    float m, o, z, t;
};
__device__ __forceinline__ Sums sums_empty() { return Sums{-INFINITY, -INFINITY, 0.0f, 0.0f}; }

// K values with maximum `top` into the sums, S = `factor`.  A -inf logit leaves a
// t that is not finite, and a maximum so large that o's rounding reaches float32's
// exponents any z: absorb_any then does the thread's part once more (sums_lost).
template <int K>
__device__ __forceinline__ void absorb_fast(Sums& s, const float* x, float top, float factor) {
    s.m = fmax_nan(s.m, top);
    const float o = s.m * factor;
    const float d = fmaxf(s.o - o, kNegBig);  // NaN where both are infinite: kNegBig
    const float sc = exp2_hw(d);
    float z0 = sc * s.z, z1 = 0.0f;
    float t0 = sc * fmaf(d, s.z, s.t), t1 = 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float u = fmaf(x[j], factor, -o);
        const float e = exp2_hw(u);
        if (j & 1) {
            z1 += e;
            t1 = fmaf(u, e, t1);
        } else {
            z0 += e;
            t0 = fmaf(u, e, t0);
        }
    }
    s.o = o;
    s.z = z0 + z1;
    s.t = t0 + t1;
}
// Offsets whose rounding could reach float32's exponents, and those that
// overflow: the sums are relative to m S itself.
__device__ __forceinline__ bool huge_offset(float o) { return !(fabsf(o) < 0x1p31f); }
// (A maximum that was huge on the way left nothing beside one that is not, or a z
// or t that is not finite.)
__device__ __forceinline__ bool sums_lost(const Sums& s) {
    return !(s.z < INFINITY) || !(s.t > -INFINITY) ||
           (huge_offset(s.o) && s.m != -INFINITY);
}
// What sums relative to a state's maximum a are moved by to another's, b >= a.
// Unequal floats whose product with S lies there are at least 64 apart in it: next
// to the larger one's weight the other's is nothing.  (2^-2^20 is 0, and -2^20
// times any z finite.)
__device__ __forceinline__ float offset_difference(float a, float b, float factor) {
    const float oa = a * factor, ob = b * factor;
    if (!huge_offset(oa) && !huge_offset(ob)) return oa - ob;
    return a == b ? 0.0f : -0x1p20f;
}
// The same for any values; -inf adds nothing.
template <int K>
__device__ __forceinline__ void absorb_any(Sums& s, const float* x, float top, float factor) {
    const float c = fmax_nan(s.m, top);
    if (c == -INFINITY) return;
    const float o = c * factor;
    const float d = offset_difference(s.m, c, factor);
    const float sc = exp2_hw(d);
    float z = sc * s.z, t = sc * fmaf(d, s.z, s.t);
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float u = fmax_nan(huge_offset(o) ? (x[j] - c) * factor : fmaf(x[j], factor, -o),
                                 kNegBig);
        const float e = exp2_hw(u);
        z += e;
        t = fmaf(u, e, t);
    }
    s = Sums{c, o, z, t};
}

__device__ __forceinline__ Stat wave_reduce_scaled(const Stat& s, float factor) {
    const float m = xrow_max(row_max16(s.m));
    const bool live = s.m != -INFINITY;
    const float d = live ? offset_difference(s.m, m, factor) : 0.0f;
    const float sc = live ? exp2_hw(d) : 0.0f;
    const float z = live ? sc * s.z : 0.0f;
    const float t = live ? sc * fmaf(d, s.z, s.t) : 0.0f;
    return Stat{m, xrow_sum(row_sum16(z)), xrow_sum(row_sum16(t))};
}

// What a row's log-probabilities are made of: y - lse = (x - m) / T - l.
struct RowEnd {
    float m, l, ent;
    bool bad;  // a NaN or +inf logit: no distribution
};
__device__ __forceinline__ RowEnd row_end(const Stat& s, float factor) {
    const float lnz = logf(s.z);
    const float o = s.m * factor;
    const float rho = huge_offset(o) ? 0.0f : -fmaf(s.m, factor, -o);
    return RowEnd{s.m, fmaf(rho, kLn2, lnz), fmaf(-kLn2, s.t / s.z, lnz),
                  !(s.m < INFINITY)};
}

__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);   // quad_perm [1, 0, 3, 2]
    v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);   // quad_perm [2, 3, 0, 1]
    v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);  // row_half_mirror
    v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);  // row_mirror
    const auto q = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = q[0] + q[1];
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] + r[1];
}
__device__ __forceinline__ unsigned long long two_words(uint32_t low, uint32_t high) {
    return static_cast<unsigned long long>(high) << 32 | low;
}

// A workgroup's part of a row: elements [begin, end), its 16-byte vectors
// [vb, ve) of those from element `head` on.
struct Piece {
    int head, begin, end;
    int vb, ve;
};

template <int WAVES, bool kSplit>
struct TopShared {
    static constexpr int NT = WAVES * 64;
    // Pieces' lists together, of which the merge keeps at most all.
    static constexpr int kList = kSplit ? kTopMergeKeys : WAVES <= 2 ? kTopListSmall : kTopList;
    uint16_t record[kRecords][NT];  // histograms of the radix search later
    union {
        unsigned long long list[kList];
        float thread_max[NT];
    };
    unsigned long long sorted[kSplit ? kTopMax : 1];  // a piece's
    uint16_t found[WAVES][64];  // a wave's records to read again
    Stat wave_stat[WAVES];
    uint32_t wave_count[WAVES];
    uint32_t n_list, before, arrived;
    float tau;
    Stat total;
    __device__ __forceinline__ int listed() const {
        return static_cast<int>(n_list < static_cast<uint32_t>(kList) ? n_list : kList);
    }
};

template <int DT>
__device__ __forceinline__ float element(const typename Traits<DT>::elem* rp, int i) {
    return to_f32<DT>(rp[i]);
}

// The piece's k first elements in the order into sh.list (sh.n_list of them,
// not in order): digits of the k-th value from the top by histograms, then its
// ties in index order.  All threads call it; elements are read as they come,
// and again in each step: logits that another stream writes meanwhile may leave
// any list, but none beyond its end.
template <int DT, int WAVES, bool kSplit>
__device__ __forceinline__ void select_exact(TopShared<WAVES, kSplit>& sh,
                                             const typename Traits<DT>::elem* rp, const Piece& pc,
                                             int k) {
    constexpr int NT = WAVES * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t* hist = reinterpret_cast<uint32_t*>(&sh.record[0][0]);  // 256 bins
    uint32_t* found = hist + 256;                                    // digit, count above, total
    uint32_t prefix = 0, left = static_cast<uint32_t>(k);
    bool all = false;  // fewer than k elements have a probability
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += NT) hist[b] = 0;
        __syncthreads();
        for (int i = pc.begin + tid; i < pc.end; i += NT) {
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
    auto list = [&](float x, int i) {
        const uint32_t at = atomicAdd(&sh.n_list, 1u);
        if (at < static_cast<uint32_t>(TopShared<WAVES, kSplit>::kList))
            sh.list[at] = order_key(x, static_cast<uint32_t>(i));
    };
    for (int i = pc.begin + tid; i < pc.end; i += NT) {
        const float x = element<DT>(rp, i);
        if (ordered(x) > bound) list(x, i);
    }
    __syncthreads();
    if (all) return;
    // The first `left` of the elements equal to it.
    for (int base = pc.begin; base < pc.end && left > 0; base += NT) {
        const int i = base + tid;
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
        if (tie && before < left) list(x, i);
        left -= here < left ? here : left;
        __syncthreads();
    }
}

// Places in the order of the list's n keys: f(place, key) for each of the
// first k.  Four lanes share a key's comparisons, and a key that is read is
// compared with as many of a lane's own as there are, up to 4: LDS reads bound
// it (4096 rows of 1000 bf16, k = 128: 28 us with one key at a time, 23 so; 64
// rows of 152064: 22.6 and 20.5).
template <int NT, int G, typename F>
__device__ __forceinline__ void rank_keys(const unsigned long long* list, int n, int k, int base,
                                          F f) {
    const int q = threadIdx.x & 3;
    unsigned long long mine[G];
    uint32_t place[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int i = base + g * (NT / 4) + (threadIdx.x >> 2);
        mine[g] = list[i < n ? i : 0];
        place[g] = 0;
    }
#pragma unroll 4
    for (int j = q; j < n; j += 4) {
        const unsigned long long other = list[j];
#pragma unroll
        for (int g = 0; g < G; ++g) place[g] += other > mine[g] ? 1u : 0u;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        uint32_t at = place[g];
        at += __builtin_amdgcn_update_dpp(0, at, 0xB1, 0xF, 0xF, false);
        at += __builtin_amdgcn_update_dpp(0, at, 0x4E, 0xF, 0xF, false);
        if (q == 0 && base + g * (NT / 4) + static_cast<int>(threadIdx.x >> 2) < n &&
            at < static_cast<uint32_t>(k))
            f(static_cast<int>(at), mine[g]);
    }
}
template <int NT, typename F>
__device__ __forceinline__ void ranked(const unsigned long long* list, int n, int k, F f) {
    int base = 0;  // whole waves all the way
    for (; n - base > NT / 2; base += NT) rank_keys<NT, 4>(list, n, k, base, f);
    if (n - base > NT / 4) rank_keys<NT, 2>(list, n, k, base, f);
    else if (n > base) rank_keys<NT, 1>(list, n, k, base, f);
}

// A row's outputs, from its sums and the list that holds its first k.
template <int NT>
__device__ __forceinline__ void put_row(const TopParams& p, int64_t row,
                                        const unsigned long long* list, int n, const Stat& total,
                                        bool has_target, float x_t, uint32_t before) {
    const int tid = threadIdx.x, k = p.k;
    const RowEnd e = row_end(total, p.factor);
    if (tid == 0) {
        // (A far row's m / T as the backward rounds the logits': far_row.)
        const float y = e.m * p.inv_t;
        p.lse[row] = far_row(y) ? y + e.l : fmaf(e.m, p.inv_t, e.l);
        p.entropy[row] = e.ent;
        p.logprob[row] = fmaf(x_t - e.m, p.inv_t, -e.l);
        p.rank[row] = has_target && !e.bad ? static_cast<int64_t>(before) : -1;
    }
    int64_t* ids = p.top_ids + row * k;
    float* logps = p.top_logprob + row * k;
    ranked<NT>(list, n, k, [&](int place, unsigned long long key) {
        ids[place] = key_index(key);
        logps[place] = fmaf(key_value(key) - e.m, p.inv_t, -e.l);
    });
    for (int j = n + tid; j < k; j += NT) {
        ids[j] = -1;
        logps[j] = e.bad ? NAN : -INFINITY;
    }
}

// A lower bound (finite) that at least k elements of the part
// reach: one that k or few more of 64 R maxima do, each of the maxima of WAVES /
// R threads, found bit by bit below the maxima's common ones.  One wave calls
// it.  64 R is at least 2 k where there are that many threads, so that few more
// than k elements reach it: where the large ones lie anywhere, 64 R ln(64 R / (64
// R - k)) of them.
template <int WAVES, int R>
__device__ __forceinline__ float bound_of(const float* thread_max, int k) {
    const int lane = threadIdx.x & 63;
    float most = -INFINITY, least = INFINITY;
    uint32_t mine[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float m = thread_max[r * 64 + lane];
#pragma unroll
        for (int w = r + R; w < WAVES; w += R) m = fmax_nan(m, thread_max[w * 64 + lane]);
        mine[r] = ordered(m);
        most = fmax_nan(most, m);
        least = fmax_nan(-m, -least) * -1.0f;
    }
    most = xrow_max(row_max16(most));
    least = -xrow_max(row_max16(-least));
    uint32_t bound = __builtin_amdgcn_readfirstlane(ordered(least));
    const uint32_t differ = bound ^ __builtin_amdgcn_readfirstlane(ordered(most));
    // All 64 R maxima reach the least of them.
    if (64 * R > k && differ != 0) {
        uint32_t bit = 0x80000000u >> __builtin_clz(differ);
        bound &= ~(2 * bit - 1);
        for (; bit != 0; bit >>= 1) {
            const uint32_t b = bound | bit;
            int n = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) n += __popcll(__ballot(mine[r] >= b));
            if (n >= k) {
                bound = b;
                if (n <= k + (k >> 2)) break;
            }
        }
    }
    return from_ordered(bound > kOrderedNegInf ? bound : kOrderedNegInf + 1);
}

// count += x[j] >= from for 4 or 8 values, all skipped where no lane's `top`
// reaches `gate`.  In one block: the compiler's own form holds a mask for each
// value at a time, and a branch of its own costs the loop its registers.  A vector
// read of VCC behind a vector write of it takes two wait states, which the compiler
// does not add in here.  (Four masks in SGPR pairs and their additions behind them
// need none, and take 1 to 4% longer: 1024 rows of 152064 bf16 53.9 us, so 52.6.)
__device__ __forceinline__ void count_from(uint32_t& count, float top, float gate, float from,
                                           const float (&x)[4]) {
    asm("v_cmp_ge_f32 vcc, %1, %2\n\t"
        "s_cbranch_vccz .LBBnone%=\n\t"
        "v_cmp_ge_f32 vcc, %4, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %5, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %6, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %7, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n"
        ".LBBnone%=:"
        : "+v"(count)
        : "v"(top), "v"(gate), "v"(from), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3])
        : "vcc");
}
__device__ __forceinline__ void count_from(uint32_t& count, float top, float gate, float from,
                                           const float (&x)[8]) {
    asm("v_cmp_ge_f32 vcc, %1, %2\n\t"
        "s_cbranch_vccz .LBBnone%=\n\t"
        "v_cmp_ge_f32 vcc, %4, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %5, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %6, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %7, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %8, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %9, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %10, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n\t"
        "v_cmp_ge_f32 vcc, %11, %3\n\ts_nop 1\n\tv_addc_co_u32 %0, vcc, 0, %0, vcc\n"
        ".LBBnone%=:"
        : "+v"(count)
        : "v"(top), "v"(gate), "v"(from), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]),
          "v"(x[5]), "v"(x[6]), "v"(x[7])
        : "vcc");
}
template <int DT, int WAVES, int U, bool kSplit>
__global__ __launch_bounds__(WAVES * 64, kSplit ? 2 : 8) void klp_top_kernel(TopParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int NT = WAVES * 64;
    constexpr int EPV = Traits<DT>::kPerVec;
    constexpr int ESZ = 16 / EPV;
    __shared__ TopShared<WAVES, kSplit> sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = kSplit ? static_cast<int64_t>(blockIdx.x) / p.splits : blockIdx.x;
    const int split = kSplit ? static_cast<int>(blockIdx.x - row * p.splits) : 0;
    const int splits = kSplit ? p.splits : 1;
    const int vocab = static_cast<int>(p.vocab);  // at most 2^26
    const int k = p.k;
    const elem* rp = static_cast<const elem*>(p.logits) + row_offset(p.rm, row);

    Piece pc;
    pc.head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(rp) & 15u)) & 15u) / ESZ);
    if (pc.head > vocab) pc.head = vocab;
    const int nvec = (vocab - pc.head) / EPV;
    const int tail_begin = pc.head + nvec * EPV;
    const int per = (nvec + splits - 1) / splits;
    pc.vb = split * per < nvec ? split * per : nvec;
    pc.ve = pc.vb + per < nvec ? pc.vb + per : nvec;
    pc.begin = split == 0 ? 0 : pc.head + pc.vb * EPV;
    pc.end = split == splits - 1 ? vocab : pc.head + pc.ve * EPV;
    const u32x4* vp = reinterpret_cast<const u32x4*>(rp + pc.head) + pc.vb;
    const int nv = pc.ve - pc.vb;

    constexpr int kStep = NT * U;  // vectors of a chunk
    const int n_full = nv / kStep;
    const int n_chunks = (nv + kStep - 1) / kStep;
    int shift = 0;  // chunks of a record, as a power of two
    while (((n_chunks - 1) >> shift) >= kRecords) ++shift;
    const int records = n_chunks > 0 ? ((n_chunks - 1) >> shift) + 1 : 0;

    // Whole chunks, kFwdRing - 1 in flight; loads past them are out of the
    // buffer's range and are not used.
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<u32x4*>(vp), 0, n_full * kStep * 16, 0x00020000);
    u32x4 set[kFwdRing][U];
    auto load = [&](u32x4 (&dst)[U], int c) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            dst[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, ((c * U + u) * NT + tid) * 16, 0,
                                                           kSplit ? 0 : kBufNonTemporal);
    };
#pragma unroll
    for (int r = 0; r < kFwdRing - 1; ++r) load(set[r], r);
    __builtin_amdgcn_sched_barrier(0);

    const int64_t given = p.targets[row];
    const bool has_target = given >= 0 && given < vocab;
    const int target = has_target ? static_cast<int>(given) : 0;
    // A target outside the row counts as a logit of 0.
    const float x_t = has_target ? element<DT>(rp, target) : 0.0f;
    // What lies before it in the order: from its value up in vectors before its
    // own (t_vec of the piece's), above its value elsewhere.
    const float above_t = has_target ? from_ordered(ordered(x_t) + 1u) : INFINITY;
    int t_vec = 0;
    if (has_target && target >= pc.head) {
        const int v = (target - pc.head) / EPV - pc.vb;
        t_vec = v < 0 ? 0 : v < nv ? v : nv;
    }
    uint32_t count = 0;

    const float gate = has_target ? x_t : INFINITY;

    Sums s = sums_empty();
    float current = -INFINITY;
    const int last = (1 << shift) - 1;
    auto take = [&](const u32x4 (&v)[U], int c, auto whole) {
        float x[U][EPV];
#pragma unroll
        for (int u = 0; u < U; ++u) unpack<DT>(v[u], x[u]);
        float top = x[0][0];
#pragma unroll
        for (int j = 1; j < U * EPV; ++j) top = fmax_nan(top, x[j / EPV][j % EPV]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            count_from(count, top, gate, (c * U + u) * NT + tid < t_vec ? x_t : above_t, x[u]);
        __builtin_amdgcn_sched_barrier(0);
        if (decltype(whole)::value) absorb_fast<U * EPV>(s, &x[0][0], top, p.factor);
        else absorb_any<U * EPV>(s, &x[0][0], top, p.factor);
        current = (c & last) == 0 ? top : fmax_nan(current, top);
        sh.record[c >> shift][tid] = record_of<DT>(current);
    };
    int c = 0;
    for (; c + kFwdRing <= n_full; c += kFwdRing) {
#pragma unroll
        for (int r = 0; r < kFwdRing; ++r) {
            load(set[(r + kFwdRing - 1) % kFwdRing], c + r + kFwdRing - 1);
            __builtin_amdgcn_sched_barrier(0);
            take(set[r], c + r, std::true_type{});
        }
    }
#pragma unroll
    for (int r = 0; r < kFwdRing - 1; ++r)
        if (c + r < n_full) take(set[r], c + r, std::true_type{});
    if (n_full < n_chunks) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (n_full * U + u) * NT + tid;
            const uint32_t w = Traits<DT>::kNegInfWord;
            v[u] = u32x4{w, w, w, w};
            if (i < nv) v[u] = load16<true>(vp + i);
        }
        take(v, n_full, std::false_type{});
    }
    if (sums_lost(s) && s.m < INFINITY) {  // (a NaN or +inf row needs none)
        s = sums_empty();
        for (int i = tid; i < nv; i += NT) {
            float x[EPV];
            unpack<DT>(vp[i], x);
            float top = x[0];
#pragma unroll
            for (int j = 1; j < EPV; ++j) top = fmax_nan(top, x[j]);
            absorb_any<EPV>(s, x, top, p.factor);
        }
    }
    // The elements before the first vector and behind the last.
    const int n_head = split == 0 ? pc.head : 0;
    const int n_edge = n_head + (split == splits - 1 ? vocab - tail_begin : 0);
    float x_edge = -INFINITY;
    int i_edge = 0;
    bool edge_before = false, tie_before = false;
    if (tid < n_edge) {
        i_edge = tid < n_head ? tid : tail_begin + (tid - n_head);
        x_edge = element<DT>(rp, i_edge);
        absorb_any<1>(s, &x_edge, x_edge, p.factor);
        edge_before = x_edge >= (i_edge < target ? x_t : above_t);
    }
    // Ties before the target in its own vector.
    if (has_target && target >= pc.head && target < tail_begin && tid < EPV) {
        const int v = (target - pc.head) / EPV;
        const int i = pc.head + v * EPV + tid;
        if (v >= pc.vb && v < pc.ve && i < target) tie_before = element<DT>(rp, i) == x_t;
    }
    count += (edge_before ? 1u : 0u) + (tie_before ? 1u : 0u);
    count = wave_sum_u32(count);

    const float best = s.m;
    const Stat of_wave = wave_reduce_scaled(Stat{s.m, s.z, s.t}, p.factor);
    sh.thread_max[tid] = best;
    if (lane == 0) {
        sh.wave_stat[wave] = of_wave;
        sh.wave_count[wave] = count;
    }
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    if (wave == 0) {
        const float bound = k <= 32 ? bound_of<WAVES, 1>(sh.thread_max, k)
                               : k <= 64 ? bound_of<WAVES, 2>(sh.thread_max, k)
                               : k <= 128 || WAVES == 4
                                   ? bound_of<WAVES, 4>(sh.thread_max, k)
                                   : bound_of<WAVES, WAVES>(sh.thread_max, k);
        if (lane == 0) sh.tau = bound;
    } else if (wave == 1) {
        const Stat total =
            wave_reduce_scaled(lane < WAVES ? sh.wave_stat[lane] : stat_empty(), p.factor);
        if (lane == 0) {
            sh.total = total;
            uint32_t n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += sh.wave_count[w];
            sh.before = n;
        }
    }
    __syncthreads();
    const float tau = sh.tau;
    const bool bad_piece = !(sh.total.m < INFINITY);
    if (!bad_piece) {
        // n elements from at[0] on that reach tau go to the list.
        auto keep = [&](auto& x, int at) {
            constexpr int kN = sizeof(x) / sizeof(float);
            uint32_t n = 0;
#pragma unroll
            for (int e = 0; e < kN; ++e) n += x[e] >= tau ? 1u : 0u;
            if (n == 0) return;
            uint32_t to = atomicAdd(&sh.n_list, n);
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                if (!(x[e] >= tau)) continue;
                if (to < static_cast<uint32_t>(TopShared<WAVES, kSplit>::kList))
                    sh.list[to] = order_key(x[e], static_cast<uint32_t>(at + e));
                ++to;
            }
        };
        if (tid < n_edge) {
            float x[1] = {x_edge};
            keep(x, i_edge);
        }
        // The records that reach tau: a wave's go round by round, one of each
        // lane that has any, with a lane for each of their vectors.
        uint32_t reach = 0;
        if (best >= tau) {
#pragma unroll
            for (int r = 0; r < kRecords; ++r)
                reach |= r < records && record_value(sh.record[r][tid]) >= tau ? 1u << r : 0u;
        }
        const int of_record = U << shift;
        for (;;) {
            const unsigned long long has = __ballot(reach != 0);
            if (has == 0) break;
            const int n = __popcll(has);
            if (reach != 0) {
                const int r = __builtin_ctz(reach);
                reach &= reach - 1;
                sh.found[wave][__popcll(has & ((1ull << lane) - 1ull))] =
                    static_cast<uint16_t>(r << 6 | lane);
            }
            __builtin_amdgcn_wave_barrier();
            for (int w = lane; w < n * of_record; w += 64) {
                const int item = sh.found[wave][w / of_record];
                const int i = ((item >> 6 << shift) * U + w % of_record) * NT + wave * 64 +
                              (item & 63);
                if (i < nv) {
                    float x[EPV];
                    unpack<DT>(vp[i], x);
                    keep(x, pc.head + (pc.vb + i) * EPV);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        const bool overflow = sh.n_list > static_cast<uint32_t>(TopShared<WAVES, kSplit>::kList);
        if (overflow) {
            __syncthreads();
            select_exact<DT, WAVES, kSplit>(sh, rp, pc, k);
        }
        __syncthreads();
    }
    int n = bad_piece ? 0 : sh.listed();
    Stat total = sh.total;
    uint32_t before = sh.before;

    if constexpr (kSplit) {
        // This piece's state and its k keys in order, side by side, then its
        // arrival: agent-scope stores, which write through to the device's
        // coherence point, and a wait for them before the count.
        const int words = k + 2;
        unsigned long long* mine = p.words + (row * splits + split) * words;
        for (int j = tid; j < k; j += NT) sh.sorted[j] = kNoKey;
        __syncthreads();
        ranked<NT>(sh.list, n, k,
                   [&](int place, unsigned long long key) { sh.sorted[place] = key; });
        __syncthreads();
        for (int j = tid; j < words; j += NT) {
            const unsigned long long w =
                j == 0   ? two_words(__float_as_uint(total.m), __float_as_uint(total.z))
                : j == 1 ? two_words(__float_as_uint(total.t), before)
                         : sh.sorted[j - 2];
            __hip_atomic_store(mine + j, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        unsigned int* counter = p.counters + row * kTopCounterStride;
        if (tid == 0)
            sh.arrived =
                __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (sh.arrived != static_cast<uint32_t>(splits - 1)) return;
        // Agent-scope loads, which no cache answers, see every piece's words: an
        // acquire fence would drop the XCD's L2 under the other rows' workgroups
        // (the loads of 64 rows then took 4 us, of one row 1.4).
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        auto word = [](const unsigned long long* w) {
            return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        if (tid == 0) {
            __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.n_list = 0;
        }
        // Of the pieces' keys, those from the least value of their ceil(k /
        // splits)-th up hold the row's k first, and so do those from the largest
        // k-th up.  Every load starts before the first wait.
        const unsigned long long* all = p.words + row * splits * words;
        constexpr int kKeys = (kTopMergeKeys + 128 + NT - 1) / NT;
        unsigned long long held[kKeys];
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            held[j] = kNoKey;
            if (j * NT + tid < splits * words) held[j] = word(all + j * NT + tid);
        }
        // Lane l merges piece l (at most 64).
        if (wave == 0) {
            Stat a = stat_empty();
            uint32_t cnt = 0;
            float least = INFINITY, most = -INFINITY;
            if (lane < splits) {
                const unsigned long long* of = all + lane * words;
                const unsigned long long first = word(of), second = word(of + 1),
                                         l = word(of + 1 + (k + splits - 1) / splits),
                                         h = word(of + k + 1);
                a = Stat{__uint_as_float(static_cast<uint32_t>(first)),
                         __uint_as_float(static_cast<uint32_t>(first >> 32)),
                         __uint_as_float(static_cast<uint32_t>(second))};
                cnt = static_cast<uint32_t>(second >> 32);
                least = l == kNoKey ? -INFINITY : key_value(l);
                most = h == kNoKey ? -INFINITY : key_value(h);
            }
            a = wave_reduce_scaled(a, p.factor);
            cnt = wave_sum_u32(cnt);
            least = -xrow_max(row_max16(-least));
            most = xrow_max(row_max16(most));
            if (lane == 0) {
                sh.total = a;
                sh.before = cnt;
                sh.tau = fmaxf(least, most);
            }
        }
        __syncthreads();
        total = sh.total;
        before = sh.before;
        if (total.m < INFINITY) {
            const float from = sh.tau;
#pragma unroll
            for (int j = 0; j < kKeys; ++j) {
                const int w = j * NT + tid;
                if (w < splits * words && w % words >= 2 && held[j] != kNoKey &&
                    key_value(held[j]) >= from)
                    sh.list[atomicAdd(&sh.n_list, 1u)] = held[j];
            }
        }
        __syncthreads();
        n = total.m < INFINITY ? static_cast<int>(sh.n_list) : 0;
    }

    put_row<NT>(p, row, sh.list, n, total, has_target, x_t, before);
}

// Rows of at most 1024 WAVES elements, 16 of them and one of the row's edges in
// a lane's registers: one load, nothing read again.  Bound by its own steps, not
// by bytes: the target's two dependent loads, the bound's search bit by bit and
// the ranking.  Next to klp_top_kernel on the same rows (us, bf16; k = 5 / 64 / 128):
//   rows x vocab   here                other
//   4096 x 500     10.3  16.0  23.1    16.1  127   128
//   4096 x 1000    10.7  15.5  22.7    17.1  28.3  470
//   4096 x 2000    12.9  19.2  29.8    19.2  28.1  45.2
//   4096 x 4000    19.2  25.0  37.9    18.9  30.2  49.2
//   4096 x 5000    35 (k = 20)         24
//   16 x 1000      5.6   11.1  18.3    5.8   9.3   87.4
template <int DT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 4) void klp_top_short_kernel(TopParams p) {
    typedef typename Traits<DT>::elem elem;
    constexpr int NT = WAVES * 64;
    constexpr int EPV = Traits<DT>::kPerVec;
    constexpr int ESZ = 16 / EPV;
    constexpr int kHeld = 16, U = kHeld / EPV;
    typedef TopShared<WAVES, false> Shared;
    __shared__ Shared sh;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const int vocab = static_cast<int>(p.vocab);
    const int k = p.k;
    const elem* rp = static_cast<const elem*>(p.logits) + row_offset(p.rm, row);
    int head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(rp) & 15u)) & 15u) / ESZ);
    if (head > vocab) head = vocab;
    const int nv = (vocab - head) / EPV;
    const int tail_begin = head + nv * EPV;
    const u32x4* vp = reinterpret_cast<const u32x4*>(rp + head);
    const int n_edge = head + (vocab - tail_begin);
    const int i_edge = tid < head ? tid : tail_begin + (tid - head);

    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t w = Traits<DT>::kNegInfWord;
        v[u] = u32x4{w, w, w, w};
        if (u * NT + tid < nv) v[u] = vp[u * NT + tid];
    }
    float x_edge[1] = {-INFINITY};
    if (tid < n_edge) x_edge[0] = element<DT>(rp, i_edge);
    const int64_t given = p.targets[row];
    const bool has_target = given >= 0 && given < vocab;
    const int target = has_target ? static_cast<int>(given) : 0;
    const float x_t = has_target ? element<DT>(rp, target) : 0.0f;
    const float above_t = has_target ? from_ordered(ordered(x_t) + 1u) : INFINITY;

    float x[kHeld];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float part[EPV];
        unpack<DT>(v[u], part);
#pragma unroll
        for (int j = 0; j < EPV; ++j) x[u * EPV + j] = part[j];
    }
    // The row's element x[e] is index(e).
    auto index = [&](int e) { return head + (e / EPV * NT + tid) * EPV + e % EPV; };
    float top = x_edge[0];
#pragma unroll
    for (int e = 0; e < kHeld; ++e) top = fmax_nan(top, x[e]);
    Sums s = sums_empty();
    absorb_any<kHeld>(s, x, top, p.factor);
    absorb_any<1>(s, x_edge, x_edge[0], p.factor);
    uint32_t count = has_target && x_edge[0] >= (i_edge < target ? x_t : above_t) ? 1u : 0u;
    // (Lanes without a vector stand behind tail_begin with -inf.)
    const int ties_to = target < tail_begin ? target : tail_begin;
#pragma unroll
    for (int e = 0; e < kHeld; ++e)
        count += has_target && x[e] >= (index(e) < ties_to ? x_t : above_t) ? 1u : 0u;
    count = wave_sum_u32(count);
    const Stat of_wave = wave_reduce_scaled(Stat{s.m, s.z, s.t}, p.factor);

    // 64 R maxima of 16 WAVES / R elements.  With fewer than k of them above -inf
    // the whole row, of less than 64 k / R elements, is listed; all the elements
    // themselves, or 512 maxima and more, where that would be many.
    float* maxima = reinterpret_cast<float*>(sh.list);
    auto leave = [&](auto of_thread) {
        constexpr int kOf = decltype(of_thread)::value, kEach = kHeld / kOf;
#pragma unroll
        for (int q = 0; q < kOf; ++q) {
            float m = q == 0 ? fmax_nan(x[0], x_edge[0]) : x[q * kEach];
#pragma unroll
            for (int e = 1; e < kEach; ++e) m = fmax_nan(m, x[q * kEach + e]);
            maxima[q * NT + tid] = m;
        }
    };
    constexpr int kFew = WAVES < 4 ? 4 : WAVES, kMany = 16;
    const bool few = k <= 64;
    if (few) leave(std::integral_constant<int, kFew / WAVES>{});
    else leave(std::integral_constant<int, kMany / WAVES>{});
    if (lane == 0) {
        sh.wave_stat[wave] = of_wave;
        sh.wave_count[wave] = count;
    }
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    if (wave == 0) {
        const float bound = few ? bound_of<kFew, kFew>(maxima, k) : bound_of<kMany, kMany>(maxima, k);
        if (lane == 0) sh.tau = bound;
    }
    if (wave == WAVES - 1) {
        const Stat total =
            wave_reduce_scaled(lane < WAVES ? sh.wave_stat[lane] : stat_empty(), p.factor);
        if (lane == 0) {
            sh.total = total;
            uint32_t n = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) n += sh.wave_count[w];
            sh.before = n;
        }
    }
    __syncthreads();
    const Stat total = sh.total;
    const float tau = sh.tau;
    int n = 0;
    if (total.m < INFINITY) {
        uint32_t mine = x_edge[0] >= tau ? 1u : 0u;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) mine += x[e] >= tau ? 1u : 0u;
        if (mine != 0) {
            uint32_t to = atomicAdd(&sh.n_list, mine);
            auto keep = [&](float value, int at) {
                if (!(value >= tau)) return;
                if (to < static_cast<uint32_t>(Shared::kList))
                    sh.list[to] = order_key(value, static_cast<uint32_t>(at));
                ++to;
            };
            keep(x_edge[0], i_edge);
#pragma unroll
            for (int e = 0; e < kHeld; ++e) keep(x[e], index(e));
        }
        __syncthreads();
        if (sh.n_list > static_cast<uint32_t>(Shared::kList)) {
            __syncthreads();
            select_exact<DT, WAVES, false>(sh, rp, Piece{head, 0, vocab, 0, nv}, k);
        }
        __syncthreads();
        n = sh.listed();
    }
    put_row<NT>(p, row, sh.list, n, total, has_target, x_t, sh.before);
}

template <int DT, int WAVES, int U>
hipError_t launch_top_t(const TopParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.n_rows * p.splits)), block(WAVES * 64);
    return p.splits > 1 ? launch_kernel(klp_top_kernel<DT, WAVES, U, true>, grid, block, stream, p)
                        : launch_kernel(klp_top_kernel<DT, WAVES, U, false>, grid, block, stream,
                                        p);
}

template <int DT, int WAVES>
hipError_t launch_top_short(const TopParams& p, hipStream_t stream) {
    return launch_kernel(klp_top_short_kernel<DT, WAVES>, dim3(static_cast<unsigned>(p.n_rows)),
                         dim3(WAVES * 64), stream, p);
}

template <int DT>
hipError_t launch_top_dt(const TopParams& p, hipStream_t stream) {
    if (p.vocab <= kTopShort) {
        if (p.vocab <= 1024) return launch_top_short<DT, 1>(p, stream);
        if (p.vocab <= 2048) return launch_top_short<DT, 2>(p, stream);
        return launch_top_short<DT, 4>(p, stream);
    }
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
