// klp_sample.hip — a token a row drawn from its logits by inverse transform of
// one uniform number, with temperature, top-k, top-p and min-p, and the
// token's log-probabilities, for gfx950.
//
//   y_v = (x_v - max x) / T,  w_v = exp(y_v)
//   order: x falling, equal ones by index; K its first top_k; P those of K
//   before which less than top_p mass(K) lies (the first always); M those of
//   P with w >= min_p (the first always);
//   token: the lowest index whose running sum of M's weights exceeds
//   uniform mass(M);  logp = y - ln sum w,  sample_logp = y - ln mass(M).
//
// Precision.  The token and the kept set are decided where a running sum over
// the whole row crosses a border, and a row of 10^5 comparable weights has
// 10^5 such borders: sums off by 10^-7 (float32) pick another token in one of
// 100 rows.  So weights are computed in float64 (2^f by a polynomial of
// degree 8, off by 2 10^-12 at most) and added in float64, or, in histograms,
// as 64-bit integers of 2^-44, whose sums do not depend on the order of the
// atomics.
//
// No row is sorted.  The kept set is {key > tau} and the first r of
// {key == tau}, key the logit's bits in order; tau is found with a histogram
// of counts and masses over 2048 buckets, linear in y, and then inside the
// bucket that holds the border by histograms over the key's bits, 11 at a
// time, of the bucket's elements: from a list in LDS, or of the whole row
// where the list overflows (a row of equal logits).
#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBucketBits = 11;
constexpr int kBuckets = 1 << kBucketBits;
constexpr int kPerThread = kBuckets / kThreads;
constexpr int kList = 4096;
// Range of the first histogram, in units of log2 of the weight; lighter
// elements share the last bucket.
constexpr float kRangeBits = 44.0f;
constexpr double kLog2eD = 1.44269504088896340736;
constexpr double kLn2D = 0.69314718055994530942;

// 2^y for y <= 0: 2^f with f = y - rint(y) as 1 + f q(f), q interpolating
// (2^f - 1) / f at the Chebyshev points of [-1/2, 1/2].
__device__ __forceinline__ double exp2_d(double y) {
    y = fmax(y, -1100.0);  // 0 from there on, -inf included
    const double n = rint(y);
    const double f = y - n;
    double q = 0x1.63b2dp-20;
    q = fma(q, f, 0x1.00c0e454p-16);
    q = fma(q, f, 0x1.4308c71ep-13);
    q = fma(q, f, 0x1.5d87759912p-10);
    q = fma(q, f, 0x1.3b2ab70adp-7);
    q = fma(q, f, 0x1.c6b08da70c1c8p-5);
    q = fma(q, f, 0x1.ebfbdff82a73dp-3);
    q = fma(q, f, 0x1.62e42fef9cc6cp-1);
    return ldexp(fma(q, f, 1.0), static_cast<int>(n));
}

// Bits in the order of the values; -0 becomes +0, which it equals.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

struct Shared {
    uint32_t count[kBuckets];
    unsigned long long mass[kBuckets];
    uint32_t list[kList];
    unsigned long long wave_mass[kWaves];
    double wave_sum[kWaves];
    double wave_all[kWaves];
    uint32_t wave_count[kWaves];
    uint32_t n_list, key_min, key_max;
    // find()'s answer
    uint32_t at, at_count, above_count;
    unsigned long long above_mass;
    // the token
    int token, last;
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ uint32_t wave_sum_u(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <int DT>
struct Row {
    typedef typename Traits<DT>::elem elem;
    const elem* x;
    int vocab;
    int span;  // elements of a wave: a contiguous part of the row

    __device__ __forceinline__ void load(int at, float (&v)[kChunk]) const {
        load_chunk<DT>(x + at, vocab - at, -INFINITY, v);
    }
    // f(first element, 8 values) for each chunk of this wave's part.  Values
    // behind the row's end are -inf.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const int begin = wave * span;
        int end = begin + span;
        if (end > vocab) end = vocab;
        for (int at = begin + lane * kChunk; at < end; at += 64 * kChunk) {
            float v[kChunk];
            load(at, v);
            f(at, v);
        }
    }
};

// The first bucket, in order, at which the running count reaches `count` (or,
// with by_mass, the running mass reaches `mass`); the last one with anything
// in it when none does.  Into s.at, with what lies before it.
__device__ __forceinline__ void find(Shared& s, bool by_mass, uint32_t count, double mass) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = threadIdx.x * kPerThread;
    uint32_t c[kPerThread], c_sum = 0;
    unsigned long long m[kPerThread], m_sum = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        c[i] = s.count[first + i];
        m[i] = s.mass[first + i];
        c_sum += c[i];
        m_sum += m[i];
    }
    uint32_t c_run = c_sum;
    unsigned long long m_run = m_sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cu = __shfl_up(c_run, o, 64);
        const unsigned long long mu = __shfl_up(m_run, o, 64);
        if (lane >= o) {
            c_run += cu;
            m_run += mu;
        }
    }
    if (lane == 63) {
        s.wave_count[wave] = c_run;
        s.wave_mass[wave] = m_run;
    }
    __syncthreads();
    uint32_t c_all = 0;
    unsigned long long m_all = 0;
    c_run -= c_sum;
    m_run -= m_sum;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) {
            c_run += c_all;
            m_run += m_all;
        }
        c_all += s.wave_count[i];
        m_all += s.wave_mass[i];
    }
    // A target that rounding left above the total is the total.
    const double want = fmin(mass, static_cast<double>(m_all));
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const bool before = by_mass ? static_cast<double>(m_run) < want : c_run < count;
        const bool here = by_mass ? static_cast<double>(m_run + m[i]) >= want
                                  : c_run + c[i] >= count;
        if (before && here) {
            s.at = first + i;
            s.at_count = c[i];
            s.above_count = c_run;
            s.above_mass = m_run;
        }
        c_run += c[i];
        m_run += m[i];
    }
    __syncthreads();
}

struct Border {
    uint32_t tau;        // key
    uint32_t ties;       // elements of that key
    uint32_t above;      // elements of larger keys
    unsigned long long above_mass;
};

// What a row's passes share.
template <int DT>
struct Sampler {
    Row<DT> row;
    Shared& s;
    float top;           // max x
    double c;            // log2(e) / T
    float bucket_scale;
    double fixed_one;    // added to a weight, it leaves its fixed-point value in the low bits

    __device__ __forceinline__ double weight(float x) const {
        return exp2_d((static_cast<double>(x) - static_cast<double>(top)) * c);
    }
    __device__ __forceinline__ unsigned long long fixed(double w) const {
        return static_cast<unsigned long long>(__double_as_longlong(w + fixed_one)) &
               ((1ull << 52) - 1);
    }
    // Monotone in x: equal logits share a bucket.
    __device__ __forceinline__ uint32_t bucket(float x) const {
        return static_cast<uint32_t>(fminf((top - x) * bucket_scale, kBuckets - 1.0f));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            s.count[threadIdx.x + i * kThreads] = 0;
            s.mass[threadIdx.x + i * kThreads] = 0;
        }
    }

    // The border inside first-histogram bucket b, among keys >= floor, with
    // `above` elements and above_mass before the bucket.
    __device__ Border resolve(uint32_t b, uint32_t floor, uint32_t above,
                              unsigned long long above_mass, bool by_mass, uint32_t count,
                              double mass) {
        if (threadIdx.x == 0) {
            s.n_list = 0;
            s.key_min = 0xFFFFFFFFu;
            s.key_max = 0;
        }
        __syncthreads();
        row.each([&](int at, const float (&v)[kChunk]) {
            uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                if (bucket(v[j]) != b || at + j >= row.vocab) continue;
                const uint32_t k = key_of(v[j]);
                if (k < floor) continue;
                lo = min(lo, k);
                hi = max(hi, k);
                const uint32_t i = atomicAdd(&s.n_list, 1u);
                if (i < kList) s.list[i] = k;
            }
            if (hi >= lo) {
                atomicMin(&s.key_min, lo);
                atomicMax(&s.key_max, hi);
            }
        });
        __syncthreads();
        const uint32_t n = s.n_list;
        uint32_t lo = s.key_min, hi = s.key_max;
        uint32_t ties = n;
        while (lo != hi) {  // at most 3 times: 32 bits, 11 at a time
            const int bits = 32 - __clz(hi - lo);
            const int shift = bits > kBucketBits ? bits - kBucketBits : 0;
            __syncthreads();
            clear();
            __syncthreads();
            auto add = [&](uint32_t k) {
                if (k < lo || k > hi) return;
                const uint32_t i = (hi - k) >> shift;
                atomicAdd(&s.count[i], 1u);
                atomicAdd(&s.mass[i], fixed(weight(value_of(k))));
            };
            if (n <= kList) {
                for (uint32_t i = threadIdx.x; i < n; i += kThreads) add(s.list[i]);
            } else {
                row.each([&](int at, const float (&v)[kChunk]) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j)
                        if (at + j < row.vocab) add(key_of(v[j]));
                });
            }
            __syncthreads();
            find(s, by_mass, by_mass ? 0 : count - above,
                 by_mass ? mass - static_cast<double>(above_mass) : 0.0);
            above += s.above_count;
            above_mass += s.above_mass;
            ties = s.at_count;
            hi -= s.at << shift;
            const uint32_t low = hi - ((1u << shift) - 1);
            if (low > lo && low <= hi) lo = low;  // hi - low may pass below 0
        }
        __syncthreads();
        return Border{lo, ties, above, above_mass};
    }
};

template <int DT>
__global__ __launch_bounds__(kThreads) void klp_sample_kernel(SampleParams p) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int vocab = static_cast<int>(p.vocab);
    Row<DT> row;
    row.x = static_cast<const typename Traits<DT>::elem*>(p.logits) + row_offset(p.rm, r);
    row.vocab = vocab;
    row.span = (vocab + kWaves * 64 * kChunk - 1) / (kWaves * 64 * kChunk) * 64 * kChunk;

    // The largest logit; NaN where there is one.
    float top = -INFINITY;
    row.each([&](int, const float (&v)[kChunk]) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) top = fmax_nan(top, v[j]);
    });
    top = xrow_max(row_max16(top));
    float* tops = reinterpret_cast<float*>(s.count);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmax_nan(top, tops[i]);
    __syncthreads();
    top += 0.0f;

    float t = p.temperatures != nullptr ? p.temperatures[r] : p.temperature;
    const float top_p = p.top_ps != nullptr ? p.top_ps[r] : p.top_p;
    const float min_p_raw = p.min_ps != nullptr ? p.min_ps[r] : p.min_p;
    int top_k = p.top_ks != nullptr ? p.top_ks[r] : p.top_k;
    const bool greedy = t == 0.0f;
    if (greedy) {
        t = 1.0f;
        top_k = 1;
    }
    if (!(fabsf(top) < INFINITY) || !(t > 0.0f && t < INFINITY)) {
        if (threadIdx.x == 0) {
            const float none = top == -INFINITY ? -INFINITY : NAN;
            p.tokens[r] = -1;
            p.logp[r] = none;
            p.sample_logp[r] = none;
        }
        return;
    }
    const double c = kLog2eD / static_cast<double>(t);
    const float bucket_scale =
        fminf(static_cast<float>(c) * ((kBuckets - 1) / kRangeBits), 1e30f);
    // Fixed point: sums of `vocab` weights of at most 1 stay below 2^63.
    int frac = 62 - (32 - __clz(vocab));
    if (frac > 44) frac = 44;
    const double fixed_one = ldexp(1.0, 52 - frac);
    Sampler<DT> sm{row, s, top, c, bucket_scale, fixed_one};

    const bool by_k = top_k > 0 && top_k < vocab;
    const bool by_p = top_p < 1.0f;  // a NaN is no filter
    const bool by_m = min_p_raw > 0.0f;
    const double min_w = by_m ? fmin(static_cast<double>(min_p_raw), 1.0) : 0.0;

    // Weights of the whole row: their sum, and their histogram where a border
    // is to be found.
    double all = 0.0, kept = 0.0;
    if (by_k || by_p) {
        sm.clear();
        __syncthreads();
    }
    row.each([&](int at, const float (&v)[kChunk]) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const double w = sm.weight(v[j]);
            all += w;
            if (by_k || by_p) {
                if (at + j < vocab) {
                    const uint32_t b = sm.bucket(v[j]);
                    atomicAdd(&s.count[b], 1u);
                    atomicAdd(&s.mass[b], sm.fixed(w));
                }
            } else if (w >= min_w) {
                kept += w;
            }
        }
    });

    uint32_t tau = 0, keep_ties = 0xFFFFFFFFu;
    double tau_w = 0.0;
    if (by_k || by_p) {
        __syncthreads();
        uint32_t floor = 0, floor_bucket = kBuckets, k_ties = 0xFFFFFFFFu;
        double share = 0.0;
        unsigned long long total = 0;
        if (by_p) {  // the whole row's mass, for want of a top-k
            find(s, true, 0, 1e30);
            total = s.above_mass + s.mass[s.at];
            __syncthreads();
        }
        uint32_t p_at = 0, p_above = 0;
        unsigned long long p_above_mass = 0;
        bool p_early = false;
        if (by_k) {
            find(s, false, static_cast<uint32_t>(top_k), 0.0);
            floor_bucket = s.at;
            const uint32_t above = s.above_count;
            const unsigned long long above_mass = s.above_mass;
            // The first histogram is needed again for top-p: its border is
            // looked for in it once the mass of K is known.
            uint32_t hold_c[kPerThread];
            unsigned long long hold_m[kPerThread];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                hold_c[i] = s.count[threadIdx.x + i * kThreads];
                hold_m[i] = s.mass[threadIdx.x + i * kThreads];
            }
            __syncthreads();
            const Border k = sm.resolve(floor_bucket, 0, above, above_mass, false,
                                        static_cast<uint32_t>(top_k), 0.0);
            floor = tau = k.tau;
            k_ties = keep_ties = static_cast<uint32_t>(top_k) - k.above;
            tau_w = sm.weight(value_of(tau));
            if (by_p) {
                total = k.above_mass + k_ties * sm.fixed(tau_w);
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    s.count[threadIdx.x + i * kThreads] = hold_c[i];
                    s.mass[threadIdx.x + i * kThreads] = hold_m[i];
                }
                __syncthreads();
            }
        }
        if (by_p) {
            share = static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(total);
            // The first element is always kept.
            share = fmax(share, 1.0);
            find(s, true, 0, share);
            p_at = s.at;
            p_above = s.above_count;
            p_above_mass = s.above_mass;
            __syncthreads();
            p_early = p_at < floor_bucket;
            const Border b = sm.resolve(p_at, p_early ? 0 : floor, p_above, p_above_mass, true, 0,
                                        share);
            uint32_t limit = b.ties;
            if (b.tau == floor && by_k) limit = min(limit, k_ties);
            tau = b.tau;
            tau_w = sm.weight(value_of(tau));
            const double one = static_cast<double>(sm.fixed(tau_w));
            const double left = share - static_cast<double>(b.above_mass);
            const double need = one > 0.0 ? ceil(left / one) : 1.0;
            keep_ties = need < 1.0 ? 1u : need < limit ? static_cast<uint32_t>(need) : limit;
        }
        // Sums of what is kept, a wave's part each; equal keys at the border
        // are counted and shared out in index order below.
        uint32_t ties = 0;
        row.each([&](int at, const float (&v)[kChunk]) {
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                const uint32_t k = key_of(v[j]);
                if (k < tau || at + j >= vocab) continue;
                if (k == tau) {
                    ++ties;
                } else {
                    const double w = sm.weight(v[j]);
                    if (w >= min_w) kept += w;
                }
            }
        });
        ties = wave_sum_u(ties);
        if (lane == 0) s.wave_count[wave] = ties;
    } else if (lane == 0) {
        s.wave_count[wave] = 0;
    }
    if (tau_w < min_w) tau_w = 0.0;

    all = wave_sum_d(all);
    kept = wave_sum_d(kept);
    if (lane == 0) {
        s.wave_all[wave] = all;
        s.wave_sum[wave] = kept;
    }
    if (threadIdx.x == 0) {
        s.token = 0x7FFFFFFF;
        s.last = -1;
    }
    __syncthreads();
    all = 0.0;
    double mass = 0.0;
    uint32_t ties_before = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const uint32_t n = s.wave_count[i];
        const uint32_t left = keep_ties - min(keep_ties, ties_before);
        all += s.wave_all[i];
        mass += s.wave_sum[i] + min(n, left) * tau_w;
        ties_before += n;
    }
    float u = p.uniform[r];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    const double target = static_cast<double>(u) * mass;
    // The part of the row in which the running sum crosses the target: the
    // last one that holds anything if rounding (or u = 1) lets none.
    int part = 0;
    double before = 0.0, run = 0.0;
    uint32_t part_ties = 0;
    ties_before = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const uint32_t n = s.wave_count[i];
        const uint32_t left = keep_ties - min(keep_ties, ties_before);
        const double m = s.wave_sum[i] + min(n, left) * tau_w;
        if (!found && m > 0.0) {
            part = i;
            before = run;
            part_ties = ties_before;
            found = run + m > target;
        }
        run += m;
        ties_before += n;
    }

    // That part again, 8 consecutive elements a thread.
    double base = before;
    uint32_t base_ties = part_ties;
    int begin = part * row.span, end = begin + row.span;
    if (end > vocab) end = vocab;
    for (int first = begin; first < end; first += kThreads * kChunk) {
        const int at = first + threadIdx.x * kChunk;
        float v[kChunk];
        double w[kChunk];
        uint32_t n_ties = 0;
        row.load(at < end ? at : vocab, v);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            const uint32_t k = key_of(v[j]);
            const bool in = at + j < end;
            w[j] = in && k > tau ? sm.weight(v[j]) : 0.0;
            if (w[j] < min_w) w[j] = 0.0;
            if (in && k == tau && tau != 0) ++n_ties;
        }
        // Ties before this thread's elements.
        uint32_t t_run = n_ties;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(t_run, o, 64);
            if (lane >= o) t_run += x;
        }
        __syncthreads();
        if (lane == 63) s.wave_count[wave] = t_run;
        __syncthreads();
        uint32_t rank = base_ties + t_run - n_ties;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) rank += s.wave_count[i];
            base_ties += s.wave_count[i];
        }
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            if (at + j < end && key_of(v[j]) == tau && tau != 0) {
                if (rank < keep_ties) w[j] = tau_w;
                ++rank;
            }
            sum += w[j];
        }
        double s_run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(s_run, o, 64);
            if (lane >= o) s_run += x;
        }
        __syncthreads();
        if (lane == 63) s.wave_sum[wave] = s_run;
        __syncthreads();
        double pos = base + (s_run - sum);
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) pos += s.wave_sum[i];
            base += s.wave_sum[i];
        }
        int mine = 0x7FFFFFFF, last = -1;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
            pos += w[j];
            if (w[j] > 0.0) {
                last = at + j;
                if (pos > target && mine == 0x7FFFFFFF) mine = at + j;
            }
        }
        if (mine != 0x7FFFFFFF) atomicMin(&s.token, mine);
        if (last >= 0) atomicMax(&s.last, last);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int token = s.token != 0x7FFFFFFF ? s.token : s.last;
        const float x = to_f32<DT>(row.x[token]);
        const double y = (static_cast<double>(x) - static_cast<double>(top)) * c * kLn2D;
        p.tokens[r] = token;
        p.logp[r] = static_cast<float>(y - log(all));
        p.sample_logp[r] = static_cast<float>(y - log(mass));
    }
}

}  // namespace

hipError_t launch_sample(int dtype, const SampleParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.n_rows));
    switch (dtype) {
        case kBF16: return launch_kernel(klp_sample_kernel<kBF16>, grid, dim3(kThreads), stream, p);
        case kFP16: return launch_kernel(klp_sample_kernel<kFP16>, grid, dim3(kThreads), stream, p);
        case kFP32: return launch_kernel(klp_sample_kernel<kFP32>, grid, dim3(kThreads), stream, p);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
