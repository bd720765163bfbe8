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
// 100 rows.  So weights are computed in float64 (off by 1.04 10^-10 at most and,
// since that error changes sign with the logit, far less in a sum) and added in
// float64, or, in histograms, as 64-bit integers of 2^-44, whose sums do not
// depend on the order of the atomics.
//
// A row is read by one workgroup, a contiguous part of it by each wave.
//   No filter: one pass sums the weights, relative to one of the row's first
// logits (or, where those are masked or far below the row's largest, a second
// one relative to that); the part whose running sum crosses the target is read
// again.
//   Filters: one pass for the maximum, then one that collects, in LDS, every
// logit that could be kept, and is followed by work on that list alone: an
// entry's rank, or the mass before it, in falling order says whether it is
// kept, and the kept mass before it by index whether it is drawn.  Up to 256
// entries are compared with each other; of more, those in the buckets of a
// histogram that hold the borders.  What could be kept is bounded beforehand
// by a bucket of a scale that is linear in y: for top-k the bucket of the k-th
// largest of the threads' maxima (k of the logits are at least that large; for
// a k above a quarter of the threads a histogram of the counts, since the k-th
// of few maxima is low), for min-p that of its border, for top-p without a
// top-k that in which a histogram of the masses, one more pass, reaches top_p.
//   Top-p alone: two passes.  A histogram of counts, in float32, whose masses
// say near which bucket the border lies; then the float64 sums of what lies
// before that bucket, and a list of what lies in it.
//   Where the list overflows (more than 4096 logits above the bound: a row of
// equal logits, a wide nucleus) the kept set is {key > tau} and the first r of
// {key == tau}, key the logit's bits in order; tau is found with histograms of
// counts and masses, first over the linear buckets, then inside the bucket
// that holds the border over the key's bits, 11 at a time, and the kept
// weights are summed and searched as those of an unfiltered row.  64 rows of
// 152064 bf16 with top_k = 50 take 23 us at T = 0.7 (greedy: 21), but 135 at T
// = 0.3 and 247 at 0.1: where the k-th largest weighs less than 2^-63 no bucket
// bounds it and the whole row is listed.
#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

namespace {

constexpr int kMaxWaves = 16;
constexpr int kBucketBits = 11;
constexpr int kBuckets = 1 << kBucketBits;
constexpr int kList = 4096;
// Lists whose entries are compared with each other; longer ones go through
// histograms.
constexpr int kRanked = 256;
// The histogram for top-p counts one of so many chunks, to foresee the list's length.
constexpr int kCountEvery = 8;
// Buckets of the first histogram to a factor of 2 of the weight; elements of
// less than 2^-64 share the last bucket.
constexpr int kPerBit = kBuckets / 64;
constexpr uint32_t kAnyBucket = kBuckets;
// A nucleus' border by a float32 histogram: buckets to a factor of 2, bits of
// the place in a bucket, and the factors of 2 by which a logit may exceed the
// one that the buckets are relative to.
constexpr int kNear = kList;  // buckets, in the list's place
constexpr int kNearPerBit = kNear / 64;
constexpr int kNearBits = 8;
constexpr int kNearRoom = 24;
constexpr double kLog2eD = 1.44269504088896340736;
constexpr double kLn2D = 0.69314718055994530942;

// Weights below this one are none: exp2's smallest is 2^-1000, for a logit
// of -inf too, and a row of 2^26 of those sums to less than this.
constexpr double kNothing = 0x1p-960;

// 2^y for |y| <= 1000 as t g: t = 2^(n / 256), n = rint(256 y), from a table
// of 2^(i / 256), i < 256, and g = 2^f, f = y - n / 256, as 1 + f q(f), q
// interpolating (2^f - 1) / f where the cubic Chebyshev polynomial of [-1/512,
// 1/512] is 0 (besides f = 0): g is off by (ln 2 / 512)^3 / 24, 1.04 10^-10
// with the terms behind.
// Adding kRound rounds to n / 256 and leaves n in the sum's low word.  An entry
// lacks i 2^12 in its high word, which n 2^12 = (n / 256) 2^20 + (n % 256) 2^12
// puts back along with the exponent.  256 entries: n's low byte is an operand
// of its own, so one shift makes it an address, and 2 products suffice.
// Arithmetic is the bound, and LDS has the room: 1024 rows of 128256 (fp16,
// unfiltered) 81.5 us, with 32 entries (in different banks, 3 products, one
// operation more for the address) 89, with a polynomial of degree 7 100.
constexpr double kRound = 0x1.8p44;
constexpr int kExp2Entries = 256;
__device__ const unsigned long long kExp2Table[kExp2Entries] = {
    0x3ff0000000000000ull, 0x3feffb1afa5abcbfull, 0x3feff63da9fb3335ull, 0x3feff168143b0281ull,
    0x3fefec9a3e778061ull, 0x3fefe7d42e11bbccull, 0x3fefe315e86e7f85ull, 0x3fefde5f72f654b1ull,
    0x3fefd9b0d3158574ull, 0x3fefd50a0e3c1f89ull, 0x3fefd06b29ddf6deull, 0x3fefcbd42b72a836ull,
    0x3fefc74518759bc8ull, 0x3fefc2bdf66607e0ull, 0x3fefbe3ecac6f383ull, 0x3fefb9c79b1f3919ull,
    0x3fefb5586cf9890full, 0x3fefb0f145e46c85ull, 0x3fefac922b7247f7ull, 0x3fefa83b23395decull,
    0x3fefa3ec32d3d1a2ull, 0x3fef9fa55fdfa9c5ull, 0x3fef9b66affed31bull, 0x3fef973028d7233eull,
    0x3fef9301d0125b51ull, 0x3fef8edbab5e2ab6ull, 0x3fef8abdc06c31ccull, 0x3fef86a814f204abull,
    0x3fef829aaea92de0ull, 0x3fef7e95934f312eull, 0x3fef7a98c8a58e51ull, 0x3fef76a45471c3c2ull,
    0x3fef72b83c7d517bull, 0x3fef6ed48695bbc0ull, 0x3fef6af9388c8deaull, 0x3fef672658375d2full,
    0x3fef635beb6fcb75ull, 0x3fef5f99f8138a1cull, 0x3fef5be084045cd4ull, 0x3fef582f95281c6bull,
    0x3fef54873168b9aaull, 0x3fef50e75eb44027ull, 0x3fef4d5022fcd91dull, 0x3fef49c18438ce4dull,
    0x3fef463b88628cd6ull, 0x3fef42be3578a819ull, 0x3fef3f49917ddc96ull, 0x3fef3bdda27912d1ull,
    0x3fef387a6e756238ull, 0x3fef351ffb82140aull, 0x3fef31ce4fb2a63full, 0x3fef2e85711ece75ull,
    0x3fef2b4565e27cddull, 0x3fef280e341ddf29ull, 0x3fef24dfe1f56381ull, 0x3fef21ba7591bb70ull,
    0x3fef1e9df51fdee1ull, 0x3fef1b8a66d10f13ull, 0x3fef187fd0dad990ull, 0x3fef157e39771b2full,
    0x3fef1285a6e4030bull, 0x3fef0f961f641589ull, 0x3fef0cafa93e2f56ull, 0x3fef09d24abd886bull,
    0x3fef06fe0a31b715ull, 0x3fef0432edeeb2fdull, 0x3fef0170fc4cd831ull, 0x3feefeb83ba8ea32ull,
    0x3feefc08b26416ffull, 0x3feef96266e3fa2dull, 0x3feef6c55f929ff1ull, 0x3feef431a2de883bull,
    0x3feef1a7373aa9cbull, 0x3feeef26231e754aull, 0x3feeecae6d05d866ull, 0x3feeea401b7140efull,
    0x3feee7db34e59ff7ull, 0x3feee57fbfec6cf4ull, 0x3feee32dc313a8e5ull, 0x3feee0e544ede173ull,
    0x3feedea64c123422ull, 0x3feedc70df1c5175ull, 0x3feeda4504ac801cull, 0x3feed822c367a024ull,
    0x3feed60a21f72e2aull, 0x3feed3fb2709468aull, 0x3feed1f5d950a897ull, 0x3feecffa3f84b9d4ull,
    0x3feece086061892dull, 0x3feecc2042a7d232ull, 0x3feeca41ed1d0057ull, 0x3feec86d668b3237ull,
    0x3feec6a2b5c13cd0ull, 0x3feec4e1e192aed2ull, 0x3feec32af0d7d3deull, 0x3feec17dea6db7d7ull,
    0x3feebfdad5362a27ull, 0x3feebe41b817c114ull, 0x3feebcb299fddd0dull, 0x3feebb2d81d8abffull,
    0x3feeb9b2769d2ca7ull, 0x3feeb8417f4531eeull, 0x3feeb6daa2cf6642ull, 0x3feeb57de83f4eefull,
    0x3feeb42b569d4f82ull, 0x3feeb2e2f4f6ad27ull, 0x3feeb1a4ca5d920full, 0x3feeb070dde910d2ull,
    0x3feeaf4736b527daull, 0x3feeae27dbe2c4cfull, 0x3feead12d497c7fdull, 0x3feeac0827ff07ccull,
    0x3feeab07dd485429ull, 0x3feeaa11fba87a03ull, 0x3feea9268a5946b7ull, 0x3feea84590998b93ull,
    0x3feea76f15ad2148ull, 0x3feea6a320dceb71ull, 0x3feea5e1b976dc09ull, 0x3feea52ae6cdf6f4ull,
    0x3feea47eb03a5585ull, 0x3feea3dd1d1929fdull, 0x3feea34634ccc320ull, 0x3feea2b9febc8fb7ull,
    0x3feea23882552225ull, 0x3feea1c1c70833f6ull, 0x3feea155d44ca973ull, 0x3feea0f4b19e9538ull,
    0x3feea09e667f3bcdull, 0x3feea052fa75173eull, 0x3feea012750bdabfull, 0x3fee9fdcddd47645ull,
    0x3fee9fb23c651a2full, 0x3fee9f9298593ae5ull, 0x3fee9f7df9519484ull, 0x3fee9f7466f42e87ull,
    0x3fee9f75e8ec5f74ull, 0x3fee9f8286ead08aull, 0x3fee9f9a48a58174ull, 0x3fee9fbd35d7cbfdull,
    0x3fee9feb564267c9ull, 0x3feea024b1ab6e09ull, 0x3feea0694fde5d3full, 0x3feea0b938ac1cf6ull,
    0x3feea11473eb0187ull, 0x3feea17b0976cfdbull, 0x3feea1ed0130c132ull, 0x3feea26a62ff86f0ull,
    0x3feea2f336cf4e62ull, 0x3feea3878491c491ull, 0x3feea427543e1a12ull, 0x3feea4d2add106d9ull,
    0x3feea589994cce13ull, 0x3feea64c1eb941f7ull, 0x3feea71a4623c7adull, 0x3feea7f4179f5b21ull,
    0x3feea8d99b4492edull, 0x3feea9cad931a436ull, 0x3feeaac7d98a6699ull, 0x3feeabd0a478580full,
    0x3feeace5422aa0dbull, 0x3feeae05bad61778ull, 0x3feeaf3216b5448cull, 0x3feeb06a5e0866d9ull,
    0x3feeb1ae99157736ull, 0x3feeb2fed0282c8aull, 0x3feeb45b0b91ffc6ull, 0x3feeb5c353aa2fe2ull,
    0x3feeb737b0cdc5e5ull, 0x3feeb8b82b5f98e5ull, 0x3feeba44cbc8520full, 0x3feebbdd9a7670b3ull,
    0x3feebd829fde4e50ull, 0x3feebf33e47a22a2ull, 0x3feec0f170ca07baull, 0x3feec2bb4d53fe0dull,
    0x3feec49182a3f090ull, 0x3feec674194bb8d5ull, 0x3feec86319e32323ull, 0x3feeca5e8d07f29eull,
    0x3feecc667b5de565ull, 0x3feece7aed8eb8bbull, 0x3feed09bec4a2d33ull, 0x3feed2c980460ad8ull,
    0x3feed503b23e255dull, 0x3feed74a8af46052ull, 0x3feed99e1330b358ull, 0x3feedbfe53c12e59ull,
    0x3feede6b5579fdbfull, 0x3feee0e521356ebaull, 0x3feee36bbfd3f37aull, 0x3feee5ff3a3c2774ull,
    0x3feee89f995ad3adull, 0x3feeeb4ce622f2ffull, 0x3feeee07298db666ull, 0x3feef0ce6c9a8952ull,
    0x3feef3a2b84f15fbull, 0x3feef68415b749b1ull, 0x3feef9728de5593aull, 0x3feefc6e29f1c52aull,
    0x3feeff76f2fb5e47ull, 0x3fef028cf22749e4ull, 0x3fef05b030a1064aull, 0x3fef08e0b79a6f1full,
    0x3fef0c1e904bc1d2ull, 0x3fef0f69c3f3a207ull, 0x3fef12c25bd71e09ull, 0x3fef16286141b33dull,
    0x3fef199bdd85529cull, 0x3fef1d1cd9fa652cull, 0x3fef20ab5fffd07aull, 0x3fef244778fafb22ull,
    0x3fef27f12e57d14bull, 0x3fef2ba88988c933ull, 0x3fef2f6d9406e7b5ull, 0x3fef33405751c4dbull,
    0x3fef3720dcef9069ull, 0x3fef3b0f2e6d1675ull, 0x3fef3f0b555dc3faull, 0x3fef43155b5bab74ull,
    0x3fef472d4a07897cull, 0x3fef4b532b08c968ull, 0x3fef4f87080d89f2ull, 0x3fef53c8eacaa1d6ull,
    0x3fef5818dcfba487ull, 0x3fef5c76e862e6d3ull, 0x3fef60e316c98398ull, 0x3fef655d71ff6075ull,
    0x3fef69e603db3285ull, 0x3fef6e7cd63a8315ull, 0x3fef7321f301b460ull, 0x3fef77d5641c0658ull,
    0x3fef7c97337b9b5full, 0x3fef81676b197d17ull, 0x3fef864614f5a129ull, 0x3fef8b333b16ee12ull,
    0x3fef902ee78b3ff6ull, 0x3fef953924676d76ull, 0x3fef9a51fbc74c83ull, 0x3fef9f7977cdb740ull,
    0x3fefa4afa2a490daull, 0x3fefa9f4867cca6eull, 0x3fefaf482d8e67f1ull, 0x3fefb4aaa2188510ull,
    0x3fefba1bee615a27ull, 0x3fefbf9c1cb6412aull, 0x3fefc52b376bba97ull, 0x3fefcac948dd7274ull,
    0x3fefd0765b6e4540ull, 0x3fefd632798844f8ull, 0x3fefdbfdad9cbe14ull, 0x3fefe1d802243c89ull,
    0x3fefe7c1819e90d8ull, 0x3fefedba3692d514ull, 0x3feff3c22b8f71f1ull, 0x3feff9d96b2a23d9ull};

struct Exp2 {
    double t, g;
};
__device__ __forceinline__ Exp2 exp2_parts(const unsigned long long* table, double y) {
    const double rounded = y + kRound;
    const double f = y - (rounded - kRound);
    const int n = __double2loint(rounded);
    const double t = __longlong_as_double(static_cast<long long>(table[n & (kExp2Entries - 1)]));
    const double q = fma(0x1.ebfbe3a9ac80bp-3, f, 0x1.62e43543b54d7p-1);
    return Exp2{__hiloint2double(__double2hiint(t) + (n << 12), __double2loint(t)),
                fma(q, f, 1.0)};
}

// The largest, a NaN where there is one: three operands an instruction.
__device__ __forceinline__ float chunk_max(const float (&v)[kChunk]) {
    const float a = fmax_nan(fmax_nan(v[0], v[1]), v[2]);
    const float b = fmax_nan(fmax_nan(v[3], v[4]), v[5]);
    return fmax_nan(fmax_nan(a, b), fmax_nan(v[6], v[7]));
}

// Bits in the order of the values; -0 becomes +0, which it equals.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// kFilters: with the histograms and the list, which leave room for two
// workgroups of 512 threads a CU; without them registers set their number.
template <bool kFilters>
struct Shared {
    unsigned long long exp2_table[kExp2Entries];
    uint32_t count[kFilters ? kBuckets : 1];
    unsigned long long mass[kFilters ? kBuckets : 1];
    uint2 list[kFilters ? kList : 1];  // (~key, index): in falling order, x before y
    uint2 few[kFilters ? kRanked : 1];  // those of one bucket
    unsigned long long few_mass[kFilters ? kRanked : 1];
    uint32_t few_kept[kFilters ? kRanked : 1];
    uint32_t n_few;
    unsigned long long wave_mass[kMaxWaves];
    double wave_sum[kMaxWaves];
    double wave_all[kMaxWaves];
    float wave_top[kMaxWaves];
    uint32_t wave_count[kMaxWaves];
    uint32_t n_list, key_min, key_max, key_count;
    // find()'s answer
    uint32_t at, at_count, above_count;
    unsigned long long above_mass;
    // search()'s first and last thread with weight
    int first, last;
};

// v from the lane that DPP control Ctrl names, 0 where there is none.
template <int Ctrl, int Rows>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t v) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), Ctrl, Rows, 0xF, false));
}
template <int Ctrl, int Rows>
__device__ __forceinline__ unsigned long long dpp_or_0(unsigned long long v) {
    const uint32_t lo = dpp_or_0<Ctrl, Rows>(static_cast<uint32_t>(v));
    const uint32_t hi = dpp_or_0<Ctrl, Rows>(static_cast<uint32_t>(v >> 32));
    return static_cast<unsigned long long>(hi) << 32 | lo;
}
template <int Ctrl, int Rows>
__device__ __forceinline__ double dpp_or_0(double v) {
    return __longlong_as_double(static_cast<long long>(
        dpp_or_0<Ctrl, Rows>(static_cast<unsigned long long>(__double_as_longlong(v)))));
}

// What the lanes up to this one have of v: shifts within rows of 16 lanes,
// then the first and third row's last lane to the row behind it, and the
// second row's to the wave's second half.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    v += dpp_or_0<0x111, 0xF>(v);
    v += dpp_or_0<0x112, 0xF>(v);
    v += dpp_or_0<0x114, 0xF>(v);
    v += dpp_or_0<0x118, 0xF>(v);
    v += dpp_or_0<0x142, 0xA>(v);
    v += dpp_or_0<0x143, 0xC>(v);
    return v;
}
// What the lanes before this one have of v; `total`: what the wave has.
template <typename V>
__device__ __forceinline__ V wave_before(V v, V& total) {
    const V run = wave_scan(v);
    total = __shfl(run, 63, 64);
    return run - v;
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
    return __shfl(wave_scan(v), 63, 64);
}

// What the threads before this one have of v; `total`: what all have.
template <int T, typename V>
__device__ __forceinline__ V block_before(V (&lds)[kMaxWaves], V v, V& total) {
    constexpr int kWaves = T / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const V run = wave_scan(v);
    __syncthreads();  // the last call's readers
    if (lane == 63) lds[wave] = run;
    __syncthreads();
    V before = run - v;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) before += total;
        total += lds[i];
    }
    return before;
}

template <int DT>
struct Row {
    typedef typename Traits<DT>::elem elem;
    const elem* x;
    int vocab;
    int span;  // elements of a wave: a contiguous part of the row
    // Chunks of a lane in flight, 32 bytes: with 64 the passes' code is twice as
    // long for nothing (256 rows of 152064 bf16 with a top-k 37 against 35 us).
    static constexpr int kBatch = DT == kFP32 ? 1 : 2;

    __device__ __forceinline__ void load(int at, float (&v)[kChunk]) const {
        load_chunk<DT, true>(x + at, vocab - at, v);
    }
    // f(first element, 8 values) for each chunk of this wave's part, the next
    // kBatch of them being loaded.  Values behind the row's end are -inf.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        constexpr int kStep = 64 * kChunk;
        const int begin = wave * span;
        int end = begin + span;
        if (end > vocab) end = vocab;
        typedef Unaligned16<elem> Vec;
        constexpr int kVecs = DT == kFP32 ? 2 : 1;
        const int batches = end > begin ? (end - begin) / (kBatch * kStep) : 0;
        int at = begin + lane * kChunk;
        if (batches > 0) {
            u32x4 raw[kBatch][kVecs];
            auto fetch = [&](int i, int from) {
#pragma unroll
                for (int k = 0; k < kVecs; ++k)
                    raw[i][k] = reinterpret_cast<const Vec*>(x + from + i * kStep)[k].v;
            };
#pragma unroll
            for (int i = 0; i < kBatch; ++i) fetch(i, at);
            for (int b = 1; b <= batches; ++b) {
                const int next = b < batches ? at + kBatch * kStep : at;  // or the last again
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    float v[kChunk];
                    unpack<DT>(raw[i][0], v);
                    if constexpr (DT == kFP32) unpack<DT>(raw[i][1], v + 4);
                    fetch(i, next);
                    f(at + i * kStep, v);
                    __builtin_amdgcn_sched_barrier(0);
                }
                at += kBatch * kStep;
            }
        }
        for (; at < end; at += kStep) {
            float v[kChunk];
            load(at, v);
            f(at, v);
        }
    }
    // The same for the passes that few rows take: a chunk at a time and f's
    // code once, since all passes with theirs five times over are more than a
    // branch of the kernel can span.
    template <typename F>
    __device__ __forceinline__ void each_small(F f) const {
        const int begin = (threadIdx.x >> 6) * span;
        const int end = min(begin + span, vocab);
#pragma unroll 1
        for (int at = begin + static_cast<int>(threadIdx.x & 63) * kChunk; at < end;
             at += 64 * kChunk) {
            float v[kChunk];
            load(at, v);
            f(at, v);
        }
    }
};

// The first bucket, in order, at which the running count reaches `count` (or,
// with by_mass, the running mass reaches `mass`); the last one with anything
// in it when none does.  Into s.at, with what lies before it.
template <int T>
__device__ __forceinline__ void find(Shared<true>& s, bool by_mass, uint32_t count,
                                     unsigned long long mass) {
    constexpr int kPerThread = kBuckets / T;
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
    uint32_t c_all;
    unsigned long long m_all;
    uint32_t c_run = block_before<T>(s.wave_count, c_sum, c_all);
    unsigned long long m_run = block_before<T>(s.wave_mass, m_sum, m_all);
    // A target that rounding left above the total is the total.
    mass = min(mass, m_all);
    count = min(count, c_all);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const bool before = by_mass ? m_run < mass : c_run < count;
        const bool here = by_mass ? m_run + m[i] >= mass : c_run + c[i] >= count;
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

// x cut to a whole number, 0 below 0 and for a NaN, 2^32 - 1 above that.
__device__ __forceinline__ uint32_t whole_part(float x) {
    uint32_t v;
    asm("v_cvt_u32_f32 %0, %1" : "=v"(v) : "v"(x));
    return v;
}

struct Border {
    uint32_t tau;        // key
    uint32_t ties;       // elements of that key
    uint32_t above;      // elements of larger keys
    unsigned long long above_mass;
};

// What a row's passes share.
template <int DT, int T, bool kFilters>
struct Sampler {
    static constexpr int kWaves = T / 64, kPerThread = kBuckets / T;
    Row<DT> row;
    Shared<kFilters>& s;
    float top;           // weights are relative to this logit
    double c;            // log2(e) / T
    float c32;
    double fixed_one;    // added to a weight, it leaves its fixed-point value in the low bits

    // Exactly 0 for x = top, whose weight is exactly 1.  16-bit logits have 11
    // bits at most and their c 42: both products are exact.
    __device__ __forceinline__ double log2_weight(float x) const {
        if constexpr (DT == kFP32) return (static_cast<double>(x) - static_cast<double>(top)) * c;
        return fma(static_cast<double>(x), c, -static_cast<double>(top) * c);
    }
    __device__ __forceinline__ Exp2 parts(double log2_w) const {
        return exp2_parts(s.exp2_table, fmax(log2_w, -1000.0));
    }
    __device__ __forceinline__ double exp2(double log2_w) const {
        const Exp2 e = parts(log2_w);
        return e.t * e.g;
    }
    __device__ __forceinline__ double weight(float x) const { return exp2(log2_weight(x)); }
    __device__ __forceinline__ unsigned long long fixed(double w) const {
        return static_cast<unsigned long long>(__double_as_longlong(w + fixed_one)) &
               ((1ull << 52) - 1);
    }
    // By -log2 of the weight, which adding 1.5 2^52 / kPerBit rounds to whole
    // buckets: monotone in x, so that equal logits share one.
    __device__ __forceinline__ uint32_t bucket_of(double log2_w) const {
        const int n = __double2loint(fmax(log2_w, -1000.0) + 0x1.8p52 / kPerBit);
        return static_cast<uint32_t>(min(-n, kBuckets - 1));
    }
    __device__ __forceinline__ uint32_t bucket(float x) const {
        return bucket_of(log2_weight(x));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            s.count[threadIdx.x + i * T] = 0;
            s.mass[threadIdx.x + i * T] = 0;
        }
        __syncthreads();
    }

    // Threads that share one of n <= kRanked entries: 2 at least, neighbours.
    static __device__ __forceinline__ uint32_t threads_for(uint32_t n) {
        uint32_t per = 64;
        while (per * n > T) per >>= 1;
        return per;
    }
    static __device__ __forceinline__ unsigned long long over_group(unsigned long long v,
                                                                    uint32_t per) {
        for (uint32_t o = per >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        return v;
    }

    // f(key) for every element of the list, or of the row.
    template <typename F>
    __device__ __forceinline__ void candidates(bool listed, F f) {
        if (listed) {
            const uint32_t n = s.n_list;
            for (uint32_t i = threadIdx.x; i < n; i += T) f(~s.list[i].x);
        } else {
            row.each_small([&](int, const float (&v)[kChunk]) {
#pragma unroll
                for (int j = 0; j < kChunk; ++j) f(key_of(v[j]));
            });
        }
    }

    // The border inside first-histogram bucket b (or kAnyBucket), among keys >= floor, with
    // `above` elements and above_mass before the bucket.
    __device__ __forceinline__ Border resolve(bool listed, uint32_t b, uint32_t floor,
                                              uint32_t above, unsigned long long above_mass,
                                              bool by_mass, uint32_t count,
                                              unsigned long long mass) {
        __syncthreads();
        if (threadIdx.x == 0) {
            s.key_count = 0;
            s.key_min = 0xFFFFFFFFu;
            s.key_max = 0;
        }
        __syncthreads();
        uint32_t lo = 0xFFFFFFFFu, hi = 0, n = 0;
        candidates(listed, [&](uint32_t k) {
            if (k < floor || (b != kAnyBucket && bucket(value_of(k)) != b)) return;
            lo = min(lo, k);
            hi = max(hi, k);
            ++n;
        });
        if (n > 0) {
            atomicMin(&s.key_min, lo);
            atomicMax(&s.key_max, hi);
            atomicAdd(&s.key_count, n);
        }
        __syncthreads();
        lo = s.key_min;
        hi = s.key_max;
        uint32_t ties = s.key_count;
        while (lo != hi) {  // at most 3 times: 32 bits, 11 at a time
            const int bits = 32 - __clz(hi - lo);
            const int shift = bits > kBucketBits ? bits - kBucketBits : 0;
            __syncthreads();
            clear();
            candidates(listed, [&](uint32_t k) {
                if (k < lo || k > hi) return;
                const uint32_t i = (hi - k) >> shift;
                atomicAdd(&s.count[i], 1u);
                if (by_mass) atomicAdd(&s.mass[i], fixed(weight(value_of(k))));
            });
            __syncthreads();
            find<T>(s, by_mass, by_mass ? 0 : count - above, by_mass ? mass - above_mass : 0);
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

    // Each wave's part of the row: its sum of kept weights above the border,
    // and its count of ties.
    __device__ __forceinline__ void set_parts(double kept, uint32_t ties) {
        kept = wave_sum(kept);
        ties = wave_sum(ties);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            s.wave_sum[threadIdx.x >> 6] = kept;
            s.wave_count[threadIdx.x >> 6] = ties;
        }
    }

    // The token of {key > tau, or one of the first keep_ties of {key == tau},
    // with a weight of at least min_w}, by the parts set before: the part whose
    // running sum crosses the target, in it the thread whose run of elements
    // does, and among those the element.  Where rounding (or u = 1) lets none
    // cross, the last that has a weight.  The wave of that thread returns the
    // token, the others -1.
    __device__ __forceinline__ int search(float u, uint32_t tau, uint32_t keep_ties, double min_w,
                                          double& mass) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        double tau_w = keep_ties > 0 ? weight(value_of(tau)) : 0.0;
        if (tau_w < min_w) tau_w = 0.0;
        if (threadIdx.x == 0) {
            s.first = T;
            s.last = -1;
        }
        __syncthreads();
        // Lane i holds part i, in every wave.
        uint32_t ties = lane < kWaves ? s.wave_count[lane] : 0, all_ties;
        uint32_t rank = wave_before(ties, all_ties);
        auto kept_ties = [&]() { return min(ties, keep_ties - min(keep_ties, rank)) * tau_w; };
        double sum = (lane < kWaves ? s.wave_sum[lane] : 0.0) + kept_ties();
        double pos = wave_before(sum, mass);
        const double target = static_cast<double>(u) * mass;
        auto choose = [&](bool has, bool crosses) {
            const uint64_t c = __ballot(has && crosses), h = __ballot(has);
            return c != 0 ? __ffsll(static_cast<unsigned long long>(c)) - 1
                          : 63 - __clzll(static_cast<long long>(h));
        };
        const int part = choose(sum > kNothing, pos + sum > target);
        // The row's largest weighs 2^-300 at least: there is such a part.
        if (part < 0) return wave == 0 ? 0 : -1;
        pos = __shfl(pos, part, 64);
        rank = __shfl(rank, part, 64);

        const int per = (row.span / kChunk + T - 1) / T * kChunk;  // elements a thread
        const int end = min((part + 1) * row.span, row.vocab);
        const int begin = part * row.span + static_cast<int>(threadIdx.x) * per;
        sum = 0.0;
        ties = 0;
        for (int at = begin; at < begin + per && at < end; at += kChunk) {
            float v[kChunk];
            row.load(at, v);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                if (at + j >= end) continue;
                const uint32_t k = key_of(v[j]);
                if (k > tau) {
                    const double w = weight(v[j]);
                    if (w >= min_w) sum += w;
                }
                if (k == tau) ++ties;
            }
        }
        double total;
        if (keep_ties > 0) {
            rank += block_before<T>(s.wave_count, ties, all_ties);
            sum += kept_ties();
        }
        pos += block_before<T>(s.wave_sum, sum, total);
        const uint64_t has = __ballot(sum > kNothing);
        const uint64_t crosses = __ballot(sum > kNothing && pos + sum > target);
        if (lane == 0 && has != 0)
            atomicMax(&s.last, wave * 64 + 63 - __clzll(static_cast<long long>(has)));
        if (lane == 0 && crosses != 0)
            atomicMin(&s.first, wave * 64 + __ffsll(static_cast<unsigned long long>(crosses)) - 1);
        __syncthreads();
        const int thread = s.first < T ? s.first : s.last;
        if (thread < 0) return wave == 0 ? part * row.span : -1;
        if (thread >> 6 != wave) return -1;
        pos = __shfl(pos, thread & 63, 64);
        rank = __shfl(rank, thread & 63, 64);

        int token = -1;
        const int first = __shfl(begin, thread & 63, 64), stop = min(first + per, end);
        for (int from = first; from < stop; from += 64) {
            const int at = from + lane;
            const bool in = at < stop;
            const float v = in ? to_f32<DT>(row.x[at]) : -INFINITY;
            const uint32_t k = key_of(v);
            double w = in && k > tau ? weight(v) : 0.0;
            if (w < min_w) w = 0.0;
            const uint64_t tie = __ballot(in && k == tau);
            if (tie >> lane & 1) {
                const uint32_t mine = rank + __popcll(tie & ((1ull << lane) - 1));
                if (mine < keep_ties) w = tau_w;
            }
            rank += __popcll(tie);
            const double before = pos + wave_before(w, total);
            const int at_lane = choose(w > kNothing, before + w > target);
            const bool found = __ballot(w > kNothing && before + w > target) != 0;
            if (at_lane >= 0) token = from + at_lane;
            if (found) break;
            pos += total;
        }
        return token >= 0 ? token : first;
    }
};

// What rows may have: no filter and no temperature of 0; no filter but top-p
// (a row's temperature of 0 is then a top-p of 0); any.  (In one kernel the passes of top-p alone would spill registers.)
enum SampleMode { kPlain, kTopP, kAny };

template <int DT, int T, int kMode>
__global__ __launch_bounds__(T, kMode != kPlain ? 4 : 6) void klp_sample_kernel(SampleParams p) {
    constexpr int kWaves = T / 64;
    constexpr bool kFilters = kMode != kPlain;
    __shared__ Shared<kFilters> s;
    const int64_t r = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int vocab = static_cast<int>(p.vocab);
    Row<DT> row;
    row.x = static_cast<const typename Traits<DT>::elem*>(p.logits) + row_offset(p.rm, r);
    row.vocab = vocab;
    row.span = (vocab + kWaves * 64 * kChunk - 1) / (kWaves * 64 * kChunk) * 64 * kChunk;

    float t = p.temperatures != nullptr ? p.temperatures[r] : p.temperature;
    float top_p = p.top_ps != nullptr ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps != nullptr ? p.min_ps[r] : p.min_p;
    int top_k = p.top_ks != nullptr ? p.top_ks[r] : p.top_k;
    float u = p.uniform[r];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    if (t == 0.0f) {
        t = 1.0f;
        top_k = 1;
        if (kMode == kTopP) top_p = 0.0f;  // keeps the same one
    }
    const bool bad_t = !(t > 0.0f && t < INFINITY);
    if (bad_t) t = 1.0f;
    const bool by_k = kMode == kAny && top_k > 0 && top_k < vocab;
    const bool by_p = top_p < 1.0f;  // a NaN is no filter
    const bool by_m = kMode == kAny && min_p > 0.0f;
    const uint32_t k_left = by_k ? static_cast<uint32_t>(top_k) : 0xFFFFFFFFu;
    // A mass before which top-p keeps what it does, of whole masses: the first
    // element always.
    auto share_of = [&](double mass) {
        const double m = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * mass);
        return m > 1.0 ? static_cast<unsigned long long>(m) : 1ull;
    };
    const double min_w = by_m ? fmin(static_cast<double>(min_p), 1.0) : 0.0;

    // Fixed point: sums of `vocab` weights of at most 1 stay below 2^63.
    int frac = 62 - (32 - __clz(vocab));
    if (frac > 44) frac = 44;
    double c = kLog2eD / static_cast<double>(t);
    if constexpr (DT != kFP32)  // 42 bits, 2^-42 of it off at most
        c = __longlong_as_double(__double_as_longlong(c) & ~0x7FFll);
    Sampler<DT, T, kFilters> sm{row, s, 0.0f, c, fminf(static_cast<float>(c), 1e30f),
                      ldexp(1.0, 52 - frac)};

    float top = -INFINITY;  // the largest logit; NaN where there is one
    auto over_row = [&]() {
        top = xrow_max(row_max16(top));
        __syncthreads();
        if (lane == 0) s.wave_top[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmax_nan(top, s.wave_top[i]);
        if (fabsf(top) < INFINITY && !bad_t) return true;
        if (threadIdx.x == 0) {
            const float none = top == -INFINITY && !bad_t ? -INFINITY : NAN;
            p.tokens[r] = -1;
            p.logp[r] = none;
            p.sample_logp[r] = none;
        }
        return false;
    };
    auto over_waves = [&](double v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) s.wave_all[wave] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v += s.wave_all[i];
        return v;
    };
    // A running sum of whole masses crosses uniform * mass where it exceeds this.
    auto target_of = [&](unsigned long long mass) {
        return static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(mass));
    };
    // By an even lane and the next one, each with one of the logarithms.
    auto finish = [&](int token, double all, double mass) {
        const double y = sm.log2_weight(to_f32<DT>(row.x[token])) * kLn2D;
        const float out = static_cast<float>(y - log(lane & 1 ? mass : all));
        (lane & 1 ? p.sample_logp : p.logp)[r] = out;
        if (!(lane & 1)) p.tokens[r] = token;
    };

    if (threadIdx.x < kExp2Entries) s.exp2_table[threadIdx.x] = kExp2Table[threadIdx.x];
    if (!kFilters || (!by_k && !by_p && !by_m)) {
        // Weights relative to the largest of the first 64 logits, or to 0 where
        // those are all masked; again, to the row's largest, where that
        // outranges float64 (by 2^900) or lies so far below such a 0 (2^300)
        // that the row's own weights would come near to counting as none.
        // (1024 rows of 128256 fp16, the first 64 masked: 86 us, 132 twice.)
        float first = lane < vocab ? to_f32<DT>(row.x[lane]) : -INFINITY;
        first = xrow_max(row_max16(first));
        __syncthreads();
        double sum;
        auto add_up = [&]() {
            sum = 0.0;
            row.each([&](int, const float (&v)[kChunk]) {
                top = fmax_nan(top, chunk_max(v));
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const Exp2 e = sm.parts(sm.log2_weight(v[j]));
                    sum = fma(e.t, e.g, sum);
                }
            });
        };
        sm.top = fabsf(first) < INFINITY ? first : 0.0f;
        add_up();
        if (!over_row()) return;
        const double ahead = sm.log2_weight(top);
        if (ahead > 900.0 || ahead < -300.0) {
            sm.top = top;
            add_up();
        }
        sm.set_parts(sum, 0);
        double mass;
        const int token = sm.search(u, 0, 0, 0.0, mass);
        if (token >= 0 && lane < 2) finish(token, mass, mass);
        return;
    }
    if constexpr (kFilters) {
        uint32_t bound = 0, p_at = kBuckets;
        double all = 0.0, kept = 0.0;
        unsigned long long share = 0, p_above = 0;
        uint32_t tau = 0, keep_ties = 0;
        bool wide = false;  // what lies before p_at's bucket is kept, that one's elements listed
        auto append = [&](uint32_t in, int at, const float (&v)[kChunk]) {
            // Past kList only the count matters, and not how far.
            if (in == 0 || *static_cast<volatile uint32_t*>(&s.n_list) > kList) return;
            uint32_t i = atomicAdd(&s.n_list, static_cast<uint32_t>(__popc(in)));
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                if (!(in >> j & 1)) continue;
                if (i < kList) s.list[i] = make_uint2(~key_of(v[j]), at + j);
                ++i;
            }
        };

        // Top-p alone: one pass finds the border's bucket in float32, another
        // sums in float64 what lies before it and lists what lies in it.  The
        // bucket's two ends count as the ends of x that they come to; that the
        // border lies between them is checked with the float64 sums.  False
        // where it does not, or the list overflows.  (The row's maximum, then
        // an exact histogram, then this pass, as where top-p is not alone:
        // 184 against 131 us for 200 rows of 262144 fp32, 114 against 88 for
        // 256 of 152064 bf16; 18 against 22 for one of 32000.)
        //   The histogram holds a bucket's count and its elements' summed
        // places in it: its mass is the count times the weight of the mean
        // place, up to the square of a bucket's width (10^-5).
        auto nucleus = [&]() {
            float near[kChunk];
            row.load(wave * row.span + lane * kChunk, near);
            float from = xrow_max(row_max16(chunk_max(near)));
            if (lane == 0) s.wave_top[wave] = from;
            __syncthreads();
            for (int i = 0; i < kWaves; ++i) from = fmax_nan(from, s.wave_top[i]);
            constexpr int kPlaces = 1 << kNearBits;
            constexpr float kSteps = kNearPerBit * kPlaces;
            constexpr uint32_t kLast = kNear * kPlaces - 1;
            auto* bucket = reinterpret_cast<unsigned long long*>(s.list);
            const float scale = sm.c32 * kSteps;
            float offset;
            for (;;) {
                offset = fmaf(from, scale, kNearRoom * kSteps);
                // No steps finer than float32's, no NaN, and no sum of places
                // that reaches the count.
                if (!(fabsf(offset) < 0x1p23f) || vocab > 1 << (32 - kNearBits)) return false;
                __syncthreads();
                for (int i = threadIdx.x; i < kNear; i += T) bucket[i] = 0;
                __syncthreads();
                top = -INFINITY;
                row.each([&](int, const float (&v)[kChunk]) {
                    top = fmax_nan(top, chunk_max(v));
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) {
                        const uint32_t at = min(whole_part(fmaf(-v[j], scale, offset)), kLast);
                        atomicAdd(&bucket[at >> kNearBits],
                                  (1ull << 32) + (at & (kPlaces - 1)));
                    }
                });
                if (!over_row()) return true;
                if ((top - from) * sm.c32 < kNearRoom - 1) break;
                from = top;  // it exceeds the room: once more
            }
            sm.top = top + 0.0f;
            // Masses in fixed point, as everywhere relative to the maximum; the
            // first bucket begins at `first`.
            constexpr int kOwn = kNear / T;
            const double first = kNearRoom + frac - (static_cast<double>(top) - from) * c;
            unsigned long long m[kOwn], own = 0, mass;
            uint32_t k[kOwn], own_count = 0, total;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                const int b = threadIdx.x * kOwn + i;
                const uint32_t count = static_cast<uint32_t>(bucket[b] >> 32);
                const double place =
                    (static_cast<uint32_t>(bucket[b]) + 0.5 * count) / (kPlaces * max(count, 1u));
                const double w = sm.exp2(first - (b + place) / kNearPerBit);
                m[i] = static_cast<unsigned long long>(count * w);
                own += m[i];
                own_count += k[i] = count;
            }
            uint32_t run_count = block_before<T>(s.wave_count, own_count, total);
            unsigned long long run = block_before<T>(s.wave_mass, own, mass);
            const unsigned long long target = share_of(static_cast<double>(mass));
            // What the sums may be off by: their fractions, a bucket's width.
            const unsigned long long off = (mass >> 13) + kNear;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                if (run < target && run + m[i] >= target) {
                    s.at = threadIdx.x * kOwn + i;
                    s.key_min = target - run <= off;
                    s.key_max = run + m[i] <= target + off;
                    s.at_count = run_count + k[i];
                }
                run += m[i];
                run_count += k[i];
            }
            __syncthreads();
            const uint32_t at = s.at;
            const bool early = s.key_min, late = s.key_max;
            if (at + late >= kNear - 1) return false;
            // A list of all that could be kept, where it is short.
            const bool whole = !late && s.at_count <= kRanked;
            const float high =
                at == 0 || whole ? INFINITY : (offset - (at - early) * kPlaces) / scale;
            const float low = (offset - (at + late + 1) * kPlaces) / scale;
            __syncthreads();
            if (threadIdx.x == 0) s.n_list = 0;
            __syncthreads();
            row.each([&](int first, const float (&v)[kChunk]) {
                uint32_t in = 0;
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    // Without its high word a weight is less than 2^-1042.
                    const Exp2 e = sm.parts(sm.log2_weight(v[j]));
                    all = fma(e.t, e.g, all);
                    kept = fma(__hiloint2double(v[j] > high ? __double2hiint(e.t) : 0,
                                                __double2loint(e.t)),
                               e.g, kept);
                    if (v[j] <= high && v[j] >= low) in |= 1u << j;
                }
                // Added here, or the sums of several chunks wait in registers.
                asm volatile("" : "+v"(all), "+v"(kept));
                append(in, first, v);
            });
            all = over_waves(all);
            const double before = over_waves(kept);
            const uint32_t n = s.n_list;
            if (n > kList) return false;
            share = share_of(all * ldexp(1.0, frac));
            p_above = static_cast<unsigned long long>(rint(before * ldexp(1.0, frac)));
            own = 0;
            for (uint32_t i = threadIdx.x; i < n; i += T)
                own += sm.fixed(sm.weight(value_of(~s.list[i].x)));
            block_before<T>(s.wave_mass, own, mass);
            if (!(p_above < share && p_above + mass >= share)) return false;
            if (whole) return n <= kRanked;
            wide = true;
            if (n > kRanked) {
                bound = p_at = kAnyBucket;
                return true;
            }
            // The border of a short list: the last entry before which less
            // than the share lies, and those kept of its equals.
            if (threadIdx.x < n)
                s.few_mass[threadIdx.x] = sm.fixed(sm.weight(value_of(~s.list[threadIdx.x].x)));
            if (threadIdx.x == 0) s.key_max = s.key_count = 0;
            __syncthreads();
            const uint32_t per = sm.threads_for(n);
            const uint32_t i = threadIdx.x / per, g = threadIdx.x % per;
            const uint2 e = i < n ? s.list[i] : make_uint2(0, 0);
            own = 0;
            for (uint32_t j = g; j < n; j += per) {
                const uint2 o = s.list[j];
                if (o.x < e.x || (o.x == e.x && o.y < e.y)) own += s.few_mass[j];
            }
            const bool keep = p_above + sm.over_group(own, per) < share && i < n && g == 0;
            if (keep) atomicMax(&s.key_max, e.x);
            __syncthreads();
            if (keep && e.x == s.key_max) atomicAdd(&s.key_count, 1u);
            __syncthreads();
            tau = ~s.key_max;
            keep_ties = s.key_count;
            bound = 0;
            return true;
        };
        if (kMode == kTopP && !bad_t && nucleus()) {
            if (!(fabsf(top) < INFINITY)) return;  // no distribution
        } else {
        top = -INFINITY;
        row.each([&](int, const float (&v)[kChunk]) { top = fmax_nan(top, chunk_max(v)); });
        const float thread_top = top;
        if (!over_row()) return;
        sm.top = top + 0.0f;
        // What could be kept lies in buckets up to `bound`.
        bound = kBuckets - 1;
        all = kept = 0.0;
        if (by_k) {
            sm.clear();
            if (top_k <= T / 4) {
                if (thread_top != -INFINITY) atomicAdd(&s.count[sm.bucket(thread_top)], 1u);
            } else {
                row.each([&](int, const float (&v)[kChunk]) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) atomicAdd(&s.count[sm.bucket(v[j])], 1u);
                });
            }
            __syncthreads();
            find<T>(s, false, k_left, 0);
            // Fewer threads than top_k have a logit: no bound from them.
            if (s.above_count + s.at_count >= k_left) bound = s.at;
        } else if (by_p) {
            sm.clear();
            row.each([&](int at, const float (&v)[kChunk]) {
                const bool counted = (at / (64 * kChunk)) % kCountEvery == 0;
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const double y = sm.log2_weight(v[j]);
                    const double w = sm.exp2(y);
                    const uint32_t b = sm.bucket_of(y);
                    all += w;
                    atomicAdd(&s.mass[b], sm.fixed(w));
                    if (counted) atomicAdd(&s.count[b], 1u);
                }
            });
            all = over_waves(all);
            share = share_of(all * ldexp(1.0, frac));
            find<T>(s, true, 0, share);
            bound = p_at = s.at;
            p_above = s.above_mass;
            wide = (s.above_count + s.at_count) * kCountEvery > kList * 3 / 4;
        }
        if (by_m && !(by_k && by_p)) {
            // One bucket on for the rounding of its border's logarithm.
            const double b = 1.0 - log2(min_w) * kPerBit;
            if (b < bound) {
                bound = static_cast<uint32_t>(b);
                wide = false;
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) s.n_list = 0;
        __syncthreads();
        if (wide) {
            // What lies before the border's bucket is kept; the bucket's
            // elements are listed.
            row.each([&](int at, const float (&v)[kChunk]) {
                uint32_t in = 0;
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const double y = sm.log2_weight(v[j]);
                    const uint32_t b = sm.bucket_of(y);
                    if (b < bound) {
                        const double w = sm.exp2(y);
                        if (w >= min_w) kept += w;
                    }
                    if (b == bound && at + j < vocab) in |= 1u << j;
                }
                append(in, at, v);
            });
            __syncthreads();
        } else {
            // Float32 weights relative to 2^offset, offset the rounded log2 of
            // the largest one's: sums of every token's weight serve logp
            // alone.  And logits of the bound's bucket, or a little less.
            const float offset = sm.top * sm.c32;
            const float least =
                bound < kBuckets - 1
                    ? sm.top - static_cast<float>((bound + 1) / (kPerBit * c)) -
                          fabsf(sm.top) * 0x1p-22f
                    : -INFINITY;
            bool summed = !by_k && by_p;
            if (!summed && !(fabsf(offset) < 0x1p20f)) {  // a temperature near 0
                row.each_small([&](int, const float (&v)[kChunk]) {
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) all += sm.weight(v[j]);
                });
                all = over_waves(all);
                summed = true;
            }
            row.each([&](int at, const float (&v)[kChunk]) {
                if (!summed) {
                    float w[kChunk];
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) w[j] = exp2_hw(fmaf(v[j], sm.c32, -offset));
                    all += static_cast<double>(((w[0] + w[1]) + (w[2] + w[3])) +
                                               ((w[4] + w[5]) + (w[6] + w[7])));
                }
                if (chunk_max(v) < least) return;
                uint32_t in = 0;
#pragma unroll
                for (int j = 0; j < kChunk; ++j)
                    if (v[j] >= least && v[j] > -INFINITY) in |= 1u << j;
                append(in, at, v);
            });
            if (!summed)  // what the rounding of the offset left out
                all = over_waves(all) *
                      sm.exp2(static_cast<double>(offset) -
                             static_cast<double>(sm.top) * static_cast<double>(sm.c32));
            else __syncthreads();
        }
        }
        const uint32_t n = s.n_list;
        if (!wide && n <= kRanked) {
            // Every entry against every other, by a group of threads each: the
            // mass before it in falling order decides whether it is kept, the
            // kept mass before it by index whether it is drawn.  In fixed
            // point, since the list's order depends on timing.
            if (threadIdx.x < n) {
                const double w = sm.weight(value_of(~s.list[threadIdx.x].x));
                const unsigned long long f = sm.fixed(w);
                s.mass[threadIdx.x] = f == 0 && w > kNothing ? 1 : f;
            }
            if (threadIdx.x == 0) s.above_mass = 0;
            __syncthreads();
            const uint32_t per = sm.threads_for(n);
            const uint32_t i = threadIdx.x / per, g = threadIdx.x % per;
            const uint2 e = i < n ? s.list[i] : make_uint2(0, 0);
            const unsigned long long w = i < n ? s.mass[i] : 0;
            const bool light = i >= n || sm.weight(value_of(~e.x)) < min_w;
            unsigned long long rank = 0, before = 0;
            for (uint32_t j = g; j < n; j += per) {
                const uint2 o = s.list[j];
                if (o.x < e.x || (o.x == e.x && o.y < e.y)) {
                    ++rank;
                    before += s.mass[j];
                }
            }
            rank = sm.over_group(rank, per);
            before = sm.over_group(before, per);
            if (by_k && by_p) {
                if (i < n && g == 0 && rank < k_left) atomicAdd(&s.above_mass, w);
                __syncthreads();
                share = share_of(static_cast<double>(s.above_mass));
            }
            const bool keep =
                i < n && rank < k_left &&
                (rank == 0 || ((!by_p || before < share) && !light));
            __syncthreads();
            if (i < n && g == 0 && !keep) s.mass[i] = 0;
            __syncthreads();
            unsigned long long mass = 0;
            before = 0;
            for (uint32_t j = g; j < n; j += per) {
                const unsigned long long m = s.mass[j];
                mass += m;
                if (s.list[j].y < e.y) before += m;
            }
            mass = sm.over_group(mass, per);
            before = sm.over_group(before, per);
            const unsigned long long target = target_of(mass);
            // One entry's: the first past the target, or the last for u = 1.
            if (keep && w > 0 && before <= target && (before + w > target || before + w == mass) &&
                g < 2)
                finish(static_cast<int>(e.y), all,
                       static_cast<double>(mass) * ldexp(1.0, -frac));
            return;
        }
        const bool listed = n <= kList;
        while (listed && !wide) {  // once; left where a bucket holds too many
            // Up to kList / T entries a thread.  A border's bucket is found by
            // histogram, its few entries are ranked; the token's likewise,
            // with buckets of the index.
            constexpr int kOwn = kList / T;
            uint2 e[kOwn];
            unsigned long long w[kOwn];
            uint32_t b[kOwn];  // its bucket; kBuckets: not kept
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const uint32_t i = threadIdx.x + j * T;
                e[j] = i < n ? s.list[i] : make_uint2(0, 0);
                const double y = i < n ? sm.log2_weight(value_of(~e[j].x)) : 0.0;
                const double x = sm.exp2(y);
                const unsigned long long f = sm.fixed(x);
                b[j] = i < n ? sm.bucket_of(y) : kBuckets;
                w[j] = i < n ? (f == 0 && x > kNothing ? 1 : f) : 0;
            }
            // The few entries of bucket `at` in s.few, and each one's place.
            uint32_t place[kOwn];
            auto pick = [&](uint32_t at, auto bucket) {
                __syncthreads();
                if (threadIdx.x == 0) s.n_few = 0;
                __syncthreads();
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    place[j] = kRanked;
                    if (b[j] == kBuckets || bucket(j) != at) continue;
                    place[j] = atomicAdd(&s.n_few, 1u);
                    if (place[j] >= kRanked) continue;
                    s.few[place[j]] = e[j];
                    s.few_mass[place[j]] = w[j];
                }
                __syncthreads();
                return s.n_few <= kRanked;
            };
            auto own_bucket = [&](int j) { return b[j]; };
            // Keeps what lies before the border in bucket `at`, of the entries
            // in it `left` by count, or those before which less than `share` lies.
            auto cut = [&](uint32_t at, bool by_mass, uint32_t left,
                           unsigned long long share_left) {
                if (!pick(at, own_bucket)) return false;
                const uint32_t m = s.n_few, per = sm.threads_for(m);
                const uint32_t i = threadIdx.x / per, g = threadIdx.x % per;
                const uint2 o = i < m ? s.few[i] : make_uint2(0, 0);
                unsigned long long rank = 0, before = 0;
                for (uint32_t j = g; j < m; j += per) {
                    const uint2 q = s.few[j];
                    if (q.x < o.x || (q.x == o.x && q.y < o.y)) {
                        ++rank;
                        before += s.few_mass[j];
                    }
                }
                rank = sm.over_group(rank, per);
                before = sm.over_group(before, per);
                if (i < m && g == 0)
                    s.few_kept[i] = by_mass ? before < share_left : rank < left;
                __syncthreads();
#pragma unroll
                for (int j = 0; j < kOwn; ++j)
                    if (b[j] > at || (b[j] == at && !s.few_kept[place[j]])) b[j] = kBuckets;
                return true;
            };
            if (by_k) {
                sm.clear();
#pragma unroll
                for (int j = 0; j < kOwn; ++j)
                    if (b[j] < kBuckets) atomicAdd(&s.count[b[j]], 1u);
                __syncthreads();
                find<T>(s, false, k_left, 0);
                const uint32_t at = s.at, left = k_left - s.above_count;
                if (!cut(at, false, left, 0)) break;
            }
            if (by_p && by_k) {
                __syncthreads();
                sm.clear();
                unsigned long long own = 0, total;
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    if (b[j] == kBuckets) continue;
                    atomicAdd(&s.mass[b[j]], w[j]);
                    own += w[j];
                }
                block_before<T>(s.wave_mass, own, total);
                const unsigned long long part = share_of(static_cast<double>(total));
                find<T>(s, true, 0, part);
                const uint32_t at = s.at;
                const unsigned long long left = part - s.above_mass;
                if (!cut(at, true, 0, left)) break;
            } else if (by_p && bound == p_at) {
                if (!cut(p_at, true, 0, share - p_above)) break;
            }
            // By index.
            const int shift = max(0, 32 - __clz(vocab - 1) - kBucketBits);
            __syncthreads();
            sm.clear();
            unsigned long long own = 0, mass;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                if (by_m && b[j] < kBuckets && sm.weight(value_of(~e[j].x)) < min_w)
                    b[j] = kBuckets;
                if (b[j] == kBuckets) continue;
                atomicAdd(&s.mass[e[j].y >> shift], w[j]);
                own += w[j];
            }
            block_before<T>(s.wave_mass, own, mass);
            const unsigned long long target = target_of(mass);
            find<T>(s, true, 0, target + 1);
            const uint32_t at = s.at;
            const unsigned long long above = s.above_mass;
            if (!pick(at, [&](int j) { return e[j].y >> shift; })) break;
            const uint32_t m = s.n_few, per = sm.threads_for(m);
            const uint32_t i = threadIdx.x / per, g = threadIdx.x % per;
            const uint2 o = i < m ? s.few[i] : make_uint2(0, 0);
            const unsigned long long mine = i < m ? s.few_mass[i] : 0;
            unsigned long long before = 0;
            for (uint32_t j = g; j < m; j += per)
                if (s.few[j].y < o.y) before += s.few_mass[j];
            before = above + sm.over_group(before, per);
            const unsigned long long to = before + mine;
            if (mine > 0 && g < 2 && before <= target && (to > target || to == mass))
                finish(static_cast<int>(o.y), all,
                       static_cast<double>(mass) * ldexp(1.0, -frac));
            return;
        }
        if (by_k) {
            sm.clear();
            sm.candidates(listed, [&](uint32_t k) {
                atomicAdd(&s.count[sm.bucket(value_of(k))], 1u);
            });
            __syncthreads();
            find<T>(s, false, k_left, 0);
            const uint32_t b = s.at, above = s.above_count;
            const Border k = sm.resolve(listed, b, 0, above, 0, false, k_left, 0);
            tau = k.tau;
            // A list may end before top_k: what is not in it has no weight.
            keep_ties = min(k_left - k.above, k.ties);
        }
        // Where min-p's bound lies before top-p's border, that keeps all.
        if (by_p && (by_k || bound == p_at)) {
            const uint32_t floor = tau, most_ties = keep_ties;
            if (by_k) {
                // The masses of K.
                sm.clear();
                double part = 0.0;
                sm.candidates(listed, [&](uint32_t k) {
                    if (k <= tau) return;
                    const double w = sm.weight(value_of(k));
                    part += w;
                    atomicAdd(&s.mass[sm.bucket(value_of(k))], sm.fixed(w));
                });
                if (threadIdx.x == 0) {
                    const double w = sm.weight(value_of(tau));
                    part += keep_ties * w;
                    atomicAdd(&s.mass[sm.bucket(value_of(tau))], keep_ties * sm.fixed(w));
                }
                share = share_of(over_waves(part) * ldexp(1.0, frac));
                find<T>(s, true, 0, share);
                p_at = s.at;
                p_above = s.above_mass;
            }
            const Border q = sm.resolve(listed, p_at, floor, 0, p_above, true, 0, share);
            tau = q.tau;
            const double one = static_cast<double>(sm.fixed(sm.weight(value_of(tau))));
            const double left = static_cast<double>(share - q.above_mass);
            const double need = one > 0.0 ? ceil(left / one) : 1.0;
            uint32_t limit = q.ties;
            if (by_k && tau == floor) limit = min(limit, most_ties);
            keep_ties = need < 1.0 ? 1u : need < limit ? static_cast<uint32_t>(need) : limit;
        }
        uint32_t ties = 0;
        if (listed) {
            // The list's kept weights by part of the row, in fixed point.
            __syncthreads();
            sm.clear();
            for (uint32_t i = threadIdx.x; i < n; i += T) {
                const uint32_t k = ~s.list[i].x;
                if (k < tau) continue;
                const int part = static_cast<int>(s.list[i].y) / row.span;
                if (k == tau) {
                    atomicAdd(&s.count[part], 1u);
                } else {
                    const double w = sm.weight(value_of(k));
                    if (w >= min_w) atomicAdd(&s.mass[part], sm.fixed(w));
                }
            }
            __syncthreads();
            if (lane == 0) {
                kept += static_cast<double>(s.mass[wave]) * ldexp(1.0, -frac);
                ties = s.count[wave];
            }
        } else {
            kept = 0.0;
            row.each_small([&](int, const float (&v)[kChunk]) {
#pragma unroll
                for (int j = 0; j < kChunk; ++j) {
                    const uint32_t k = key_of(v[j]);
                    if (k < tau) continue;
                    if (k == tau) {
                        ++ties;
                    } else {
                        const double w = sm.weight(v[j]);
                        if (w >= min_w) kept += w;
                    }
                }
            });
        }
        sm.set_parts(kept, ties);
        double mass;
        const int token = sm.search(u, tau, keep_ties, min_w, mass);
        if (token >= 0 && lane < 2) finish(token, all, mass);
    }
}

}  // namespace

namespace {

template <int DT, int T>
hipError_t launch_sample_threads(const SampleParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.n_rows)), block(T);
    const bool k = p.top_ks != nullptr || (p.top_k > 0 && p.top_k < p.vocab);
    const bool m = p.min_ps != nullptr || p.min_p > 0.0f;
    const bool greedy = p.temperatures == nullptr && p.temperature == 0.0f;
    const bool by_p = p.top_ps != nullptr || p.top_p < 1.0f;
    if (by_p && !k && !m && !greedy)
        return launch_kernel(klp_sample_kernel<DT, T, kTopP>, grid, block, stream, p);
    if (by_p || k || m || greedy || p.temperatures != nullptr)
        return launch_kernel(klp_sample_kernel<DT, T, kAny>, grid, block, stream, p);
    return launch_kernel(klp_sample_kernel<DT, T, kPlain>, grid, block, stream, p);
}

// A row's passes are short of arithmetic while its workgroup is alone on a CU,
// so 1024 threads; with more rows than CUs two workgroups share one, and 512
// leave fewer idle at a row's barriers.  (us, 1024 and 512 threads: 256 rows
// of 152064 unfiltered 28 and 31, 200 of 262144 fp32 with top-p 131 and 143;
// 300 rows of 32000 unfiltered 18 and 15, 1024 of 128256 fp16 with top-p 283
// and 212.)
template <int DT>
hipError_t launch_sample_dt(const SampleParams& p, hipStream_t stream) {
    if (p.n_rows > kHeadGemmCus) return launch_sample_threads<DT, 512>(p, stream);
    return launch_sample_threads<DT, 1024>(p, stream);
}

}  // namespace

hipError_t launch_sample(int dtype, const SampleParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_sample_dt<kBF16>(p, stream);
        case kFP16: return launch_sample_dt<kFP16>(p, stream);
        case kFP32: return launch_sample_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
