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
#include "klp_mfma.h"
#include "klp_rows.h"

namespace klp {

namespace {

using mfma::f32x4;
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kK = kScaleBlock;
// The longest row stride whose 256 rows 32-bit byte offsets reach.
constexpr int64_t kFp8TileMaxStride = INT32_MAX / 256;

// A scale block's products and sums, in one of two ways.
//
// The e4m3 instruction aligns the products of 8 consecutive k to the largest
// of their exponents and drops what lies more than 13 bits below it, before
// its float32 sums (measured with two and with 128 products of chosen
// exponents): off by up to 7 2^-13 of a group's largest product, 1.5 to 5
// 10^-5 of a result (2-norm) on normal data.  A 16-bit output's own rounding
// is 10 to 100 times that; a float32 output's is 1000 times less.  kExact
// converts the codes to bf16 (exactly) and takes four bf16 instructions, whose
// products are exact and whose sums are float32: half the peak rate.
template <bool kExact> struct Operand;
template <> struct Operand<false> {
    i32x8 v;
    __device__ __forceinline__ static Operand from(i32x8 x) { return Operand{x}; }
};
template <> struct Operand<true> {
    bf16x8 v[4];
    __device__ __forceinline__ static Operand from(i32x8 x) {
        Operand o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t w = static_cast<uint32_t>(x[i]);
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
            const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
            const int at = 4 * (i & 1);
            o.v[i >> 1][at] = lo[0];
            o.v[i >> 1][at + 1] = lo[1];
            o.v[i >> 1][at + 2] = hi[0];
            o.v[i >> 1][at + 3] = hi[1];
        }
        return o;
    }
};
__device__ __forceinline__ f32x4 mul_block(const Operand<false>& a, const Operand<false>& b) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    // Constant block scales of 0 select the instruction without any.
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mul_block(const Operand<true>& a, const Operand<true>& b) {
    f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
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

// Small products: a workgroup's waves share the K of 16 weight rows and 16 MB
// tokens, both straight from memory to registers (the tokens' rows stay in the
// caches); their sums meet in LDS and are added in order.
constexpr int kSplit = 4;
template <int DT, int MB, bool kExact>
__global__ __launch_bounds__(64 * kSplit) void klp_fp8_stream_kernel(Fp8LinearParams p) {
    __shared__ f32x4 part[(kSplit - 1) * MB * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * 16;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * 16 * MB;
    const int lrow = lane & 15, lq = lane >> 4;

    // Rows past the end repeat the last one; their outputs are not stored.
    const int64_t wrow = v0 + lrow < p.n ? v0 + lrow : p.n - 1;
    const uint8_t* w = p.w + wrow * p.ld_w + 16 * lq;
    const uint8_t* x[MB];
    const float* xs[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t r = t0 + 16 * j + lrow;
        const int64_t m = r < p.m ? r : p.m - 1;
        x[j] = p.x + m * p.ld_x + 16 * lq;
        xs[j] = p.xs + m * p.n_blocks;
    }
    const float* ws = p.ws + v0 / kScaleBlock * p.n_blocks;

    const int nb = static_cast<int>(p.n_blocks);
    const int first = static_cast<int>(static_cast<int64_t>(nb) * wave / kSplit);
    const int end = static_cast<int>(static_cast<int64_t>(nb) * (wave + 1) / kSplit);
    f32x4 acc[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto fold = [&](i32x8 a, const i32x8 (&b)[MB], const float (&s)[MB], float g) {
        const Operand<kExact> row = Operand<kExact>::from(a);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const f32x4 c = mul_block(row, Operand<kExact>::from(b[j]));
            const float f = s[j] * g;
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(c[r], f, acc[j][r]);
        }
    };
    auto load = [&](int b, i32x8& a, i32x8 (&c)[MB], float (&s)[MB], float& g) {
        const int64_t k0 = static_cast<int64_t>(b) * kK;
        a = load_operand(w, k0);
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
    i32x8 a[2], c[2][MB];
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
        a[0] = load_operand_tail(w, k0, left);
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            c[0][j] = load_operand_tail(x[j], k0, left);
            s[0][j] = xs[j][whole];
        }
        fold(a[0], c[0], s[0], ws[whole]);
    }

    if (wave > 0) {
#pragma unroll
        for (int j = 0; j < MB; ++j) part[((wave - 1) * MB + j) * 64 + lane] = acc[j];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int z = 0; z < kSplit - 1; ++z)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[j] += part[(z * MB + j) * 64 + lane];

    typedef typename Traits<DT>::elem elem;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t m = t0 + 16 * j + lrow;
        const int64_t n = v0 + 4 * lq;
        if (m < p.m) store4<DT>(static_cast<elem*>(p.out) + m * p.ld_out + n, p.n - n, acc[j]);
    }
}

// Many tokens: a workgroup of 8 waves computes 256 outputs of a token for
// 16 MB * kTokenWaves tokens.  Both operands go through LDS, two stages of one
// scale block each: 128-byte rows, their 16-byte chunks swizzled (swz), and
// the tokens' scales of the block behind them.  A wave reads 16 VB weight rows
// and 16 MB token rows a stage.
//
// A stage's token rows are held in registers, its weight rows read as they are
// needed.  Twice a stage the workgroup meets, each time before the last row of
// blocks of a half: every wave has then read that half's weight rows (and, at
// the first meeting, the token rows, long since).  Behind the first meeting
// go the copies of the first half's weight rows and the token rows of the
// stage after the next, into the slots just read; behind the second those of
// the second half's weight rows.  The meetings wait for the copies that the
// next half reads, which were started one and a half stages before.
//
// LDS is the bound that can be counted: a stage of a 256 x 256 tile reads 192
// KB (128 bytes a clock) and receives 64 KB (64 a clock), 2560 clocks against
// 2048 of matrix instructions, beside which the four FMAs of a scale run for
// nothing (4780 TFLOP/s for a loop of one and four).  4096 tokens of a [152064,
// 3584] head: 2150 us, 2.08 PFLOP/s, 58 us a tile of which that makes 39 at
// 1.83 GHz; matrix units 56% busy, 80% if it were all.  The rest is not
// accounted for: one workgroup fills a CU's LDS, so nothing runs under a tile's
// first copies and its stores (without stores 2016 us, without copies 1717).
// 16 tokens: 100 us, the weight read at 5.5 TB/s.  float32 outputs: 4336 us,
// and 110 for 16 tokens.
template <int VB_, int MB_, int kTokenWaves_>
struct TileShape {
    static constexpr int VB = VB_, MB = MB_, kTokenWaves = kTokenWaves_;
    static constexpr int kVocabWaves = 8 / kTokenWaves;
    static constexpr int kRowsV = 16 * VB * kVocabWaves;
    static constexpr int kRowsM = 16 * MB * kTokenWaves;
    static constexpr int kSlotV = kRowsV * kK;
    static constexpr int kSlotM = kRowsM * kK;
    static constexpr int kSlotS = kRowsM * 4;
    static constexpr int kLds = 2 * (kSlotV + kSlotM + kSlotS);
    // Registers for two workgroups a CU (float32 outputs' operands need more).
    static constexpr bool kSmall = VB * MB <= 8;
    static constexpr int kHalfV = kRowsV / 128;  // copies of 1 KB, a wave
    static constexpr int kCopiesM = kRowsM / 64;
    static constexpr int kFirst = kHalfV + kCopiesM + 1;
    static constexpr int kSecond = kHalfV;
};
constexpr int kTileThreads = 512;

// 64 lanes' dwords to LDS byte offset `lds` + 4 lane; as mfma::copy_to_lds.
__device__ __forceinline__ void copy_dwords_to_lds(u32x4 rsrc, uint32_t lds, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc), "s"(0u)
                 : "memory");
}

template <int DT, typename Shape>
__global__
__launch_bounds__(kTileThreads, Shape::kSmall && DT != kFP32 ? 4 : 2) void klp_fp8_tile_kernel(
    Fp8LinearParams p) {
    using namespace mfma;
    constexpr int VB = Shape::VB, MB = Shape::MB;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[Shape::kLds];
    constexpr int kAt_m = 2 * Shape::kSlotV;
    constexpr int kAt_s = kAt_m + 2 * Shape::kSlotM;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wv = wave % Shape::kVocabWaves, wm = wave / Shape::kVocabWaves;

    // Workgroup b runs on XCD b % 8; each XCD takes one contiguous range of
    // tiles: groups of 8 weight tiles, in each the weight tiles fastest, then
    // the token tiles, so that its 32 workgroups share 8 and 4 of them.
    const uint32_t per_xcd = gridDim.x / 8;
    const uint32_t item = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    const uint32_t v_tiles = static_cast<uint32_t>((p.n + Shape::kRowsV - 1) / Shape::kRowsV);
    const uint32_t m_tiles = static_cast<uint32_t>((p.m + Shape::kRowsM - 1) / Shape::kRowsM);
    if (item >= v_tiles * m_tiles) return;
    constexpr uint32_t kGroup = 8;
    const uint32_t group = item / (kGroup * m_tiles);
    const uint32_t in = item - group * (kGroup * m_tiles);
    const uint32_t width = v_tiles - group * kGroup < kGroup ? v_tiles - group * kGroup : kGroup;
    const uint32_t m_tile = in / width;
    const int64_t v0 = static_cast<int64_t>(group * kGroup + in - m_tile * width) * Shape::kRowsV;
    const int64_t t0 = static_cast<int64_t>(m_tile) * Shape::kRowsM;
    const int rows_v = static_cast<int>(p.n - v0 < Shape::kRowsV ? p.n - v0 : Shape::kRowsV);
    const int rows_m = static_cast<int>(p.m - t0 < Shape::kRowsM ? p.m - t0 : Shape::kRowsM);
    const int nb = static_cast<int>(p.n_blocks);

    // A copy fills 8 slot rows: lane l chunk l % 8 of row l / 8, which holds
    // the row's chunk (l % 8) ^ swz(row).  Token rows: copy j of wave w rows
    // 64 j + 8 w.  Weight rows: a half is 8 VB rows of each of the 16 VB that
    // a vocabulary wave reads, copy j of wave w takes rows 128 j + wrow of it.
    constexpr uint32_t kNowhere = 0x80000000u;  // past every descriptor
    const int crow = wave * 8 + (lane >> 3);
    const int cchunk = (lane & 7) ^ swz(crow);
    const int wrow = wave / VB * (16 * VB) + wave % VB * 8;
    static_assert(VB == 4 || VB == 8, "8 waves fill 128 rows' half");
    const uint32_t ld_v = static_cast<uint32_t>(p.ld_w), ld_m = static_cast<uint32_t>(p.ld_x);
    constexpr int kScaleWaves = Shape::kRowsM / 64;  // the others copy the same again
    const uint32_t stok = static_cast<uint32_t>((wave % kScaleWaves) * 64 + lane);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)lds));

    // Copies of block b into slot b % 2.  Chunks past K, and all of a block
    // past the last, come from past the descriptors: zeros, and the count of
    // copies in flight stays the same.
    const uint32_t k = static_cast<uint32_t>(p.k);
    const u32x4 rs_v = bytes_rsrc(p.w + v0 * p.ld_w, (rows_v - 1) * ld_v + k);
    const u32x4 rs_m = bytes_rsrc(p.x + t0 * p.ld_x, (rows_m - 1) * ld_m + k);
    const u32x4 rs_s = bytes_rsrc(p.xs + t0 * p.n_blocks, static_cast<uint32_t>(rows_m) * nb * 4);
    const uint32_t lane_v = static_cast<uint32_t>(wrow + (lane >> 3)) * ld_v + cchunk * 16;
    const uint32_t lane_m = static_cast<uint32_t>(crow) * ld_m + cchunk * 16;
    const uint32_t lane_s = stok * static_cast<uint32_t>(nb) * 4;
    // Blocks with this chunk.
    const int chunks = static_cast<int>((p.k - cchunk * 16 + kK - 1) / kK);
    int block[2] = {0, 0};  // the first and second copies' next
    auto copy_v = [&](int half, int j) {
        const int b = block[half];
        copy_to_lds(rs_v, lds0 + (b & 1) * Shape::kSlotV + (wrow + 128 * j + 8 * VB * half) * kK,
                    b < chunks ? lane_v + (128 * j + 8 * VB * half) * ld_v + b * kK : kNowhere, 0);
    };
    auto copy_first = [&](int z) {
        const int b = block[0];
        if (z < Shape::kHalfV) {
            copy_v(0, z);
        } else if (z < Shape::kHalfV + Shape::kCopiesM) {
            const int j = z - Shape::kHalfV;
            copy_to_lds(rs_m, lds0 + kAt_m + (b & 1) * Shape::kSlotM + (wave + 8 * j) * 1024,
                        b < chunks ? lane_m + j * 64 * ld_m + b * kK : kNowhere, 0);
        } else {
            copy_dwords_to_lds(rs_s, lds0 + kAt_s + (b & 1) * Shape::kSlotS +
                                         (wave % kScaleWaves) * 256,
                               b < nb ? lane_s + b * 4 : kNowhere);
            ++block[0];
        }
    };
    auto copy_second = [&](int z) {
        copy_v(1, z);
        if (z == Shape::kSecond - 1) ++block[1];
    };

    // Operands: lane l holds row l % 16 of a block, chunks l / 16 and 4 + l / 16.
    const int lrow = lane & 15, lq = lane >> 4;
    const int lchunk = (lq ^ swz(lrow)) * 16;
    const int base_v = wv * (16 * VB) * kK + lrow * kK;
    const int base_m = kAt_m + wm * (16 * MB) * kK + lrow * kK;
    auto read = [&](int at) {
        union {
            u32x4 h[2];
            i32x8 v;
        } u;
        u.h[0] = *reinterpret_cast<const u32x4*>(lds + at + lchunk);
        u.h[1] = *reinterpret_cast<const u32x4*>(lds + at + (lchunk ^ 64));
        return Operand<DT == kFP32>::from(u.v);
    };
    auto read_v = [&](int slot, int i) {
        return read(slot * Shape::kSlotV + base_v + i * 16 * kK);
    };
    auto read_m = [&](int slot, int j) {
        return read(slot * Shape::kSlotM + base_m + j * 16 * kK);
    };
    auto read_s = [&](int slot, int j) {
        return *reinterpret_cast<const float*>(lds + kAt_s + slot * Shape::kSlotS +
                                               (wm * 16 * MB + 16 * j + lrow) * 4);
    };
    int64_t first_row = v0 + wv * (16 * VB);
    if (first_row >= p.n) first_row = 0;  // a wave past the weight: its outputs are not stored
    // Constant memory: a scalar load.  A vector load's wait would also wait for
    // the copies before it.
    typedef __attribute__((address_space(4))) const float const_float;
    const const_float* ws =
        (const const_float*)(uintptr_t)(p.ws + first_row / kScaleBlock * p.n_blocks);

    f32x4 acc[VB][MB];
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int z = 0; z < Shape::kFirst; ++z) copy_first(z);
#pragma unroll
        for (int z = 0; z < Shape::kSecond; ++z) copy_second(z);
    }
    constexpr int kStage = Shape::kFirst + Shape::kSecond;
    auto meet = [&](auto in_flight) {
        pin();
        __builtin_amdgcn_s_waitcnt(waitcnt(decltype(in_flight)::value, 0));
        __builtin_amdgcn_s_barrier();
        pin();
    };
    meet(std::integral_constant<int, kStage + Shape::kSecond>{});

    typedef Operand<DT == kFP32> Op;
    Op av[2], bv[MB];
    float f[MB];
    av[0] = read_v(0, 0);
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        bv[j] = read_m(0, j);
        f[j] = read_s(0, j);
    }
    float g = ws[0];
    // The sums of a matrix instruction are scaled and added kLag instructions
    // later: 2 (4 + 1) + 1 instructions lie between, the 11 wait states of an
    // 8-pass instruction's result.
    constexpr int kLag = 3;
    constexpr int kSteps = VB * MB, kMeet = kSteps - MB, kMid = kSteps / 2 - MB;
    static_assert(Shape::kSecond <= MB, "before the next meeting");
    constexpr bool kFits = kMid + Shape::kFirst <= kMeet;  // a copy an instruction
    f32x4 c[kLag + 1];
    int slot = 0;
    for (int b = 0; b < nb; ++b) {
        const float g_next = ws[b + 1 < nb ? b + 1 : b];
#pragma unroll
        for (int j = 0; j < MB; ++j) f[j] *= g;
        g = g_next;
        float f_next[MB];
        auto fold = [&](int q) {
            const int i = q / MB, j = q % MB;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[i][j][r] = fmaf(c[q % (kLag + 1)][r], f[j], acc[i][j][r]);
        };
#pragma unroll
        for (int q = 0; q < kSteps; ++q) {
            const int i = q / MB, j = q % MB;
            if (q == kMid || q == kMeet) meet(std::integral_constant<int, kStage>{});
            if (q == kMeet) slot ^= 1;
            c[q % (kLag + 1)] = mul_block(av[i & 1], bv[j]);
            pin();
            if (j == 0) av[(i + 1) & 1] = read_v(slot, (i + 1) % VB);
            if (i == VB - 1) {
                bv[j] = read_m(slot, j);
                f_next[j] = read_s(slot, j);
            }
#pragma unroll
            for (int z = 0; z < Shape::kFirst; ++z)
                if (q == kMid + (kFits ? z : z * (kMeet - kMid) / Shape::kFirst)) copy_first(z);
            if (q >= kMeet && q - kMeet < Shape::kSecond) copy_second(q - kMeet);
            if (q >= kLag) fold(q - kLag);
            pin();
        }
#pragma unroll
        for (int z = kSteps - kLag; z < kSteps; ++z) fold(z);
#pragma unroll
        for (int j = 0; j < MB; ++j) f[j] = f_next[j];
    }
    // The last copies write zeros to LDS: before the workgroup gives it up.
    __builtin_amdgcn_s_waitcnt(waitcnt(0, 15));

    typedef typename Traits<DT>::elem elem;
    const int64_t n0 = v0 + wv * (16 * VB);
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t m = t0 + wm * (16 * MB) + 16 * j + lrow;
        elem* out = static_cast<elem*>(p.out) + m * p.ld_out;
#pragma unroll
        for (int i = 0; i < VB; ++i) {
            const int64_t n = n0 + 16 * i + 4 * lq;
            if (m < p.m) store4<DT>(out + n, p.n - n, acc[i][j]);
        }
    }
}

template <int DT, typename Shape>
hipError_t launch_tile(const Fp8LinearParams& p, hipStream_t stream) {
    const int64_t tiles = ((p.n + Shape::kRowsV - 1) / Shape::kRowsV) *
                          ((p.m + Shape::kRowsM - 1) / Shape::kRowsM);
    const dim3 grid(static_cast<unsigned>((tiles + 7) / 8 * 8));
    return launch_kernel(klp_fp8_tile_kernel<DT, Shape>, grid, dim3(kTileThreads), stream, p);
}

template <int DT, int MB>
hipError_t launch_stream(const Fp8LinearParams& p, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>((p.n + 15) / 16),
                    static_cast<unsigned>((p.m + 16 * MB - 1) / (16 * MB)));
    return launch_kernel(klp_fp8_stream_kernel<DT, MB, DT == kFP32>, grid, dim3(256), stream, p);
}

template <typename Shape>
int64_t tiles_of(const Fp8LinearParams& p) {
    return ((p.n + Shape::kRowsV - 1) / Shape::kRowsV) *
           ((p.m + Shape::kRowsM - 1) / Shape::kRowsM);
}
// Rounds of one tile a CU, times a round's time.
template <typename Shape>
int64_t cost_of(const Fp8LinearParams& p, int round) {
    return (tiles_of<Shape>(p) + kHeadGemmCus - 1) / kHeadGemmCus * round;
}

// Tiles of 256 x 256, 256 x 128, 128 x 128 and 128 x 64 (weight rows x
// tokens) take 64, 39, 25 and 18 us a round at k = 4096: the wider a tile, the
// fewer bytes it moves through LDS for its products, the narrower, the more
// CUs a small product fills.  (us, bf16 out:)
//   m     n       k       256x256  256x128  128x128  128x64  split
//   16    152064  3584    128      108      104      100     137
//   64    152064  3584    143      124      124      122     322
//   128   152064  3584    171      148      164      193     633
//   256   152064  3584    197      218      260              1250
//   512   152064  3584    319      403      452              2493
//   64    32000   4096    44       28       23       23      90
//   256   32000   4096    56       40       51       68      351
//   1024  32000   4096    133      149      192              1362
//   512   4096    4096    50       33       25       21      90
//   1024  4096    4096    51       33       27       35      177
//   2048  4096    4096    52       40       49       67      351
//   64    4096    4096    42       27       20       18      14.6
//   16    8192    8192             47       34       32      19
//   512   512     4096    47       29       20       18      14
// With at most 4 blocks of 16 x 16 outputs a CU, splitting their K over a
// workgroup's waves is faster than any tile.
template <int DT>
hipError_t launch_fp8_linear_dt(const Fp8LinearParams& p, hipStream_t stream) {
    // 32-bit offsets within a tile's rows.
    const bool near = p.ld_x <= kFp8TileMaxStride && p.ld_w <= kFp8TileMaxStride;
    if (!near || ((p.n + 15) / 16) * ((p.m + 15) / 16) <= 4 * kHeadGemmCus) {
        if (p.m <= 16) return launch_stream<DT, 1>(p, stream);
        if (p.m <= 32) return launch_stream<DT, 2>(p, stream);
        return launch_stream<DT, 4>(p, stream);
    }
    typedef TileShape<8, 4, 4> Wide;
    typedef TileShape<4, 4, 2> Half;
    typedef TileShape<4, 2, 4> Square;
    typedef TileShape<4, 1, 4> Narrow;
    const int64_t half = cost_of<Half>(p, 39), square = cost_of<Square>(p, 25),
                  narrow = cost_of<Narrow>(p, 18);
    // The exact operands of a 256 x 256 tile do not fit the registers.
    if constexpr (DT != kFP32) {
        const int64_t wide = cost_of<Wide>(p, 64);
        if (wide <= half && wide <= square && wide <= narrow)
            return launch_tile<DT, Wide>(p, stream);
    }
    if (half <= square && half <= narrow) return launch_tile<DT, Half>(p, stream);
    if (square <= narrow) return launch_tile<DT, Square>(p, stream);
    return launch_tile<DT, Narrow>(p, stream);
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
