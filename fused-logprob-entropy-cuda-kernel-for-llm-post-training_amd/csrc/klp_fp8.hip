// klp_fp8.hip — e4m3 quantization with a scale per block, for gfx950.
//
//   a = max |x| of a block, scale = a / 448, q = e4m3(x (448 / a))
//
// Blocks are 128 elements of a row (activations: 16 lanes a block, one pass)
// or 128 x 128 elements (weights: a workgroup a block, held in registers
// between its maximum and its codes).  Bound by memory: every element is read
// once and its code written once.  Measured: 152064 x 3584 bf16 in 128 x 128
// blocks 293 us (5.6 TB/s), 4096 x 3584 fp16 in rows 9.2 us (4.8 TB/s); a copy
// runs at 5.9.
#include "klp_launch.h"
#include "klp_rows.h"

namespace klp {

namespace {

constexpr int kQuantThreads = 256;
constexpr int kLanes = kScaleBlock / kChunk;               // 16 lanes a block's row
constexpr int kRowsAtOnce = kQuantThreads / kLanes;        // 16
constexpr int kTileRows = kScaleBlock / kRowsAtOnce;       // 8 rows a lane of a 128 x 128 block

// One 128-element block per 16 lanes.
template <int DT>
__global__ __launch_bounds__(kQuantThreads) void klp_quantize_rows_kernel(QuantizeParams p,
                                                                          uint32_t n_items) {
    typedef typename Traits<DT>::elem elem;
    const uint32_t item = blockIdx.x * kRowsAtOnce + threadIdx.x / kLanes;
    if (item >= n_items) return;
    const uint32_t nb = static_cast<uint32_t>(p.n_blocks);
    const uint32_t row = item / nb;
    const uint32_t b = item - row * nb;
    const int64_t c = static_cast<int64_t>(b) * kScaleBlock + (threadIdx.x % kLanes) * kChunk;
    float x[kChunk];
    load_chunk<DT>(static_cast<const elem*>(p.x) + row * p.ld_x + c, p.dim - c, x);
    const E4m3Scale e = e4m3_scale(row_max16(chunk_amax(x)));
    store_codes(p.q + row * p.dim + c, p.dim - c, e4m3_pack8(x, e.inv));
    if (threadIdx.x % kLanes == 0) p.scales[item] = e.scale;
}

// One 128 x 128 block per workgroup.
template <int DT>
__global__ __launch_bounds__(kQuantThreads) void klp_quantize_tile_kernel(QuantizeParams p) {
    typedef typename Traits<DT>::elem elem;
    __shared__ float part[kQuantThreads / 64];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kScaleBlock +
                      (threadIdx.x % kLanes) * kChunk;
    const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kScaleBlock + threadIdx.x / kLanes;
    float x[kTileRows][kChunk];
#pragma unroll
    for (int i = 0; i < kTileRows; ++i) {
        const int64_t row = row0 + i * kRowsAtOnce;
        load_chunk<DT>(static_cast<const elem*>(p.x) + row * p.ld_x + c,
                       row < p.rows ? p.dim - c : 0, x[i]);
    }
    float a = chunk_amax(x[0]);
#pragma unroll
    for (int i = 1; i < kTileRows; ++i) a = fmax_nan(a, chunk_amax(x[i]));
    a = xrow_max(row_max16(a));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int i = 1; i < kQuantThreads / 64; ++i) a = fmax_nan(a, part[i]);
    const E4m3Scale e = e4m3_scale(a);
#pragma unroll
    for (int i = 0; i < kTileRows; ++i) {
        const int64_t row = row0 + i * kRowsAtOnce;
        if (row < p.rows) store_codes(p.q + row * p.dim + c, p.dim - c, e4m3_pack8(x[i], e.inv));
    }
    if (threadIdx.x == 0) p.scales[blockIdx.y * p.n_blocks + blockIdx.x] = e.scale;
}

template <int DT>
hipError_t launch_quantize_dt(const QuantizeParams& p, hipStream_t stream) {
    if (p.block_rows == 1) {
        const int64_t n = p.rows * p.n_blocks;  // below 2^31 (klp_quantize_fp8)
        const dim3 grid(static_cast<unsigned>((n + kRowsAtOnce - 1) / kRowsAtOnce));
        return launch_kernel(klp_quantize_rows_kernel<DT>, grid, dim3(kQuantThreads), stream, p,
                             static_cast<uint32_t>(n));
    }
    const dim3 grid(static_cast<unsigned>(p.n_blocks),
                    static_cast<unsigned>((p.rows + kScaleBlock - 1) / kScaleBlock));
    return launch_kernel(klp_quantize_tile_kernel<DT>, grid, dim3(kQuantThreads), stream, p);
}

}  // namespace

hipError_t launch_quantize(int dtype, const QuantizeParams& p, hipStream_t stream) {
    switch (dtype) {
        case kBF16: return launch_quantize_dt<kBF16>(p, stream);
        case kFP16: return launch_quantize_dt<kFP16>(p, stream);
        case kFP32: return launch_quantize_dt<kFP32>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace klp
