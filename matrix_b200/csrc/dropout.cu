// Dropout from a counter-based generator for sm_100a: dst = keep ? src * 65536 / kept : 0, the mask made
// again wherever it is needed and never stored.
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;

// A thread takes the eight columns of one counter.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(T* dst, const T* src, uint64_t blocks_per_row, uint64_t items, uint32_t width, uint64_t ds,
                   uint64_t ss, const DropArgs d) {
    const Philox rng(d);
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < items; i += (uint64_t)gridDim.x * kThreads) {
        const uint64_t row = i / blocks_per_row;
        const uint32_t block = (uint32_t)(i - row * blocks_per_row);
        const uint4 w = rng(block, (uint32_t)row);
        const T* x = src + row * ss;
        T* y = dst + row * ds;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t c = block * 8 + j;
            if (c < width) y[c] = from_float<T>(Philox::lane(w, j) < d.kept ? to_float(x[c]) * d.scale : 0.0f);
        }
    }
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_dropout(int dtype, void* dst, const void* src, uint64_t rows, uint64_t width,
                            uint64_t dst_row_stride, uint64_t src_row_stride, const mtxc_dropout_state* drop) {
    if (int rc = require_init()) return rc;
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, std::string("mtxc_dropout: no kernel for dtype ") + dtype_name(dtype));
    if (!drop) return fail(MTXC_ERR_INVALID_ARGUMENT, "mtxc_dropout: null dropout state");
    DropArgs d;
    if (int rc = drop_args(*drop, "mtxc_dropout", &d)) return rc;
    if (rows >> 31 || width >> 31) return fail(MTXC_ERR_SHAPE, "mtxc_dropout: rows and width must be below 2^31");
    if (rows == 0 || width == 0) return MTXC_OK;
    if (!dst || !src) return fail(MTXC_ERR_INVALID_ARGUMENT, "mtxc_dropout: null buffer");
    const uint64_t blocks = (width + 7) / 8, items = rows * blocks;
    const unsigned grid = (unsigned)std::min<uint64_t>((items + kThreads - 1) / kThreads, (uint64_t)ctx().sm_count * 8);
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        dropout_kernel<T><<<grid, kThreads, 0, ctx().stream()>>>(static_cast<T*>(dst), static_cast<const T*>(src), blocks,
                                                                 items, (uint32_t)width, dst_row_stride,
                                                                 src_row_stride, d);
    });
    return check_launch("dropout_kernel");
}
