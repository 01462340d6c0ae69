// Dropout from a counter-based generator for sm_100a: dst = keep ? src * 65536 / kept : 0, the mask made
// again wherever it is needed and never stored.
//
// Bound by HBM where an element is 4 bytes; where it is 2, the generator (one counter for eight elements)
// costs about as many instructions as the memory leaves time for.
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;

struct Dropout {
    void* dst;
    const void* src;
    uint64_t ds, ss;
    uint64_t first;  // the launch's first element in contiguous tensors
    uint32_t first_row, items, width;  // items: counters of this launch, row by row
    FastDiv per_row;                   // counters per row
    DropArgs drop;
};

// Rows that take Eight's accesses: a thread takes kUnroll counters, a block's width apart, and has all
// their loads in flight before it makes the first mask.
// FLAT: both tensors are contiguous.  [16384, 8192] bf16 87 us, 6.2 TB/s; [4096, 8192] float 41 us, 6.5 TB/s (B200).
constexpr int kUnroll = 4;
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kThreads) dropout_vec_kernel(const Dropout a) {
    const Philox rng(a.drop);
    const uint32_t first = blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
    Eight<T> x[kUnroll];
    uint32_t row[kUnroll] = {}, block[kUnroll] = {};
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint32_t i = first + k * kThreads;
        if (i >= a.items) continue;
        a.per_row.divmod(i, row[k], block[k]);
        row[k] += a.first_row;
        x[k].load(static_cast<const T*>(a.src) + (FLAT ? a.first + (uint64_t)i * 8 : row[k] * a.ss + block[k] * 8));
    }
    if (a.drop.on) {
        Lanes w[kUnroll];
        rng.make(block, row, w);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = x[k].get(2 * j) * a.drop.scale, v = x[k].get(2 * j + 1) * a.drop.scale;
                x[k].set2(j, w[k].keeps(a.drop, 2 * j) ? u : 0.0f, w[k].keeps(a.drop, 2 * j + 1) ? v : 0.0f);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint32_t i = first + k * kThreads;
        if (i < a.items)
            x[k].store(static_cast<T*>(a.dst) + (FLAT ? a.first + (uint64_t)i * 8 : row[k] * a.ds + block[k] * 8));
    }
}

// Any width, stride and alignment.  A lane makes the mask of one counter; the warp's 32 x 8 elements are then
// read and written 32 consecutive slots at a time (slot s belongs to the counter of lane s / 8), with the mask
// bits of a slot from the lane that owns it.  Where the warp's counters are all of one row the slots' places need no
// exchange.  Bound by the scalar accesses: [8192, 4099] float 48 us, 5.7 TB/s; bf16 45 us, 3.0 TB/s.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_any_kernel(const Dropout a) {
    const Philox rng(a.drop);
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    uint32_t row = a.first_row, block = 0;
    if (i < a.items) {
        a.per_row.divmod(i, row, block);
        row += a.first_row;
    }
    T x[8];
    uint64_t to[8];
    uint32_t valid = 0;
    const uint32_t row0 = __shfl_sync(0xffffffffu, row, 0), block0 = __shfl_sync(0xffffffffu, block, 0);
    if (__all_sync(0xffffffffu, i < a.items && row == row0)) {
        const uint32_t c0 = block0 * 8 + lane;
        const T* src = static_cast<const T*>(a.src) + row0 * a.ss + c0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) to[j] = row0 * a.ds + c0 + 32 * j;
        if (block0 * 8 + 256 <= a.width) {  // the whole warp inside the row: no comparisons
            valid = 0xFF;
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) x[j] = src[32 * j];
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (c0 + 32 * j < a.width) {
                    valid |= 1u << j;
                    x[j] = src[32 * j];
                }
        }
    } else {
        const uint32_t inside = i < a.items ? min(8u, a.width - block * 8) : 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t from = j * 4 + lane / 8, e = lane % 8;
            const uint32_t r = __shfl_sync(0xffffffffu, row, from), c = __shfl_sync(0xffffffffu, block, from) * 8 + e;
            to[j] = r * a.ds + c;
            if (e < __shfl_sync(0xffffffffu, inside, from)) {
                valid |= 1u << j;
                x[j] = static_cast<const T*>(a.src)[r * a.ss + c];
            }
        }
    }
    uint32_t keep = 0xFF;  // bit j for element j of this lane's counter
    if (a.drop.on) {
        const Lanes w = rng(block, row);
        keep = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) keep |= (uint32_t)w.keeps(a.drop, j) << j;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const bool kept = __shfl_sync(0xffffffffu, keep, j * 4 + lane / 8) >> (lane % 8) & 1u;
        if (valid >> j & 1u)
            static_cast<T*>(a.dst)[to[j]] = from_float<T>(kept ? to_float(x[j]) * a.drop.scale : 0.0f);
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
    Dropout a{};
    if (int rc = drop_args(*drop, "mtxc_dropout", &a.drop)) return rc;
    if (rows >> 31 || width >> 31) return fail(MTXC_ERR_SHAPE, "mtxc_dropout: rows and width must be below 2^31");
    if (rows == 0 || width == 0) return MTXC_OK;
    if (!dst || !src) return fail(MTXC_ERR_INVALID_ARGUMENT, "mtxc_dropout: null buffer");
    const uint32_t per_row = (uint32_t)((width + 7) / 8);
    a.dst = dst;
    a.src = src;
    a.ds = rows == 1 ? 0 : dst_row_stride;
    a.ss = rows == 1 ? 0 : src_row_stride;
    a.width = (uint32_t)width;
    a.per_row = FastDiv(per_row);
    // launches of fewer than 2^31 counters (one, but for tensors of 2^34 elements)
    const uint64_t most = std::max<uint64_t>(1, ((1ull << 31) - 1) / per_row);
    for (uint64_t row = 0; row < rows; row += most) {
        a.first_row = (uint32_t)row;
        a.items = (uint32_t)(std::min(most, rows - row) * per_row);
        a.first = row * width;
        dispatch_float(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            const unsigned grid = (a.items + kThreads * kUnroll - 1) / (kThreads * kUnroll);
            if (width % 8 || !eight_aligned<T>(dst, a.ds) || !eight_aligned<T>(src, a.ss))
                dropout_any_kernel<T><<<(a.items + kThreads - 1) / kThreads, kThreads, 0, ctx().stream()>>>(a);
            else if (rows == 1 || (a.ds == width && a.ss == width))
                dropout_vec_kernel<T, true><<<grid, kThreads, 0, ctx().stream()>>>(a);
            else dropout_vec_kernel<T, false><<<grid, kThreads, 0, ctx().stream()>>>(a);
        });
        if (int rc = check_launch("dropout_kernel")) return rc;
    }
    return MTXC_OK;
}
