// Rotary positions for sm_100a: pairs of a head's elements turned by position * frequency, for queries and
// keys in one launch.
//
// The angle: position * frequency / (2 pi) is the number of turns, in 64 bits; its whole part is dropped
// there, and the rest, at most half a turn, goes to sincospif in 32 bits.  At position 10^6 a product in
// 32 bits would be off by up to 0.03 radians.
#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;

struct Rotary {
    uint64_t batch, length, tokens;
    uint32_t head, half, heads0, heads;  // heads0: the first tensor's; heads: both tensors'
    const void* src[2];
    void* dst[2];
    uint64_t ss[2][3], ds[2][3];
    const void* positions;
    bool wide_positions;
    uint64_t ps[2];
    const double* freq;
    float scale;
    bool interleaved, inverse;
};

__device__ __forceinline__ double position_of(const Rotary& r, uint64_t b, uint64_t s) {
    const uint64_t at = b * r.ps[0] + s * r.ps[1];
    return r.wide_positions ? (double)static_cast<const long long*>(r.positions)[at]
                            : (double)static_cast<const int*>(r.positions)[at];
}

// cos and sin of position * frequency, times scale, sin negated for the inverse.
__device__ __forceinline__ void turn(const Rotary& r, double position, uint32_t j, float& cs, float& sn) {
    const double turns = position * r.freq[j] * 0.15915494309189533576888376337251;  // 1 / (2 pi)
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    cs *= r.scale;
    sn *= r.inverse ? -r.scale : r.scale;
}

// A block per token; a thread takes pairs and passed-on elements of its heads one by one.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r) {
    const uint32_t rest = r.head - 2 * r.half, per_head = r.half + rest, items = per_head * r.heads;
    for (uint64_t token = blockIdx.x; token < r.tokens; token += gridDim.x) {
        const uint64_t b = token / r.length, s = token - b * r.length;
        const double position = position_of(r, b, s);
        for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
            const uint32_t h = i / per_head, j = i - h * per_head;
            const int k = h >= r.heads0;
            const uint32_t hh = k ? h - r.heads0 : h;
            const T* x = static_cast<const T*>(r.src[k]) + b * r.ss[k][0] + s * r.ss[k][1] + hh * r.ss[k][2];
            T* y = static_cast<T*>(r.dst[k]) + b * r.ds[k][0] + s * r.ds[k][1] + hh * r.ds[k][2];
            if (j >= r.half) {
                y[r.half + j] = x[r.half + j];
                continue;
            }
            float cs, sn;
            turn(r, position, j, cs, sn);
            const uint32_t p = r.interleaved ? 2 * j : j, q = r.interleaved ? 2 * j + 1 : j + r.half;
            const float u = to_float(x[p]), v = to_float(x[q]);
            y[p] = from_float<T>(u * cs - v * sn);
            y[q] = from_float<T>(u * sn + v * cs);
        }
    }
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_rotary(int dtype, const mtxc_rotary_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_rotary";
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": rotary_dim must be even and at most head_dim");
    if (a->position_dtype != MTXC_INT32 && a->position_dtype != MTXC_INT64)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": positions must be Int32 or Int64");
    const uint64_t heads = (uint64_t)a->heads[0] + a->heads[1];
    if (heads * a->head_dim >> 31 || (a->length && a->batch > (1ull << 40) / a->length))
        return fail(MTXC_ERR_SHAPE, who + ": a token's elements must be below 2^31, the tokens at most 2^40");
    if (a->batch == 0 || a->length == 0 || a->head_dim == 0 || heads == 0) return MTXC_OK;
    Rotary r{};
    r.batch = a->batch;
    r.length = a->length;
    r.tokens = a->batch * a->length;
    r.head = a->head_dim;
    r.half = a->rotary_dim / 2;
    r.heads0 = a->heads[0];
    r.heads = (uint32_t)heads;
    for (int k = 0; k < 2; ++k) {
        if (!a->heads[k]) continue;
        if (!a->src[k] || !a->dst[k]) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tensor");
        r.src[k] = a->src[k];
        r.dst[k] = a->dst[k];
        for (int i = 0; i < 3; ++i) r.ss[k][i] = a->src_strides[k][i], r.ds[k][i] = a->dst_strides[k][i];
    }
    if (r.half && (!a->positions || !a->frequencies))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null positions or frequencies");
    r.positions = a->positions;
    r.wide_positions = a->position_dtype == MTXC_INT64;
    r.ps[0] = a->position_strides[0];
    r.ps[1] = a->position_strides[1];
    r.freq = a->frequencies;
    r.scale = a->scale;
    r.interleaved = a->interleaved != 0;
    r.inverse = a->inverse != 0;
    const unsigned grid = (unsigned)std::min<uint64_t>(r.tokens, (uint64_t)ctx().sm_count * 16);
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        rotary_kernel<T><<<grid, kThreads, 0, ctx().stream()>>>(r);
    });
    return check_launch("rotary_kernel");
}

extern "C" int mtxc_rotary_frequencies(int scaling, uint32_t rotary_dim, double base, double factor,
                                       double original_length, double fast_turns, double slow_turns,
                                       double* frequencies, double* scale) {
    const std::string who = "mtxc_rotary_frequencies";
    if (!scale || (!frequencies && rotary_dim)) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null pointer");
    if (rotary_dim % 2 || !(base > 0) || !(factor > 0))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": rotary_dim must be even, base and factor positive");
    if (scaling < MTXC_ROTARY_NONE || scaling > MTXC_ROTARY_BY_PARTS)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": unknown scaling");
    if (scaling == MTXC_ROTARY_BASE && rotary_dim == 2)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": the base scaling needs rotary_dim above 2");
    if (scaling == MTXC_ROTARY_BY_PARTS && (!(original_length > 0) || !(fast_turns > slow_turns)))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": needs original_length > 0 and fast_turns > slow_turns");
    if (scaling == MTXC_ROTARY_BASE && rotary_dim) base *= std::pow(factor, rotary_dim / (rotary_dim - 2.0));
    *scale = scaling == MTXC_ROTARY_BY_PARTS ? 0.1 * std::log(factor) + 1.0 : 1.0;
    for (uint32_t j = 0; j < rotary_dim / 2; ++j) {
        double w = std::pow(base, -2.0 * j / rotary_dim);
        if (scaling == MTXC_ROTARY_LINEAR) w /= factor;
        if (scaling == MTXC_ROTARY_BY_PARTS) {
            const double turns = original_length * w / 6.283185307179586476925286766559;
            const double keep = std::min(1.0, std::max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)));
            w = keep * w + (1.0 - keep) * w / factor;
        }
        frequencies[j] = w;
    }
    return MTXC_OK;
}
