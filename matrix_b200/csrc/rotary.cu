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
constexpr int kUnroll = 2;              // units of a thread whose loads are in flight together
constexpr uint32_t kMaxHalf = 4096;     // a token's cosines and sines: 32 KB of shared memory
constexpr uint32_t kTableEntries = 2048;  // what a block's tokens share otherwise
constexpr uint32_t kTileUnits = 4;        // units of a thread in all

struct Rotary {
    uint32_t tokens, tile;  // tokens of this launch, tokens of a block
    uint32_t half, heads0, items_per_token;
    FastDiv length, units, heads, half_div;  // units of a head, heads of both tensors
    uint64_t first_batch;  // where the launch starts
    const void* src[2];
    void* dst[2];
    uint64_t ss[2][3], ds[2][3];
    const void* positions;
    bool wide_positions;
    uint64_t ps[2];
    const double* freq;
    float scale, sin_scale;  // sin_scale: -scale for the inverse
};

// cos and sin of position * frequency, times scale.
__device__ __forceinline__ void turn(const Rotary& r, double position, uint32_t j, float& cs, float& sn) {
    const double turns = position * r.freq[j] * 0.15915494309189533576888376337251;  // 1 / (2 pi)
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    cs *= r.scale;
    sn *= r.sin_scale;
}

// A block takes `tile` tokens.  It makes their cosines and sines once, in shared memory, for all heads -- with its
// first loads already in flight -- and then turns units: VEC, eight pairs (two accesses of eight elements, half
// a head apart) or, PAIRS (interleaved), eight elements of four pairs; else one pair.  What is not turned is copied in
// units of eight elements, or one.
template <typename T, bool VEC, bool PAIRS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r) {
    extern __shared__ float table[];  // [tile][half] cosines, then sines
    const uint32_t first = blockIdx.x * r.tile, n = min(r.tile, r.tokens - first);
    float* const cosines = table;
    float* const sines = table + r.tile * r.half;
    const uint32_t items = n * r.items_per_token;
    const uint32_t turned = VEC ? (PAIRS ? r.half / 4 : r.half / 8) : r.half;  // units of a head that are turned

    auto batch_and_s = [&](uint32_t token, uint64_t& b, uint64_t& s) {
        uint32_t q, m;
        r.length.divmod(token, q, m);
        b = r.first_batch + q;
        s = m;
    };
    struct Unit {
        uint64_t from, to;
        uint32_t at;  // into the table; only for turned units
        bool k, copy;
        Eight<T> a, b;
        T u, v;
    };
    auto load = [&](uint32_t i, Unit& x) {
        uint32_t q, unit, token, h;
        r.units.divmod(i, q, unit);
        r.heads.divmod(q, token, h);
        uint64_t b, s;
        batch_and_s(first + token, b, s);
        x.k = h >= r.heads0;
        const int k = x.k;
        const uint64_t hh = k ? h - r.heads0 : h;
        x.copy = unit >= turned;
        // the unit's first element: turned units from 0 (half layout: their second half r.half further), copied
        // ones from 2 * half
        uint32_t c;
        if (x.copy) c = 2 * r.half + (unit - turned) * (VEC ? 8 : 1);
        else c = unit * (VEC ? 8 : PAIRS ? 2 : 1);
        x.at = token * r.half + (VEC ? (PAIRS ? unit * 4 : unit * 8) : unit);
        x.from = b * r.ss[k][0] + s * r.ss[k][1] + hh * r.ss[k][2] + c;
        x.to = b * r.ds[k][0] + s * r.ds[k][1] + hh * r.ds[k][2] + c;
        const T* src = static_cast<const T*>(r.src[k]) + x.from;
        if constexpr (VEC) {
            x.a.load(src);
            if (!PAIRS && !x.copy) x.b.load(src + r.half);
        } else {
            x.u = src[0];
            if (!x.copy) x.v = src[PAIRS ? 1 : r.half];
        }
    };
    auto finish = [&](Unit& x) {
        T* dst = static_cast<T*>(r.dst[x.k]) + x.to;
        if constexpr (VEC) {
            if (!x.copy) {
                const float4* c4 = reinterpret_cast<const float4*>(cosines + x.at);
                const float4* s4 = reinterpret_cast<const float4*>(sines + x.at);
                if constexpr (PAIRS) {
                    const float4 c = c4[0], s = s4[0];
                    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 p = x.a.get2(j);
                        x.a.set2(j, p.x * cs[j] - p.y * sn[j], p.x * sn[j] + p.y * cs[j]);
                    }
                } else {
                    const float4 c0 = c4[0], c1 = c4[1], s0 = s4[0], s1 = s4[1];
                    const float2 cs[4] = {{c0.x, c0.y}, {c0.z, c0.w}, {c1.x, c1.y}, {c1.z, c1.w}};
                    const float2 sn[4] = {{s0.x, s0.y}, {s0.z, s0.w}, {s1.x, s1.y}, {s1.z, s1.w}};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 u = x.a.get2(j), v = x.b.get2(j);
                        const float2 vs = __fmul2_rn(v, sn[j]), vc = __fmul2_rn(v, cs[j]);
                        const float2 p = __ffma2_rn(u, cs[j], make_float2(-vs.x, -vs.y)), q = __ffma2_rn(u, sn[j], vc);
                        x.a.set2(j, p.x, p.y);
                        x.b.set2(j, q.x, q.y);
                    }
                    x.b.store(dst + r.half);
                }
            }
            x.a.store(dst);
        } else if (x.copy) dst[0] = x.u;
        else {
            const float cs = cosines[x.at], sn = sines[x.at], u = to_float(x.u), v = to_float(x.v);
            dst[0] = from_float<T>(u * cs - v * sn);
            dst[PAIRS ? 1 : r.half] = from_float<T>(u * sn + v * cs);
        }
    };

    Unit x[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint32_t i = threadIdx.x + k * kThreads;
        if (i < items) load(i, x[k]);
    }
    for (uint32_t e = threadIdx.x; e < n * r.half; e += kThreads) {
        uint32_t token, j;
        r.half_div.divmod(e, token, j);
        uint64_t b, s;
        batch_and_s(first + token, b, s);
        const uint64_t at = b * r.ps[0] + s * r.ps[1];
        const double position = r.wide_positions ? (double)static_cast<const long long*>(r.positions)[at]
                                                 : (double)static_cast<const int*>(r.positions)[at];
        turn(r, position, j, cosines[e], sines[e]);
    }
    __syncthreads();
    for (uint32_t base = threadIdx.x;; base += kUnroll * kThreads) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (base + k * kThreads < items) finish(x[k]);
        if (base + kUnroll * kThreads >= items) break;
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = base + (kUnroll + k) * kThreads;
            if (i < items) load(i, x[k]);
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
    if (a->rotary_dim % 2 || a->rotary_dim > a->head_dim || a->rotary_dim > 2 * kMaxHalf)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": rotary_dim must be even, at most head_dim and at most " +
                                                   std::to_string(2 * kMaxHalf));
    if (a->position_dtype != MTXC_INT32 && a->position_dtype != MTXC_INT64)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": positions must be Int32 or Int64");
    const uint64_t heads = (uint64_t)a->heads[0] + a->heads[1];
    if (heads * a->head_dim >> 27 || a->length >> 31)
        return fail(MTXC_ERR_SHAPE, who + ": a token's elements must be below 2^27, the length below 2^31");
    if (a->batch == 0 || a->length == 0 || a->head_dim == 0 || heads == 0) return MTXC_OK;
    Rotary r{};
    r.half = a->rotary_dim / 2;
    r.heads0 = a->heads[0];
    const uint32_t rest = a->head_dim - a->rotary_dim;
    bool in_place = true;
    for (int k = 0; k < 2; ++k) {
        if (!a->heads[k]) continue;
        if (!a->src[k] || !a->dst[k]) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tensor");
        r.src[k] = a->src[k];
        r.dst[k] = a->dst[k];
        in_place = in_place && a->src[k] == a->dst[k];
        for (int i = 0; i < 3; ++i) {
            r.ss[k][i] = a->src_strides[k][i], r.ds[k][i] = a->dst_strides[k][i];
            in_place = in_place && r.ss[k][i] == r.ds[k][i];
        }
    }
    if (r.half && (!a->positions || !a->frequencies))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null positions or frequencies");
    const uint32_t copied = in_place ? 0 : rest;
    if (r.half == 0 && copied == 0) return MTXC_OK;
    r.positions = a->positions;
    r.wide_positions = a->position_dtype == MTXC_INT64;
    r.ps[0] = a->position_strides[0];
    r.ps[1] = a->position_strides[1];
    r.freq = a->frequencies;
    r.scale = a->scale;
    r.sin_scale = a->inverse ? -a->scale : a->scale;
    const bool pairs = a->interleaved != 0;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        bool vec = r.half % (pairs ? 4 : 8) == 0 && copied % 8 == 0;
        for (int k = 0; k < 2; ++k)
            for (int i = 0; a->heads[k] && i < 3; ++i)
                vec = vec && eight_aligned<T>(r.src[k], r.ss[k][i]) && eight_aligned<T>(r.dst[k], r.ds[k][i]);
        const uint32_t units = vec ? r.half / (pairs ? 4 : 8) + copied / 8 : r.half + copied;
        r.units = FastDiv(units);
        r.heads = FastDiv((uint32_t)heads);
        r.half_div = FastDiv(std::max(1u, r.half));
        r.items_per_token = units * (uint32_t)heads;
        // launches of fewer than 2^31 tokens, whole sequences each
        const uint64_t most = std::max<uint64_t>(1, ((1ull << 31) - 1) / a->length);
        for (uint64_t batch = 0; batch < a->batch && rc == MTXC_OK; batch += most) {
            r.first_batch = batch;
            r.tokens = (uint32_t)(std::min(most, a->batch - batch) * a->length);
            r.length = FastDiv((uint32_t)a->length);
            // tokens of a block: what gives a thread kTileUnits units, while all SMs still have blocks and the table fits
            uint32_t tile = std::max(1u, kThreads * kTileUnits / r.items_per_token);
            tile = std::min(tile, std::max(1u, r.tokens / (4 * (uint32_t)ctx().sm_count)));
            tile = std::min(tile, std::max(1u, kTableEntries / std::max(1u, r.half)));
            r.tile = tile;
            const unsigned grid = (r.tokens + tile - 1) / tile;
            const size_t smem = 2 * sizeof(float) * tile * r.half;
            cudaStream_t st = ctx().stream();
            if (vec && pairs) rotary_kernel<T, true, true><<<grid, kThreads, smem, st>>>(r);
            else if (vec) rotary_kernel<T, true, false><<<grid, kThreads, smem, st>>>(r);
            else if (pairs) rotary_kernel<T, false, true><<<grid, kThreads, smem, st>>>(r);
            else rotary_kernel<T, false, false><<<grid, kThreads, smem, st>>>(r);
            rc = check_launch("rotary_kernel");
        }
    });
    return rc;
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
