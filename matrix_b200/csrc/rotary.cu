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
constexpr uint32_t kMaxHalf = 4096;       // a token's cosines and sines: 32 KB of shared memory
constexpr uint32_t kTableEntries = 2048;  // what a block's tokens share otherwise
constexpr uint32_t kBlocksPerSm = 4;

struct Rotary {
    uint32_t length, tile, tiles;  // tokens of a sequence, of a block; blocks of a sequence
    uint32_t half, heads0, far;    // far: between the two accesses of a copied unit, 0: it has one
    uint32_t items, lanes, rows;   // units of a token; threads that take them side by side, and tokens side by side
    FastDiv tiles_div, units, lanes_div, half_div;  // units: of a head
    uint64_t first_batch;          // where the launch starts
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

template <int M>
__device__ __forceinline__ void read_table(const float* p, float (&v)[M]) {
    if constexpr (M % 4 == 0) {
#pragma unroll
        for (int i = 0; i < M; i += 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + i);
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
    } else if constexpr (M == 2) {
        const float2 q = *reinterpret_cast<const float2*>(p);
        v[0] = q.x, v[1] = q.y;
    } else v[0] = p[0];
}

// A block takes `tile` tokens of a sequence.  It makes their cosines and sines once, in shared memory, for all
// heads -- with its first loads already in flight -- and then turns units: N pairs (two accesses of N = 8 or 4
// elements, half a head apart) or, PAIRS (interleaved), N elements of N / 2 pairs; N = 0: one pair.  What is not
// turned is copied in units of N elements, without PAIRS two such r.far apart where they divide so, or one
// element.  A thread stays with one unit of one head for all its tokens, kUnroll at a time, so that a unit's place
// is worked out once (worked out for each, it was two thirds of the instructions).  Bound by HBM: 16,384 tokens x
// 40 heads of 128 bf16 56 us, 6.0 TB/s.
template <typename T, int N, bool PAIRS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r) {
    constexpr int kUnroll = N && !PAIRS ? 2 : 4;
    constexpr int kStep = N ? N : 1, kPairs = N == 0 ? 1 : PAIRS ? N / 2 : N;  // elements of a copy, pairs of a unit
    extern __shared__ float table[];  // [tile][half] cosines, then sines
    float* const cosines = table;
    float* const sines = table + r.tile * r.half;
    uint32_t batch, t0;
    r.tiles_div.divmod(blockIdx.x, batch, t0);
    t0 *= r.tile;
    const uint32_t n = min(r.tile, r.length - t0);
    const uint64_t b = r.first_batch + batch;
    const uint32_t turned = r.half / kPairs;  // units of a head that are turned
    uint32_t lane, token0;  // this thread's first unit and token
    r.lanes_div.divmod(threadIdx.x, token0, lane);
    const bool idle = token0 >= r.rows;

    struct Unit {
        Few<T, N ? N : 4> a, b;
        T u, v;
    };
    const T* src = nullptr;
    T* dst = nullptr;
    uint64_t src_step = 0, dst_step = 0;
    uint32_t at = 0, far = 0;  // the unit's first pair; from its first access to its second (0: none)
    bool copy = false;
    // places a unit of the tile's first token
    auto place = [&](uint32_t item) {
        uint32_t h, unit;
        r.units.divmod(item, h, unit);
        const int k = h >= r.heads0;
        const uint64_t hh = k ? h - r.heads0 : h;
        copy = unit >= turned;
        far = copy ? r.far : PAIRS ? (N ? 0 : 1) : r.half;
        at = unit * kPairs;
        const uint32_t c = copy ? 2 * r.half + (unit - turned) * kStep : at * (PAIRS ? 2 : 1);
        src = static_cast<const T*>(r.src[k]) + b * r.ss[k][0] + t0 * r.ss[k][1] + hh * r.ss[k][2] + c;
        dst = static_cast<T*>(r.dst[k]) + b * r.ds[k][0] + t0 * r.ds[k][1] + hh * r.ds[k][2] + c;
        src_step = r.ss[k][1];
        dst_step = r.ds[k][1];
    };
    auto load = [&](uint32_t token, Unit& x) {
        const T* p = src + token * src_step;
        if constexpr (N) {
            x.a.load(p);
            if (!PAIRS && far) x.b.load(p + far);
        } else {
            x.u = p[0];
            if (far) x.v = p[far];
        }
    };
    auto finish = [&](uint32_t token, Unit& x) {
        T* p = dst + token * dst_step;
        if (!copy) {
            float cs[kPairs], sn[kPairs];
            read_table(cosines + token * r.half + at, cs);
            read_table(sines + token * r.half + at, sn);
            if constexpr (N == 0) {
                const float u = to_float(x.u), v = to_float(x.v);
                x.u = from_float<T>(u * cs[0] - v * sn[0]);
                x.v = from_float<T>(u * sn[0] + v * cs[0]);
            } else if constexpr (PAIRS) {
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float2 q = x.a.get2(j);
                    const float2 o = __ffma2_rn(make_float2(q.x, q.x), make_float2(cs[j], sn[j]),
                                                __fmul2_rn(make_float2(q.y, q.y), make_float2(-sn[j], cs[j])));
                    x.a.set2(j, o.x, o.y);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kPairs / 2; ++j) {
                    const float2 u = x.a.get2(j), v = x.b.get2(j);
                    const float2 c = make_float2(cs[2 * j], cs[2 * j + 1]), s = make_float2(sn[2 * j], sn[2 * j + 1]);
                    const float2 p = __ffma2_rn(u, c, __fmul2_rn(v, make_float2(-s.x, -s.y)));
                    const float2 q = __ffma2_rn(u, s, __fmul2_rn(v, c));
                    x.a.set2(j, p.x, p.y);
                    x.b.set2(j, q.x, q.y);
                }
            }
        }
        if constexpr (N) {
            x.a.store(p);
            if (!PAIRS && far) x.b.store(p + far);
        } else {
            p[0] = x.u;
            if (far) p[far] = x.v;
        }
    };

    Unit x[kUnroll];
    uint32_t item = blockIdx.y * r.lanes + lane;  // blocks along y share a tile's units
    const bool any = !idle && item < r.items;
    if (any) {
        place(item);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (token0 + k * r.rows < n) load(token0 + k * r.rows, x[k]);
    }
    for (uint32_t e = threadIdx.x; e < n * r.half; e += blockDim.x) {
        uint32_t token, j;
        r.half_div.divmod(e, token, j);
        const uint64_t p = b * r.ps[0] + (t0 + token) * r.ps[1];
        const double position = r.wide_positions ? (double)static_cast<const long long*>(r.positions)[p]
                                                 : (double)static_cast<const int*>(r.positions)[p];
        turn(r, position, j, cosines[e], sines[e]);
    }
    __syncthreads();
    if (!any) return;
    for (uint32_t token = token0;;) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (token + k * r.rows < n) finish(token + k * r.rows, x[k]);
        token += kUnroll * r.rows;
        if (token >= n) {
            item += gridDim.y * r.lanes;
            if (item >= r.items) break;
            place(item);
            token = token0;
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (token + k * r.rows < n) load(token + k * r.rows, x[k]);
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
    if (heads * a->head_dim >> 27 || a->length >> 31 || (a->length && a->batch > (1ull << 40) / a->length))
        return fail(MTXC_ERR_SHAPE, who + ": a token's elements must be below 2^27, the length below 2^31, the tokens at most 2^40");
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
    if (int rc = distinct(who, {r.dst[0], r.dst[1]})) return rc;
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
        // elements of an access: what the sizes, strides and addresses all divide by
        auto fits = [&](auto count) {
            constexpr int N = decltype(count)::value;
            bool ok = r.half % (pairs ? N / 2 : N) == 0 && copied % N == 0;
            for (int k = 0; k < 2; ++k)
                for (int i = 0; a->heads[k] && i < 3; ++i)
                    ok = ok && few_aligned<T, N>(r.src[k], r.ss[k][i]) && few_aligned<T, N>(r.dst[k], r.ds[k][i]);
            return ok;
        };
        const uint32_t step = fits(std::integral_constant<int, 8>()) ? 8 : fits(std::integral_constant<int, 4>()) ? 4 : 1;
        r.far = !pairs && copied % (2 * step) == 0 ? copied / 2 : 0;
        const uint32_t units = r.half / (step == 1 ? 1 : pairs ? step / 2 : step) + copied / step / (r.far ? 2 : 1);
        r.units = FastDiv(units);
        r.half_div = FastDiv(std::max(1u, r.half));
        r.items = units * (uint32_t)heads;
        r.length = (uint32_t)a->length;
        // threads side by side: a token's units evenly in as few rounds as 256 threads allow, and as many tokens
        // as fit
        const uint32_t rounds = std::min<uint32_t>((r.items + kThreads - 1) / kThreads, 65535);
        r.lanes = std::min<uint32_t>((r.items + rounds - 1) / rounds, kThreads);
        r.lanes_div = FastDiv(r.lanes);
        // tokens of a block: what gives a thread 6 units of two accesses or 10 of one, in whole rounds of the
        // unrolled loads, while every SM still has kBlocksPerSm blocks and the table fits (16,384 tokens x 40
        // heads of 128 bf16: 57 us with 6, 63 with 8, 66 with 12; interleaved 56 us with 10, 60 with 16, 98 with
        // 4)
        const uint64_t tokens = a->batch * a->length;
        const uint32_t round = std::max(1u, kThreads / r.lanes) * (step > 1 && !pairs ? 2 : 4);
        uint64_t tile = std::max<uint64_t>(1, (step > 1 && !pairs ? 6 : 10) * kThreads / r.items);
        tile = std::min(tile, std::max<uint64_t>(1, tokens / (kBlocksPerSm * (uint64_t)ctx().sm_count)));
        tile = std::min<uint64_t>({tile, std::max(1u, kTableEntries / std::max(1u, r.half)), r.length});
        if (tile > round) tile = tile / round * round;
        r.tile = (uint32_t)tile;
        r.tiles = (r.length + r.tile - 1) / r.tile;
        r.tiles_div = FastDiv(r.tiles);
        r.rows = std::min(kThreads / r.lanes, r.tile);
        const unsigned threads = (r.lanes * r.rows + 31) / 32 * 32;
        const size_t smem = 2 * sizeof(float) * r.tile * r.half;
        // launches of fewer than 2^31 blocks, whole sequences each
        const uint64_t most = std::max<uint64_t>(1, ((1ull << 31) - 1) / r.tiles);
        for (uint64_t batch = 0; batch < a->batch && rc == MTXC_OK; batch += most) {
            r.first_batch = batch;
            const unsigned blocks = (unsigned)(std::min(most, a->batch - batch) * r.tiles);
            const dim3 grid(blocks, blocks < (unsigned)ctx().sm_count ? rounds : 1);  // few tokens: no second round
            cudaStream_t st = ctx().stream();
            auto run = [&](auto count) {
                if (pairs) rotary_kernel<T, decltype(count)::value, true><<<grid, threads, smem, st>>>(r);
                else rotary_kernel<T, decltype(count)::value, false><<<grid, threads, smem, st>>>(r);
            };
            if (step == 8) run(std::integral_constant<int, 8>());
            else if (step == 4) run(std::integral_constant<int, 4>());
            else run(std::integral_constant<int, 0>());
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
