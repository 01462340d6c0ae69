// Norms of queries and keys for each head with their rotary positions, forward and backward, for sm_100a.
//
//   n = x r w',  r = 1 / sqrt(mean(x^2) + eps),  w' = weight_offset + w;   y = scale * turn(n), the rest of the head n
//   backward: g = turn back (scale included) of dy, u = g w':  dx = r (u - x r^2 mean(u x)),  dw = sum of g x r
//
// Bound by HBM: x (and dy) read once, y (dx) written once.  A group of lanes holds a head in registers between the
// reduction and the store; its blocks work on queries alone or keys alone, so that a lane meets one piece of one weight
// (and adds to one piece of its gradient) for all its heads.
#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxHead = 1024;
constexpr uint32_t kTableEntries = 2048;  // cosines of a tile; as many sines

struct Side {  // queries or keys
    uint32_t heads, tile, blocks, first_block;  // tokens of a tile
    uint64_t tiles;
    FastDiv heads_div;
    const void *x, *dy, *weight;
    void* out;               // y or dx
    uint64_t xs[3], ys[3], os[3];
    float* rstd;             // written forward (or NULL), read backward
    float* d_weight;         // partial rows [blocks][head], or NULL
};

struct HeadNorm {
    uint64_t tokens;
    uint64_t length;         // tokens of a sequence
    uint32_t head, half, lanes_log, units, turned, second;  // second: from a copied unit's first access to its second
    FastDiv half_div;
    int weight_dtype;
    const void* positions;
    bool wide_positions;
    uint64_t ps[2];
    const double* freq;
    float scale, sin_scale, weight_offset, eps, inv_head;
    Side side[2];
};

__device__ __forceinline__ void turn(const HeadNorm& r, double position, uint32_t j, float& cs, float& sn) {
    const double turns = position * r.freq[j] * 0.15915494309189533576888376337251;  // 1 / (2 pi)
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    cs *= r.scale;
    sn *= r.sin_scale;
}

__device__ __forceinline__ double position_of(const HeadNorm& r, uint64_t b, uint64_t t) {
    const uint64_t p = b * r.ps[0] + t * r.ps[1];
    return r.wide_positions ? (double)static_cast<const long long*>(r.positions)[p]
                            : (double)static_cast<const int*>(r.positions)[p];
}

__device__ __forceinline__ float weight_at(const HeadNorm& r, const Side& s, uint32_t d) {
    if (!s.weight) return 1.0f;
    const float w = r.weight_dtype == MTXC_FLOAT ? static_cast<const float*>(s.weight)[d]
                    : r.weight_dtype == MTXC_FLOAT16 ? __half2float(static_cast<const __half*>(s.weight)[d])
                                                     : __bfloat162float(static_cast<const __nv_bfloat16*>(s.weight)[d]);
    return r.weight_offset + w;
}

// ------------------------------------------------------------------------------------------
// Any head: a warp per head, which it reads twice; the angles made where they are used.
// ------------------------------------------------------------------------------------------
template <typename T, bool PAIRS, bool BACKWARD>
__global__ void __launch_bounds__(kThreads) head_norm_any_kernel(const HeadNorm r) {
    extern __shared__ float sums[];  // BACKWARD: [warps][head], a lane adds to its own columns
    const int k = blockIdx.x >= r.side[1].first_block;
    const Side& s = r.side[k];
    const uint32_t block = blockIdx.x - s.first_block, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr uint32_t kWarps = kThreads / 32;
    float* const mine = sums + warp * r.head;
    const bool weighed = BACKWARD && s.d_weight;
    if (weighed)
        for (uint32_t d = lane; d < r.head; d += 32) mine[d] = 0.0f;
    __syncwarp();  // the columns of a pair need not be those that the lane has cleared
    const uint32_t rest = r.head - 2 * r.half;
    for (uint64_t i = (uint64_t)block * kWarps + warp; i < r.tokens * s.heads; i += (uint64_t)s.blocks * kWarps) {
        const uint64_t token = i / s.heads, h = i % s.heads, b = token / r.length, t = token % r.length;
        const T* x = static_cast<const T*>(s.x) + b * s.xs[0] + t * s.xs[1] + h * s.xs[2];
        T* out = static_cast<T*>(s.out) + b * s.os[0] + t * s.os[1] + h * s.os[2];
        const double position = r.half ? position_of(r, b, t) : 0.0;
        if constexpr (!BACKWARD) {
            float sum = 0.0f;
            for (uint32_t d = lane; d < r.head; d += 32) {
                const float v = to_float(x[d]);
                sum = fmaf(v, v, sum);
            }
#pragma unroll
            for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
            const float rstd = rsqrtf(fmaf(sum, r.inv_head, r.eps));
            if (s.rstd && lane == 0) s.rstd[i] = rstd;
            for (uint32_t j = lane; j < r.half; j += 32) {
                const uint32_t a = PAIRS ? 2 * j : j, c = PAIRS ? a + 1 : j + r.half;
                float cs, sn;
                turn(r, position, j, cs, sn);
                const float u = to_float(x[a]) * rstd * weight_at(r, s, a), v = to_float(x[c]) * rstd * weight_at(r, s, c);
                out[a] = from_float<T>(u * cs - v * sn);
                out[c] = from_float<T>(u * sn + v * cs);
            }
            for (uint32_t j = lane; j < rest; j += 32) {
                const uint32_t a = 2 * r.half + j;
                out[a] = from_float<T>(to_float(x[a]) * rstd * weight_at(r, s, a));
            }
        } else {
            const T* dy = static_cast<const T*>(s.dy) + b * s.ys[0] + t * s.ys[1] + h * s.ys[2];
            const float rstd = s.rstd[i];
            // visit(column, x r, gradient at n)
            auto each = [&](auto&& visit) {
                for (uint32_t j = lane; j < r.half; j += 32) {
                    const uint32_t a = PAIRS ? 2 * j : j, c = PAIRS ? a + 1 : j + r.half;
                    float cs, sn;
                    turn(r, position, j, cs, sn);
                    const float u = to_float(dy[a]), v = to_float(dy[c]), xa = to_float(x[a]), xc = to_float(x[c]);
                    visit(a, xa * rstd, u * cs - v * sn);
                    visit(c, xc * rstd, u * sn + v * cs);
                }
                for (uint32_t j = lane; j < rest; j += 32) {
                    const uint32_t a = 2 * r.half + j;
                    visit(a, to_float(x[a]) * rstd, to_float(dy[a]));
                }
            };
            float sum = 0.0f;
            each([&](uint32_t d, float e, float g) {
                sum = fmaf(g * weight_at(r, s, d), e, sum);
                if (weighed) mine[d] = fmaf(g, e, mine[d]);
            });
#pragma unroll
            for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
            sum *= r.inv_head;
            // a pair's elements are read before either is written: dx may be dy or x
            for (uint32_t j = lane; j < r.half; j += 32) {
                const uint32_t a = PAIRS ? 2 * j : j, c = PAIRS ? a + 1 : j + r.half;
                float cs, sn;
                turn(r, position, j, cs, sn);
                const float u = to_float(dy[a]), v = to_float(dy[c]);
                const float ea = to_float(x[a]) * rstd, ec = to_float(x[c]) * rstd;
                out[a] = from_float<T>(rstd * ((u * cs - v * sn) * weight_at(r, s, a) - ea * sum));
                out[c] = from_float<T>(rstd * ((u * sn + v * cs) * weight_at(r, s, c) - ec * sum));
            }
            for (uint32_t j = lane; j < rest; j += 32) {
                const uint32_t a = 2 * r.half + j;
                out[a] = from_float<T>(rstd * (to_float(dy[a]) * weight_at(r, s, a) - to_float(x[a]) * rstd * sum));
            }
        }
    }
    if (weighed) {
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < r.head; d += kThreads) {
            float sum = 0.0f;
            for (uint32_t w = 0; w < kWarps; ++w) sum += sums[w * r.head + d];
            s.d_weight[(uint64_t)block * r.head + d] = sum;
        }
    }
}

// ------------------------------------------------------------------------------------------
// The weights' gradients from the blocks' partial rows, added in a fixed order: 32 columns a block, 32 threads a
// column.
// ------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) head_norm_finish_kernel(const float* p0, uint32_t rows0, float* d0, const float* p1,
                                                                uint32_t rows1, float* d1, uint32_t head) {
    __shared__ float sums[32][33];
    const float* p = blockIdx.y ? p1 : p0;
    float* d = blockIdx.y ? d1 : d0;
    if (!d) return;
    const uint32_t rows = blockIdx.y ? rows1 : rows0, x = threadIdx.x % 32, y = threadIdx.x / 32, c = blockIdx.x * 32 + x;
    float sum = 0.0f;
    if (c < head)
        for (uint32_t i = y; i < rows; i += 32) sum += p[(uint64_t)i * head + c];
    sums[y][x] = sum;
    __syncthreads();
    sum = sums[x][y];
#pragma unroll
    for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
    if (x == 0 && blockIdx.x * 32 + y < head) d[blockIdx.x * 32 + y] = sum;
}

int check_args(const std::string& who, int dtype, const mtxc_head_norm_args* a) {
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (a->head_dim > kMaxHead) return fail(MTXC_ERR_SHAPE, who + ": head_dim must be at most " + std::to_string(kMaxHead));
    if (a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": rotary_dim must be even and at most head_dim");
    if (a->position_dtype != MTXC_INT32 && a->position_dtype != MTXC_INT64)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": positions must be Int32 or Int64");
    if (!is_float_like(a->weight_dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": weights must be Float, Float16 or BFloat16");
    if (a->heads[0] >> 16 || a->heads[1] >> 16 || a->length >> 31 || (a->length && a->batch > (1ull << 40) / a->length))
        return fail(MTXC_ERR_SHAPE, who + ": heads must be below 65,536, the length below 2^31, the tokens at most 2^40");
    const uint64_t tokens = a->batch * a->length;
    for (int k = 0; k < 2 && tokens && a->head_dim; ++k)
        if (a->heads[k] && (!a->src[k] || !a->dst[k])) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tensor");
    if (tokens && a->rotary_dim && (!a->positions || !a->frequencies))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null positions or frequencies");
    return distinct(who, {a->heads[0] ? a->dst[0] : nullptr, a->heads[1] ? a->dst[1] : nullptr});
}

// The call's arguments as the kernels take them, and its plan; blocks: all that the launch needs.
struct Plan {
    HeadNorm r{};
    bool vector = false;
    uint32_t blocks = 0;
};

Plan plan(int dtype, const mtxc_head_norm_args* a, bool backward) {
    Plan p;
    HeadNorm& r = p.r;
    r.tokens = a->batch * a->length;
    r.length = std::max<uint64_t>(1, a->length);
    r.head = a->head_dim;
    r.half = a->rotary_dim / 2;
    r.weight_dtype = a->weight_dtype;
    r.positions = a->positions;
    r.wide_positions = a->position_dtype == MTXC_INT64;
    r.ps[0] = a->position_strides[0];
    r.ps[1] = a->position_strides[1];
    r.freq = a->frequencies;
    r.scale = a->scale;
    r.sin_scale = backward ? -a->scale : a->scale;
    r.weight_offset = a->weight_offset;
    r.eps = a->eps;
    r.inv_head = 1.0f / (float)std::max(1u, r.head);
    for (int k = 0; k < 2; ++k) {
        Side& s = r.side[k];
        s.heads = a->heads[k];
        s.heads_div = FastDiv(std::max(1u, s.heads));
        s.x = a->src[k];
        s.dy = a->d_out[k];
        s.weight = a->weight[k];
        s.out = a->dst[k];
        s.rstd = a->rstd[k];
        for (int i = 0; i < 3; ++i)
            s.xs[i] = a->src_strides[k][i], s.ys[i] = a->d_out_strides[k][i], s.os[i] = a->dst_strides[k][i];
        const uint64_t warps = r.tokens * s.heads;
        s.blocks = (uint32_t)std::min<uint64_t>((warps + kThreads / 32 - 1) / (kThreads / 32), 4u * ctx().sm_count);
        s.first_block = p.blocks;
        p.blocks += s.blocks;
    }
    return p;
}

template <bool BACKWARD>
int launch(int dtype, const mtxc_head_norm_args* a, const Plan& p) {
    const HeadNorm& r = p.r;
    const size_t smem = BACKWARD ? sizeof(float) * (kThreads / 32) * r.head : 0;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a->interleaved) head_norm_any_kernel<T, true, BACKWARD><<<p.blocks, kThreads, smem, ctx().stream()>>>(r);
        else head_norm_any_kernel<T, false, BACKWARD><<<p.blocks, kThreads, smem, ctx().stream()>>>(r);
    });
    return check_launch("head_norm_kernel");
}

// Bytes of partial rows that a backward call wants (its sides' d_weight may be NULL).
size_t partial_bytes(const Plan& p, const mtxc_head_norm_args* a) {
    size_t n = 0;
    for (int k = 0; k < 2; ++k)
        if (a->d_weight[k]) n += (size_t)p.r.side[k].blocks * p.r.head;
    return (n * sizeof(float) + 255) / 256 * 256;
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_head_norm_rotary(int dtype, const mtxc_head_norm_args* a) {
    if (int rc = require_init()) return rc;
    if (int rc = check_args("mtxc_head_norm_rotary", dtype, a)) return rc;
    if (int rc = distinct("mtxc_head_norm_rotary", {a->dst[0], a->dst[1], a->rstd[0], a->rstd[1]})) return rc;
    const Plan p = plan(dtype, a, false);
    if (!p.blocks || !a->head_dim) return MTXC_OK;
    return launch<false>(dtype, a, p);
}

extern "C" int mtxc_head_norm_rotary_backward_workspace(int dtype, const mtxc_head_norm_args* a, size_t* bytes) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_head_norm_rotary_backward_workspace";
    if (!bytes) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null pointer");
    if (int rc = check_args(who, dtype, a)) return rc;
    *bytes = partial_bytes(plan(dtype, a, true), a);
    return MTXC_OK;
}

extern "C" int mtxc_head_norm_rotary_backward(int dtype, const mtxc_head_norm_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_head_norm_rotary_backward";
    if (int rc = check_args(who, dtype, a)) return rc;
    if (int rc = distinct(who, {a->dst[0], a->dst[1], a->d_weight[0], a->d_weight[1]})) return rc;
    Plan p = plan(dtype, a, true);
    for (int k = 0; k < 2; ++k) {
        if (p.r.side[k].blocks && a->head_dim && (!a->d_out[k] || !a->rstd[k]))
            return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null d_out or rstd");
    }
    if (!a->head_dim) return MTXC_OK;
    const size_t bytes = partial_bytes(p, a);
    float* partial = static_cast<float*>(a->workspace ? a->workspace : ctx().workspace);
    if (bytes > (a->workspace ? a->workspace_bytes : ctx().workspace_bytes))
        return fail(MTXC_ERR_WORKSPACE, who + ": the partial sums need " + std::to_string(bytes) + " bytes of workspace");
    const float* rows[2] = {nullptr, nullptr};
    for (int k = 0; k < 2; ++k) {
        if (!a->d_weight[k]) continue;
        rows[k] = p.r.side[k].d_weight = partial;
        partial += (size_t)p.r.side[k].blocks * a->head_dim;
    }
    if (p.blocks)
        if (int rc = launch<true>(dtype, a, p)) return rc;
    if (a->d_weight[0] || a->d_weight[1]) {
        const dim3 grid((a->head_dim + 31) / 32, 2);
        head_norm_finish_kernel<<<grid, 1024, 0, ctx().stream()>>>(rows[0], p.r.side[0].blocks, a->d_weight[0], rows[1],
                                                                   p.r.side[1].blocks, a->d_weight[1], a->head_dim);
        return check_launch("head_norm_finish_kernel");
    }
    return MTXC_OK;
}
