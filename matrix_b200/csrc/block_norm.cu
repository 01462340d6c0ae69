// The norms after and before a transformer block, fused with its gate, dropout and residual (forward and
// backward), for sm_100a.
//
//   forward   n = b r w_post,  h = alpha x + beta g drop(n),  a = h s w_next
//   backward  H = dh + s p - h kappa,  p = da w_next,  kappa = s^3 mean(p h)
//             dx = alpha H;  t = beta mask H;  u = t g w_post;  db = r u - b r^3 mean(u b)
//             dw_next += da h s;  S += t b r (per gate row);  dw_post += g S;  dg = w_post S
//
// mean(u b) needs H, which needs mean(p h): with e = beta mask g w_post b it is
// mean(e (dh + s p)) - kappa mean(e h), so one reduction of three sums serves both.  (kappa h is the
// projection of s p on h, never longer than s p: the difference loses no more than H itself does.)
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float param(const void* p, uint64_t i, bool is_float) {
    return is_float ? __ldg(static_cast<const float*>(p) + i) : to_float(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Sums N values over the block; every thread gets the totals.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* part) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    __syncthreads();  // part may still be read from the last sum
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) part[i * 32 + warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? part[i * 32 + lane] : 0.0f);
}

struct Forward {
    const void *x, *b, *w_post, *w_next, *gate;
    void *h, *a;
    float *post_rstd, *next_rstd;
    uint64_t xs, bs, gs, hs, as;
    uint32_t rows, width, gate_rows;
    bool w_float, g_float;
    float alpha, beta, w0, eps;
    DropArgs drop;
};

// Any width, stride and alignment: a block per row, which reads its row once for each sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_any_kernel(const Forward f) {
    __shared__ float part[32];
    const Philox rng(f.drop);
    for (uint32_t row = blockIdx.x; row < f.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(f.x) + row * f.xs;
        const T* b = static_cast<const T*>(f.b) + row * f.bs;
        const uint64_t g0 = f.gate ? row / f.gate_rows * f.gs : 0;
        float r = 1.0f, s = 1.0f;
        if (f.w_post) {
            float sum[1] = {0.0f};
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) sum[0] += to_float(b[c]) * to_float(b[c]);
            block_sum(sum, part);
            r = rsqrtf(sum[0] / f.width + f.eps);
        }
        auto at = [&](uint32_t c) {
            float h = f.alpha * to_float(x[c]);
            if (!f.b) return h;
            float n = to_float(b[c]);
            if (f.w_post) n *= r * (f.w0 + param<T>(f.w_post, c, f.w_float));
            if (f.drop.on) n = Philox::lane(rng(c / 8, row), c % 8) < f.drop.kept ? n * f.drop.scale : 0.0f;
            if (f.gate) n *= param<T>(f.gate, g0 + c, f.g_float);
            return h + f.beta * n;
        };
        if (f.w_next) {
            float sum[1] = {0.0f};
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float h = at(c);
                sum[0] += h * h;
            }
            block_sum(sum, part);
            s = rsqrtf(sum[0] / f.width + f.eps);
        }
        for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
            const float h = at(c);
            if (f.a) static_cast<T*>(f.a)[row * f.as + c] = from_float<T>(h * s * (f.w0 + param<T>(f.w_next, c, f.w_float)));
            if (f.h) static_cast<T*>(f.h)[row * f.hs + c] = from_float<T>(h);
        }
        if (threadIdx.x == 0) {
            if (f.post_rstd) f.post_rstd[row] = r;
            if (f.next_rstd) f.next_rstd[row] = s;
        }
    }
}

// ------------------------------------------------------------------------------------------
// Backward.  The rows are cut into one contiguous run for each block; a block adds its rows' shares of the
// sums over rows into rows of its own in the workspace, and a second kernel adds the blocks' in order.  Where
// there is a gate, runs respect its rows: either a block has whole gate rows (parts == 1) and writes their
// gradients itself, or `parts` blocks share one gate row and leave their S to the second kernel.
// ------------------------------------------------------------------------------------------
struct Backward {
    const void *dh, *da, *h, *b, *w_post, *w_next, *gate;
    const float *post_rstd, *next_rstd;
    void *dx, *db, *dgate;
    uint64_t dhs, das, hs, bs, gs, dxs, dbs, dgs;
    uint32_t rows, width, gate_rows;
    bool w_float, g_float;
    float alpha, beta, w0;
    DropArgs drop;
    // partial sums, one row of `width` floats per block each; NULL: not wanted
    float *part_next, *part_post, *part_gate;
    uint32_t groups, parts;  // gate rows (1 without a gate), blocks per gate row (1: blocks take whole gate rows)
    uint32_t runs;           // blocks
};

// The rows of block `run`, gate row by gate row: calls fn(group, first, last) for each.
template <typename Fn>
__device__ __forceinline__ void for_each_segment(const Backward& f, uint32_t run, Fn&& fn) {
    if (f.parts > 1) {
        const uint32_t group = run / f.parts, part = run % f.parts;
        const uint64_t first = (uint64_t)group * f.gate_rows, n = min((uint64_t)f.gate_rows, f.rows - first);
        fn(group, (uint32_t)(first + n * part / f.parts), (uint32_t)(first + n * (part + 1) / f.parts));
    } else {
        const uint32_t begin = (uint32_t)((uint64_t)f.groups * run / f.runs);
        const uint32_t end = (uint32_t)((uint64_t)f.groups * (run + 1) / f.runs);
        for (uint32_t group = begin; group < end; ++group) {
            const uint64_t first = (uint64_t)group * f.gate_rows;
            fn(group, (uint32_t)first, (uint32_t)min(first + f.gate_rows, (uint64_t)f.rows));
        }
    }
}

// Any width, stride and alignment: the rows are read twice and the sums over rows live in the workspace.
template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_backward_any_kernel(const Backward f) {
    __shared__ float part[3 * 32];
    const Philox rng(f.drop);
    const uint64_t own = (uint64_t)blockIdx.x * f.width;
    for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
        if (f.part_next) f.part_next[own + c] = 0.0f;
        if (f.part_post) f.part_post[own + c] = 0.0f;
    }
    const bool want_s = f.part_post || f.dgate;
    for_each_segment(f, blockIdx.x, [&](uint32_t group, uint32_t first, uint32_t last) {
        auto gate = [&](uint32_t c) { return f.gate ? param<T>(f.gate, group * f.gs + c, f.g_float) : 1.0f; };
        auto post = [&](uint32_t c) { return f.w_post ? f.w0 + param<T>(f.w_post, c, f.w_float) : 1.0f; };
        if (f.part_gate)
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) f.part_gate[own + c] = 0.0f;
        for (uint32_t row = first; row < last; ++row) {
            const T* dh = static_cast<const T*>(f.dh) + row * f.dhs;
            const T* da = static_cast<const T*>(f.da) + row * f.das;
            const T* h = static_cast<const T*>(f.h) + row * f.hs;
            const T* b = static_cast<const T*>(f.b) + row * f.bs;
            const float r = f.w_post ? f.post_rstd[row] : 1.0f, s = f.w_next ? f.next_rstd[row] : 0.0f;
            auto upper = [&](uint32_t c) { return f.dh ? to_float(dh[c]) : 0.0f; };
            auto p_of = [&](uint32_t c) {
                return f.w_next ? to_float(da[c]) * (f.w0 + param<T>(f.w_next, c, f.w_float)) : 0.0f;
            };
            auto mask = [&](uint32_t c) {
                if (!f.drop.on) return f.beta;
                return Philox::lane(rng(c / 8, row), c % 8) < f.drop.kept ? f.beta * f.drop.scale : 0.0f;
            };
            float sum[3] = {0.0f, 0.0f, 0.0f};
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float p = p_of(c), hv = to_float(h[c]);
                sum[0] += p * hv;
                if (f.w_post) {
                    const float e = mask(c) * gate(c) * post(c) * to_float(b[c]);
                    sum[1] += e * (upper(c) + s * p);
                    sum[2] += e * hv;
                }
            }
            block_sum(sum, part);
            const float kappa = s * s * s * (sum[0] / f.width);
            const float c2 = (sum[1] - kappa * sum[2]) / f.width;
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float hv = to_float(h[c]);
                const float g_next = f.w_next ? to_float(da[c]) * hv * s : 0.0f;
                const float H = upper(c) + s * p_of(c) - hv * kappa;
                if (f.b) {
                    const float bv = to_float(b[c]), t = mask(c) * H, u = t * gate(c) * post(c);
                    if (f.db)
                        static_cast<T*>(f.db)[row * f.dbs + c] = from_float<T>(f.w_post ? r * u - bv * (r * r * r * c2) : u);
                    if (want_s) {
                        // one row's S at a time is enough where the run's S is not kept
                        const float S = t * (bv * r);
                        if (f.part_gate) f.part_gate[own + c] += S;
                        else if (f.part_post) f.part_post[own + c] += gate(c) * S;
                    }
                }
                if (f.dx) static_cast<T*>(f.dx)[row * f.dxs + c] = from_float<T>(f.alpha * H);
                if (f.part_next) f.part_next[own + c] += g_next;
            }
        }
        if (f.part_gate) {
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float S = f.part_gate[own + c];
                if (f.part_post) f.part_post[own + c] += gate(c) * S;
                if (f.parts == 1) {
                    const float d = post(c) * S;
                    if (f.g_float) static_cast<float*>(f.dgate)[group * f.dgs + c] = d;
                    else static_cast<T*>(f.dgate)[group * f.dgs + c] = from_float<T>(d);
                }
            }
        }
    });
}

// Adds the blocks' partial sums in order: first the plain sums (dw_next, dw_post), then each gate row's.
struct Finish {
    const float* part[2];
    float* dst[2];
    uint32_t plain;  // plain sums, `runs` partial rows each
    uint32_t runs;
    const float* part_gate;  // groups x parts partial rows
    uint32_t parts;
    void* dgate;
    uint64_t dgs;
    const void* w_post;
    uint32_t width;
    bool w_float, g_float;
    float w0;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_finish_kernel(const Finish f) {
    __shared__ float sums[kThreads / 32][32];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = kThreads / 32;
    const uint32_t c = blockIdx.x * 32 + lane;
    const bool plain = blockIdx.y < f.plain;
    const uint32_t group = blockIdx.y - f.plain, n = plain ? f.runs : f.parts;
    const float* part = plain ? f.part[blockIdx.y] : f.part_gate + (uint64_t)group * f.parts * f.width;
    float v = 0.0f;
    if (c < f.width) {
        const uint32_t end = (uint32_t)((uint64_t)n * (warp + 1) / warps);
        for (uint32_t i = (uint32_t)((uint64_t)n * warp / warps); i < end; ++i) v += part[(uint64_t)i * f.width + c];
    }
    sums[warp][lane] = v;
    __syncthreads();
    if (warp || c >= f.width) return;
    v = sums[0][lane];
#pragma unroll
    for (uint32_t i = 1; i < warps; ++i) v += sums[i][lane];
    if (plain) f.dst[blockIdx.y][c] = v;
    else {
        if (f.w_post) v *= f.w0 + param<T>(f.w_post, c, f.w_float);
        if (f.g_float) static_cast<float*>(f.dgate)[group * f.dgs + c] = v;
        else static_cast<T*>(f.dgate)[group * f.dgs + c] = from_float<T>(v);
    }
}

// Checks what both directions share; returns MTXC_OK or an error status.
int check_common(const std::string& who, int dtype, uint64_t rows, uint64_t width, bool branch, const void* post_weight,
                 const void* next_weight, const void* gate, uint64_t gate_rows, int weight_dtype, int gate_dtype) {
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (rows >> 31 || width >> 31) return fail(MTXC_ERR_SHAPE, who + ": rows and width must be below 2^31");
    if ((post_weight || next_weight) && weight_dtype != dtype && weight_dtype != MTXC_FLOAT)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": weights must have the tensors' dtype or Float");
    if (gate && gate_dtype != dtype && gate_dtype != MTXC_FLOAT)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": the gate must have the tensors' dtype or Float");
    if (rows == 0 || width == 0) return MTXC_OK;  // an empty tensor's pointer may be NULL
    if (!branch && (post_weight || gate))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": post_weight and gate need a branch");
    if (gate && gate_rows == 0) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": gate_rows must be positive");
    return MTXC_OK;
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_block_norm(int dtype, const mtxc_block_norm_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_block_norm";
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (int rc = check_common(who, dtype, a->rows, a->width, a->branch, a->post_weight, a->next_weight, a->gate,
                              a->gate_rows, a->weight_dtype, a->gate_dtype))
        return rc;
    Forward f{};
    if (int rc = drop_args(a->drop, who.c_str(), &f.drop)) return rc;
    if (a->rows == 0 || a->width == 0) {  // the mean over no elements is NaN
        for (float* r : {a->post_rstd, a->next_rstd})
            if (r && a->rows)
                if (cudaError_t err = cudaMemsetAsync(r, 0xFF, a->rows * sizeof(float), ctx().stream()); err != cudaSuccess)
                    return cuda_fail(err, "cudaMemsetAsync");
        return MTXC_OK;
    }
    if (!a->residual) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null residual");
    if ((a->normed || a->next_rstd) && !a->next_weight)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": normed and next_rstd need next_weight");
    if (a->post_rstd && !a->post_weight) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": post_rstd needs post_weight");
    f.x = a->residual;
    f.xs = a->residual_stride;
    f.b = a->branch;
    f.bs = a->branch_stride;
    f.w_post = a->post_weight;
    f.w_next = a->next_weight;
    f.gate = a->gate;
    f.gs = a->gate_stride;
    f.gate_rows = a->gate ? (uint32_t)std::min<uint64_t>(a->gate_rows, a->rows) : 1;
    f.h = a->residual_out;
    f.hs = a->residual_out_stride;
    f.a = a->normed;
    f.as = a->normed_stride;
    f.post_rstd = a->post_rstd;
    f.next_rstd = a->next_rstd;
    f.rows = (uint32_t)a->rows;
    f.width = (uint32_t)a->width;
    f.w_float = a->weight_dtype == MTXC_FLOAT;
    f.g_float = a->gate_dtype == MTXC_FLOAT;
    f.alpha = a->residual_scale;
    f.beta = a->branch_scale;
    f.w0 = a->weight_offset;
    f.eps = a->eps;
    const unsigned grid = (unsigned)std::min<uint64_t>(f.rows, (uint64_t)ctx().sm_count * 8);
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        block_norm_any_kernel<T><<<grid, kThreads, 0, ctx().stream()>>>(f);
    });
    return check_launch("block_norm_any_kernel");
}

extern "C" int mtxc_block_norm_backward(int dtype, const mtxc_block_norm_backward_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_block_norm_backward";
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (int rc = check_common(who, dtype, a->rows, a->width, a->branch, a->post_weight, a->next_weight, a->gate,
                              a->gate_rows, a->weight_dtype, a->gate_dtype))
        return rc;
    Backward f{};
    if (int rc = drop_args(a->drop, who.c_str(), &f.drop)) return rc;
    cudaStream_t st = ctx().stream();
    if (a->rows == 0 || a->width == 0) {  // sums over no rows
        for (float* d : {a->d_post_weight, a->d_next_weight})
            if (d && a->width)
                if (cudaError_t err = cudaMemsetAsync(d, 0, a->width * sizeof(float), st); err != cudaSuccess)
                    return cuda_fail(err, "cudaMemsetAsync");
        return MTXC_OK;
    }
    if (!a->d_normed != !a->next_weight)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": d_normed and next_weight go together");
    if ((a->d_branch && !a->branch) || (a->d_post_weight && !a->post_weight) || (a->d_next_weight && !a->next_weight) ||
        (a->d_gate && !a->gate))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": a gradient is asked for that the forward call has no input for");
    if (!a->residual_out && (a->next_weight || a->branch)) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null residual_out");
    if ((a->next_weight && !a->next_rstd) || (a->post_weight && !a->post_rstd))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": a norm's rstd is missing");
    f.dh = a->d_residual_out;
    f.dhs = a->d_residual_out_stride;
    f.da = a->d_normed;
    f.das = a->d_normed_stride;
    f.h = a->residual_out;
    f.hs = a->residual_out_stride;
    f.b = a->branch;
    f.bs = a->branch_stride;
    f.post_rstd = a->post_rstd;
    f.next_rstd = a->next_rstd;
    f.w_post = a->post_weight;
    f.w_next = a->next_weight;
    f.gate = a->gate;
    f.gs = a->gate_stride;
    f.dx = a->d_residual;
    f.dxs = a->d_residual_stride;
    f.db = a->d_branch;
    f.dbs = a->d_branch_stride;
    f.dgate = a->d_gate;
    f.dgs = a->d_gate_stride;
    f.rows = (uint32_t)a->rows;
    f.width = (uint32_t)a->width;
    f.gate_rows = a->gate ? (uint32_t)std::min<uint64_t>(a->gate_rows, a->rows) : f.rows;
    f.w_float = a->weight_dtype == MTXC_FLOAT;
    f.g_float = a->gate_dtype == MTXC_FLOAT;
    f.alpha = a->residual_scale;
    f.beta = a->branch_scale;
    f.w0 = a->weight_offset;

    // blocks: two per SM, as many as there are rows and the workspace holds partial sums for
    const int sums = !!a->d_next_weight + !!a->d_post_weight + !!a->d_gate;
    const uint64_t row_bytes = (uint64_t)f.width * sizeof(float) * sums;
    uint64_t runs = std::min<uint64_t>(f.rows, (uint64_t)ctx().sm_count * 2);
    if (row_bytes) runs = std::min<uint64_t>(runs, ctx().workspace_bytes / row_bytes);
    if (runs == 0)
        return fail(MTXC_ERR_WORKSPACE, who + ": one block's partial sums need " + std::to_string(row_bytes) +
                                            " bytes of workspace, the thread has " + std::to_string(ctx().workspace_bytes));
    f.groups = (uint32_t)(((uint64_t)f.rows + f.gate_rows - 1) / f.gate_rows);
    f.parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(runs / f.groups, f.gate_rows));
    f.runs = f.parts > 1 ? f.groups * f.parts : (uint32_t)std::min<uint64_t>(runs, f.groups);
    float* ws = static_cast<float*>(ctx().workspace);
    auto take = [&](bool wanted) {
        float* p = wanted ? ws : nullptr;
        if (wanted) ws += (uint64_t)f.runs * f.width;
        return p;
    };
    f.part_next = take(a->d_next_weight);
    f.part_post = take(a->d_post_weight);
    f.part_gate = take(a->d_gate);
    Finish e{};
    if (f.part_next) e.part[e.plain] = f.part_next, e.dst[e.plain++] = a->d_next_weight;
    if (f.part_post) e.part[e.plain] = f.part_post, e.dst[e.plain++] = a->d_post_weight;
    e.runs = f.runs;
    e.part_gate = f.part_gate;
    e.parts = f.parts;
    e.dgate = f.dgate;
    e.dgs = f.dgs;
    e.w_post = f.w_post;
    e.width = f.width;
    e.w_float = f.w_float;
    e.g_float = f.g_float;
    e.w0 = f.w0;
    const uint32_t jobs = e.plain + (f.part_gate && f.parts > 1 ? f.groups : 0);
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        block_norm_backward_any_kernel<T><<<f.runs, kThreads, 0, st>>>(f);
        if (jobs) block_norm_finish_kernel<T><<<dim3((f.width + 31) / 32, jobs), kThreads, 0, st>>>(e);
    });
    return check_launch("block_norm_backward");
}
