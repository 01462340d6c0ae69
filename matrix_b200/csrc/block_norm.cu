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
// A deviation's cube passes the range of 32 bits where a row's root mean square passes 1e12 either way, and the
// gradients do not: kappa is made one factor at a time, and b r^3 mean(u b) as (b r) (r (r mean(u b))).
#include <algorithm>

#include <cooperative_groups.h>

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

// ------------------------------------------------------------------------------------------
// A thread's share of a row: chunks of eight elements.  VEC: eight consecutive columns, one access per chunk
// (16 bytes of a half type, 32 of float); else a warp takes 256 consecutive columns and a lane every 32nd of
// them, so that scalar accesses of rows of any width and alignment are contiguous across the warp.
// ------------------------------------------------------------------------------------------
template <typename T, bool VEC>
struct Chunk {
    uint32_t c;  // first column
    // chunk k of thread `tid` of `threads` that share the columns from `from` (a multiple of 256)
    __device__ __forceinline__ Chunk(uint32_t k, uint32_t threads, uint32_t tid, uint32_t from = 0)
        : c(from + (VEC ? (k * threads + tid) * 8 : (k * threads + (tid & ~31u)) * 8 + tid % 32)) {}
    __device__ __forceinline__ uint32_t column(int j) const { return VEC ? c + j : c + 32 * j; }
    // whether element j lies in the row (VEC: all eight do or none)
    __device__ __forceinline__ bool inside(int j, uint32_t width) const { return VEC ? c < width : c + 32 * j < width; }

    // whether the warp's 256 columns all lie in the row: then scalar accesses need no comparisons, which were a
    // third of the instructions of a row of half types
    __device__ __forceinline__ bool whole(uint32_t width) const { return c - threadIdx.x % 32 + 256 <= width; }

    __device__ __forceinline__ Eight<T> load(const T* row, uint32_t width) const {
        Eight<T> v;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)(2 * sizeof(T)); ++i) v.w[i] = 0;
            if (c < width) v.load(row + c);
        } else {
            T e[8];
            const T* p = row + c;
            if (whole(width)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = p[32 * j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = inside(j, width) ? p[32 * j] : T(0.0f);
            }
            memcpy(v.w, e, sizeof(e));
        }
        return v;
    }
    __device__ __forceinline__ void store(T* row, uint32_t width, const float2 (&v)[4]) const {
        Eight<T> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o.set2(j, v[j].x, v[j].y);
        if constexpr (VEC) {
            if (c < width) o.store(row + c);
        } else {
            T e[8];
            memcpy(e, o.w, sizeof(e));
            T* p = row + c;
            if (whole(width)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[32 * j] = e[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (inside(j, width)) p[32 * j] = e[j];
            }
        }
    }
    // Eight values of a weight or gate row, shared by many rows and so left in L1 (0 outside the row).
    __device__ __forceinline__ void param(const void* p, uint64_t at, bool is_float, uint32_t width, float2 (&v)[4]) const {
        if constexpr (VEC) {
            if (c >= width) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = make_float2(0.0f, 0.0f);
            } else if (std::is_same_v<T, float> || is_float) {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + c);
                const float4 a = __ldg(q), b = __ldg(q + 1);
                v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w);
                v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
            } else if constexpr (sizeof(T) == 2) {
                const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + at + c));
                const Eight<T> e{{a.x, a.y, a.z, a.w}};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = e.get2(j);
            }
        } else {
            auto all = [&](auto* q) {
                q += at + c;
                if (whole(width)) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = make_float2(to_float(q[64 * j]), to_float(q[64 * j + 32]));
                } else {
                    auto one = [&](int j) { return inside(j, width) ? to_float(q[32 * j]) : 0.0f; };
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = make_float2(one(2 * j), one(2 * j + 1));
                }
            };
            if (is_float) all(static_cast<const float*>(p));
            else all(static_cast<const T*>(p));
        }
    }
    // The column block whose counter this lane makes: its own, or one of the warp's 32.
    __device__ __forceinline__ uint32_t block() const { return VEC ? c / 8 : c / 8 - threadIdx.x % 32 / 8 + threadIdx.x % 32; }
};

// Zeroes the dropped ones of a thread's K chunks of a row; the whole warp takes part.  Counters are made two
// at a time: more would hold too many registers.
template <typename T, bool VEC, int K>
__device__ __forceinline__ void drop(const DropArgs& d, uint32_t row, uint32_t threads, uint32_t tid, float2 (&v)[K][4]) {
    constexpr int N = K < 2 ? K : 2;
    const Philox rng(d);
    const uint32_t lane = threadIdx.x % 32;
#pragma unroll
    for (int k = 0; k < K; k += N) {
        uint32_t block[N], rows[N];
#pragma unroll
        for (int i = 0; i < N; ++i) block[i] = Chunk<T, VEC>(k + i, threads, tid).block(), rows[i] = row;
        Lanes l[N];
        rng.make(block, rows, l);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[k + i][j].x = l[i].keeps(d, 2 * j) ? v[k + i][j].x : 0.0f;
                    v[k + i][j].y = l[i].keeps(d, 2 * j + 1) ? v[k + i][j].y : 0.0f;
                }
            } else {  // each lane's eight bits go to the eight lanes that hold their columns
                uint32_t own = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) own |= l[i].keeps(d, j) ? 1u << j : 0u;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t bits = __shfl_sync(0xffffffffu, own, j * 4 + lane / 8);
                    float& e = j % 2 ? v[k + i][j / 2].y : v[k + i][j / 2].x;
                    e = bits >> (lane % 8) & 1u ? e : 0.0f;
                }
            }
        }
    }
}

// Which of a thread's K chunks of a row are kept, held for several uses: the lanes themselves where a chunk is one
// counter's columns, else bits.  The whole warp makes them.
template <typename T, int K, bool VEC>
struct Kept {
    Lanes lanes[VEC ? K : 1];
    uint32_t bits = 0;

    __device__ __forceinline__ void make(const DropArgs& d, uint32_t row, uint32_t threads, uint32_t tid, uint32_t from) {
        const Philox rng(d);
        uint32_t block[K], rows[K];
#pragma unroll
        for (int k = 0; k < K; ++k) block[k] = Chunk<T, VEC>(k, threads, tid, from).block(), rows[k] = row;
        if constexpr (VEC) rng.make(block, rows, lanes);
        else {
            Lanes l[K];
            rng.make(block, rows, l);
            uint32_t own = 0;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) own |= l[k].keeps(d, j) ? 1u << (8 * k + j) : 0u;
            const uint32_t lane = threadIdx.x % 32;
            bits = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // each lane's bits go to the eight lanes that hold their columns
                const uint32_t from = __shfl_sync(0xffffffffu, own, j * 4 + lane / 8) >> (lane % 8);
#pragma unroll
                for (int k = 0; k < K; ++k) bits |= (from >> (8 * k) & 1u) << (8 * k + j);
            }
        }
    }
    __device__ __forceinline__ bool at(const DropArgs& d, int k, int j) const {
        if constexpr (VEC) return lanes[k].keeps(d, j);
        else return bits >> (8 * k + j) & 1u;
    }
    __device__ __forceinline__ void zero_others(const DropArgs& d, int k, Eight<T>& v) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (sizeof(T) == 4) v.w[j] = at(d, k, j) ? v.w[j] : 0;
            else v.w[j / 2] &= at(d, k, j) ? 0xFFFFFFFFu : j % 2 ? 0xFFFFu : 0xFFFF0000u;
        }
    }
    __device__ __forceinline__ void zero_others(const DropArgs& d, int k, float2 (&v)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j].x = at(d, k, 2 * j) ? v[j].x : 0.0f;
            v[j].y = at(d, k, 2 * j + 1) ? v[j].y : 0.0f;
        }
    }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Sums N values over the threads that share a row: a warp (part unused), or a team of `threads` (a block, or several
// warps of one that have a named barrier of their own) through part[N][32], which no earlier sum of the row has used.
template <int N, bool WARP>
__device__ __forceinline__ void row_sum(float (&v)[N], float* part, uint32_t threads, uint32_t team) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if constexpr (!WARP) {
        const uint32_t lane = threadIdx.x % 32, warps = threads / 32, base = team * warps;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[i * 32 + threadIdx.x / 32] = v[i];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? part[i * 32 + base + lane] : 0.0f);
    }
}

// Rows held in registers, E elements per thread: read once, written once.  WARP: a warp per row, eight rows per
// block; else a block per row.  Bound by HBM without dropout ([8192, 4096] bf16 43 us, 6.2 TB/s).  With it neither
// issue (61 %) nor HBM is full: a block's phases follow one another, and the mask is made after the first reduction,
// when little is on its way ([8192, 8192] bf16 with a gate per channel 108 us, 5.0 TB/s).  A grid of resident blocks that
// copies the next row ahead was slower (47 -> 51 us, 109 -> 122): more blocks hide a row's two reductions better.
template <typename T, int E, bool VEC, bool WARP, int BLOCK, int MIN>
__global__ void __launch_bounds__(BLOCK, MIN) block_norm_kernel(const Forward f) {
    constexpr int K = E / 8;
    __shared__ float part[2][32];
    const uint32_t threads = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x % 32 : threadIdx.x;
    const uint32_t row = WARP ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (WARP && row >= f.rows) return;
    const uint32_t width = f.width;
    Eight<T> x[K];
    float2 h[K][4];  // first the branch, stage by stage, then h; arithmetic two elements at a time
    if (f.b) {
        Eight<T> b[K];
#pragma unroll
        for (int k = 0; k < K; ++k)
            b[k] = Chunk<T, VEC>(k, threads, tid).load(static_cast<const T*>(f.b) + row * f.bs, width);
#pragma unroll
        for (int k = 0; k < K; ++k)
            x[k] = Chunk<T, VEC>(k, threads, tid).load(static_cast<const T*>(f.x) + row * f.xs, width);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) h[k][j] = b[k].get2(j);
        if (f.w_post) {
            float2 q = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) q = __ffma2_rn(h[k][j], h[k][j], q);
            float sum[1] = {q.x + q.y};
            row_sum<1, WARP>(sum, part[0], threads, 0);
            const float r = rsqrtf(sum[0] / width + f.eps);
            if (f.post_rstd && tid == 0) f.post_rstd[row] = r;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float2 w[4];
                Chunk<T, VEC>(k, threads, tid).param(f.w_post, 0, f.w_float, width, w);
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = __fmul2_rn(h[k][j], __ffma2_rn(both(r), w[j], both(r * f.w0)));
            }
        }
        float beta = f.beta;
        if (f.drop.on) {
            beta *= f.drop.scale;
            drop<T, VEC>(f.drop, row, threads, tid, h);
        }
        if (f.gate) {
            const uint64_t g0 = row / f.gate_rows * f.gs;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float2 w[4];
                Chunk<T, VEC>(k, threads, tid).param(f.gate, g0, f.g_float, width, w);
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = __fmul2_rn(h[k][j], w[j]);
            }
        }
        if (f.alpha == 1.0f) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = __ffma2_rn(both(beta), h[k][j], x[k].get2(j));
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = __ffma2_rn(both(beta), h[k][j], __fmul2_rn(both(f.alpha), x[k].get2(j)));
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
            x[k] = Chunk<T, VEC>(k, threads, tid).load(static_cast<const T*>(f.x) + row * f.xs, width);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) h[k][j] = __fmul2_rn(both(f.alpha), x[k].get2(j));
    }
    if (f.h) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            Chunk<T, VEC>(k, threads, tid).store(static_cast<T*>(f.h) + row * f.hs, width, h[k]);
    }
    if (!f.w_next) return;
    float2 q = both(0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) q = __ffma2_rn(h[k][j], h[k][j], q);
    float sum[1] = {q.x + q.y};
    row_sum<1, WARP>(sum, part[1], threads, 0);
    const float s = rsqrtf(sum[0] / width + f.eps);
    if (f.a) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Chunk<T, VEC> ch(k, threads, tid);
            float2 w[4];
            ch.param(f.w_next, 0, f.w_float, width, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[k][j] = __fmul2_rn(h[k][j], __ffma2_rn(both(s), w[j], both(s * f.w0)));
            ch.store(static_cast<T*>(f.a) + row * f.as, width, h[k]);
        }
    }
    if (f.next_rstd && tid == 0) f.next_rstd[row] = s;
}

// Elements per thread E, threads and blocks per SM (measured on a B200, the best against the next):
//   a warp per row to 256 columns, and to 512 for vectors of half types ([32768, 512] bf16 5446 GB/s, a block 4699)
//   few elements, up to 10,240 per SM: E = 8, the shortest way through one row ([300, 2048] bf16 3.2 us on the device,
//     E = 16 3.6, E = 32 4.4; [300, 8192], which is more, 7.8, 6.4 and 6.0)
//   half types, vectors: E = 16 to 1024 columns ([16384, 1024] bf16 with dropout 4471 GB/s, E = 8 3847, a warp 3902) and
//     up to 57,344 elements per SM ([2000, 4096] 13.3 us, E = 32 13.6, E = 8 14.7; [4000, 4096] 26.9, 22.9, 28.5), then
//     32, whose blocks hold more of a row in their registers ([16384, 2048] 5647 GB/s, E = 16 5352, E = 8 4722)
//   float, and scalar accesses: E = 8 to 4096 ([16384, 2047] bf16 2780 GB/s, E = 16 2563, E = 32 1320), which needs
//     the fewest registers, then 16 ([8192, 4097] bf16 2893, E = 8 in blocks of 1024 2340)
// Wider rows return -1.
template <typename T, bool VEC>
int launch_forward(const Forward& f, cudaStream_t st, int sms) {
    auto threads = [&](uint32_t e) { return (f.width + 32 * e - 1) / (32 * e) * 32; };
    const unsigned warps = (f.rows + 7) / 8;
    const uint64_t per_sm = (uint64_t)f.rows * f.width / sms;
    constexpr bool kHalfVec = VEC && sizeof(T) == 2;
    if (f.width <= 256) block_norm_kernel<T, 8, VEC, true, 256, 1><<<warps, 256, 0, st>>>(f);
    else if (f.width > 16384) return -1;
    else if (f.width <= 8192 && per_sm <= 10240) block_norm_kernel<T, 8, VEC, false, 1024, 1><<<f.rows, threads(8), 0, st>>>(f);
    else if constexpr (kHalfVec) {
        if (f.width <= 512) block_norm_kernel<T, 16, VEC, true, 256, 1><<<warps, 256, 0, st>>>(f);
        else if (f.width <= 1024 || per_sm <= 57344) block_norm_kernel<T, 16, VEC, false, 1024, 1><<<f.rows, threads(16), 0, st>>>(f);
        else if (f.width <= 8192) block_norm_kernel<T, 32, VEC, false, 256, 3><<<f.rows, threads(32), 0, st>>>(f);
        else block_norm_kernel<T, 32, VEC, false, 512, 2><<<f.rows, threads(32), 0, st>>>(f);
    } else {
        if (f.width <= 4096) block_norm_kernel<T, 8, VEC, false, 512, 3><<<f.rows, threads(8), 0, st>>>(f);
        else block_norm_kernel<T, 16, VEC, false, 1024, 1><<<f.rows, threads(16), 0, st>>>(f);
    }
    return check_launch("block_norm_kernel");
}

// Any width (in use: above 16,384), stride and alignment: a block per row, which reads its row once for each sum.
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
            if (f.drop.on) n = rng(c / 8, row).at(c % 8) < f.drop.kept ? n * f.drop.scale : 0.0f;
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
// Backward.  The rows are cut into contiguous runs, one for each team of threads (a block, or a part of one); a
// block leaves its teams' sums over rows as one row of partial sums in the workspace, and a second kernel adds the
// blocks' in order.  Where there is a gate, runs respect its rows: either a run has whole gate rows (parts == 1) and
// writes their gradients itself, or `parts` runs share one gate row and leave their S to the second kernel.
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
    // partial sums, one row of `width` floats per block each; NULL: not wanted.  Where runs share gate rows there is
    // no part_post: S, in part_gate, gives both sums.
    float *part_next, *part_post, *part_gate;
    uint32_t groups, parts;  // gate rows (1 without a gate), runs per gate row (1: runs take whole gate rows)
    uint32_t runs;
    uint32_t cluster, cols;  // blocks that share a row, and a block's columns
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

// Any width (in use: above 65,536, and where a gradient is written over a gate per token that the post weight's
// gradient needs, which is here read before the row's stores), stride and alignment: the rows are read twice and the
// sums over rows live in the workspace.
template <typename T>
__global__ void __launch_bounds__(kThreads) block_norm_backward_any_kernel(const Backward f) {
    __shared__ float part[3 * 32];
    const Philox rng(f.drop);
    const uint64_t own = (uint64_t)blockIdx.x * f.width;
    for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
        if (f.part_next) f.part_next[own + c] = 0.0f;
        if (f.part_post) f.part_post[own + c] = 0.0f;
    }
    const bool want_s = f.part_post || f.part_gate;
    const float cf = f.drop.on ? f.beta * f.drop.scale : f.beta;
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
            auto stream = [&](uint32_t c) { return f.w_next ? to_float(h[c]) : 0.0f; };  // serves the next norm alone
            auto p_of = [&](uint32_t c) {
                return f.w_next ? to_float(da[c]) * (f.w0 + param<T>(f.w_next, c, f.w_float)) : 0.0f;
            };
            auto keeps = [&](uint32_t c) { return !f.drop.on || rng(c / 8, row).at(c % 8) < f.drop.kept; };
            float sum[3] = {0.0f, 0.0f, 0.0f};
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float p = p_of(c), hv = stream(c);
                sum[0] += p * hv;
                if (f.w_post) {
                    const float e = keeps(c) ? cf * gate(c) * post(c) * to_float(b[c]) : 0.0f;
                    sum[1] += e * (upper(c) + s * p);
                    sum[2] += e * hv;
                }
            }
            block_sum(sum, part);
            const float kappa = s * (s * (s * (sum[0] / f.width)));
            const float c2 = r * (r * ((sum[1] - kappa * sum[2]) / f.width));
            const bool ends = f.part_gate && row + 1 == last;
            for (uint32_t c = threadIdx.x; c < f.width; c += kThreads) {
                const float hv = stream(c), g = gate(c);
                const float g_next = f.w_next ? to_float(da[c]) * hv * s : 0.0f;
                const float H = upper(c) + s * p_of(c) - hv * kappa;
                if (f.b) {
                    // what is dropped may be infinite or NaN: a zero all the same
                    const bool kept = keeps(c);
                    const float bv = to_float(b[c]), t = kept ? cf * H : 0.0f, w = post(c), u = t * g * w;
                    if (f.db)
                        static_cast<T*>(f.db)[row * f.dbs + c] = from_float<T>(f.w_post ? r * u - (bv * r) * c2 : u);
                    if (want_s) {
                        // one row's S at a time is enough where the run's S is not kept
                        float S = kept ? t * (bv * r) : 0.0f;
                        if (f.part_gate) S = f.part_gate[own + c] += S;
                        if (f.part_post && (ends || !f.part_gate)) f.part_post[own + c] += g * S;
                        if (ends && f.parts == 1) {
                            if (f.g_float) static_cast<float*>(f.dgate)[group * f.dgs + c] = w * S;
                            else static_cast<T*>(f.dgate)[group * f.dgs + c] = from_float<T>(w * S);
                        }
                    }
                }
                if (f.dx) static_cast<T*>(f.dx)[row * f.dxs + c] = from_float<T>(f.alpha * H);
                if (f.part_next) f.part_next[own + c] += g_next;
            }
        }
    });
}

constexpr uint32_t kMaxCluster = 8;

// The rows of a run: contiguous, so that the next ones can be fetched ahead across gate rows.
__device__ __forceinline__ void run_rows(const Backward& f, uint32_t run, uint32_t& first, uint32_t& last) {
    if (f.parts > 1) {
        const uint64_t start = (uint64_t)(run / f.parts) * f.gate_rows, n = min((uint64_t)f.gate_rows, f.rows - start);
        const uint32_t part = run % f.parts;
        first = (uint32_t)(start + n * part / f.parts);
        last = (uint32_t)(start + n * (part + 1) / f.parts);
    } else {
        first = (uint32_t)((uint64_t)f.groups * run / f.runs * f.gate_rows);
        last = (uint32_t)min((uint64_t)f.groups * (run + 1) / f.runs * f.gate_rows, (uint64_t)f.rows);
    }
}

__device__ __forceinline__ void copy16(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// The four rows that a row of the backward pass reads, as one thread's chunks.  VEC: copied to shared memory
// `stages` rows ahead by the thread that reads them, which therefore needs no barrier; else in registers.
template <typename T, int K, bool VEC>
struct Inputs {
    static constexpr int kPieces = sizeof(Eight<T>) / 16;
    uint4* ring;  // this thread's first slot; slots of a block's threads lie side by side
    uint32_t stride;
    Eight<T> regs[VEC ? 1 : 4][VEC ? 1 : K];

    // h serves the next norm alone (and the post norm's sums where there is one): without it, it is not read
    __device__ __forceinline__ static const T* base(const Backward& f, int i) {
        return static_cast<const T*>(i == 0 ? f.dh : i == 1 ? f.da : i == 2 ? (f.w_next ? f.h : nullptr) : f.b);
    }
    __device__ __forceinline__ static uint64_t row_stride(const Backward& f, int i) {
        return i == 0 ? f.dhs : i == 1 ? f.das : i == 2 ? f.hs : f.bs;
    }
    // Zeros for what is never fetched: absent rows, and chunks outside the row.
    __device__ __forceinline__ void absent(const Backward& f, uint32_t stages) {
        if constexpr (VEC) {
            for (uint32_t i = 0; i < stages * 4 * K * kPieces; ++i) ring[i * stride] = make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < K; ++k) regs[i][k] = Eight<T>{};
        }
    }
    __device__ __forceinline__ void fetch(const Backward& f, uint32_t row, uint32_t stage, uint32_t threads, uint32_t tid,
                                          uint32_t from, uint32_t limit) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T* p = base(f, i);
            if (!p) continue;
            p += row * row_stride(f, i);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Chunk<T, VEC> ch(k, threads, tid, from);
                if constexpr (VEC) {
                    if (ch.c >= limit) continue;
#pragma unroll
                    for (int v = 0; v < kPieces; ++v)
                        copy16(ring + (((stage * 4 + i) * K + k) * kPieces + v) * stride,
                               reinterpret_cast<const uint4*>(p + ch.c) + v);
                } else regs[i][k] = ch.load(p, limit);
            }
        }
    }
    __device__ __forceinline__ Eight<T> get(int i, int k, uint32_t stage) const {
        if constexpr (VEC) {
            Eight<T> e;
#pragma unroll
            for (int v = 0; v < kPieces; ++v) {
                const uint4 q = ring[(((stage * 4 + i) * K + k) * kPieces + v) * stride];
                e.w[4 * v] = q.x, e.w[4 * v + 1] = q.y, e.w[4 * v + 2] = q.z, e.w[4 * v + 3] = q.w;
            }
            return e;
        } else return regs[i][k];
    }
    __device__ __forceinline__ void put(int i, int k, uint32_t stage, const Eight<T>& e) {
        if constexpr (VEC) {
#pragma unroll
            for (int v = 0; v < kPieces; ++v)
                ring[(((stage * 4 + i) * K + k) * kPieces + v) * stride] =
                    make_uint4(e.w[4 * v], e.w[4 * v + 1], e.w[4 * v + 2], e.w[4 * v + 3]);
        } else regs[i][k] = e;
    }
};

// A thread's share of a partial-sum row.
template <typename T, bool VEC>
__device__ __forceinline__ void store_sums(const Chunk<T, VEC>& ch, float* row, uint32_t width, const float2 (&v)[4]) {
    if constexpr (VEC) {
        if (ch.c >= width) return;
        float4* p = reinterpret_cast<float4*>(row + ch.c);
        p[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        p[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (ch.inside(j, width)) row[ch.column(j)] = j % 2 ? v[j / 2].y : v[j / 2].x;
    }
}

// Rows read once: E elements per thread, the sums over rows in registers.  A run of rows for each team: a warp
// (WARP), or `threads` threads; a block's teams add their sums in shared memory, so that there is one row of
// partial sums for each block.  MULTI: a run has whole gate rows and writes their gradients; else it has (part of)
// one gate row.  CLUSTER: a row's columns are shared by the blocks of a cluster (one team each), f.cols to a
// block, which exchange their sums through distributed shared memory: one cluster barrier per row.  A thread keeps
// its columns' w_next' and gate * w_post' in shared memory, as floats ready for use, for the run (or the gate
// row).  Inputs that the call does not have read as zeros, weights as ones: fewer branches.  Bound by latency at
// 16 warps per SM (vectors of half types at 4,096 and 8,192 columns; 9 to 14 at most widths between): [8192, 4096] bf16
// with gate and dropout 89 us with the finish, 4.5 TB/s.  The kernels of scalar accesses hold 64 registers and spill
// (up to 490 bytes with several gate rows a run), as those of a warp per row with several gate rows do at 128.
template <typename T, int E, bool VEC, bool WARP, bool MULTI, bool CLUSTER, int BLOCK, int MIN>
__global__ void __launch_bounds__(BLOCK, MIN) block_norm_backward_kernel(const Backward f, uint32_t team_threads, uint32_t stages) {
    constexpr int K = E / 8;
    extern __shared__ uint4 ring[];
    __shared__ float part[2][3 * 32];
    __shared__ float from_rank[2][kMaxCluster][3];  // CLUSTER: the blocks' sums of a row
    const uint32_t threads = WARP ? 32 : team_threads, teams = blockDim.x / threads;
    const uint32_t team = threadIdx.x / threads, tid = threadIdx.x - team * threads;
    const uint32_t rank = CLUSTER ? blockIdx.x % f.cluster : 0;
    const uint32_t run = CLUSTER ? blockIdx.x / f.cluster : blockIdx.x * teams + team;
    const uint32_t from = CLUSTER ? rank * f.cols : 0, limit = CLUSTER ? min(f.width, from + f.cols) : f.width;
    const bool has_b = f.b, has_post = f.w_post, has_next = f.w_next, has_gate = f.gate, drops = f.drop.on && has_b;
    const bool want_s = f.part_post || f.dgate;
    const float cf = drops ? f.beta * f.drop.scale : f.beta;
    uint32_t first = 0, last = 0;
    if (run < f.runs) run_rows(f, run, first, last);
    uint32_t group = first / f.gate_rows, group_left = f.gate_rows - first % f.gate_rows;

    Inputs<T, K, VEC> in;
    in.ring = ring + threadIdx.x;
    in.stride = blockDim.x;
    uint4* const weights = in.ring + (VEC ? stages * 4 * K * Inputs<T, K, VEC>::kPieces : 0) * blockDim.x;
    in.absent(f, stages);
    if constexpr (VEC) {
        for (uint32_t i = 0; i < stages; ++i) {
            if (first + i < last) in.fetch(f, first + i, i, threads, tid, from, limit);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    // which = 0: w_next', 1: gate * w_post'
    auto make_weights = [&](int which, int k, float2 (&w)[4]) {
        const Chunk<T, VEC> ch(k, threads, tid, from);
        const void* p = which ? f.w_post : f.w_next;
        if (p) {
            ch.param(p, 0, f.w_float, limit, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __fadd2_rn(both(f.w0), w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = both(1.0f);
        }
        if (which && has_gate) {
            float2 g[4];
            ch.param(f.gate, group * f.gs, f.g_float, limit, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __fmul2_rn(g[j], w[j]);
        }
    };
    auto keep_weights = [&](int which) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float2 w[4];
            make_weights(which, k, w);
            float4* q = reinterpret_cast<float4*>(weights + (which * K + k) * 2 * blockDim.x);
            q[0] = make_float4(w[0].x, w[0].y, w[1].x, w[1].y);
            q[blockDim.x] = make_float4(w[2].x, w[2].y, w[3].x, w[3].y);
        }
    };
    auto get_weights = [&](int which, int k, float2 (&w)[4]) {
        const float4* q = reinterpret_cast<const float4*>(weights + (which * K + k) * 2 * blockDim.x);
        const float4 a = q[0], b = q[blockDim.x];
        w[0] = make_float2(a.x, a.y), w[1] = make_float2(a.z, a.w);
        w[2] = make_float2(b.x, b.y), w[3] = make_float2(b.z, b.w);
    };
    keep_weights(0), keep_weights(1);

    float2 A[K][4], S[K][4], W[MULTI ? K : 1][4];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            A[k][j] = S[k][j] = both(0.0f);
            if (MULTI) W[k][j] = both(0.0f);
        }
    // the next row's deviations are on their way while a row is worked on
    float next_r = 1.0f, next_s = 0.0f;
    auto load_rstd = [&](uint32_t row) {
        if (has_post) next_r = __ldg(f.post_rstd + row);
        if (has_next) next_s = __ldg(f.next_rstd + row);
    };
    if (first < last) load_rstd(first);
    if constexpr (CLUSTER) cooperative_groups::this_cluster().sync();  // every block runs before the first is written to
    for (uint32_t row = first, stage = 0; row < last; ++row) {
        const float r = next_r, s = next_s;
        if (row + 1 < last) load_rstd(row + 1);
        if constexpr (VEC) {
            if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
        } else in.fetch(f, row, 0, threads, tid, from, limit);
        // a gate row that ends with this row: the next one's way from HBM starts now
        if (MULTI && group_left == 1 && row + 1 < last) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Chunk<T, VEC> ch(k, threads, tid, from);
                const uint64_t at = (group + 1) * f.gs + ch.c;
                const void* p = f.g_float ? static_cast<const void*>(static_cast<const float*>(f.gate) + at)
                                          : static_cast<const void*>(static_cast<const T*>(f.gate) + at);
                if (ch.c < limit) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
            }
        }
        Kept<T, K, VEC> kept;
        if (drops) {
            kept.make(f.drop, row, threads, tid, from);
            // What is dropped may be infinite or NaN: a zero to the gate's sums below all the same.  (With a post norm such
            // an element has spoilt its whole row's deviation already.)
            if (want_s && !has_post) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    Eight<T> b = in.get(3, k, stage);
                    kept.zero_others(f.drop, k, b);
                    in.put(3, k, stage, b);
                }
            }
        }
        float2 c1 = both(0.0f), su = both(0.0f), sv = both(0.0f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Eight<T> dh = in.get(0, k, stage), da = in.get(1, k, stage), h = in.get(2, k, stage),
                           b = in.get(3, k, stage);
            float2 p[4], e[4];
            get_weights(0, k, p);
            get_weights(1, k, e);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[j] = __fmul2_rn(da.get2(j), p[j]);
                e[j] = __fmul2_rn(b.get2(j), e[j]);
            }
            if (drops) kept.zero_others(f.drop, k, e);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c1 = __ffma2_rn(p[j], h.get2(j), c1);
                su = __ffma2_rn(e[j], __ffma2_rn(both(s), p[j], dh.get2(j)), su);
                sv = __ffma2_rn(e[j], h.get2(j), sv);
            }
        }
        float sum[3] = {c1.x + c1.y, su.x + su.y, sv.x + sv.y};
        row_sum<3, WARP>(sum, part[(row - first) % 2], threads, team);
        if constexpr (CLUSTER) {
            // double buffered like part: a block that writes a row's slots again has passed the barrier of the row
            // between
            cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            float(&slots)[kMaxCluster][3] = from_rank[(row - first) % 2];
            if (threadIdx.x < f.cluster) {
                float* to = cluster.map_shared_rank(slots[rank], threadIdx.x);
                to[0] = sum[0], to[1] = sum[1], to[2] = sum[2];
            }
            cluster.sync();
            sum[0] = sum[1] = sum[2] = 0.0f;
            for (uint32_t i = 0; i < f.cluster; ++i) sum[0] += slots[i][0], sum[1] += slots[i][1], sum[2] += slots[i][2];
        }
        const float kappa = s * (s * (s * (sum[0] / f.width)));
        const float c2 = r * (r * (cf * (sum[1] - kappa * sum[2]) / f.width));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Chunk<T, VEC> ch(k, threads, tid, from);
            const Eight<T> dh = in.get(0, k, stage), da = in.get(1, k, stage), h = in.get(2, k, stage),
                           b = in.get(3, k, stage);
            float2 H[4], w[4], o[4];
            get_weights(0, k, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 d = __fmul2_rn(both(s), da.get2(j));
                A[k][j] = __ffma2_rn(d, h.get2(j), A[k][j]);
                H[j] = __ffma2_rn(d, w[j], __ffma2_rn(both(-kappa), h.get2(j), dh.get2(j)));
                o[j] = __fmul2_rn(both(f.alpha), H[j]);
            }
            if (f.dx) ch.store(static_cast<T*>(f.dx) + row * f.dxs, limit, o);
            if (!has_b) continue;
            if (drops) kept.zero_others(f.drop, k, H);
            get_weights(1, k, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                H[j] = __fmul2_rn(both(cf * r), H[j]);
                S[k][j] = __ffma2_rn(H[j], b.get2(j), S[k][j]);
                H[j] = __fmul2_rn(H[j], w[j]);
            }
            if (has_post) {
#pragma unroll
                for (int j = 0; j < 4; ++j) H[j] = __ffma2_rn(both(-c2), __fmul2_rn(both(r), b.get2(j)), H[j]);
            }
            if (f.db) ch.store(static_cast<T*>(f.db) + row * f.dbs, limit, H);
        }
        if constexpr (VEC) {
            if (row + stages < last) in.fetch(f, row + stages, stage, threads, tid, from, limit);
            asm volatile("cp.async.commit_group;" ::: "memory");
            stage = stage + 1 == stages ? 0 : stage + 1;
        }
        if (MULTI && (--group_left == 0 || row + 1 == last)) {  // the last of the gate row's rows in this run
            if (want_s) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const Chunk<T, VEC> ch(k, threads, tid, from);
                    float2 w[4];
                    ch.param(f.gate, group * f.gs, f.g_float, limit, w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) W[MULTI ? k : 0][j] = __ffma2_rn(w[j], S[k][j], W[MULTI ? k : 0][j]);
                    if (f.dgate) {
                        if (has_post) {
                            ch.param(f.w_post, 0, f.w_float, limit, w);
#pragma unroll
                            for (int j = 0; j < 4; ++j) S[k][j] = __fmul2_rn(S[k][j], __fadd2_rn(both(f.w0), w[j]));
                        }
                        if (f.g_float) store_sums(ch, static_cast<float*>(f.dgate) + group * f.dgs, limit, S[k]);
                        else ch.store(static_cast<T*>(f.dgate) + group * f.dgs, limit, S[k]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) S[k][j] = both(0.0f);
                }
            }
            if (row + 1 < last) {
                ++group, group_left = f.gate_rows;
                keep_weights(1);
            }
        }
    }
    if constexpr (VEC) asm volatile("cp.async.wait_all;" ::: "memory");
    float* const out_a = f.part_next ? f.part_next + (uint64_t)(CLUSTER ? run : blockIdx.x) * f.width : nullptr;
    float* out_s = MULTI || !f.part_gate ? f.part_post : f.part_gate;
    if (out_s) out_s += (uint64_t)(CLUSTER ? run : blockIdx.x) * f.width;
    if (CLUSTER || teams == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Chunk<T, VEC> ch(k, threads, tid, from);
            if (out_a) store_sums(ch, out_a, limit, A[k]);
            if (out_s) store_sums(ch, out_s, limit, MULTI ? W[MULTI ? k : 0] : S[k]);
        }
        return;
    }
    // each thread's sums into its own slots of the weights, then piece by piece over the teams, in order
    float4* const own = reinterpret_cast<float4*>(weights);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const float2(&v)[4] = MULTI ? W[MULTI ? k : 0] : S[k];
        own[(2 * k) * blockDim.x] = make_float4(A[k][0].x, A[k][0].y, A[k][1].x, A[k][1].y);
        own[(2 * k + 1) * blockDim.x] = make_float4(A[k][2].x, A[k][2].y, A[k][3].x, A[k][3].y);
        own[(2 * K + 2 * k) * blockDim.x] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        own[(2 * K + 2 * k + 1) * blockDim.x] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    __syncthreads();
    for (uint32_t piece = team; piece < 4 * K; piece += teams) {
        float* out = piece < 2 * K ? out_a : out_s;
        if (!out) continue;
        const Chunk<T, VEC> ch(piece / 2 % K, threads, tid, from);
        const float4* slot = own + piece * blockDim.x - team * threads;
        float4 sum = slot[0];
        for (uint32_t t = 1; t < teams; ++t) {
            const float4 o = slot[t * threads];
            sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
        }
        const int j = piece % 2 * 4;
        if constexpr (VEC) {
            if (ch.c < limit) *reinterpret_cast<float4*>(out + ch.c + j) = sum;
        } else {
            const float e[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ch.inside(j + i, limit)) out[ch.column(j + i)] = e[i];
        }
    }
}

// Adds the blocks' partial sums in order.  A job is one row of sums: dw_next; dw_post, from its own partial sums or,
// where runs share gate rows, from the S of every run times the run's gate row; or the gradient of one gate row.
struct Finish {
    const float *part_next, *part_post, *part_gate;
    float *d_next, *d_post;
    void* dgate;  // NULL: not wanted, or written by the runs
    const void *w_post, *gate;
    uint64_t dgs, gs;
    uint32_t width, runs, parts;  // rows of partial sums in all, and for a gate row
    uint32_t split_log;
    bool w_float, g_float;
    float w0;
};

constexpr uint32_t kFinishThreads = 1024;
// A block takes kFinishThreads >> split_log columns of a job, whose partial rows it shares out over 1 << split_log
// groups of threads: 32 for the plain sums, fewer for gate rows of few partial rows.
template <typename T>
__global__ void __launch_bounds__(kFinishThreads) block_norm_finish_kernel(const Finish f) {
    __shared__ float sums[kFinishThreads];
    const uint32_t plain = (f.part_next ? 1 : 0) + (f.d_post ? 1 : 0), plain_blocks = (f.width + 31) / 32;
    uint32_t job, block = blockIdx.x, split_log = 5;  // job 0: next, 1: post, 2 + g: gate row g
    if (block < plain * plain_blocks) {
        job = block / plain_blocks + (f.part_next ? 0 : 1);
        block %= plain_blocks;
    } else {
        block -= plain * plain_blocks;
        split_log = f.split_log;
        const uint32_t blocks = (uint32_t)((((uint64_t)f.width << split_log) + kFinishThreads - 1) / kFinishThreads);
        job = 2 + block / blocks;
        block %= blocks;
    }
    const uint32_t cols = kFinishThreads >> split_log, part_of = threadIdx.x >> (10 - split_log);
    const uint32_t c = block * cols + (threadIdx.x & (cols - 1));
    const bool weighted = job == 1 && !f.part_post;
    const uint32_t n = job < 2 ? f.runs : f.parts;
    const float* part = job == 0 ? f.part_next : job == 1 && !weighted ? f.part_post : f.part_gate;
    if (job >= 2) part += (uint64_t)(job - 2) * f.parts * f.width;
    float v = 0.0f;
    if (c < f.width) {
        const uint32_t begin = n * part_of >> split_log, end = n * (part_of + 1) >> split_log;
        if (weighted) {
            for (uint32_t i = begin; i < end; ++i)
                v += param<T>(f.gate, i / f.parts * f.gs + c, f.g_float) * part[(uint64_t)i * f.width + c];
        } else {
#pragma unroll 8
            for (uint32_t i = begin; i < end; ++i) v += part[(uint64_t)i * f.width + c];
        }
    }
    sums[threadIdx.x] = v;
    __syncthreads();
    if (part_of || c >= f.width) return;
    if (split_log == 5) {
#pragma unroll
        for (uint32_t i = 1; i < 32; ++i) v += sums[i * 32 + threadIdx.x];
    } else {
        for (uint32_t i = 1; i < 1u << split_log; ++i) v += sums[i * cols + threadIdx.x];
    }
    if (job == 0) f.d_next[c] = v;
    else if (job == 1) f.d_post[c] = v;
    else {
        if (f.w_post) v *= f.w0 + param<T>(f.w_post, c, f.w_float);
        const uint64_t at = (job - 2) * f.dgs + c;
        if (f.g_float) static_cast<float*>(f.dgate)[at] = v;
        else static_cast<T*>(f.dgate)[at] = from_float<T>(v);
    }
}

// Which backward kernel serves a width, and with what blocks.  Rows of more than 8192 elements go to clusters of 2
// to 8 blocks, each with 4,352 to 8,192 columns (kinds 2 and 4: the cluster kernels have their elements per
// thread), of more than 65,536 to block_norm_backward_any_kernel.  Larger clusters than a width needs measured
// slower ([2048, 8192] bf16 48 us with one block, 59 with two, 86 with four).  Vectors take 16 elements a thread
// at 128 registers ([8192, 4096] bf16 with gate and dropout 98 us when 8 at 64 registers took 115, 16 at 80
// registers 124), scalar accesses 8 at 64 ([8192, 1001] bf16 45 us, with the next row ahead in registers and half
// the blocks 57).
struct Plan {
    int kind = -1;  // -1: block_norm_backward_any_kernel
    uint32_t team = kThreads, teams = 1, blocks_per_sm = 2, stages = 1, cluster = 1, cols = 0;
    size_t team_smem = 0;
};

constexpr size_t kMaxShared = 227 * 1024 - 2048;  // less the kernels' static part

template <typename T>
Plan plan_backward(uint32_t width, bool vec) {
    Plan p;
    while (p.cluster < kMaxCluster && width > 8192 * p.cluster) p.cluster *= 2;
    p.cols = p.cluster > 1 ? ((width + p.cluster - 1) / p.cluster + 255) / 256 * 256 : width;
    if (p.cols > 8192) return Plan();
    uint32_t e = 16, block = 512, regs = 128;  // elements of a thread, threads of a block, registers
    if (p.cols <= 256) p.kind = 0, e = 8, block = 256;
    else if (vec && p.cols <= 512) p.kind = 1, block = 256;
    else if (vec) p.kind = 2;
    else if (p.cols <= 4096) p.kind = 3, e = 8, regs = 64;
    else p.kind = 4, e = 8, block = 1024, regs = 64;
    p.team = p.kind <= 1 ? 32 : (p.cols + 32 * e - 1) / (32 * e) * 32;
    // the rows of a stage, and the weights
    const size_t stage = vec ? (size_t)p.team * 4 * e * sizeof(T) : 0, weights = p.team * 2 * e * sizeof(float);
    p.stages = 2 * stage + weights <= kMaxShared ? 2 : 1;
    p.team_smem = p.stages * stage + weights;
    if (p.cluster == 1) p.teams = (uint32_t)std::min<size_t>({block / p.team, kMaxShared / p.team_smem, 15});
    const uint32_t threads = p.team * p.teams;
    p.blocks_per_sm = std::max<uint32_t>(
        1, std::min<size_t>({2048 / threads, 65536 / (threads * regs), kMaxShared / (p.team_smem * p.teams + 2048)}));
    return p;
}

template <typename T, int E, bool VEC, bool WARP, bool MULTI, bool CLUSTER, int BLOCK, int MIN>
int launch_backward_kernel(const Backward& f, const Plan& p, cudaStream_t st) {
    auto kernel = block_norm_backward_kernel<T, E, VEC, WARP, MULTI, CLUSTER, BLOCK, MIN>;
    const size_t smem = p.team_smem * p.teams;
    cudaError_t err = cudaSuccess;
    // The limit belongs to the kernel, not to the call, and several threads may call: always the same one, which never
    // undoes another's.  (46 KB: the kernel has static shared memory too.)
    if (smem > 46 * 1024)
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxShared);
    if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute(block_norm_backward_kernel)");
    if constexpr (CLUSTER) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = p.cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(f.runs * p.cluster);
        config.blockDim = dim3(p.team);
        config.dynamicSmemBytes = smem;
        config.stream = st;
        config.attrs = &attr;
        config.numAttrs = 1;
        err = cudaLaunchKernelEx(&config, kernel, f, p.team, p.stages);
        if (err != cudaSuccess) return cuda_fail(err, "block_norm_backward_kernel");
        return MTXC_OK;
    } else {
        kernel<<<(f.runs + p.teams - 1) / p.teams, p.team * p.teams, smem, st>>>(f, p.team, p.stages);
        return check_launch("block_norm_backward_kernel");
    }
}

template <typename T, bool MULTI>
int launch_backward(const Backward& f, const Plan& p, bool vec, cudaStream_t st) {
    if (p.cluster > 1) {
        if (vec) return launch_backward_kernel<T, 16, true, false, MULTI, true, 512, 1>(f, p, st);
        return launch_backward_kernel<T, 8, false, false, MULTI, true, 1024, 1>(f, p, st);
    }
    switch (p.kind) {
        case 0:
            return vec ? launch_backward_kernel<T, 8, true, true, MULTI, false, 256, 2>(f, p, st)
                       : launch_backward_kernel<T, 8, false, true, MULTI, false, 256, 2>(f, p, st);
        case 1: return launch_backward_kernel<T, 16, true, true, MULTI, false, 256, 2>(f, p, st);
        case 2: return launch_backward_kernel<T, 16, true, false, MULTI, false, 512, 1>(f, p, st);
        case 3: return launch_backward_kernel<T, 8, false, false, MULTI, false, 512, 2>(f, p, st);
        case 4: return launch_backward_kernel<T, 8, false, false, MULTI, false, 1024, 1>(f, p, st);
        default:
            block_norm_backward_any_kernel<T><<<f.runs, kThreads, 0, st>>>(f);
            return check_launch("block_norm_backward_any_kernel");
    }
}

// What eight consecutive parameters need for 16-byte accesses (any of the float-like types).
bool param_aligned(const void* p, uint64_t stride) { return aligned16(p) && stride % 8 == 0; }

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
    if (int rc = distinct(who, {a->residual_out, a->normed, a->post_rstd, a->next_rstd})) return rc;
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
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool vec = f.width % 8 == 0 && eight_aligned<T>(f.x, f.xs) && eight_aligned<T>(f.b, f.bs) &&
                         eight_aligned<T>(f.h, f.hs) && eight_aligned<T>(f.a, f.as) && param_aligned(f.w_post, 0) &&
                         param_aligned(f.w_next, 0) && param_aligned(f.gate, f.gs);
        rc = vec ? launch_forward<T, true>(f, ctx().stream(), ctx().sm_count)
                 : launch_forward<T, false>(f, ctx().stream(), ctx().sm_count);
        if (rc == -1) {
            block_norm_any_kernel<T><<<grid, kThreads, 0, ctx().stream()>>>(f);
            rc = check_launch("block_norm_any_kernel");
        }
    });
    return rc;
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
    if (int rc = distinct(who, {a->d_residual, a->d_branch, a->d_post_weight, a->d_next_weight, a->d_gate})) return rc;
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

    // runs of rows: what fills the GPU, no more than there are rows and the workspace holds partial sums for
    bool vec = false;
    Plan plan;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        vec = f.width % 8 == 0 && eight_aligned<T>(f.dh, f.dhs) && eight_aligned<T>(f.da, f.das) &&
              eight_aligned<T>(f.h, f.hs) && eight_aligned<T>(f.b, f.bs) && eight_aligned<T>(f.dx, f.dxs) &&
              eight_aligned<T>(f.db, f.dbs) && param_aligned(f.w_post, 0) && param_aligned(f.w_next, 0) &&
              param_aligned(f.gate, f.gs) && eight_aligned<T>(f.dgate, f.dgs);
        plan = plan_backward<T>(f.width, vec);
    });
    // For the post weight's gradient the other kernels read a gate row once more after its rows' stores: read before
    // them it is held across the row's work, which cost the kernels of scalar accesses 10 to 22 % in spills ([8192,
    // 1001] f16 77 -> 93 us).  This one takes 711 us for [4096, 4096] bf16, 84 with tensors apart.
    if (f.gate && a->d_post_weight && (f.dx == f.gate || f.db == f.gate)) plan = Plan();
    const int sums = !!a->d_next_weight + !!a->d_post_weight + !!a->d_gate;
    const uint64_t row_bytes = (uint64_t)f.width * sizeof(float) * sums;
    // teams that the GPU holds; a block's teams share a gate row, or each has whole ones; few rows: fewer teams in a
    // block, so that all SMs have some
    f.cluster = plan.cluster;
    f.cols = plan.cols;
    const uint64_t most = std::max<uint64_t>(1, (uint64_t)ctx().sm_count * plan.blocks_per_sm * plan.teams / plan.cluster);
    f.groups = (uint32_t)(((uint64_t)f.rows + f.gate_rows - 1) / f.gate_rows);
    plan.teams = (uint32_t)std::min<uint64_t>(plan.teams, std::max<uint64_t>(1, f.rows / ctx().sm_count));
    if (f.gate && most >= f.groups) plan.teams = (uint32_t)std::min<uint64_t>(plan.teams, most / f.groups);
    uint64_t blocks = most / plan.teams;
    if (row_bytes) blocks = std::min<uint64_t>(blocks, ctx().workspace_bytes / row_bytes);
    if (blocks == 0)
        return fail(MTXC_ERR_WORKSPACE, who + ": one block's partial sums need " + std::to_string(row_bytes) +
                                            " bytes of workspace, the thread has " + std::to_string(ctx().workspace_bytes));
    const uint64_t runs = std::min<uint64_t>(f.rows, blocks * plan.teams);
    f.parts = (uint32_t)(std::min<uint64_t>(runs / f.groups, f.gate_rows) / plan.teams * plan.teams);
    if (f.parts <= 1) f.parts = 1;
    f.runs = f.parts > 1 ? f.groups * f.parts : (uint32_t)std::min<uint64_t>(runs, f.groups);
    const uint32_t partial_rows = (f.runs + plan.teams - 1) / plan.teams;
    float* ws = static_cast<float*>(ctx().workspace);
    auto take = [&](bool wanted) {
        float* p = wanted ? ws : nullptr;
        if (wanted) ws += (uint64_t)partial_rows * f.width;
        return p;
    };
    const bool shared_gate = f.gate && f.parts > 1;  // then S of each run gives both sums
    f.part_next = take(a->d_next_weight);
    f.part_post = take(a->d_post_weight && !shared_gate);
    f.part_gate = take(a->d_gate || (a->d_post_weight && shared_gate));
    Finish e{};
    e.part_next = f.part_next;
    e.part_post = f.part_post;
    e.part_gate = f.part_gate;
    e.d_next = a->d_next_weight;
    e.d_post = a->d_post_weight;
    e.dgate = shared_gate ? f.dgate : nullptr;
    e.w_post = f.w_post;
    e.gate = f.gate;
    e.dgs = f.dgs;
    e.gs = f.gs;
    e.width = f.width;
    e.runs = partial_rows;
    e.parts = std::max(1u, f.parts / plan.teams);
    e.w_float = f.w_float;
    e.g_float = f.g_float;
    e.w0 = f.w0;
    while (e.split_log < 5 && 4u << e.split_log < e.parts) ++e.split_log;
    const uint64_t finish = (uint64_t)(!!e.part_next + !!e.d_post) * ((f.width + 31) / 32) +
                            (e.dgate ? (uint64_t)f.groups * ((((uint64_t)f.width << e.split_log) + kFinishThreads - 1) / kFinishThreads) : 0);
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        rc = f.gate && f.parts == 1 ? launch_backward<T, true>(f, plan, vec, st) : launch_backward<T, false>(f, plan, vec, st);
        if (rc == MTXC_OK && finish) block_norm_finish_kernel<T><<<(unsigned)finish, kFinishThreads, 0, st>>>(e);
    });
    return rc == MTXC_OK ? check_launch("block_norm_finish_kernel") : rc;
}
