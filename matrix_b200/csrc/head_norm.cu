// Norms of queries and keys for each head with their rotary positions, forward and backward, for sm_100a.
//
//   n = x r w',  r = 1 / sqrt(mean(x^2) + eps),  w' = weight_offset + w;   y = scale * turn(n), the rest of the head n
//   backward: g = turn back (scale included) of dy, u = g w':  dx = r (u - x r^2 mean(u x)),  dw = sum of g x r
//
// x (and dy) are read once, y (dx) written once.  A group of lanes holds a head in registers between the reduction and the
// store; its blocks work on queries alone or keys alone, so that a lane meets one piece of one weight (and adds to one piece of
// its gradient) for all its heads.  Measured: 16,384 tokens x 40 heads of 128 bf16 forward 70 us, 4.8 TB/s, backward 107 us, 4.7;
// f32 8,192 tokens 58 and 91 us, 5.7 and 5.5.  Half types are bound by their instructions (issue 57 and 52 %, about 260 and 350
// for a warp's four heads) behind one another's latency at 24 and 16 warps an SM; 32 warps of 64 registers measured the same.
#include <algorithm>
#include <cmath>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxHead = 1024;
constexpr uint32_t kTableEntries = 2048;  // cosines of a tile; as many sines
constexpr uint32_t kResident = 2;         // blocks an SM of the backward pass

struct Side {  // queries or keys
    uint32_t heads, blocks, first_block;
    uint32_t tile, tiles;  // tokens of a tile, tiles of a sequence
    FastDiv heads_div, tiles_div;
    const void *x, *dy, *weight;
    void* out;               // y or dx
    uint64_t xs[3], ys[3], os[3];
    float* rstd;             // written forward (or NULL), read backward
    float* d_weight;         // partial rows [blocks][head], or NULL
    bool whole_weight;       // of the heads' dtype and aligned as they are
};

struct HeadNorm {
    uint64_t tokens;
    uint64_t length;         // tokens of a sequence
    uint32_t batch, head, half, lanes_log;
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
// Heads by accesses of N elements: a group of up to 32 lanes holds a head, a lane two accesses of it (half a head apart where
// they are turned against each other, or, PAIRS, where each is turned in itself).  A block takes tiles of tokens of a sequence:
// it makes their cosines and sines once, in shared memory, for all heads, with its first loads already in flight, and each group
// loads its next head before it works on the one at hand.  Forward a tile a block; backward the blocks stay, since they keep
// the sums for the weight's gradient in registers.
// ------------------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void read_table(const float* p, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + i);
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
    } else {
        const float2 q = *reinterpret_cast<const float2*>(p);
        v[0] = q.x, v[1] = q.y;
    }
}

template <typename T, int N, bool PAIRS, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, BACKWARD ? 2 : 3) head_norm_kernel(const HeadNorm r) {
    constexpr int kAngles = PAIRS ? N / 2 : N;  // of an access
    extern __shared__ float4 table4[];
    float* const table = reinterpret_cast<float*>(table4);
    const int k = blockIdx.x >= r.side[1].first_block;
    const Side& s = r.side[k];
    const uint32_t block = blockIdx.x - s.first_block;
    float* const cosines = table;
    float* const sines = table + s.tile * r.half;
    const uint32_t lanes = 1u << r.lanes_log, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> r.lanes_log;
    const uint32_t groups = kThreads >> r.lanes_log;
    // this lane's accesses: their first elements, whether they are there and turned, and their first angles
    uint32_t at[2];
    bool there[2], turns[2];
    if (PAIRS) {
        const uint32_t all = r.head / N, first = (all + 1) / 2;
        at[0] = lane * N, at[1] = (lane + first) * N;
        there[0] = lane < first, there[1] = lane < first && lane + first < all;
        turns[0] = at[0] < 2 * r.half, turns[1] = at[1] < 2 * r.half;
    } else {
        const uint32_t turned = r.half / N, rest = r.head / N - 2 * turned, first = (rest + 1) / 2, i = lane - turned;
        const bool t = lane < turned;
        at[0] = t ? lane * N : 2 * r.half + i * N, at[1] = at[0] + (t ? r.half : first * N);
        there[0] = t || i < first, there[1] = t || (i < first && i + first < rest);
        turns[0] = turns[1] = t;
    }
    float2 w[2][N / 2], dw[2][N / 2];  // two elements at a time: two products an instruction
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[a][i] = s.weight ? make_float2(0.0f, 0.0f) : make_float2(1.0f, 1.0f), dw[a][i] = make_float2(0.0f, 0.0f);
    if (s.weight && s.whole_weight) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            Few<T, N> v;
            if (!there[a]) continue;
            v.load(static_cast<const T*>(s.weight) + at[a]);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) w[a][i] = __fadd2_rn(make_float2(r.weight_offset, r.weight_offset), v.get2(i));
        }
    } else if (s.weight) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (there[a]) w[a][i] = make_float2(weight_at(r, s, at[a] + 2 * i), weight_at(r, s, at[a] + 2 * i + 1));
    }

    struct Head {
        Few<T, N> x[2], dy[BACKWARD ? 2 : 1];
        float rstd;
    };
    // accesses that are not there stay zeros
    Head next{};
    uint32_t token_step, head_step;  // from a group's head to its next one
    s.heads_div.divmod(groups, token_step, head_step);
    const uint32_t all_tiles = r.batch * s.tiles;
    for (uint32_t tile = block; tile < all_tiles; tile += s.blocks) {
        uint32_t b, t0;
        s.tiles_div.divmod(tile, b, t0);
        t0 *= s.tile;
        const uint32_t n = (uint32_t)min((uint64_t)s.tile, r.length - t0), items = n * s.heads;
        const T* const x = static_cast<const T*>(s.x) + b * s.xs[0] + t0 * s.xs[1];
        const T* const dy = BACKWARD ? static_cast<const T*>(s.dy) + b * s.ys[0] + t0 * s.ys[1] : nullptr;
        T* const out = static_cast<T*>(s.out) + b * s.os[0] + t0 * s.os[1];
        float* const rstd = s.rstd ? s.rstd + (b * r.length + t0) * s.heads : nullptr;
        auto load = [&](uint32_t item, uint32_t token, uint32_t h, Head& v) {
            const T* const px = x + token * s.xs[1] + h * s.xs[2];
            const T* const py = BACKWARD ? dy + token * s.ys[1] + h * s.ys[2] : nullptr;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                if (!there[a]) continue;
                v.x[a].load(px + at[a]);
                if constexpr (BACKWARD) v.dy[a].load(py + at[a]);
            }
            if constexpr (BACKWARD) v.rstd = rstd[item];
        };
        // the angles of access a, of which `first` is the value in the first place of its pair
        auto turn_all = [&](uint32_t token, float2 (&v)[2][N / 2]) {
            float cs[kAngles], sn[kAngles];
            if constexpr (PAIRS) {
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    if (!turns[a] || !there[a]) continue;
                    read_table(cosines + token * r.half + at[a] / 2, cs);
                    read_table(sines + token * r.half + at[a] / 2, sn);
#pragma unroll
                    for (int j = 0; j < kAngles; ++j) {
                        const float2 q = v[a][j];
                        v[a][j] = __ffma2_rn(make_float2(q.x, q.x), make_float2(cs[j], sn[j]),
                                             __fmul2_rn(make_float2(q.y, q.y), make_float2(-sn[j], cs[j])));
                    }
                }
            } else if (turns[0]) {
                read_table(cosines + token * r.half + at[0], cs);
                read_table(sines + token * r.half + at[0], sn);
#pragma unroll
                for (int j = 0; j < kAngles / 2; ++j) {
                    const float2 p = v[0][j], q = v[1][j], c = make_float2(cs[2 * j], cs[2 * j + 1]), d = make_float2(sn[2 * j], sn[2 * j + 1]);
                    v[0][j] = __ffma2_rn(p, c, __fmul2_rn(q, make_float2(-d.x, -d.y)));
                    v[1][j] = __ffma2_rn(p, d, __fmul2_rn(q, c));
                }
            }
        };
        uint32_t token, h;
        s.heads_div.divmod(group, token, h);
        if (group < items) load(group, token, h, next);
        __syncthreads();  // the tile before is done with the table
        for (uint32_t e = threadIdx.x; e < n * r.half; e += kThreads) {
            uint32_t t, j;
            r.half_div.divmod(e, t, j);
            turn(r, position_of(r, b, t0 + t), j, cosines[e], sines[e]);
        }
        __syncthreads();
        for (uint32_t base = 0; base < items; base += groups) {  // the same for all lanes of a warp
            const uint32_t item = base + group;
            const bool mine = item < items;
            const Head v = next;
            const uint32_t token_now = token, h_now = h;
            token += token_step, h += head_step;
            if (h >= s.heads) h -= s.heads, ++token;
            if (item + groups < items) load(item + groups, token, h, next);
            float2 y[2][N / 2], sums = make_float2(0.0f, 0.0f);
            if constexpr (!BACKWARD) {
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        y[a][i] = v.x[a].get2(i);
                        sums = __ffma2_rn(y[a][i], y[a][i], sums);
                    }
                float sum = sums.x + sums.y;
#pragma unroll
                for (uint32_t m = 16; m; m /= 2)
                    if (m < lanes) sum += __shfl_xor_sync(~0u, sum, m);
                const float scale = rsqrtf(fmaf(sum, r.inv_head, r.eps));
                if (!mine) continue;
                if (rstd && lane == 0) rstd[item] = scale;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) y[a][i] = __fmul2_rn(__fmul2_rn(y[a][i], make_float2(scale, scale)), w[a][i]);
                turn_all(token_now, y);
            } else {
                float2 e[2][N / 2];
                const float2 scale = make_float2(v.rstd, v.rstd);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        y[a][i] = v.dy[a].get2(i);
                        e[a][i] = __fmul2_rn(v.x[a].get2(i), scale);
                    }
                if (mine) {
                    turn_all(token_now, y);
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int i = 0; i < N / 2; ++i) {
                            dw[a][i] = __ffma2_rn(y[a][i], e[a][i], dw[a][i]);
                            y[a][i] = __fmul2_rn(y[a][i], w[a][i]);
                            sums = __ffma2_rn(y[a][i], e[a][i], sums);
                        }
                }
                float sum = sums.x + sums.y;
#pragma unroll
                for (uint32_t m = 16; m; m /= 2)
                    if (m < lanes) sum += __shfl_xor_sync(~0u, sum, m);
                if (!mine) continue;
                sum *= -r.inv_head;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) y[a][i] = __fmul2_rn(scale, __ffma2_rn(e[a][i], make_float2(sum, sum), y[a][i]));
            }
            T* const to = out + token_now * s.os[1] + h_now * s.os[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                if (!there[a]) continue;
                Few<T, N> o;
#pragma unroll
                for (int i = 0; i < N / 2; ++i) o.set2(i, y[a][i].x, y[a][i].y);
                o.store(to + at[a]);
            }
        }
    }
    if constexpr (BACKWARD) {
        if (!s.d_weight) return;
        // the groups of a warp, then the warps, in order
        const uint32_t warp = threadIdx.x / 32;
        __syncthreads();
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float v = i % 2 ? dw[a][i / 2].y : dw[a][i / 2].x;
                for (uint32_t m = 16; m >= lanes; m /= 2) v += __shfl_xor_sync(~0u, v, m);
                if (threadIdx.x % 32 < lanes && there[a]) table[warp * r.head + at[a] + i] = v;
            }
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < r.head; d += kThreads) {
            float sum = 0.0f;
            for (uint32_t i = 0; i < kThreads / 32; ++i) sum += table[i * r.head + d];
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
    // queries and keys are worked on at the same time: an output may be its own input, not the other's
    for (int k = 0; k < 2; ++k) {
        if (!a->heads[k]) continue;
        if (int rc = apart(who, {a->dst[k]}, {a->heads[1 - k] ? a->src[1 - k] : nullptr, a->weight[0], a->weight[1]})) return rc;
        if (int rc = laid_alike(who, a->dst[k], a->dst_strides[k], a->src[k], a->src_strides[k], {a->batch, a->length, a->heads[k]})) return rc;
    }
    if (tokens && a->rotary_dim && (!a->positions || !a->frequencies))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null positions or frequencies");
    return distinct(who, {a->heads[0] ? a->dst[0] : nullptr, a->heads[1] ? a->dst[1] : nullptr});
}

// The call's arguments as the kernels take them, and its plan; blocks: all that the launch needs; access: elements, 0: any.
struct Plan {
    HeadNorm r{};
    uint32_t access = 0, blocks = 0;
};

// Whether a call's heads go by accesses of N elements.
template <typename T, int N>
bool fits(const mtxc_head_norm_args* a, bool backward) {
    const uint32_t half = a->rotary_dim / 2, head = a->head_dim;
    if (head % N || (a->interleaved ? a->rotary_dim % N : half % N)) return false;
    const uint32_t lanes = a->interleaved ? (head / N + 1) / 2 : half / N + (head / N - 2 * (half / N) + 1) / 2;
    bool ok = lanes <= 32 && a->length < 1ull << 31 && a->batch < 1ull << 31;
    for (int k = 0; k < 2; ++k)
        for (int i = 0; a->heads[k] && i < 3; ++i) {
            ok = ok && few_aligned<T, N>(a->src[k], a->src_strides[k][i]) && few_aligned<T, N>(a->dst[k], a->dst_strides[k][i]);
            if (backward) ok = ok && few_aligned<T, N>(a->d_out[k], a->d_out_strides[k][i]);
        }
    return ok;
}

Plan plan(int dtype, const mtxc_head_norm_args* a, bool backward) {
    Plan p;
    HeadNorm& r = p.r;
    r.tokens = a->batch * a->length;
    r.length = std::max<uint64_t>(1, a->length);
    r.batch = (uint32_t)a->batch;
    r.head = a->head_dim;
    r.half = a->rotary_dim / 2;
    r.half_div = FastDiv(std::max(1u, r.half));
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
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        p.access = fits<T, 8>(a, backward) ? 8 : fits<T, 4>(a, backward) ? 4 : 0;
    });
    if (!r.tokens || !r.head) p.access = 0;
    for (int k = 0; k < 2; ++k)
        r.side[k].whole_weight = a->weight_dtype == dtype && reinterpret_cast<uintptr_t>(a->weight[k]) % 32 == 0;
    uint32_t lanes = 1;
    if (p.access) {
        const uint32_t n = p.access, turned = r.half / n;
        const uint32_t want = a->interleaved ? (r.head / n + 1) / 2 : turned + (r.head / n - 2 * turned + 1) / 2;
        while (lanes < want) lanes *= 2, ++r.lanes_log;
    }
    const uint32_t groups = kThreads / lanes, all_heads = a->heads[0] + a->heads[1], sms = (uint32_t)ctx().sm_count;
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
        s.tile = s.tiles = 1;
        if (!s.heads || !r.tokens) {
            s.blocks = 0;
        } else if (p.access) {
            // tokens of a tile: eight heads a group, while every SM has four blocks and the table fits
            uint64_t tile = std::max<uint64_t>(1, 8 * groups / s.heads);
            tile = std::min(tile, std::max<uint64_t>(1, r.tokens * all_heads / (4ull * sms * s.heads)));
            tile = std::min<uint64_t>({tile, std::max(1u, kTableEntries / std::max(1u, r.half)), r.length});
            s.tile = (uint32_t)tile;
            s.tiles = (uint32_t)((r.length + tile - 1) / tile);
            const uint64_t all = (uint64_t)s.tiles * a->batch;
            if (all >> 31) p.access = 0;
            // backward: as many blocks as are resident, shared by heads
            const uint64_t most = backward ? std::max<uint64_t>(1, (uint64_t)kResident * sms * s.heads / all_heads) : 1u << 30;
            s.blocks = (uint32_t)std::min(all, most);
        }
        s.tiles_div = FastDiv(s.tiles);
    }
    for (int k = 0; k < 2; ++k) {
        Side& s = r.side[k];
        if (!p.access) {
            const uint64_t warps = r.tokens * s.heads;
            s.blocks = (uint32_t)std::min<uint64_t>((warps + kThreads / 32 - 1) / (kThreads / 32), 4u * sms);
        }
        s.first_block = p.blocks;
        p.blocks += s.blocks;
    }
    return p;
}

template <bool BACKWARD>
int launch(int dtype, const mtxc_head_norm_args* a, const Plan& p) {
    const HeadNorm& r = p.r;
    const size_t sums = BACKWARD ? sizeof(float) * (kThreads / 32) * r.head : 0;
    const size_t table = 2 * sizeof(float) * r.half * std::max(r.side[0].tile, r.side[1].tile);
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        cudaStream_t st = ctx().stream();
        auto run = [&](auto pairs) {
            constexpr bool P = decltype(pairs)::value;
            if (p.access == 8) head_norm_kernel<T, 8, P, BACKWARD><<<p.blocks, kThreads, std::max(sums, table), st>>>(r);
            else if (p.access == 4) head_norm_kernel<T, 4, P, BACKWARD><<<p.blocks, kThreads, std::max(sums, table), st>>>(r);
            else head_norm_any_kernel<T, P, BACKWARD><<<p.blocks, kThreads, sums, st>>>(r);
        };
        if (a->interleaved) run(std::true_type());
        else run(std::false_type());
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
    if (int rc = apart("mtxc_head_norm_rotary", {a->rstd[0], a->rstd[1]}, {a->src[0], a->src[1], a->weight[0], a->weight[1]})) return rc;
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
    for (int k = 0; k < 2; ++k) {
        if (!a->heads[k]) continue;
        if (int rc = apart(who, {a->dst[k]}, {a->heads[1 - k] ? a->d_out[1 - k] : nullptr, a->rstd[0], a->rstd[1]})) return rc;
        if (int rc = laid_alike(who, a->dst[k], a->dst_strides[k], a->d_out[k], a->d_out_strides[k], {a->batch, a->length, a->heads[k]})) return rc;
    }
    if (int rc = apart(who, {a->d_weight[0], a->d_weight[1]},
                       {a->src[0], a->src[1], a->d_out[0], a->d_out[1], a->rstd[0], a->rstd[1], a->weight[0], a->weight[1]}))
        return rc;
    Plan p = plan(dtype, a, true);
    for (int k = 0; k < 2; ++k) {
        if (p.r.side[k].blocks && a->head_dim && (!a->d_out[k] || !a->rstd[k]))
            return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null d_out or rstd");
    }
    if (!a->head_dim) return MTXC_OK;
    const size_t bytes = partial_bytes(p, a);
    float* partial = static_cast<float*>(a->workspace ? a->workspace : ctx().workspace);
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": the workspace must be aligned to 256 bytes");
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
