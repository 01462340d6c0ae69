// Attention over whole prompts, for sm_100a: packed sequences of different lengths, grouped heads, causal or not.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j,  m_i a running maximum
//
// over the keys j <= i + (m - n) of a sequence of n queries and m keys (causal) or all of them.
#include <algorithm>
#include <cmath>

#include "attention.cuh"

namespace mtxc {
namespace {

constexpr uint32_t kMaxHead = 256;
constexpr float kLowest = -3.402823466e+38f;
constexpr int kAnyThreads = 256;
constexpr uint32_t kAnyTile = 64;  // queries, and keys

struct Prompt {
    const void *q, *k, *v;
    void* out;
    uint64_t qs[2], ks[2], vs[2], os[2];  // token, head
    uint32_t tokens, k_tokens, sequences, heads, group, head;
    const int *starts, *k_starts;
    FastDiv group_div;
    float scale;  // times log2(e)
    bool causal;
};

// Rows [first, first + count) of a sequence, within what there is.
__device__ __forceinline__ void rows_of(const int* starts, uint32_t i, uint32_t tokens, uint32_t& first, uint32_t& count) {
    const uint32_t lo = (uint32_t)min(max(starts[i], 0), (int)tokens), hi = (uint32_t)min(max(starts[i + 1], 0), (int)tokens);
    first = lo;
    count = hi > lo ? hi - lo : 0;
}

// ------------------------------------------------------------------------------------------
// Any head and type: 64 queries and 64 keys at a time, products in 32 bits.
// ------------------------------------------------------------------------------------------
__host__ __device__ inline uint32_t pitch_of(uint32_t head) { return (head + 3) / 8 * 8 + 4; }  // an odd number of 16-byte units

template <typename T>
__global__ void __launch_bounds__(kAnyThreads) prompt_any_kernel(const Prompt p) {
    extern __shared__ float4 smem4[];
    __shared__ uint64_t buf[33];
    __shared__ Found found;
    constexpr uint32_t kTilePitch = kAnyTile + 4;
    const uint32_t pitch = pitch_of(p.head), quads = (p.head + 3) / 4;
    float* const q = reinterpret_cast<float*>(smem4);    // [64][pitch]
    float* const kv = q + kAnyTile * pitch;              // [64][pitch]: keys, then values
    float* const weights = kv + kAnyTile * pitch;        // [64][kTilePitch]
    // the last sequence first, and in each the last tile first: of causal ones the longest
    auto count = [&](uint32_t i) {
        uint32_t first, n;
        rows_of(p.starts, p.sequences - 1 - i, p.tokens, first, n);
        return (uint64_t)(n + kAnyTile - 1) / kAnyTile;
    };
    const Found f = find(p.sequences, blockIdx.x, count, buf, &found);
    if (!f.any) return;
    const uint32_t i = p.sequences - 1 - f.i, h = blockIdx.y, kh = p.group_div.div(h);
    uint32_t q_first, n, k_first, m;
    rows_of(p.starts, i, p.tokens, q_first, n);
    rows_of(p.k_starts, i, p.k_tokens, k_first, m);
    const uint32_t row0 = ((n + kAnyTile - 1) / kAnyTile - 1 - (uint32_t)(blockIdx.x - f.first)) * kAnyTile;
    const int64_t ahead = (int64_t)m - n;  // a query sees keys up to its own index plus this
    auto load = [&](float* to, const void* from, const uint64_t (&s)[2], uint32_t first, uint32_t head, uint32_t rows) {
        const T* x = static_cast<const T*>(from) + head * s[1];
        for (uint32_t e = threadIdx.x; e < kAnyTile * quads * 4; e += kAnyThreads) {
            const uint32_t r = e / (quads * 4), c = e - r * (quads * 4);
            to[r * pitch + c] = r < rows && c < p.head ? to_float(x[(uint64_t)(first + r) * s[0] + c]) : 0.0f;
        }
    };
    load(q, p.q, p.qs, q_first + row0, h, min(kAnyTile, n - row0));
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;  // rows 4 ty .., keys tx + 16 j, columns 4 tx + 64 c
    float top[4], sum[4];
    float4 acc[4][kMaxHead / 64];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        top[a] = -INFINITY, sum[a] = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < kMaxHead / 64; ++c) acc[a][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    int64_t last = p.causal ? min((int64_t)m, (int64_t)min(row0 + kAnyTile, n) + ahead) : (int64_t)m;  // keys seen by any row
    for (int64_t k0 = 0; k0 < last; k0 += kAnyTile) {
        const uint32_t keys = (uint32_t)min((int64_t)kAnyTile, m - k0);
        __syncthreads();
        load(kv, p.k, p.ks, k_first + (uint32_t)k0, kh, keys);
        __syncthreads();
        float s[4][4] = {};
        for (uint32_t c = 0; c < quads; ++c) {
            float4 x[4], y[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4*>(q + (4 * ty + a) * pitch + 4 * c);
#pragma unroll
            for (int b = 0; b < 4; ++b) y[b] = *reinterpret_cast<const float4*>(kv + (tx + 16 * b) * pitch + 4 * c);
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    s[a][b] = fmaf(x[a].x, y[b].x, s[a][b]);
                    s[a][b] = fmaf(x[a].y, y[b].y, s[a][b]);
                    s[a][b] = fmaf(x[a].z, y[b].z, s[a][b]);
                    s[a][b] = fmaf(x[a].w, y[b].w, s[a][b]);
                }
        }
        __syncthreads();
        load(kv, p.v, p.vs, k_first + (uint32_t)k0, kh, keys);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int64_t limit = p.causal ? (int64_t)row0 + 4 * ty + a + ahead : (int64_t)m - 1;
            float now = -INFINITY;
            bool seen[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int64_t j = k0 + tx + 16 * b;
                seen[b] = j < m && j <= limit;
                s[a][b] *= p.scale;
                // a key that counts lifts the maximum off -infinity even where its score is -infinity
                if (seen[b]) now = fmaxf(now, fmaxf(s[a][b], kLowest));
            }
#pragma unroll
            for (int d = 8; d; d /= 2) now = fmaxf(now, __shfl_xor_sync(~0u, now, d));
            now = fmaxf(now, top[a]);
            const float factor = now == top[a] ? 1.0f : exp2f(top[a] - now);
            top[a] = now;
            float part = 0.0f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float w = seen[b] ? exp2f(s[a][b] - now) : 0.0f;
                part += w;
                weights[(4 * ty + a) * kTilePitch + tx + 16 * b] = w;
            }
            sum[a] = sum[a] * factor + part;
#pragma unroll
            for (uint32_t c = 0; c < kMaxHead / 64; ++c) {
                acc[a][c].x *= factor, acc[a][c].y *= factor, acc[a][c].z *= factor, acc[a][c].w *= factor;
            }
        }
        __syncthreads();
        int seen_to[4];  // what a row does not see may hold anything
#pragma unroll
        for (int a = 0; a < 4; ++a)
            seen_to[a] = p.causal ? (int)max((int64_t)-1, min((int64_t)kAnyTile, (int64_t)row0 + 4 * ty + a + ahead - k0)) : (int)kAnyTile;
        for (uint32_t j = 0; j < keys; ++j) {
            float w[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) w[a] = weights[(4 * ty + a) * kTilePitch + j];
#pragma unroll
            for (uint32_t c = 0; c < kMaxHead / 64; ++c) {
                if (tx + 16 * c >= quads) break;
                const float4 y = *reinterpret_cast<const float4*>(kv + j * pitch + 4 * (tx + 16 * c));
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    if ((int)j > seen_to[a]) continue;
                    acc[a][c].x = fmaf(w[a], y.x, acc[a][c].x);
                    acc[a][c].y = fmaf(w[a], y.y, acc[a][c].y);
                    acc[a][c].z = fmaf(w[a], y.z, acc[a][c].z);
                    acc[a][c].w = fmaf(w[a], y.w, acc[a][c].w);
                }
            }
        }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
#pragma unroll
        for (int d = 8; d; d /= 2) sum[a] += __shfl_xor_sync(~0u, sum[a], d);
        const uint32_t row = row0 + 4 * ty + a;
        if (row >= n) continue;
        T* out = static_cast<T*>(p.out) + (uint64_t)(q_first + row) * p.os[0] + h * p.os[1];
        const bool any = top[a] != -INFINITY;
#pragma unroll
        for (uint32_t c = 0; c < kMaxHead / 64; ++c) {
            const uint32_t at = 4 * (tx + 16 * c);
            const float o[4] = {acc[a][c].x, acc[a][c].y, acc[a][c].z, acc[a][c].w};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (at + e < p.head) out[at + e] = from_float<T>(any ? o[e] / sum[a] : 0.0f);
        }
    }
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_prompt_attention(int dtype, const mtxc_prompt_attention_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_prompt_attention";
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (a->head_dim == 0 || a->head_dim > kMaxHead)
        return fail(MTXC_ERR_SHAPE, who + ": head_dim must be 1 to " + std::to_string(kMaxHead));
    if (a->tokens >> 30 || a->k_tokens >> 30 || a->sequences >> 30)
        return fail(MTXC_ERR_SHAPE, who + ": tokens and sequences must be below 2^30");
    if (a->heads > 65535 || (a->heads && (!a->kv_heads || a->heads % a->kv_heads)))
        return fail(MTXC_ERR_SHAPE, who + ": heads must be at most 65,535 and a multiple of the keys'");
    if (!a->tokens || !a->sequences || !a->heads) return MTXC_OK;
    if (!a->q || !a->out || !a->starts || (a->k_tokens && (!a->k || !a->v)))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tensor");
    Prompt p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out;
    for (int i = 0; i < 2; ++i)
        p.qs[i] = a->q_strides[i], p.ks[i] = a->k_strides[i], p.vs[i] = a->v_strides[i], p.os[i] = a->out_strides[i];
    p.tokens = (uint32_t)a->tokens;
    p.k_tokens = (uint32_t)a->k_tokens;
    p.sequences = (uint32_t)a->sequences;
    p.heads = a->heads;
    p.group = a->heads / a->kv_heads;
    p.group_div = FastDiv(p.group);
    p.head = a->head_dim;
    p.starts = a->starts;
    p.k_starts = a->k_starts ? a->k_starts : a->starts;
    p.scale = a->scale * 1.4426950408889634f;
    p.causal = a->causal != 0;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto smem = [](uint32_t head) { return sizeof(float) * (2 * kAnyTile * pitch_of(head) + kAnyTile * (kAnyTile + 4)); };
        // the same limit in every call: calls from several threads do not undo each other's
        cudaError_t err = cudaFuncSetAttribute(prompt_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem(kMaxHead));
        if (err != cudaSuccess) {
            rc = cuda_fail(err, "cudaFuncSetAttribute");
            return;
        }
        // as many tiles as the sequences can have: one each may be part filled
        const uint64_t tiles = a->tokens / kAnyTile + std::min(a->sequences, a->tokens);
        prompt_any_kernel<T><<<dim3((unsigned)tiles, a->heads), kAnyThreads, smem(p.head), ctx().stream()>>>(p);
        rc = check_launch("prompt_any_kernel");
    });
    return rc;
}
