// Attention of one new token of each sequence over a paged cache, for sm_100a.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m a running maximum
//
// The keys and values are read once: bound by HBM.  The work -- a tile of keys for each key head and each 16 of its query
// heads, of all sequences one after another -- is shared out evenly over a fixed number of blocks, whatever the lengths are
// (which only the device knows).  A unit (sequence, heads) that lies within one block is written there; of one that blocks
// share, each leaves its sums and maxima in the workspace, and a second launch joins them in order.
#include <algorithm>
#include <cmath>

#include "attention.cuh"

namespace mtxc {
namespace {

constexpr uint32_t kMaxHead = 256;
constexpr uint32_t kRows = 16;       // query heads of a unit
constexpr int kAnyThreads = 256;
constexpr uint32_t kAnyTile = 32;    // keys
constexpr float kLowest = -3.402823466e+38f;

struct Decode {
    Cache cache;
    uint32_t batch, heads, kv_heads, group, groups, units, head, max_pages, tile, blocks;  // groups: of 16 query heads
    const void* q;
    void* out;
    uint64_t qs[2], os[2];
    const int* table;
    uint64_t table_stride;
    const int* lengths;
    float scale;      // times log2(e)
    float* partial;   // [2 * blocks][kRows][head + 2]: sums, maximum, sum of weights
};

__device__ __forceinline__ uint32_t length_of(const Decode& d, uint32_t b) {
    const int n = d.lengths[b];
    return n < 0 ? 0u : (uint32_t)min((unsigned long long)n, (unsigned long long)d.max_pages * d.cache.page_size);
}
__device__ __forceinline__ uint32_t tiles_of(const Decode& d, uint32_t b) { return (length_of(d, b) + d.tile - 1) / d.tile; }

// The blocks that share the work: each has some.
__device__ __forceinline__ uint64_t sharing(const Decode& d, uint64_t work) { return min(work, (uint64_t)d.blocks); }

// The page and slot of key j of sequence b; false: the table names no page of the cache.
__device__ __forceinline__ bool place_of(const Decode& d, uint32_t b, uint32_t j, uint32_t& page, uint32_t& slot) {
    uint32_t i;
    d.cache.page_div.divmod(j, i, slot);
    page = (uint32_t)d.table[b * d.table_stride + i];
    return page < d.cache.pages;
}

// Rows of a unit: query heads first .. first + count - 1.
__device__ __forceinline__ uint32_t rows_of(const Decode& d, uint32_t unit, uint32_t& head, uint32_t& first) {
    head = unit / d.groups;
    const uint32_t g = unit - head * d.groups;
    first = head * d.group + g * kRows;
    return min(kRows, d.group - g * kRows);
}

// Element d of key (0) or value (1) at a page's slot.
template <typename T, bool SMALL>
__device__ __forceinline__ float element(const CacheSide& c, uint64_t at, uint32_t d, float scale) {
    if constexpr (SMALL) return from_e4m3(static_cast<const uint8_t*>(c.data)[at + d]).x * scale;
    else return to_float(static_cast<const T*>(c.data)[at + d]);
}

// ------------------------------------------------------------------------------------------
// Any head and type: keys and values as floats in shared memory, products in 32 bits.
// ------------------------------------------------------------------------------------------
template <typename T, bool SMALL>
__global__ void __launch_bounds__(kAnyThreads) decode_any_kernel(const Decode d) {
    extern __shared__ float smem[];
    __shared__ uint64_t buf[33];
    __shared__ Found found;
    __shared__ float row_max[kRows], row_sum[kRows], row_factor[kRows];
    __shared__ bool valid[kAnyTile];
    const uint32_t pitch = d.head + 1, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float* const q = smem;                       // [kRows][head]
    float* const keys = q + kRows * d.head;      // [kAnyTile][pitch]
    float* const values = keys + kAnyTile * pitch;
    float* const weights = values + kAnyTile * pitch;  // [kRows][kAnyTile]
    auto count = [&](uint32_t b) { return (uint64_t)tiles_of(d, b) * d.units; };
    const uint64_t work = total_of(d.batch, count, buf), blocks = sharing(d, work);
    if (blockIdx.x >= blocks) return;
    uint64_t at = work * blockIdx.x / blocks;
    const uint64_t end = work * (blockIdx.x + 1) / blocks;
    const Found f = find(d.batch, at, count, buf, &found);
    uint32_t b = f.i, tiles = tiles_of(d, b);
    uint32_t unit = (uint32_t)((at - f.first) / tiles), tile = (uint32_t)((at - f.first) - (uint64_t)unit * tiles);
    // this thread's column and rows of the output
    uint32_t wide = 32;
    while (wide < d.head) wide *= 2;
    const uint32_t column = threadIdx.x % wide, row0 = threadIdx.x / wide, row_step = kAnyThreads / wide;
    while (at < end) {
        uint32_t h, first;
        const uint32_t rows = rows_of(d, unit, h, first), n = length_of(d, b), tile0 = tile;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < rows * d.head; i += kAnyThreads) {
            const uint32_t r = i / d.head, c = i - r * d.head;
            q[i] = to_float(static_cast<const T*>(d.q)[b * d.qs[0] + (first + r) * d.qs[1] + c]);
        }
        if (threadIdx.x < kRows) row_max[threadIdx.x] = -INFINITY, row_sum[threadIdx.x] = 0.0f;
        float acc[kRows];
#pragma unroll
        for (uint32_t i = 0; i < kRows; ++i) acc[i] = 0.0f;
        for (; tile < tiles && at < end; ++tile, ++at) {
            __syncthreads();
            for (uint32_t j = warp; j < kAnyTile; j += kAnyThreads / 32) {
                const uint32_t key = tile * kAnyTile + j;
                uint32_t page = 0, slot = 0;
                const bool ok = key < n && place_of(d, b, key, page, slot);
                if (lane == 0) valid[j] = ok;
                float scale[2] = {1.0f, 1.0f};
                uint64_t from[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const CacheSide& c = d.cache.side[k];
                    from[k] = page * c.s[0] + slot * c.s[1] + h * c.s[2];
                    if (SMALL && ok) scale[k] = power_of_two(c.exponents[page * c.es[0] + slot * c.es[1] + h * c.es[2]]);
                }
                for (uint32_t c = lane; c < d.head; c += 32) {
                    keys[j * pitch + c] = ok ? element<T, SMALL>(d.cache.side[0], from[0], c, scale[0]) : 0.0f;
                    values[j * pitch + c] = ok ? element<T, SMALL>(d.cache.side[1], from[1], c, scale[1]) : 0.0f;
                }
            }
            __syncthreads();
            // a warp has the scores of a row, a lane that of a key
            for (uint32_t r = warp; r < rows; r += kAnyThreads / 32) {
                float s = 0.0f;
                for (uint32_t c = 0; c < d.head; ++c) s = fmaf(q[r * d.head + c], keys[lane * pitch + c], s);
                s *= d.scale;
                // a key that counts lifts the maximum off -infinity even where its score is -infinity
                float top = valid[lane] ? fmaxf(s, kLowest) : -INFINITY;
#pragma unroll
                for (int m = 16; m; m /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
                const float old = row_max[r];
                top = fmaxf(top, old);
                const float w = valid[lane] ? exp2f(s - top) : 0.0f;
                float sum = w;
#pragma unroll
                for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
                weights[r * kAnyTile + lane] = w;
                __syncwarp();
                if (lane == 0) {
                    const float factor = old == top ? 1.0f : exp2f(old - top);
                    row_factor[r] = factor;
                    row_sum[r] = row_sum[r] * factor + sum;
                    row_max[r] = top;
                }
            }
            __syncthreads();
            if (column < d.head) {
#pragma unroll
                for (uint32_t i = 0; i < kRows; ++i) {
                    const uint32_t r = row0 + i * row_step;
                    if (r < rows) {
                        float a = acc[i] * row_factor[r];
                        for (uint32_t j = 0; j < kAnyTile; ++j) a = fmaf(weights[r * kAnyTile + j], values[j * pitch + column], a);
                        acc[i] = a;
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile == tiles;
        float* const part = d.partial + (2ull * blockIdx.x + (tile0 == 0)) * kRows * (d.head + 2);
        if (column < d.head) {
#pragma unroll
            for (uint32_t i = 0; i < kRows; ++i) {
                const uint32_t r = row0 + i * row_step;
                if (r < rows) {
                    if (whole) {
                        const float o = row_max[r] == -INFINITY ? 0.0f : acc[i] / row_sum[r];
                        static_cast<T*>(d.out)[b * d.os[0] + (first + r) * d.os[1] + column] = from_float<T>(o);
                    } else {
                        part[r * (d.head + 2) + column] = acc[i];
                        if (column == 0) part[r * (d.head + 2) + d.head] = row_max[r], part[r * (d.head + 2) + d.head + 1] = row_sum[r];
                    }
                }
            }
        }
        tile = 0;
        if (at < end && ++unit == d.units) {
            unit = 0;
            do ++b; while ((tiles = tiles_of(d, b)) == 0);  // there is work left, so there is a sequence with some
        }
    }
}

// Joins the parts of a row that blocks share: block (query head, sequence), a thread a column.  A sequence without keys
// gets zeros here.
template <typename T>
__global__ void __launch_bounds__(128) decode_join_kernel(const Decode d) {
    __shared__ uint64_t buf[33];
    const uint32_t b = blockIdx.y, query = blockIdx.x, h = query / d.group, g = (query - h * d.group) / kRows;
    const uint32_t unit = h * d.groups + g, row = query - h * d.group - g * kRows, tiles = tiles_of(d, b);
    T* const out = static_cast<T*>(d.out) + b * d.os[0] + query * d.os[1];
    if (tiles == 0) {
        for (uint32_t c = threadIdx.x; c < d.head; c += blockDim.x) out[c] = from_float<T>(0.0f);
        return;
    }
    auto count = [&](uint32_t i) { return (uint64_t)tiles_of(d, i) * d.units; };
    const uint64_t before = total_of(b, count, buf), work = total_of(d.batch, count, buf);
    const uint64_t first = before + (uint64_t)unit * tiles, blocks = sharing(d, work);
    const uint32_t c0 = (uint32_t)(((first + 1) * blocks - 1) / work), c1 = (uint32_t)(((first + tiles) * blocks - 1) / work);
    if (c0 == c1) return;
    auto part = [&](uint32_t c) { return d.partial + ((2ull * c + (c == c0)) * kRows + row) * (d.head + 2); };
    float top = -INFINITY;
    for (uint32_t c = c0; c <= c1; ++c) top = fmaxf(top, part(c)[d.head]);
    float sum = 0.0f, acc[(kMaxHead + 127) / 128] = {};
    for (uint32_t c = c0; c <= c1; ++c) {
        const float* p = part(c);
        const float m = p[d.head], factor = m == top ? 1.0f : exp2f(m - top);
        sum = fmaf(p[d.head + 1], factor, sum);
#pragma unroll
        for (uint32_t i = 0; i < (kMaxHead + 127) / 128; ++i) {
            const uint32_t column = threadIdx.x + i * 128;
            if (column < d.head) acc[i] = fmaf(p[column], factor, acc[i]);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < (kMaxHead + 127) / 128; ++i) {
        const uint32_t column = threadIdx.x + i * 128;
        if (column < d.head) out[column] = from_float<T>(top == -INFINITY ? 0.0f : acc[i] / sum);
    }
}

int prepare(const std::string& who, int dtype, const mtxc_decode_attention_args* a, Decode* out) {
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    Decode& d = *out;
    if (int rc = cache_args(who, a->cache, &d.cache)) return rc;
    if (a->cache.dtype != MTXC_FLOAT8_E4M3 && a->cache.dtype != dtype)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": queries of the cache's dtype expected (any of the three for a cache in 8 bits)");
    if (a->cache.head_dim == 0 || a->cache.head_dim > kMaxHead)
        return fail(MTXC_ERR_SHAPE, who + ": head_dim must be 1 to " + std::to_string(kMaxHead));
    if (a->batch > 65535 || a->heads >> 16)
        return fail(MTXC_ERR_SHAPE, who + ": batch must be at most 65,535 and heads below 65,536");
    if (a->heads && (!a->cache.heads || a->heads % a->cache.heads))
        return fail(MTXC_ERR_SHAPE, who + ": the query heads must be a multiple of the cache's");
    if (a->max_pages >> 31 || a->max_pages * a->cache.page_size >> 31)
        return fail(MTXC_ERR_SHAPE, who + ": the slots of a sequence's pages must be below 2^31");
    d.batch = (uint32_t)a->batch;
    d.heads = a->heads;
    d.kv_heads = std::max(1u, a->cache.heads);
    d.group = d.heads / d.kv_heads;
    d.groups = (d.group + kRows - 1) / kRows;
    d.units = d.kv_heads * d.groups;
    d.head = a->cache.head_dim;
    d.max_pages = (uint32_t)a->max_pages;
    d.q = a->q;
    d.out = a->out;
    for (int i = 0; i < 2; ++i) d.qs[i] = a->q_strides[i], d.os[i] = a->out_strides[i];
    d.table = a->page_table;
    d.table_stride = a->page_table_stride;
    d.lengths = a->lengths;
    d.scale = a->scale * 1.4426950408889634f;
    d.tile = kAnyTile;
    d.blocks = 2u * ctx().sm_count;
    return MTXC_OK;
}

size_t partial_bytes(const Decode& d) { return ((size_t)2 * d.blocks * kRows * (d.head + 2) * sizeof(float) + 255) / 256 * 256; }

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_decode_attention_workspace(int dtype, const mtxc_decode_attention_args* a, size_t* bytes) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_decode_attention_workspace";
    if (!bytes) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null pointer");
    Decode d{};
    if (int rc = prepare(who, dtype, a, &d)) return rc;
    *bytes = partial_bytes(d);
    return MTXC_OK;
}

extern "C" int mtxc_decode_attention(int dtype, const mtxc_decode_attention_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_decode_attention";
    Decode d{};
    if (int rc = prepare(who, dtype, a, &d)) return rc;
    if (!d.batch || !d.heads) return MTXC_OK;
    if (!a->q || !a->out || !a->lengths || (a->max_pages && !a->page_table))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tensor");
    const size_t bytes = partial_bytes(d);
    d.partial = static_cast<float*>(a->workspace ? a->workspace : ctx().workspace);
    if (bytes > (a->workspace ? a->workspace_bytes : ctx().workspace_bytes))
        return fail(MTXC_ERR_WORKSPACE, who + ": the partial sums need " + std::to_string(bytes) + " bytes of workspace");
    const bool small = a->cache.dtype == MTXC_FLOAT8_E4M3;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const size_t smem = sizeof(float) * (kRows * d.head + 2 * kAnyTile * (d.head + 1) + kRows * kAnyTile);
        constexpr int kMost = sizeof(float) * (kRows * kMaxHead + 2 * kAnyTile * (kMaxHead + 1) + kRows * kAnyTile);
        auto kernel = small ? decode_any_kernel<T, true> : decode_any_kernel<T, false>;
        // the same limit in every call: calls from several threads do not undo each other's
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (err != cudaSuccess) {
            rc = cuda_fail(err, "cudaFuncSetAttribute");
            return;
        }
        kernel<<<d.blocks, kAnyThreads, smem, ctx().stream()>>>(d);
        if ((rc = check_launch("decode_any_kernel"))) return;
        decode_join_kernel<T><<<dim3(d.heads, d.batch), 128, 0, ctx().stream()>>>(d);
        rc = check_launch("decode_join_kernel");
    });
    return rc;
}
