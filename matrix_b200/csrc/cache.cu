// A paged cache of keys and values: rows of heads stored at slots, and read back, for sm_100a.
//
// In 8 bits a row is e4m3 bytes times 2^e, one e for a head of a token: the least with which the row's largest finite
// element is at most 448 = 1.75 * 2^8, e4m3's largest.  A power of two, because e4m3 has an exponent of its own: a scale in
// between would add no significant bit, while a power of two makes the scaling, its inverse and a bfloat16 or float copy of
// what was read exact, and fits one byte.
#include <algorithm>

#include "attention.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxTile = 64;
constexpr uint32_t kChunk = 16384;  // tokens of a launch of the write
constexpr uint32_t kMaxHead = 1024;

struct Rows {
    Cache cache;
    uint32_t tokens, heads, head, lanes_log, tile;
    FastDiv heads_div;
    void* rows[2];
    uint64_t rs[2][2];
    const void* slots;
    bool wide_slots;
    uint64_t slot_stride;
};

// The slot of a token of the launch; -1: none.
__device__ __forceinline__ int slot_of(const Rows& r, uint32_t token) {
    const long long s = r.wide_slots ? static_cast<const long long*>(r.slots)[token * r.slot_stride]
                                     : static_cast<const int*>(r.slots)[token * r.slot_stride];
    return s >= 0 && s < (long long)r.cache.slots ? (int)s : -1;
}

// N elements, read where they lie and written at once.
template <typename T, int N>
struct Piece {
    Few<T, N> v;
    __device__ __forceinline__ void load(const T* p) { v.load(p); }
    __device__ __forceinline__ void store(T* p) const { v.store(p); }
    __device__ __forceinline__ float get(int i) const { return v.get(i); }
    __device__ __forceinline__ void set2(int i, float a, float b) { v.set2(i, a, b); }
};
template <typename T>
struct Piece<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ float get(int) const { return to_float(v); }
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}

// The exponent of the scale of a row whose largest finite element has these bits.
__device__ __forceinline__ int exponent_of(uint32_t top) {
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7FFFFFu) > 0x600000u);
    return top ? max(-96, min(96, e)) : 0;
}

template <int N>
__device__ __forceinline__ void store_bytes(uint8_t* p, const float (&y)[N]) {
    if constexpr (N == 8) {
        uint2 w;
        w.x = to_e4m3(y[0], y[1]) | to_e4m3(y[2], y[3]) << 16;
        w.y = to_e4m3(y[4], y[5]) | to_e4m3(y[6], y[7]) << 16;
        *reinterpret_cast<uint2*>(p) = w;
    } else *p = (uint8_t)to_e4m3(y[0], 0.0f);
}

// A group of 2^lanes_log lanes stores the key and the value of one head of one token, a lane every N elements.  Of the
// tokens that name one slot the last is stored: a block looks for its slots among those of the tokens behind it (a bit for
// each of its slots modulo 2,048 tells nearly all of them apart at once).
template <typename T, int N, bool SMALL>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const Rows r) {
    __shared__ int slots[kMaxTile];
    __shared__ bool again[kMaxTile];
    __shared__ uint32_t seen[64];
    const uint32_t t0 = blockIdx.x * r.tile, n = min(r.tile, r.tokens - t0);
    if (threadIdx.x < 64) seen[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x < n) {
        const int s = slot_of(r, t0 + threadIdx.x);
        slots[threadIdx.x] = s;
        again[threadIdx.x] = false;
        if (s >= 0) atomicOr(&seen[s % 2048 / 32], 1u << (s % 32));
    }
    __syncthreads();
    for (uint32_t t = t0 + 1 + threadIdx.x; t < r.tokens; t += kThreads) {
        const int s = slot_of(r, t);
        if (s >= 0 && (seen[s % 2048 / 32] >> (s % 32) & 1))
            for (uint32_t i = 0; i < n && t0 + i < t; ++i)
                if (slots[i] == s) again[i] = true;
    }
    __syncthreads();
    const uint32_t lanes = 1u << r.lanes_log, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> r.lanes_log;
    const uint32_t groups = kThreads >> r.lanes_log, pieces = r.head / N, items = n * r.heads;
    for (uint32_t base = 0; base < items; base += groups) {
        const uint32_t item = base + group;
        uint32_t token, h;
        r.heads_div.divmod(item, token, h);
        const int slot = item < items && !again[token] ? slots[token] : -1;
        uint32_t page = 0, at = 0;
        if (slot >= 0) r.cache.page_div.divmod((uint32_t)slot, page, at);
        const T* src[2];
        Piece<T, N> x[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            src[k] = static_cast<const T*>(r.rows[k]) + (uint64_t)(t0 + token) * r.rs[k][0] + h * r.rs[k][1];
            if (slot >= 0 && lane < pieces) x[k].load(src[k] + lane * N);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const CacheSide& c = r.cache.side[k];
            const uint64_t to = page * c.s[0] + at * c.s[1] + h * c.s[2];
            if constexpr (SMALL) {
                uint32_t top = 0;
                if (slot >= 0)
                    for (uint32_t p = lane; p < pieces; p += lanes) {
                        Piece<T, N> y = x[k];
                        if (p != lane) y.load(src[k] + p * N);
#pragma unroll
                        for (int i = 0; i < N; ++i) top = max(top, finite_bits(y.get(i)));
                    }
                for (uint32_t m = lanes / 2; m; m /= 2) top = max(top, __shfl_xor_sync(~0u, top, m));
                if (slot < 0) continue;
                const int e = exponent_of(top);
                const float scale = power_of_two(-e);
                for (uint32_t p = lane; p < pieces; p += lanes) {
                    Piece<T, N> y = x[k];
                    if (p != lane) y.load(src[k] + p * N);
                    float q[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float v = y.get(i);
                        q[i] = fmaf(v, scale, v - v);  // an infinity becomes NaN: the type has none
                    }
                    store_bytes<N>(static_cast<uint8_t*>(c.data) + to + p * N, q);
                }
                if (lane == 0) c.exponents[page * c.es[0] + at * c.es[1] + h * c.es[2]] = (int8_t)e;
            } else {
                if (slot < 0) continue;
                for (uint32_t p = lane; p < pieces; p += lanes) {
                    Piece<T, N> y = x[k];
                    if (p != lane) y.load(src[k] + p * N);
                    y.store(static_cast<T*>(c.data) + to + p * N);
                }
            }
        }
    }
}

template <typename T, int N, bool SMALL>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const Rows r) {
    const uint32_t lanes = 1u << r.lanes_log, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> r.lanes_log;
    const uint32_t groups = kThreads >> r.lanes_log, pieces = r.head / N;
    const uint64_t items = (uint64_t)r.tokens * r.heads;
    for (uint64_t item = (uint64_t)blockIdx.x * groups + group; item < items; item += (uint64_t)gridDim.x * groups) {
        const uint32_t token = (uint32_t)(item / r.heads), h = (uint32_t)(item - (uint64_t)token * r.heads);
        const int slot = slot_of(r, token);
        uint32_t page = 0, at = 0;
        if (slot >= 0) r.cache.page_div.divmod((uint32_t)slot, page, at);
        for (uint32_t p = lane; p < pieces; p += lanes) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const CacheSide& c = r.cache.side[k];
                T* dst = static_cast<T*>(r.rows[k]) + (uint64_t)token * r.rs[k][0] + h * r.rs[k][1] + p * N;
                const uint64_t from = page * c.s[0] + at * c.s[1] + h * c.s[2] + p * N;
                if constexpr (!SMALL) {
                    Piece<T, N> y{};
                    if (slot >= 0) y.load(static_cast<const T*>(c.data) + from);
                    y.store(dst);
                } else {
                    float scale = 0.0f;
                    if (slot >= 0) scale = power_of_two(c.exponents[page * c.es[0] + at * c.es[1] + h * c.es[2]]);
                    const uint8_t* bytes = static_cast<const uint8_t*>(c.data) + from;
                    if constexpr (N == 8) {
                        uint2 w = make_uint2(0, 0);
                        if (slot >= 0) w = *reinterpret_cast<const uint2*>(bytes);
                        Few<T, 8> y;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 v = from_e4m3((i < 2 ? w.x : w.y) >> (i % 2 * 16) & 0xFFFFu);
                            y.set2(i, v.x * scale, v.y * scale);
                        }
                        y.store(dst);
                    } else *dst = from_float<T>(slot >= 0 ? from_e4m3(*bytes).x * scale : 0.0f);
                }
            }
        }
    }
}

int prepare(const std::string& who, int dtype, const mtxc_cache_rows_args* a, Rows* out) {
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    Rows& r = *out;
    if (int rc = cache_args(who, a->cache, &r.cache)) return rc;
    if (a->cache.dtype != MTXC_FLOAT8_E4M3 && a->cache.dtype != dtype)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": rows of the cache's dtype expected (any of the three for a cache in 8 bits)");
    if (a->cache.head_dim > kMaxHead) return fail(MTXC_ERR_SHAPE, who + ": head_dim must be at most " + std::to_string(kMaxHead));
    if (a->tokens >> 31) return fail(MTXC_ERR_SHAPE, who + ": tokens must be below 2^31");
    if (a->slot_dtype != MTXC_INT32 && a->slot_dtype != MTXC_INT64)
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": slots must be Int32 or Int64");
    if (a->tokens && a->cache.heads && a->cache.head_dim && (!a->rows[0] || !a->rows[1] || !a->slots))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null rows or slots");
    r.tokens = (uint32_t)a->tokens;
    r.heads = a->cache.heads;
    r.head = a->cache.head_dim;
    r.heads_div = FastDiv(std::max(1u, r.heads));
    for (int k = 0; k < 2; ++k) {
        r.rows[k] = a->rows[k];
        r.rs[k][0] = a->row_strides[k][0], r.rs[k][1] = a->row_strides[k][1];
    }
    r.slots = a->slots;
    r.wide_slots = a->slot_dtype == MTXC_INT64;
    r.slot_stride = a->slot_stride;
    return MTXC_OK;
}

// Whether rows of T and the cache's rows can be moved eight elements at a time; sets the lanes of a group.
template <typename T>
bool by_eights(Rows& r, bool small) {
    bool ok = r.head % 8 == 0;
    for (int k = 0; ok && k < 2; ++k) {
        for (int i = 0; i < 2; ++i) ok = ok && few_aligned<T, 8>(r.rows[k], r.rs[k][i]);
        const CacheSide& c = r.cache.side[k];
        for (int i = 0; i < 3; ++i)
            ok = ok && (small ? reinterpret_cast<uintptr_t>(c.data) % 8 == 0 && c.s[i] % 8 == 0 : few_aligned<T, 8>(c.data, c.s[i]));
    }
    const uint32_t pieces = ok ? r.head / 8 : r.head;
    r.lanes_log = 0;
    while (r.lanes_log < 5 && (1u << r.lanes_log) < pieces) ++r.lanes_log;
    return ok;
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_cache_write(int dtype, const mtxc_cache_rows_args* a) {
    if (int rc = require_init()) return rc;
    Rows r{};
    if (int rc = prepare("mtxc_cache_write", dtype, a, &r)) return rc;
    if (int rc = distinct("mtxc_cache_write", {a->cache.data[0], a->cache.data[1]})) return rc;
    if (!r.tokens || !r.heads || !r.head || !r.cache.slots) return MTXC_OK;
    const bool small = a->cache.dtype == MTXC_FLOAT8_E4M3;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool eights = by_eights<T>(r, small);
        // launches of kChunk tokens: a block's search through the tokens behind it stays short, and a later launch
        // overwrites an earlier one's slots
        for (uint64_t first = 0; first < a->tokens && rc == MTXC_OK; first += kChunk) {
            Rows c = r;
            c.tokens = (uint32_t)std::min<uint64_t>(kChunk, a->tokens - first);
            for (int k = 0; k < 2; ++k) c.rows[k] = static_cast<T*>(r.rows[k]) + first * r.rs[k][0];
            c.slots = static_cast<const char*>(r.slots) + first * r.slot_stride * (r.wide_slots ? 8 : 4);
            c.tile = std::max(1u, std::min(kMaxTile, c.tokens / (4u * ctx().sm_count)));
            const unsigned blocks = (c.tokens + c.tile - 1) / c.tile;
            cudaStream_t st = ctx().stream();
            auto run = [&](auto n, auto s) {
                cache_write_kernel<T, decltype(n)::value, decltype(s)::value><<<blocks, kThreads, 0, st>>>(c);
            };
            using one = std::integral_constant<int, 1>;
            using eight = std::integral_constant<int, 8>;
            if (small) eights ? run(eight(), std::true_type()) : run(one(), std::true_type());
            else eights ? run(eight(), std::false_type()) : run(one(), std::false_type());
            rc = check_launch("cache_write_kernel");
        }
    });
    return rc;
}

extern "C" int mtxc_cache_read(int dtype, const mtxc_cache_rows_args* a) {
    if (int rc = require_init()) return rc;
    Rows r{};
    if (int rc = prepare("mtxc_cache_read", dtype, a, &r)) return rc;
    if (int rc = distinct("mtxc_cache_read", {a->rows[0], a->rows[1]})) return rc;
    if (!r.tokens || !r.heads || !r.head) return MTXC_OK;
    const bool small = a->cache.dtype == MTXC_FLOAT8_E4M3;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool eights = by_eights<T>(r, small);
        const uint64_t groups = kThreads >> r.lanes_log, items = (uint64_t)r.tokens * r.heads;
        const unsigned blocks = (unsigned)std::min<uint64_t>((items + groups - 1) / groups, 8u * ctx().sm_count);
        cudaStream_t st = ctx().stream();
        auto run = [&](auto n, auto s) {
            cache_read_kernel<T, decltype(n)::value, decltype(s)::value><<<blocks, kThreads, 0, st>>>(r);
        };
        using one = std::integral_constant<int, 1>;
        using eight = std::integral_constant<int, 8>;
        if (small) eights ? run(eight(), std::true_type()) : run(one(), std::true_type());
        else eights ? run(eight(), std::false_type()) : run(one(), std::false_type());
    });
    return check_launch("cache_read_kernel");
}
