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
constexpr uint32_t kBlocksPerSm = 4;
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
    bool wide_slots, four_slots;  // four_slots: 32 bits, one after another, aligned to four
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

// Where a row lies in the cache: its elements and its exponents, of keys (0) or values (1).
__device__ __forceinline__ uint64_t row_at(const Rows& r, int k, int slot, uint32_t h) {
    uint32_t page, at;
    r.cache.page_div.divmod((uint32_t)slot, page, at);
    const CacheSide& c = r.cache.side[k];
    return page * c.s[0] + at * c.s[1] + h * c.s[2];
}
__device__ __forceinline__ int8_t* exponent_at(const Rows& r, int k, int slot, uint32_t h) {
    uint32_t page, at;
    r.cache.page_div.divmod((uint32_t)slot, page, at);
    const CacheSide& c = r.cache.side[k];
    return c.exponents + page * c.es[0] + at * c.es[1] + h * c.es[2];
}

// A group of 2^lanes_log lanes stores the key and the value of one head of one token, a lane every N elements, kAhead heads on
// their way at a time.  Of the tokens that name one slot the last is stored: a block looks for its slots among those of the
// tokens behind it (a bit for each of its slots modulo kBits tells nearly all of them apart at once; modulo 2,048, where one in
// 70 was mistaken, the search took most of the time: 70 us for [16384 tokens, 8 heads of 128]), while its first rows come.
// [16,384 tokens, 8 heads of 128] bf16 to 8 bits 41 us, 2.4 TB/s: 11 us of it is that search, and the rest is bound by its
// instructions (issue 57 %); to bf16 34 us, 4.0 TB/s.
constexpr int kAhead = 2;
constexpr uint32_t kBits = 32768;

// The largest finite magnitude of a group's row, as a float's bits; bad: some row of the warp has others.  (Of half types the
// magnitudes are compared two at a time as they are, and only where one is not finite each by itself.)
template <typename T, int N, bool ONE>
__device__ __forceinline__ uint32_t largest(const Piece<T, N>& x, const T* src, uint32_t lane, uint32_t lanes, uint32_t pieces, bool& bad) {
    if constexpr (ONE && N == 8 && sizeof(T) == 2) {
        constexpr uint32_t kInfinite = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, x.v.w[i] & 0x7FFF7FFFu);
        if (lane >= pieces) m = 0;
#pragma unroll
        for (uint32_t d = 16; d; d /= 2)
            if (d < lanes) m = __vmaxu2(m, __shfl_xor_sync(~0u, m, d));
        m = max(m & 0xFFFFu, m >> 16);
        bad = __any_sync(~0u, m >= kInfinite);
        if (!bad) return std::is_same_v<T, __half> ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))) : m << 16;
    }
    uint32_t top = 0;
    bad = true;
    for (uint32_t p = lane; p < pieces; p += lanes) {
        Piece<T, N> y = x;
        if (!ONE && p != lane) y.load(src + p * N);
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, finite_bits(y.get(i)));
    }
    __syncwarp();
    for (uint32_t d = lanes / 2; d; d /= 2) top = max(top, __shfl_xor_sync(~0u, top, d));
    return top;
}

template <typename T, int N, bool SMALL, bool ONE>  // ONE: no lane has more than one piece
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const Rows r) {
    __shared__ int slots[kMaxTile];
    __shared__ bool again[kMaxTile];
    __shared__ uint64_t places[2][kMaxTile], exponents[2][kMaxTile];  // of a token's slot
    __shared__ uint32_t seen[kBits / 32];
    const uint32_t t0 = blockIdx.x * r.tile, n = min(r.tile, r.tokens - t0);
    const uint32_t lanes = 1u << r.lanes_log, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> r.lanes_log;
    const uint32_t groups = kThreads >> r.lanes_log, pieces = r.head / N, items = n * r.heads;
    Piece<T, N> x[kAhead][2];
    auto row = [&](int k, uint32_t token, uint32_t h) {
        return static_cast<const T*>(r.rows[k]) + (uint64_t)(t0 + token) * r.rs[k][0] + h * r.rs[k][1];
    };
    auto load = [&](uint32_t first) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t item = first + a * groups + group;
            uint32_t token, h;
            r.heads_div.divmod(item, token, h);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (item < items && lane < pieces) x[a][k].load(row(k, token, h) + lane * N);
        }
    };
    load(0);
    for (uint32_t i = threadIdx.x; i < kBits / 32; i += kThreads) seen[i] = 0;
    __syncthreads();
    if (threadIdx.x < n) {
        const int s = slot_of(r, t0 + threadIdx.x);
        slots[threadIdx.x] = s;
        again[threadIdx.x] = false;
        if (s >= 0) {
            atomicOr(&seen[s % kBits / 32], 1u << (s % 32));
            uint32_t page, at;
            r.cache.page_div.divmod((uint32_t)s, page, at);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const CacheSide& c = r.cache.side[k];
                places[k][threadIdx.x] = page * c.s[0] + at * c.s[1];
                exponents[k][threadIdx.x] = page * c.es[0] + at * c.es[1];
            }
        }
    }
    __syncthreads();
    auto look = [&](uint32_t t, int s) {
        if (seen[(uint32_t)s % kBits / 32] >> (s & 31) & 1)
            for (uint32_t i = 0; i < n && t0 + i < t; ++i)
                if (slots[i] == s) again[i] = true;
    };
    uint32_t from = t0 + 1;
    if (r.four_slots) {
        // four at a time, sixteen on their way
        const uint32_t end = r.tokens / 4;
#pragma unroll 4
        for (uint32_t q = (from + 3) / 4 + threadIdx.x; q < end; q += kThreads) {
            const int4 v = __ldg(static_cast<const int4*>(r.slots) + q);
            // most often four slots of a page, one after another: their bits lie in one word
            const bool row = v.y == v.x + 1 && v.z == v.x + 2 && v.w == v.x + 3 && (v.x & 31) <= 28;
            if (row && !(seen[(uint32_t)v.x % kBits / 32] >> (v.x & 31) & 15)) continue;
            look(4 * q, v.x), look(4 * q + 1, v.y), look(4 * q + 2, v.z), look(4 * q + 3, v.w);
        }
        // what is left at both ends: fewer than eight
        const uint32_t t = threadIdx.x < 4 ? from + threadIdx.x : 4 * end + threadIdx.x - 4;
        if (threadIdx.x < 8 && t < r.tokens && (threadIdx.x >= 4 ? t >= from : t < (from + 3) / 4 * 4)) look(t, slot_of(r, t));
        from = r.tokens;
    }
#pragma unroll 4
    for (uint32_t t = from + threadIdx.x; t < r.tokens; t += kThreads) look(t, slot_of(r, t));
    __syncthreads();
    for (uint32_t first = 0; first < items; first += kAhead * groups) {
        if (first) load(first);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (first + a * groups >= items) break;  // for the whole block
            const uint32_t item = first + a * groups + group;
            uint32_t token, h;
            r.heads_div.divmod(item, token, h);
            const bool stored = item < items && !again[token] && slots[token] >= 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const CacheSide& c = r.cache.side[k];
                const T* const src = ONE ? nullptr : row(k, token, h);
                const uint32_t mine = stored ? pieces : 0;
                if constexpr (SMALL) {
                    bool bad;
                    const int e = exponent_of(largest<T, N, ONE>(x[a][k], src, lane, lanes, mine, bad));
                    if (!stored) continue;
                    const float scale = power_of_two(-e);
                    uint8_t* const to = static_cast<uint8_t*>(c.data) + places[k][token] + h * c.s[2];
                    for (uint32_t p = lane; p < pieces; p += lanes) {
                        Piece<T, N> y = x[a][k];
                        if (!ONE && p != lane) y.load(src + p * N);
                        float q[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const float v = y.get(i);
                            q[i] = bad && isinf(v) ? NAN : v * scale;  // the type has no infinities
                        }
                        store_bytes<N>(to + p * N, q);
                        if (ONE) break;
                    }
                    if (lane == 0) c.exponents[exponents[k][token] + h * c.es[2]] = (int8_t)e;
                } else {
                    T* const to = static_cast<T*>(c.data) + places[k][token] + h * c.s[2];
                    for (uint32_t p = lane; p < mine; p += lanes) {
                        Piece<T, N> y = x[a][k];
                        if (!ONE && p != lane) y.load(src + p * N);
                        y.store(to + p * N);
                        if (ONE) break;
                    }
                }
            }
        }
    }
}

// The way back: the slots of kAhead heads, then their rows, then what is stored.  [16,384 tokens, 8 heads of 128] 8 bits to bf16
// 21 us, 4.8 TB/s, bf16 23 us, 5.9; four heads on their way took 25.
template <typename T, int N, bool SMALL>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const Rows r) {
    using Held = std::conditional_t<SMALL, uint8_t, T>;
    struct Eight {  // eight bytes, or what a Piece has
        Piece<T, N> v;
        uint2 w;
    };
    const uint32_t lanes = 1u << r.lanes_log, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> r.lanes_log;
    const uint32_t groups = kThreads >> r.lanes_log, pieces = r.head / N;
    const uint64_t items = (uint64_t)r.tokens * r.heads, step = (uint64_t)gridDim.x * groups;
    for (uint64_t first = (uint64_t)blockIdx.x * groups + group; first < items; first += kAhead * step) {
        int slot[kAhead];
        uint32_t token[kAhead], h[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint64_t item = first + a * step;
            token[a] = (uint32_t)(item / r.heads), h[a] = (uint32_t)(item - (uint64_t)token[a] * r.heads);
            slot[a] = item < items ? slot_of(r, token[a]) : -2;
        }
        for (uint32_t p = lane; p < pieces; p += lanes) {
            Eight x[kAhead][2] = {};
            int8_t e[kAhead][2];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (slot[a] < 0) continue;
                    const Held* const from = static_cast<const Held*>(r.cache.side[k].data) + row_at(r, k, slot[a], h[a]) + p * N;
                    if constexpr (SMALL) {
                        e[a][k] = *exponent_at(r, k, slot[a], h[a]);
                        if constexpr (N == 8) x[a][k].w = *reinterpret_cast<const uint2*>(from);
                        else x[a][k].w.x = *from;
                    } else x[a][k].v.load(from);
                }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (slot[a] == -2) continue;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    T* const dst = static_cast<T*>(r.rows[k]) + (uint64_t)token[a] * r.rs[k][0] + h[a] * r.rs[k][1] + p * N;
                    if constexpr (SMALL) {
                        const float scale = slot[a] < 0 ? 0.0f : power_of_two(e[a][k]);
                        if constexpr (N == 8) {
                            Few<T, 8> y;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 v = from_e4m3((i < 2 ? x[a][k].w.x : x[a][k].w.y) >> (i % 2 * 16) & 0xFFFFu);
                                y.set2(i, v.x * scale, v.y * scale);
                            }
                            y.store(dst);
                        } else *dst = from_float<T>(from_e4m3(x[a][k].w.x).x * scale);
                    } else x[a][k].v.store(dst);
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
    for (int k = 0; k < 2; ++k)
        if (a->rows[k] && (a->rows[k] == a->cache.data[0] || a->rows[k] == a->cache.data[1]))
            return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": rows that are the cache itself");
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
    if (int rc = distinct("mtxc_cache_write", {a->cache.data[0], a->cache.data[1], a->cache.exponents[0], a->cache.exponents[1]})) return rc;
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
            c.four_slots = !c.wide_slots && c.slot_stride == 1 && aligned16(c.slots);
            // one wave of blocks where the tiles allow
            const uint32_t wave = kBlocksPerSm * ctx().sm_count;
            c.tile = std::min(kMaxTile, (c.tokens + wave - 1) / wave);
            const unsigned blocks = (c.tokens + c.tile - 1) / c.tile;
            cudaStream_t st = ctx().stream();
            const bool one = c.head / (eights ? 8 : 1) <= 1u << c.lanes_log;
            auto run = [&](auto n, auto s) {
                constexpr int N = decltype(n)::value;
                constexpr bool S = decltype(s)::value;
                if (one) cache_write_kernel<T, N, S, true><<<blocks, kThreads, 0, st>>>(c);
                else cache_write_kernel<T, N, S, false><<<blocks, kThreads, 0, st>>>(c);
            };
            using single = std::integral_constant<int, 1>;
            using eight = std::integral_constant<int, 8>;
            if (small) eights ? run(eight(), std::true_type()) : run(single(), std::true_type());
            else eights ? run(eight(), std::false_type()) : run(single(), std::false_type());
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
        const unsigned blocks = (unsigned)std::min<uint64_t>((items + groups - 1) / groups, (uint64_t)kBlocksPerSm * ctx().sm_count);
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
