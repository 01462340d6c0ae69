// Shared by the language-model row operators (dropout.cu, block_norm.cu, rotary.cu, logits.cu): the
// dispatch over the float-like dtypes and the dropout generator.
#pragma once

#include <cmath>
#include <initializer_list>
#include <string>

#include "mtxc_internal.cuh"

namespace mtxc {

template <typename Fn>
bool dispatch_float(int dtype, Fn&& fn) {
    switch (dtype) {
        case MTXC_FLOAT: fn((float*)nullptr); return true;
        case MTXC_FLOAT16: fn((__half*)nullptr); return true;
        case MTXC_BFLOAT16: fn((__nv_bfloat16*)nullptr); return true;
        default: return false;
    }
}

// Refuses one tensor for two outputs (NULL: not wanted); returns MTXC_OK or an error status.
inline int distinct(const std::string& who, std::initializer_list<const void*> outputs) {
    for (auto a = outputs.begin(); a != outputs.end(); ++a)
        for (auto b = outputs.begin(); *a && b != a; ++b)
            if (*a == *b) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": one tensor for two outputs");
    return MTXC_OK;
}

// Refuses an output (NULL: not wanted) that starts where an input does.
inline int apart(const std::string& who, std::initializer_list<const void*> outputs, std::initializer_list<const void*> inputs) {
    for (const void* out : outputs)
        for (const void* in : inputs)
            if (out && out == in) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": an output over a tensor that the call reads");
    return MTXC_OK;
}

// Refuses an output that starts where the input does that it may be, and lies otherwise: `strides` of axes of these sizes.
inline int laid_alike(const std::string& who, const void* out, const uint64_t* out_strides, const void* in, const uint64_t* in_strides,
                      std::initializer_list<uint64_t> sizes) {
    if (!out || out != in) return MTXC_OK;
    for (uint64_t size : sizes) {
        if (size > 1 && *out_strides != *in_strides)
            return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": an output over its input with other strides");
        ++out_strides, ++in_strides;
    }
    return MTXC_OK;
}

inline bool is_float_like(int dtype) { return dtype == MTXC_FLOAT || dtype == MTXC_FLOAT16 || dtype == MTXC_BFLOAT16; }

// ------------------------------------------------------------------------------------------
// Dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011), counter (column / 8, row, offset), key =
// seed; eight 16-bit lanes per counter, one for each of eight columns.  16 bits, not 32, per element: the
// generator is the integer work that bounds a 2-byte dropout (about 80 instructions per counter), and 2^-16
// is far below any use of p.
// ------------------------------------------------------------------------------------------
struct DropArgs {
    uint32_t on = 0;    // 0: nothing is dropped (p too small to drop in 16 bits included)
    uint32_t kept = 0;  // an element is kept when its lane is below this (0 .. 65535)
    float scale = 1.0f; // 65536 / kept
    uint64_t offset = 0;
    const uint64_t* device_offset = nullptr;
    uint32_t key[20];   // the rounds' keys: constant operands, no additions in the kernel
};

// Checks a dropout state and prepares its kernel arguments; returns MTXC_OK or an error status.
inline int drop_args(const mtxc_dropout_state& s, const char* who, DropArgs* out) {
    if (!(s.p >= 0.0 && s.p <= 1.0))
        return fail(MTXC_ERR_INVALID_ARGUMENT, std::string(who) + ": the dropout probability must be in 0 .. 1");
    DropArgs& d = *out;
    d.kept = (uint32_t)std::nearbyint((1.0 - s.p) * 65536.0);
    d.on = d.kept < 65536;
    d.scale = d.kept ? (float)(65536.0 / d.kept) : 0.0f;
    d.offset = s.offset;
    d.device_offset = s.device_offset;
    for (uint32_t i = 0; i < 10; ++i) {
        d.key[2 * i] = (uint32_t)s.seed + i * 0x9E3779B9u;
        d.key[2 * i + 1] = (uint32_t)(s.seed >> 32) + i * 0xBB67AE85u;
    }
    return MTXC_OK;
}

// Eight lanes of one counter: lane i is half i % 2 of word i / 2.
struct Lanes {
    uint32_t w[4];
    __device__ __forceinline__ uint32_t at(uint32_t i) const {
        const uint32_t lo = (i & 2) ? w[1] : w[0], hi = (i & 2) ? w[3] : w[2];
        const uint32_t v = (i & 4) ? hi : lo;
        return (i & 1) ? v >> 16 : v & 0xFFFFu;
    }
    // lane i < kept, for a constant i: compared in the upper half of a word, which spares half the masking
    __device__ __forceinline__ bool keeps(const DropArgs& d, int i) const {
        return (i % 2 ? w[i / 2] : w[i / 2] << 16) < d.kept << 16;
    }
};

struct Philox {
    const DropArgs& d;
    uint32_t c2, c3;
    __device__ __forceinline__ explicit Philox(const DropArgs& args) : d(args) {
        uint64_t off = d.offset;
        if (d.device_offset) off += __ldg(reinterpret_cast<const unsigned long long*>(d.device_offset));
        c2 = (uint32_t)off;
        c3 = (uint32_t)(off >> 32);
    }
    // The lanes of columns 8 * block[k] .. 8 * block[k] + 7 of row[k].  N counters go through the rounds together:
    // they share the loads of the keys (a fifth of the instructions of a counter by itself) and hide each
    // other's latency.
    template <int N>
    __device__ __forceinline__ void make(const uint32_t (&block)[N], const uint32_t (&row)[N], Lanes (&out)[N]) const {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = Lanes{{block[k], row[k], c2, c3}};
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint32_t a = d.key[2 * i], b = d.key[2 * i + 1];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                uint32_t(&x)[4] = out[k].w;
                const uint64_t p0 = (uint64_t)x[0] * 0xD2511F53u, p1 = (uint64_t)x[2] * 0xCD9E8D57u;
                x[0] = (uint32_t)(p1 >> 32) ^ x[1] ^ a;
                x[1] = (uint32_t)p1;
                x[2] = (uint32_t)(p0 >> 32) ^ x[3] ^ b;
                x[3] = (uint32_t)p0;
            }
        }
    }
    __device__ __forceinline__ Lanes operator()(uint32_t block, uint32_t row) const {
        const uint32_t b[1] = {block}, r[1] = {row};
        Lanes l[1];
        make(b, r, l);
        return l[0];
    }
};

// ------------------------------------------------------------------------------------------
// N consecutive elements in one access of 8, 16 or 32 bytes (eight floats: one 256-bit access).
// ------------------------------------------------------------------------------------------
template <typename T, int N>
struct Few {
    static constexpr int kBytes = N * (int)sizeof(T);
    uint32_t w[kBytes / 4];

    // Streaming read, past L1.  Not volatile, as load_stream: read before anything writes it.
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes == 32)
            asm("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                : "l"(p));
        else if constexpr (kBytes == 16)
            asm("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                : "l"(p));
        else asm("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes == 32)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        else if constexpr (kBytes == 16) __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
        else __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[i / 2]);
            return i % 2 ? __high2float(h) : __low2float(h);
        } else return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
    // Elements 2 * i and 2 * i + 1.
    __device__ __forceinline__ float2 get2(int i) const { return make_float2(get(2 * i), get(2 * i + 1)); }
    __device__ __forceinline__ void set2(int i, float a, float b) {
        if constexpr (std::is_same_v<T, float>) {
            w[2 * i] = __float_as_uint(a);
            w[2 * i + 1] = __float_as_uint(b);
        } else if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
};
template <typename T>
using Eight = Few<T, 8>;

// What a pointer and its row stride (elements) need for Few's accesses.
template <typename T, int N>
inline bool few_aligned(const void* p, uint64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % sizeof(Few<T, N>) == 0 && stride % N == 0;
}
template <typename T>
inline bool eight_aligned(const void* p, uint64_t stride) { return few_aligned<T, 8>(p, stride); }

}  // namespace mtxc
