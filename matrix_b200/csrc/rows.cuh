// Shared by the language-model row operators (dropout.cu, block_norm.cu, rotary.cu, logits.cu): the
// dispatch over the float-like dtypes and the dropout generator.
#pragma once

#include <cmath>

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

inline bool is_float_like(int dtype) { return dtype == MTXC_FLOAT || dtype == MTXC_FLOAT16 || dtype == MTXC_BFLOAT16; }

// ------------------------------------------------------------------------------------------
// Dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011), counter (column / 8, row, offset), key =
// seed; eight 16-bit lanes per counter, one for each of eight columns.  16 bits, not 32, per element: the
// generator is the integer work that bounds a 2-byte dropout (about 80 instructions per counter), and 2^-16
// is far below any use of p.
// ------------------------------------------------------------------------------------------
struct DropArgs {
    uint32_t on = 0;    // 0: nothing is dropped
    uint32_t kept = 0;  // an element is kept when its lane is below this (0 .. 65536)
    float scale = 1.0f; // 65536 / kept
    uint64_t seed = 0, offset = 0;
    const uint64_t* device_offset = nullptr;
};

// Checks a dropout state and prepares its kernel arguments; returns MTXC_OK or an error status.
inline int drop_args(const mtxc_dropout_state& s, const char* who, DropArgs* out) {
    if (!(s.p >= 0.0 && s.p <= 1.0))
        return fail(MTXC_ERR_INVALID_ARGUMENT, std::string(who) + ": the dropout probability must be in 0 .. 1");
    DropArgs d;
    d.on = s.p > 0.0;
    d.kept = (uint32_t)std::nearbyint((1.0 - s.p) * 65536.0);
    d.scale = d.kept ? (float)(65536.0 / d.kept) : 0.0f;
    d.seed = s.seed;
    d.offset = s.offset;
    d.device_offset = s.device_offset;
    *out = d;
    return MTXC_OK;
}

struct Philox {
    uint32_t k0, k1, c2, c3;
    __device__ __forceinline__ explicit Philox(const DropArgs& d) {
        uint64_t off = d.offset;
        if (d.device_offset) off += __ldg(reinterpret_cast<const unsigned long long*>(d.device_offset));
        k0 = (uint32_t)d.seed;
        k1 = (uint32_t)(d.seed >> 32);
        c2 = (uint32_t)off;
        c3 = (uint32_t)(off >> 32);
    }
    // The eight lanes of columns 8 * block .. 8 * block + 7 of `row`: lane i is half i % 2 of word i / 2.
    __device__ __forceinline__ uint4 operator()(uint32_t block, uint32_t row) const {
        uint32_t x0 = block, x1 = row, x2 = c2, x3 = c3, a = k0, b = k1;
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint64_t p0 = (uint64_t)x0 * 0xD2511F53u, p1 = (uint64_t)x2 * 0xCD9E8D57u;
            x0 = (uint32_t)(p1 >> 32) ^ x1 ^ a;
            x1 = (uint32_t)p1;
            x2 = (uint32_t)(p0 >> 32) ^ x3 ^ b;
            x3 = (uint32_t)p0;
            a += 0x9E3779B9u;
            b += 0xBB67AE85u;
        }
        return make_uint4(x0, x1, x2, x3);
    }
    // Lane i (0 .. 7) of a counter's four words.
    static __device__ __forceinline__ uint32_t lane(const uint4& w, uint32_t i) {
        const uint32_t lo = (i & 2) ? w.y : w.x, hi = (i & 2) ? w.w : w.z;
        const uint32_t v = (i & 4) ? hi : lo;
        return (i & 1) ? v >> 16 : v & 0xFFFFu;
    }
};

}  // namespace mtxc
