// Shared by the attention operators (cache.cu, decode.cu, prompt.cu): the paged cache of keys and values and its checks.
#pragma once

#include <cuda_fp8.h>

#include "rows.cuh"

namespace mtxc {

struct CacheSide {  // keys or values
    void* data;
    int8_t* exponents;
    uint64_t s[3], es[3];  // page, slot, head
};

struct Cache {
    uint32_t pages, page_size, slots;
    FastDiv page_div;
    CacheSide side[2];
};

inline bool is_cache_dtype(int dtype) { return is_float_like(dtype) || dtype == MTXC_FLOAT8_E4M3; }

// Checks a cache and prepares it for the kernels; returns MTXC_OK or an error status.
inline int cache_args(const std::string& who, const mtxc_kv_cache& a, Cache* out) {
    if (!is_cache_dtype(a.dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no cache of dtype " + std::to_string(a.dtype));
    if (a.page_size == 0 || a.page_size >> 31 || a.pages > ((1ull << 31) - 1) / a.page_size)
        return fail(MTXC_ERR_SHAPE, who + ": page_size must be positive and the slots of all pages below 2^31");
    if (a.heads >> 16) return fail(MTXC_ERR_SHAPE, who + ": heads must be below 65,536");
    Cache& c = *out;
    c.pages = (uint32_t)a.pages;
    c.page_size = a.page_size;
    c.slots = (uint32_t)(a.pages * a.page_size);
    c.page_div = FastDiv(a.page_size);
    for (int k = 0; k < 2; ++k) {
        if (c.slots && a.heads && a.head_dim && (!a.data[k] || (a.dtype == MTXC_FLOAT8_E4M3 && !a.exponents[k])))
            return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null cache");
        c.side[k].data = a.data[k];
        c.side[k].exponents = a.exponents[k];
        for (int i = 0; i < 3; ++i) c.side[k].s[i] = a.strides[k][i], c.side[k].es[i] = a.exponent_strides[k][i];
    }
    return MTXC_OK;
}

// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Two bytes of e4m3 (the lower first) as floats: exact.
__device__ __forceinline__ float2 from_e4m3(uint32_t bytes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)bytes, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t to_e4m3(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// ------------------------------------------------------------------------------------------
// Which sequence a piece of work belongs to: sequence i has count(i) pieces.
// ------------------------------------------------------------------------------------------
struct Found {
    uint32_t i;      // the sequence
    uint64_t first;  // its first piece
    bool any;        // false: there are not so many pieces
};

// The pieces of sequences 0 .. n - 1, added by the whole block (buf: a word for each of its warps).
template <typename Fn>
__device__ __forceinline__ uint64_t total_of(uint32_t n, Fn&& count, uint64_t* buf) {
    uint64_t sum = 0;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) sum += count(i);
#pragma unroll
    for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
    __syncthreads();
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = 0;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) sum += buf[w];
    return sum;
}

// The sequence of piece `target`, for the whole block.
template <typename Fn>
__device__ __forceinline__ Found find(uint32_t n, uint64_t target, Fn&& count, uint64_t* buf, Found* found) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    if (threadIdx.x == 0) found->any = false;
    uint64_t before = 0;
    for (uint32_t base = 0; base < n && before <= target; base += blockDim.x) {
        const uint32_t i = base + threadIdx.x;
        const uint64_t mine = i < n ? count(i) : 0;
        uint64_t sum = mine;
#pragma unroll
        for (int m = 1; m < 32; m *= 2) {
            const uint64_t v = __shfl_up_sync(~0u, sum, m);
            if (lane >= (uint32_t)m) sum += v;
        }
        __syncthreads();
        if (lane == 31) buf[warp] = sum;
        __syncthreads();
        uint64_t all = 0;
        for (uint32_t w = 0; w < warps; ++w) {
            if (w < warp) sum += buf[w];
            all += buf[w];
        }
        const uint64_t first = before + sum - mine;
        if (first <= target && target < first + mine) *found = Found{i, first, true};
        before += all;
    }
    __syncthreads();
    return *found;
}

// A kernel that is launched as the next one's predecessor lets it start; the next one waits until all that the first has
// written is there.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Args>
cudaError_t launch_next(void (*kernel)(Args...), dim3 grid, unsigned threads, cudaStream_t stream, const Args&... args) {
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// The same for a warp by itself.  Where one round takes all sequences their counts are read once for both.
struct Counts {
    uint64_t mine, sum;  // of sequence `lane`, and of those up to it (of at most 32 sequences)
    uint64_t total;
};
__device__ __forceinline__ uint64_t warp_sums(uint64_t sum) {
    const uint32_t lane = threadIdx.x % 32;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
        const uint64_t v = __shfl_up_sync(~0u, sum, m);
        if (lane >= (uint32_t)m) sum += v;
    }
    return sum;
}
template <typename Fn>
__device__ __forceinline__ Counts warp_counts(uint32_t n, Fn&& count) {
    const uint32_t lane = threadIdx.x % 32;
    Counts c;
    c.mine = lane < n ? count(lane) : 0;
    c.sum = warp_sums(c.mine);
    c.total = __shfl_sync(~0u, c.sum, 31);
    uint64_t rest = 0;
    for (uint32_t i = 32 + lane; i < n; i += 32) rest += count(i);
    if (n > 32) c.total += __shfl_sync(~0u, warp_sums(rest), 31);
    return c;
}
template <typename Fn>
__device__ __forceinline__ Found warp_find(uint32_t n, uint64_t target, const Counts& c, Fn&& count) {
    const uint32_t lane = threadIdx.x % 32;
    uint64_t before = 0, mine = c.mine, sum = c.sum;
    for (uint32_t base = 0; base < n; base += 32) {
        if (base) {
            mine = base + lane < n ? count(base + lane) : 0;
            sum = warp_sums(mine);
        }
        const uint32_t passed = __ballot_sync(~0u, before + sum > target);
        if (passed) {
            const int l = __ffs((int)passed) - 1;
            return Found{base + l, before + __shfl_sync(~0u, sum - mine, l), true};
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return Found{0, 0, false};
}

}  // namespace mtxc
