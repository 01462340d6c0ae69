// Rules on logits before a token is chosen (repeated-token penalties, biases, a grammar's bit mask), for
// sm_100a: one pass over the logits, no counts kept from call to call.
//
// A block takes a slice of one row's vocabulary.  Most tokens are in no list: they are only masked, and streamed
// through registers.  While their loads are on the way the block scans the row's tokens and biases (a few KB, from L2
// after the row's first block) and keeps what falls into its slice in shared memory: per token, how often it was
// generated, with the top bit for "also in the prompt"; one bit for the tokens that a bias names; and a list of the
// tokens with a count.  When the slice is written, each token of the list without a bias, and then each last entry of
// a biased token, is read again, ruled and written over; that also holds where dst is src, since an allowed token's
// first write leaves its value.  The counts are integer atomics, and the list's order changes nothing: equal calls
// give equal bits.
//
// [256, 131072] bf16 with a mask takes 18 us without lists (7.6 TB/s, partly from L2), 25 with 16 biases and 41
// with a history of 2,048 tokens a row too: the scans are what is left, and they are bound by issue.
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kChunks = 2;  // eights of a thread

struct Logits {
    uint32_t first_row, vocab;
    FastDiv slices_div;
    void* dst;
    const void* src;
    uint64_t ds, ss;
    const int32_t* tokens;
    uint64_t ts;
    uint32_t history;
    const int32_t *lengths, *prompt_lengths;
    const float *repetition, *frequency, *presence;
    const int32_t* bias_tokens;
    const float* bias_values;
    uint64_t bts, bvs;
    uint32_t biases;
    const uint32_t* mask;
    uint64_t ms;
};

// A thread's share of a list: its first four entries, whose loads start before their number is known, then the rest,
// four loads in flight.
template <int THREADS>
struct Share {
    const int32_t* list;
    int32_t t[4];
    __device__ __forceinline__ Share(const int32_t* p, uint32_t most) : list(p) {
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = threadIdx.x + k * THREADS < most ? __ldg(list + threadIdx.x + k * THREADS) : -1;
    }
    // fn(index, token) for the entries below n
    template <typename Fn>
    __device__ __forceinline__ void each(uint32_t n, Fn&& fn) {
        for (uint32_t i = threadIdx.x;;) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * THREADS < n) fn(i + k * THREADS, t[k]);
            i += 4 * THREADS;
            if (i >= n) break;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * THREADS < n) t[k] = __ldg(list + i + k * THREADS);
        }
    }
};

// One token's count: of type C in shared memory, 16 bits while the history is shorter than 2^15.
template <typename C>
struct Counts {
    static constexpr uint32_t kPrompt = 1u << (8 * sizeof(C) - 1);
    uint32_t* words;
    // Both return whether the token had no count before.
    __device__ __forceinline__ bool generated(uint32_t t) const { return add(t, false); }
    __device__ __forceinline__ bool prompt(uint32_t t) const { return add(t, true); }
    __device__ __forceinline__ uint32_t at(uint32_t t) const { return reinterpret_cast<const C*>(words)[t]; }

private:
    __device__ __forceinline__ bool add(uint32_t t, bool prompt) const {
        const uint32_t shift = sizeof(C) == 2 ? t % 2 * 16 : 0;
        uint32_t* w = words + (sizeof(C) == 2 ? t / 2 : t);
        const uint32_t old = prompt ? atomicOr(w, kPrompt << shift) : atomicAdd(w, 1u << shift);
        return (C)(old >> shift) == 0;
    }
};

// VEC: a thread's eights are eight consecutive tokens, one access each; else every 32nd of the warp's 256, so that
// scalar accesses are contiguous across the warp.  C: the counts' type.
template <typename T, bool VEC, int THREADS, typename C>
__global__ void __launch_bounds__(THREADS) logits_rules_kernel(const Logits a) {
    constexpr uint32_t kSlice = THREADS * kChunks * 8;  // tokens of a block
    static_assert(kSlice <= 65536 && THREADS <= 1024, "the list holds 16-bit positions, an entry 10-bit threads");
    extern __shared__ uint4 smem[];
    __shared__ uint32_t listed, named;
    __shared__ uint32_t entries[THREADS];  // of the biases looked at together: position << 10 | thread
    uint32_t* const biased = reinterpret_cast<uint32_t*>(smem);  // kSlice bits
    const Counts<C> count{biased + kSlice / 32};                 // kSlice counts
    uint16_t* const list = reinterpret_cast<uint16_t*>(reinterpret_cast<C*>(count.words) + kSlice);  // kSlice positions
    uint32_t row, slice;
    a.slices_div.divmod(blockIdx.x, row, slice);
    row += a.first_row;
    const uint32_t first = slice * kSlice, n = min(kSlice, a.vocab - first);
    const T* x = static_cast<const T*>(a.src) + row * a.ss + first;
    T* y = static_cast<T*>(a.dst) + row * a.ds + first;
    const uint32_t* mask = a.mask ? a.mask + row * a.ms + first / 32 : nullptr;
    const uint32_t lane = threadIdx.x % 32;
    auto at = [&](int k, int j) {  // element j of eight k, in the slice
        const uint32_t c = k * (THREADS * 8);
        return VEC ? c + threadIdx.x * 8 + j : c + (threadIdx.x - lane) * 8 + j * 32 + lane;
    };
    // scalar accesses: whether the warp's 256 tokens of eight k all lie in the slice, and need no comparisons
    auto whole = [&](int k) { return at(k, 0) - lane + 256 <= n; };
    Eight<T> v[kChunks];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        if constexpr (VEC) {
            if (at(k, 0) < n) v[k].load(x + at(k, 0));
        } else {
            T e[8];
            const T* p = x + at(k, 0);
            if (whole(k)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = p[32 * j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = at(k, j) < n ? p[32 * j] : T(0.0f);
            }
            memcpy(v[k].w, e, sizeof(e));
        }
    }
    const float rep = a.repetition ? __ldg(a.repetition + row) : 1.0f;
    const float freq = a.frequency ? __ldg(a.frequency + row) : 0.0f, pres = a.presence ? __ldg(a.presence + row) : 0.0f;
    const bool lists = a.tokens || a.bias_tokens;
    // The biases, THREADS at a time from the list's end; this thread's of these: its position (n or more: not in the
    // slice), entered for the others to see.
    const int32_t* names = a.bias_tokens + row * a.bts;
    const uint32_t last_names = a.bias_tokens ? (a.biases - 1) / THREADS * THREADS : 0;
    uint32_t named_here = 0xFFFFFFFFu;
    auto enter = [&](uint32_t t) {
        named_here = t;
        if (t < n) entries[atomicAdd(&named, 1u)] = t << 10 | threadIdx.x;
    };
    if (lists) {
        uint32_t len = a.history, prompt = 0;
        if (a.lengths) len = min((uint32_t)max(__ldg(a.lengths + row), 0), a.history);
        if (a.prompt_lengths) prompt = (uint32_t)max(__ldg(a.prompt_lengths + row), 0);
        Share<THREADS> tokens(a.tokens + row * a.ts, a.tokens ? a.history : 0);
        if (threadIdx.x == 0) listed = named = 0;
        const uint32_t bytes = kSlice / 8 + (a.tokens ? kSlice * sizeof(C) : 0);
        for (uint32_t i = threadIdx.x; i < bytes / 16; i += THREADS) smem[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (a.tokens) {
            tokens.each(len, [&](uint32_t i, int32_t token) {
                const uint32_t t = (uint32_t)token - first;
                if (t < n && (i < prompt ? count.prompt(t) : count.generated(t))) list[atomicAdd(&listed, 1u)] = (uint16_t)t;
            });
        }
        if (a.bias_tokens) {
            for (uint32_t i = threadIdx.x; i < a.biases; i += THREADS) {
                const uint32_t t = (uint32_t)__ldg(names + i) - first;
                if (t < n) atomicOr(&biased[t / 32], 1u << (t % 32));
                if (i >= last_names) enter(t);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        if constexpr (VEC) {
            if (at(k, 0) >= n) continue;
            if (mask) {
                const uint32_t allowed = __ldg(mask + at(k, 0) / 32) >> (at(k, 0) % 32);
                T e[8];
                memcpy(e, v[k].w, sizeof(e));
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(allowed >> j & 1u)) e[j] = from_float<T>(-INFINITY);
                memcpy(v[k].w, e, sizeof(e));
            }
            v[k].store(y + at(k, 0));
        } else {
            T e[8];
            memcpy(e, v[k].w, sizeof(e));
            T* p = y + at(k, 0);
            const uint32_t* m = mask ? mask + at(k, 0) / 32 : nullptr;  // the warp's eight words, one for each element
            if (whole(k)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[32 * j] = m && !(__ldg(m + j) >> lane & 1u) ? from_float<T>(-INFINITY) : e[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(k, j) < n) p[32 * j] = m && !(__ldg(m + j) >> lane & 1u) ? from_float<T>(-INFINITY) : e[j];
            }
        }
    }
    if (!lists) return;
    __syncthreads();  // the slice is written, the list and the bits are complete
    auto rule = [&](uint32_t t, float bias) {
        if (mask && !(mask[t / 32] >> (t % 32) & 1u)) return;
        float l = to_float(x[t]);
        const uint32_t c = a.tokens ? count.at(t) : 0, made = c & ~Counts<C>::kPrompt;
        if (c && a.repetition) l = l > 0.0f ? l / rep : l * rep;
        if (made) {
            if (a.frequency) l -= freq * (float)made;
            if (a.presence) l -= pres;
        }
        y[t] = from_float<T>(l + bias);
    };
    if (a.tokens) {
        for (uint32_t i = threadIdx.x, m = listed; i < m; i += THREADS) {
            const uint32_t t = list[i];
            if (!a.bias_tokens || !(biased[t / 32] >> (t % 32) & 1u)) rule(t, 0.0f);
        }
    }
    if (a.bias_tokens) {
        // an entry counts if its token still has its bit and no later entry of these names it too
        for (uint32_t base = last_names;; base -= THREADS) {
            const uint32_t t = named_here;
            bool last = t < n && (biased[t / 32] >> (t % 32) & 1u);
            for (uint32_t k = 0, m = last ? named : 0; k < m; ++k)
                if (entries[k] >> 10 == t && (entries[k] & 1023) > threadIdx.x) last = false;
            if (last) rule(t, a.bias_values[row * a.bvs + base + threadIdx.x]);
            if (base == 0) break;
            __syncthreads();
            if (last) atomicAnd(&biased[t / 32], ~(1u << (t % 32)));
            if (threadIdx.x == 0) named = 0;
            __syncthreads();
            enter((uint32_t)__ldg(names + base - THREADS + threadIdx.x) - first);
            __syncthreads();
        }
    }
}

// Launches of fewer than 2^31 blocks.
template <typename T, bool VEC, int THREADS, typename C>
int launch(Logits l, uint64_t rows, cudaStream_t st) {
    constexpr uint32_t kSlice = THREADS * kChunks * 8;
    const size_t smem = l.tokens ? kSlice / 8 + kSlice * (sizeof(C) + sizeof(uint16_t)) : l.bias_tokens ? kSlice / 8 : 0;
    auto kernel = logits_rules_kernel<T, VEC, THREADS, C>;
    if (smem > 40 * 1024) {  // the kernel has static shared memory too
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute(logits_rules_kernel)");
    }
    const uint32_t slices = (l.vocab + kSlice - 1) / kSlice;
    const uint64_t most = std::max<uint64_t>(1, ((1ull << 31) - 1) / slices);
    l.slices_div = FastDiv(slices);
    for (uint64_t row = 0; row < rows; row += most) {
        l.first_row = (uint32_t)row;
        kernel<<<(unsigned)(std::min(most, rows - row) * slices), THREADS, smem, st>>>(l);
        if (int rc = check_launch("logits_rules_kernel")) return rc;
    }
    return MTXC_OK;
}

// Threads of a block, and with them its slice: larger slices scan the lists less often, smaller ones hide the scan
// behind more blocks.  On a B200: [256, 131072] bf16 with a history of 2,048 takes 47 us with 256 threads, 42 with
// 512, 44 with 1024; [100, 131072] float with 1,000 26, 29 and 32; [256, 50257] bf16 (scalar accesses) 29, 35 and
// 41; [64, 131072] bf16 with 40,000 85, 58 and 45.
template <typename T, bool VEC>
int launch(const Logits& l, uint64_t rows, cudaStream_t st) {
    if (l.history >= 32768) return launch<T, VEC, 1024, uint32_t>(l, rows, st);
    if ((VEC && sizeof(T) == 2) || l.history > 8192) return launch<T, VEC, 512, uint16_t>(l, rows, st);
    return launch<T, VEC, 256, uint16_t>(l, rows, st);
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_logits_rules(int dtype, const mtxc_logits_args* a) {
    if (int rc = require_init()) return rc;
    const std::string who = "mtxc_logits_rules";
    if (!is_float_like(dtype))
        return fail(MTXC_ERR_UNSUPPORTED_DTYPE, who + ": no kernel for dtype " + dtype_name(dtype));
    if (!a) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null arguments");
    if (a->rows >> 31 || a->vocab >> 31 || a->history >> 31 || a->biases >> 31)
        return fail(MTXC_ERR_SHAPE, who + ": rows, vocab, history and biases must be below 2^31");
    if (a->history && !a->tokens) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null tokens");
    if (a->biases && (!a->bias_tokens || !a->bias_values))
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": bias_tokens and bias_values go together");
    if (a->rows == 0 || a->vocab == 0) return MTXC_OK;
    if (!a->dst || !a->src) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": null buffer");
    Logits l{};
    l.vocab = (uint32_t)a->vocab;
    l.dst = a->dst;
    l.src = a->src;
    l.ds = a->dst_stride;
    l.ss = a->src_stride;
    l.history = (uint32_t)a->history;
    if (a->history && (a->repetition || a->frequency || a->presence)) l.tokens = a->tokens;
    l.ts = a->tokens_stride;
    l.lengths = a->lengths;
    l.prompt_lengths = a->prompt_lengths;
    l.repetition = a->repetition;
    l.frequency = a->frequency;
    l.presence = a->presence;
    l.biases = (uint32_t)a->biases;
    if (a->biases) l.bias_tokens = a->bias_tokens;
    l.bias_values = a->bias_values;
    l.bts = a->bias_tokens_stride;
    l.bvs = a->bias_values_stride;
    l.mask = a->mask;
    l.ms = a->mask_stride;
    const bool vec_shape = l.vocab % 8 == 0;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool vec = vec_shape && eight_aligned<T>(l.src, a->rows == 1 ? 0 : l.ss) && eight_aligned<T>(l.dst, a->rows == 1 ? 0 : l.ds);
        rc = vec ? launch<T, true>(l, a->rows, ctx().stream()) : launch<T, false>(l, a->rows, ctx().stream());
    });
    return rc;
}
