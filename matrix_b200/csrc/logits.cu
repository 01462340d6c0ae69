// Rules on logits before a token is chosen (repeated-token penalties, biases, a grammar's bit mask), for
// sm_100a: one pass over the logits, no counts kept from call to call.
//
// A block takes a slice of one row's vocabulary.  Most tokens are in no list: they are only masked, and streamed
// through registers.  Meanwhile the block scans the row's tokens and biases (a few KB, from L2 after the row's
// first block) and keeps what falls into its slice in shared memory: per token, how often it was generated with the
// top bit for "also in the prompt", the last bias entry that names it, and a list of the tokens that have either.
// When the slice is written, the listed tokens, each once, are read again, ruled and written over; that also holds
// where dst is src, since an allowed token's first write leaves its value.  The counts are integer atomics, and
// the list's order changes nothing: equal calls give equal bits.
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;
constexpr int kChunks = 2;                            // eights of a thread
constexpr uint32_t kSlice = kThreads * kChunks * 8;   // tokens of a block
static_assert(kSlice <= 65536, "the list holds 16-bit positions");
constexpr uint32_t kPrompt = 1u << 31;

struct Logits {
    uint32_t first_row, vocab, slices;
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

// Calls fn(index, token) for a thread's share of a list, four tokens' loads in flight.
template <typename Fn>
__device__ __forceinline__ void scan(const int32_t* list, uint32_t n, Fn&& fn) {
    uint32_t i = threadIdx.x;
    for (; i + 3 * kThreads < n; i += 4 * kThreads) {
        int32_t t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = __ldg(list + i + k * kThreads);
#pragma unroll
        for (int k = 0; k < 4; ++k) fn(i + k * kThreads, t[k]);
    }
    for (; i < n; i += kThreads) fn(i, __ldg(list + i));
}

// VEC: a thread's eights are eight consecutive tokens, one access each; else every 32nd of the warp's 256, so that
// scalar accesses are contiguous across the warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) logits_rules_kernel(const Logits a) {
    extern __shared__ uint4 smem[];
    __shared__ uint32_t listed;
    uint32_t* const touched = reinterpret_cast<uint32_t*>(smem);  // kSlice bits: on the list
    uint32_t* const count = touched + kSlice / 32;                // kSlice words where there are tokens
    uint32_t* const entry = count + (a.tokens ? kSlice : 0);      // kSlice words where there are biases: last entry + 1
    uint16_t* const list = reinterpret_cast<uint16_t*>(entry + (a.bias_tokens ? kSlice : 0));  // kSlice halves
    uint32_t row, slice;
    a.slices_div.divmod(blockIdx.x, row, slice);
    row += a.first_row;
    const uint32_t first = slice * kSlice, n = min(kSlice, a.vocab - first);
    const T* x = static_cast<const T*>(a.src) + row * a.ss + first;
    T* y = static_cast<T*>(a.dst) + row * a.ds + first;
    const uint32_t lane = threadIdx.x % 32;
    auto at = [&](int k, int j) {  // element j of eight k, in the slice
        const uint32_t c = k * (kThreads * 8);
        return VEC ? c + threadIdx.x * 8 + j : c + (threadIdx.x - lane) * 8 + j * 32 + lane;
    };
    Eight<T> v[kChunks];
    uint32_t allowed[kChunks];  // bit j for element j
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        if constexpr (VEC) {
            if (at(k, 0) < n) v[k].load(x + at(k, 0));
        } else {
            T e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = at(k, j) < n ? x[at(k, j)] : T(0.0f);
            memcpy(v[k].w, e, sizeof(e));
        }
        allowed[k] = 0xFF;
        if (a.mask) {
            const uint32_t* m = a.mask + row * a.ms + first / 32;
            if constexpr (VEC) {
                if (at(k, 0) < n) allowed[k] = __ldg(m + at(k, 0) / 32) >> (at(k, 0) % 32) & 0xFF;
            } else {
                allowed[k] = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(k, j) < n) allowed[k] |= (__ldg(m + at(k, j) / 32) >> lane & 1u) << j;
            }
        }
    }
    const bool lists = a.tokens || a.bias_tokens;
    if (lists) {
        if (threadIdx.x == 0) listed = 0;
        const uint32_t words = kSlice / 32 + (a.tokens ? kSlice : 0) + (a.bias_tokens ? kSlice : 0);
        for (uint32_t i = threadIdx.x; i < words / 4; i += kThreads) smem[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto touch = [&](uint32_t t) {
            const uint32_t bit = 1u << (t % 32);
            if (!(atomicOr(&touched[t / 32], bit) & bit)) list[atomicAdd(&listed, 1u)] = (uint16_t)t;
        };
        if (a.tokens) {
            const uint32_t len = a.lengths ? min((uint32_t)max(a.lengths[row], 0), a.history) : a.history;
            const uint32_t prompt = a.prompt_lengths ? (uint32_t)max(a.prompt_lengths[row], 0) : 0;
            scan(a.tokens + row * a.ts, len, [&](uint32_t i, int32_t token) {
                const uint32_t t = (uint32_t)token - first;
                if (t >= n) return;
                if (i < prompt) atomicOr(&count[t], kPrompt);
                else atomicAdd(&count[t], 1u);
                touch(t);
            });
        }
        if (a.bias_tokens) {
            scan(a.bias_tokens + row * a.bts, a.biases, [&](uint32_t i, int32_t token) {
                const uint32_t t = (uint32_t)token - first;
                if (t >= n) return;
                atomicMax(&entry[t], i + 1);
                touch(t);
            });
        }
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        T e[8];
        memcpy(e, v[k].w, sizeof(e));
        if (allowed[k] != 0xFF) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(allowed[k] >> j & 1u)) e[j] = from_float<T>(-INFINITY);
        }
        if constexpr (VEC) {
            memcpy(v[k].w, e, sizeof(e));
            if (at(k, 0) < n) v[k].store(y + at(k, 0));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(k, j) < n) y[at(k, j)] = e[j];
        }
    }
    if (!lists) return;
    __syncthreads();  // the slice is written, the list complete
    const uint32_t m = listed;
    if (threadIdx.x >= m) return;
    const float rep = a.repetition ? a.repetition[row] : 1.0f;
    const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
    for (uint32_t i = threadIdx.x; i < m; i += kThreads) {
        const uint32_t t = list[i];
        if (a.mask && !(a.mask[row * a.ms + (first + t) / 32] >> (t % 32) & 1u)) continue;
        float l = to_float(x[t]);
        const uint32_t c = a.tokens ? count[t] : 0, made = c & ~kPrompt;
        if (c && a.repetition) l = l > 0.0f ? l / rep : l * rep;
        if (made) {
            if (a.frequency) l -= freq * (float)made;
            if (a.presence) l -= pres;
        }
        if (a.bias_tokens && entry[t]) l += a.bias_values[row * a.bvs + entry[t] - 1];
        y[t] = from_float<T>(l);
    }
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
    l.slices = (l.vocab + kSlice - 1) / kSlice;
    l.slices_div = FastDiv(l.slices);
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
    const int lists = (l.tokens != nullptr) + (l.bias_tokens != nullptr);
    const size_t smem = lists ? sizeof(uint32_t) * (kSlice / 32 + kSlice * lists + kSlice / 2) : 0;
    // launches of fewer than 2^31 blocks
    const uint64_t most = std::max<uint64_t>(1, ((1ull << 31) - 1) / l.slices);
    for (uint64_t row = 0; row < a->rows; row += most) {
        l.first_row = (uint32_t)row;
        const unsigned grid = (unsigned)(std::min(most, a->rows - row) * l.slices);
        dispatch_float(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (l.vocab % 8 == 0 && eight_aligned<T>(l.src, a->rows == 1 ? 0 : l.ss) &&
                eight_aligned<T>(l.dst, a->rows == 1 ? 0 : l.ds))
                logits_rules_kernel<T, true><<<grid, kThreads, smem, ctx().stream()>>>(l);
            else logits_rules_kernel<T, false><<<grid, kThreads, smem, ctx().stream()>>>(l);
        });
        if (int rc = check_launch("logits_rules_kernel")) return rc;
    }
    return MTXC_OK;
}
