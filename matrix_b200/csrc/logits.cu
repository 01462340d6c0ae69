// Rules on logits before a token is chosen (repeated-token penalties, biases, a grammar's bit mask), for
// sm_100a: one pass over the logits, no counts kept from call to call.
//
// A block takes a slice of one row's vocabulary.  It scans the row's tokens and biases once (a few KB, from
// L2 after the row's first block) and keeps what falls into its slice in shared memory: per token, how often
// it was generated with the top bit for "also in the prompt", and the last bias entry that names it.  Both are
// integer atomics, so the result does not depend on their order.  Then it streams its logits.
#include <algorithm>

#include "rows.cuh"

namespace mtxc {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kSlice = 4096;
constexpr uint32_t kPrompt = 1u << 31;

struct Logits {
    uint32_t rows, vocab, slices;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) logits_rules_kernel(const Logits a) {
    extern __shared__ uint32_t smem[];
    uint32_t* count = smem;                          // kSlice words where there are tokens
    uint32_t* entry = smem + (a.tokens ? kSlice : 0);  // kSlice words where there are biases: last entry + 1
    for (uint64_t u = blockIdx.x; u < (uint64_t)a.rows * a.slices; u += gridDim.x) {
        const uint32_t row = (uint32_t)(u / a.slices), first = (uint32_t)(u % a.slices) * kSlice;
        const uint32_t n = min(kSlice, a.vocab - first);
        __syncthreads();  // the last slice's counts are still read
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            if (a.tokens) count[i] = 0;
            if (a.bias_tokens) entry[i] = 0;
        }
        __syncthreads();
        if (a.tokens) {
            const int32_t* t = a.tokens + row * a.ts;
            const uint32_t len = a.lengths ? min((uint32_t)max(a.lengths[row], 0), a.history) : a.history;
            const uint32_t prompt = a.prompt_lengths ? (uint32_t)max(a.prompt_lengths[row], 0) : 0;
            for (uint32_t i = threadIdx.x; i < len; i += kThreads) {
                const uint32_t v = (uint32_t)t[i] - first;
                if (v < n) {
                    if (i < prompt) atomicOr(&count[v], kPrompt);
                    else atomicAdd(&count[v], 1u);
                }
            }
        }
        if (a.bias_tokens) {
            const int32_t* t = a.bias_tokens + row * a.bts;
            for (uint32_t i = threadIdx.x; i < a.biases; i += kThreads) {
                const uint32_t v = (uint32_t)t[i] - first;
                if (v < n) atomicMax(&entry[v], i + 1);
            }
        }
        __syncthreads();
        const T* x = static_cast<const T*>(a.src) + row * a.ss + first;
        T* y = static_cast<T*>(a.dst) + row * a.ds + first;
        const uint32_t* mask = a.mask ? a.mask + row * a.ms + first / 32 : nullptr;
        const float rep = a.repetition ? a.repetition[row] : 1.0f;
        const float freq = a.frequency ? a.frequency[row] : 0.0f, pres = a.presence ? a.presence[row] : 0.0f;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            float l = to_float(x[i]);
            const uint32_t c = a.tokens ? count[i] : 0;
            if (c) {
                if (a.repetition) l = l > 0.0f ? l / rep : l * rep;
                if (c & ~kPrompt) {
                    if (a.frequency) l -= freq * (float)(c & ~kPrompt);
                    if (a.presence) l -= pres;
                }
            }
            if (a.bias_tokens && entry[i]) l += a.bias_values[row * a.bvs + entry[i] - 1];
            if (mask && !(mask[i / 32] >> (i % 32) & 1u)) l = -INFINITY;
            y[i] = from_float<T>(l);
        }
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
    l.rows = (uint32_t)a->rows;
    l.vocab = (uint32_t)a->vocab;
    l.slices = (l.vocab + kSlice - 1) / kSlice;
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
    const unsigned grid = (unsigned)std::min<uint64_t>((uint64_t)l.rows * l.slices, (uint64_t)ctx().sm_count * 8);
    const size_t smem = sizeof(uint32_t) * kSlice * ((l.tokens != nullptr) + (l.bias_tokens != nullptr));
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        logits_rules_kernel<T><<<grid, kThreads, smem, ctx().stream()>>>(l);
    });
    return check_launch("logits_rules_kernel");
}
