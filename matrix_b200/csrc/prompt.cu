// Attention over whole prompts, for sm_100a: packed sequences of different lengths, grouped heads, causal or not.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j,  m_i a running maximum
//
// over the keys j <= i + (m - n) of a sequence of n queries and m keys (causal) or all of them.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "tensor.cuh"

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
    bool pairs;   // the tensor cores' kernel: two heads of a group a block, and not two tiles of a head
};

// Rows [first, first + count) of a sequence, within what there is.
__device__ __forceinline__ void rows_of(const int* starts, uint32_t i, uint32_t tokens, uint32_t& first, uint32_t& count) {
    const uint32_t lo = (uint32_t)min(max(starts[i], 0), (int)tokens), hi = (uint32_t)min(max(starts[i + 1], 0), (int)tokens);
    first = lo;
    count = hi > lo ? hi - lo : 0;
}

// ------------------------------------------------------------------------------------------
// Any head and type: 16 ROWS queries and 64 keys at a time, products in 32 bits on the multipliers, a thread ROWS rows by 4 keys
// of the scores and by up to 16 elements of the output.  The next keys come while the weights meet the values, the next values
// while the scores are made.  ROWS = 2 where there would be fewer than four blocks of 64 rows an SM: its blocks are half as long
// ([500, 228, 381] f32, 8 heads of 80: a row of tiles of 64 keys is all that the longest block has).
// ------------------------------------------------------------------------------------------
__host__ __device__ inline uint32_t pitch_of(uint32_t head) { return (head + 3) / 8 * 8 + 4; }  // an odd number of 16-byte units
constexpr uint32_t kTilePitch = kAnyTile + 4;

template <int ROWS>
uint32_t any_bytes(uint32_t head) { return (uint32_t)sizeof(float) * ((16 * ROWS + 2 * kAnyTile) * pitch_of(head) + 16 * ROWS * kTilePitch); }

template <typename T, int ROWS, int COLUMNS, bool WHOLE>  // COLUMNS: 64 elements each; WHOLE: float, by 16-byte units
__global__ void __launch_bounds__(kAnyThreads) prompt_any_kernel(const Prompt p) {
    extern __shared__ float4 smem4[];
    __shared__ uint64_t buf[kAnyThreads / 32];
    __shared__ Found found;
    constexpr uint32_t kRows = 16 * ROWS;
    const uint32_t pitch = pitch_of(p.head), quads = (p.head + 3) / 4;
    float* const q = reinterpret_cast<float*>(smem4);    // [kRows][pitch]
    float* const keys = q + kRows * pitch;               // [64][pitch]
    float* const values = keys + kAnyTile * pitch;       // [64][pitch]
    float* const weights = values + kAnyTile * pitch;    // [kRows][kTilePitch]
    // the last sequence first, and in each the last tile first: of causal ones the longest
    auto count = [&](uint32_t i) {
        uint32_t first, n;
        rows_of(p.starts, p.sequences - 1 - i, p.tokens, first, n);
        return (uint64_t)(n + kRows - 1) / kRows;
    };
    const Found f = find(p.sequences, blockIdx.x, count, buf, &found);
    if (!f.any) return;
    const uint32_t i = p.sequences - 1 - f.i, h = blockIdx.y, kh = p.group_div.div(h);
    uint32_t q_first, n, k_first, m;
    rows_of(p.starts, i, p.tokens, q_first, n);
    rows_of(p.k_starts, i, p.k_tokens, k_first, m);
    const uint32_t row0 = ((n + kRows - 1) / kRows - 1 - (uint32_t)(blockIdx.x - f.first)) * kRows;
    const int64_t ahead = (int64_t)m - n;  // a query sees keys up to its own index plus this
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    // a warp a row; rows and elements that are not there are zeros
    auto load = [&](float* to, const void* from, const uint64_t (&s)[2], uint32_t first, uint32_t head, uint32_t rows, uint32_t all) {
        const T* x = static_cast<const T*>(from) + head * s[1] + (uint64_t)first * s[0];
        for (uint32_t r = warp; r < all; r += kAnyThreads / 32) {
            if constexpr (WHOLE) {
                for (uint32_t c = lane; c < quads; c += 32)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + r * pitch + 4 * c)),
                                 "l"(r < rows ? x + (uint64_t)r * s[0] + 4 * c : static_cast<const T*>(from)), "r"(r < rows ? 16 : 0)
                                 : "memory");
            } else {
                for (uint32_t c = lane; c < 4 * quads; c += 32)
                    to[r * pitch + c] = r < rows && c < p.head ? to_float(x[(uint64_t)r * s[0] + c]) : 0.0f;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;  // rows ROWS ty .., keys tx + 16 j, columns 4 tx + 64 c
    float top[ROWS], sum[ROWS];
    float2 acc[ROWS][COLUMNS][2];
#pragma unroll
    for (int a = 0; a < ROWS; ++a) {
        top[a] = -INFINITY, sum[a] = 0.0f;
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) acc[a][c][0] = acc[a][c][1] = make_float2(0.0f, 0.0f);
    }
    const int64_t last = p.causal ? min((int64_t)m, (int64_t)min(row0 + kRows, n) + ahead) : (int64_t)m;  // keys seen by any row
    auto keys_of = [&](int64_t k0) { return (uint32_t)max((int64_t)0, min((int64_t)kAnyTile, m - k0)); };
    load(q, p.q, p.qs, q_first + row0, h, min(kRows, n - row0), kRows);
    load(keys, p.k, p.ks, k_first, kh, last > 0 ? keys_of(0) : 0, kAnyTile);
    load(values, p.v, p.vs, k_first, kh, last > 0 ? keys_of(0) : 0, kAnyTile);
    for (int64_t k0 = 0; k0 < last; k0 += kAnyTile) {
        const uint32_t there = keys_of(k0);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // all but the values
        __syncthreads();
        float2 even_odd[ROWS][4] = {};  // the products of even and of odd elements: two at a time
#pragma unroll 2
        for (uint32_t c = 0; c < quads; ++c) {
            float4 x[ROWS], y[4];
#pragma unroll
            for (int a = 0; a < ROWS; ++a) x[a] = *reinterpret_cast<const float4*>(q + (ROWS * ty + a) * pitch + 4 * c);
#pragma unroll
            for (int b = 0; b < 4; ++b) y[b] = *reinterpret_cast<const float4*>(keys + (tx + 16 * b) * pitch + 4 * c);
#pragma unroll
            for (int a = 0; a < ROWS; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    even_odd[a][b] = __ffma2_rn(make_float2(x[a].x, x[a].y), make_float2(y[b].x, y[b].y), even_odd[a][b]);
                    even_odd[a][b] = __ffma2_rn(make_float2(x[a].z, x[a].w), make_float2(y[b].z, y[b].w), even_odd[a][b]);
                }
        }
        float s[ROWS][4];
#pragma unroll
        for (int a = 0; a < ROWS; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) s[a][b] = even_odd[a][b].x + even_odd[a][b].y;
        int limit[ROWS];  // the last key of this tile that a row sees
        bool all = true;
#pragma unroll
        for (int a = 0; a < ROWS; ++a) {
            const int64_t sees = (p.causal ? min((int64_t)m - 1, (int64_t)row0 + ROWS * ty + a + ahead) : (int64_t)m - 1) - k0;
            limit[a] = (int)max((int64_t)-1, min((int64_t)kAnyTile - 1, sees));
            all = all && limit[a] == kAnyTile - 1;
            float now = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                s[a][b] *= p.scale;
                // a key that counts lifts the maximum off -infinity even where its score is -infinity
                if ((int)tx + 16 * b <= limit[a]) now = fmaxf(now, fmaxf(s[a][b], kLowest));
            }
#pragma unroll
            for (int d = 8; d; d /= 2) now = fmaxf(now, __shfl_xor_sync(~0u, now, d));
            now = fmaxf(now, top[a]);
            const float factor = now == top[a] ? 1.0f : exp2f(top[a] - now);
            top[a] = now;
            float part = 0.0f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float w = (int)tx + 16 * b <= limit[a] ? exp2f(s[a][b] - now) : 0.0f;
                part += w;
                weights[(ROWS * ty + a) * kTilePitch + tx + 16 * b] = w;
            }
            sum[a] = sum[a] * factor + part;
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) acc[a][c][e] = __fmul2_rn(acc[a][c][e], make_float2(factor, factor));
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the scores are made, the values have come
        const int64_t next = k0 + kAnyTile;
        load(keys, p.k, p.ks, k_first + (uint32_t)next, kh, next < last ? keys_of(next) : 0, next < last ? kAnyTile : 0);
        auto add = [&](float w, const float4& y, float2 (&o)[2]) {
            o[0] = __ffma2_rn(make_float2(w, w), make_float2(y.x, y.y), o[0]);
            o[1] = __ffma2_rn(make_float2(w, w), make_float2(y.z, y.w), o[1]);
        };
        for (uint32_t j = 0; j < there; j += 4) {
            float4 w[ROWS];
#pragma unroll
            for (int a = 0; a < ROWS; ++a) w[a] = *reinterpret_cast<const float4*>(weights + (ROWS * ty + a) * kTilePitch + j);
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                if (tx + 16 * c >= quads) break;
                const float* const v = values + j * pitch + 4 * (tx + 16 * c);
                float4 y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = *reinterpret_cast<const float4*>(v + e * pitch);
                if (all) {
#pragma unroll
                    for (int a = 0; a < ROWS; ++a) add(w[a].x, y[0], acc[a][c]), add(w[a].y, y[1], acc[a][c]), add(w[a].z, y[2], acc[a][c]), add(w[a].w, y[3], acc[a][c]);
                } else {
                    // what a row does not see may hold anything
#pragma unroll
                    for (int a = 0; a < ROWS; ++a) {
                        if ((int)j <= limit[a]) add(w[a].x, y[0], acc[a][c]);
                        if ((int)j + 1 <= limit[a]) add(w[a].y, y[1], acc[a][c]);
                        if ((int)j + 2 <= limit[a]) add(w[a].z, y[2], acc[a][c]);
                        if ((int)j + 3 <= limit[a]) add(w[a].w, y[3], acc[a][c]);
                    }
                }
            }
        }
        __syncthreads();
        load(values, p.v, p.vs, k_first + (uint32_t)next, kh, next < last ? keys_of(next) : 0, next < last ? kAnyTile : 0);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int a = 0; a < ROWS; ++a) {
#pragma unroll
        for (int d = 8; d; d /= 2) sum[a] += __shfl_xor_sync(~0u, sum[a], d);
        const uint32_t row = row0 + ROWS * ty + a;
        if (row >= n) continue;
        T* out = static_cast<T*>(p.out) + (uint64_t)(q_first + row) * p.os[0] + h * p.os[1];
        const bool any = top[a] != -INFINITY;
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) {
            const uint32_t at = 4 * (tx + 16 * c);
            const float o[4] = {acc[a][c][0].x, acc[a][c][0].y, acc[a][c][1].x, acc[a][c][1].y};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (at + e < p.head) out[at + e] = from_float<T>(any ? o[e] / sum[a] : 0.0f);
        }
    }
}

template <typename T, int ROWS, bool WHOLE>
int launch_any(const mtxc_prompt_attention_args* a, const Prompt& p) {
    auto kernel = p.head <= 64    ? prompt_any_kernel<T, ROWS, 1, WHOLE>
                  : p.head <= 128 ? prompt_any_kernel<T, ROWS, 2, WHOLE>
                                  : prompt_any_kernel<T, ROWS, 4, WHOLE>;
    // the same limit in every call: calls from several threads do not undo each other's
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)any_bytes<ROWS>(kMaxHead));
    if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
    // as many tiles as the sequences can have: one each may be part filled
    const uint64_t tiles = a->tokens / (16 * ROWS) + std::min(a->sequences, a->tokens);
    kernel<<<dim3((unsigned)tiles, a->heads), kAnyThreads, any_bytes<ROWS>(p.head), ctx().stream()>>>(p);
    return check_launch("prompt_any_kernel");
}

template <typename T>
int launch_any(const mtxc_prompt_attention_args* a, const Prompt& p) {
    const bool few = (a->tokens / 64 + std::min(a->sequences, a->tokens)) * a->heads < 4u * ctx().sm_count;
    if constexpr (std::is_same_v<T, float>) {
        bool whole = a->head_dim % 4 == 0;
        for (const void* x : {a->q, a->k, a->v}) whole = whole && aligned16(x);
        for (int i = 0; i < 2; ++i) whole = whole && a->q_strides[i] % 4 == 0 && a->k_strides[i] % 4 == 0 && a->v_strides[i] % 4 == 0;
        if (whole) return few ? launch_any<T, 2, true>(a, p) : launch_any<T, 4, true>(a, p);
    }
    return few ? launch_any<T, 2, false>(a, p) : launch_any<T, 4, false>(a, p);
}

// ------------------------------------------------------------------------------------------
// Half types on the tensor cores.
//
// A block has NT tiles of 128 queries (NT = 2 for heads of up to 128 elements: of two heads that share keys, or, where groups
// are odd, one behind the other of one head) and runs along the keys in tiles of 128.  Roles: four warps for each tile of
// queries, a thread a row, have its softmax; one warp issues the products, one the copies, and two clean values (below).  The
// scores S = Q K' of a tile lie in tensor memory; a row's thread reads them, writes the weights P over them in 16 bits, and the
// product with V takes them from there, so that neither passes through shared memory.  While one tile of queries is with its
// softmax the tensor cores work for the other, and the product of the first half of the keys' weights starts while the second
// half is made:
//     S0(j)  softmax 0         | P0 V(j), S0(j+1)
//     S1(j)         softmax 1         | P1 V(j), S1(j+1)
// (Scores 64 keys at a time, with two places in turn for each tile: 780 us for prompts of 8,192 and 3,903 tokens where 128 keys
// took 691, because a product of 64 columns takes the tensor cores as long as one of 128.  Blocks that stay and take one piece
// of work after another, the next one's scores made during the last one's output: 635 us where one piece a block took 597.)
//
// The output is rescaled only where the maximum has grown by more than 2^8 since it last was: until then weights stay below
// 2^8 (the sums are exact whatever the reference point is), and nearly all tiles keep the first one's.  S(j + 1) is issued
// behind P V(j), so a thread that sees S(j + 1) may touch the output.  float16 weights are taken 2^11 times and rescaled from
// 2^4 on: they end at 2^15 (the type at 65,504), and only what is below 2^-25 of the largest has fewer than 11 bits (its
// rounding is to multiples of 2^-24).  At 1 and 2^8 a key with nearly all the weight left others of 2^-25 as nothing or twice
// what they are, and those are the output where its value is 0.
//
// Measured, 32 heads of 128 over 8, bf16: two prompts of 8,192 tokens 898 us in a few calls, 1,225 TFLOP/s (0.73 of cuBLAS's
// burst), of 8,192 and 3,903 tokens 572 us, 1,180, and back to back for a second, under the power limit, 663 us, 1,015; 24 prompts
// of 105 to 777 tokens, 16 heads of 64, f16: 77 us, 237.  Heads of 80 and 96 take the work of 128, of 136 to 192 that of 256 (two
// prompts of 4,096 tokens, 16 heads of 64, 80, 96, 128, 160, 192, 256 over 4: 113, 134, 140, 140, 328, 328, 333 us).
// Weights are operands of 16 bits, which adds to the result's own rounding (relative 0.0021 against 64 bits in bfloat16, of which
// 0.0016 are that rounding; 2.6e-4 and 2.1e-4 in float16): a second operand, as in decode, would be half as many products again
// and more to make for the softmax.  Bound by the exchange of a tile between its softmax and its products: the tensor cores are
// busy for half of the time at heads of 128 and for a quarter at 64, whose products take half as long and whose softmax as long;
// the exponentials' unit for 38 %.
//
// What a row does not see gets the weight 0, which is not enough where the value is NaN or infinite (another sequence's
// row, a later token).  The two cleaning warps look through the tiles of values that some row does not see whole: rows
// behind the sequence are zeroed, and a non-finite element of a later token is zeroed and its first key noted for each
// element of the head, so that rows that do see it receive it at the end.
// ------------------------------------------------------------------------------------------
constexpr int kThreads = 384;
constexpr uint32_t kTile = 128, kHalf = 64;

struct Maps {
    CUtensorMap q, k, v;
    uint32_t tokens_last;  // bit 0, 1, 2: of q, k, v the token is the outermost axis (else the head)
};

template <int D, int NT>
struct Layout {
    static constexpr uint32_t kRowTile = kTile * 128;             // 64 elements of 128 rows
    static constexpr uint32_t kTileBytes = kRowTile * (D / 64);
    static constexpr uint32_t kSlots = D == 256 ? 2 : D == 128 ? 5 : 8;  // keys and values in turn
    static constexpr uint32_t kAgain = kSlots % 2 ? kSlots : kSlots / 2;  // tiles from one whose values have a slot to the next
    static constexpr uint32_t kBytes = kTileBytes * (NT + kSlots) + 1024;  // the tiles start at a multiple of 1,024
    // With an odd number of slots keys and values take turns in a slot.  Values that are to be cleaned arrive at `raw`, and the
    // slot's `full` misses a phase that its next keys' wait counts: (kSlots + 1) / 2 tiles further, which has to be behind the
    // last tile.  NT + 1 tiles of keys at most are seen in part by NT tiles of rows, one behind the other, and cleaned.
    static_assert(kSlots % 2 == 0 || NT + 1 <= (kSlots + 1) / 2, "keys would be waited for at a phase that their slot does not reach");
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// Whether none of eight elements is NaN or infinite: their products with 0 are added up.
template <typename T>
__device__ __forceinline__ bool all_finite(const uint4& w) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 zero = __float2half2_rn(0.0f);
        __half2 s = __hmul2(*reinterpret_cast<const __half2*>(&w.x), zero);
        s = __hfma2(*reinterpret_cast<const __half2*>(&w.y), zero, s);
        s = __hfma2(*reinterpret_cast<const __half2*>(&w.z), zero, s);
        s = __hfma2(*reinterpret_cast<const __half2*>(&w.w), zero, s);
        return __hbeq2(s, zero);
    } else {
        const __nv_bfloat162 zero = __float2bfloat162_rn(0.0f);
        __nv_bfloat162 s = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w.x), zero);
        s = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.y), zero, s);
        s = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.z), zero, s);
        s = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.w), zero, s);
        return __hbeq2(s, zero);
    }
}

// 2^x on the multipliers, for a share of the weights: the unit that has the function makes 16 a clock, which is what a tile's
// two products take.  x = n + f with n whole and |f| <= 1/2; 2^f by the polynomial of least largest relative error that is 1 at
// 0 (found by exchange of its extrema: 1.0e-4 of degree 3, 3.6e-6 of degree 4, to bfloat16's 2^-9 and float16's 2^-12 of
// rounding), n added to its exponent.  From -127 down, -infinity and NaN included, exactly 0: 1's exponent less 127.
// Of eight pairs 0, 1, 2, 3, 4 by it: four prompts of 4,096 tokens, 16 heads of 64, 237, 227, 226, 230, 242 us.
constexpr int kPolynomial = 2;
template <typename T>
__device__ __forceinline__ float2 exp2_polynomial(float2 x) {
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    const auto two = [](float v) { return make_float2(v, v); };
    x.x = fmaxf(x.x, -127.0f), x.y = fmaxf(x.y, -127.0f);
    const float2 t = __fadd2_rn(x, two(12582912.0f));  // 1.5 * 2^23: the whole part in the last bits
    const float2 f = __fadd2_rn(x, __ffma2_rn(t, two(-1.0f), two(12582912.0f)));
    float2 y;
    if constexpr (kBf16) {
        y = __ffma2_rn(f, two(0.05500893294811249f), two(0.24221095442771912f));
        y = __ffma2_rn(f, y, two(0.6932829022407532f));
    } else {
        y = __ffma2_rn(f, two(0.009782912209630013f), two(0.055976882576942444f));
        y = __ffma2_rn(f, y, two(0.24020710587501526f));
        y = __ffma2_rn(f, y, two(0.6931136250495911f));
    }
    y = __ffma2_rn(f, y, two(1.0f));
    return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)));
}

__device__ int waits_gave_up;  // since it was last looked at, in a kernel of this device

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ Maps maps, const Prompt p) {
    using L = Layout<D, NT>;
    constexpr uint32_t kSlots = L::kSlots, kScores = 0, kOutput = NT * kTile;
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr float kLazy = kBf16 ? 8.0f : 4.0f, kLifted = kBf16 ? 0.0f : 11.0f;
    extern __shared__ uint8_t dynamic[];
    __shared__ uint64_t buf[kThreads / 32];
    __shared__ Found found;
    __shared__ uint32_t tensor_base;
    __shared__ alignas(8) uint64_t bars[2 + 4 * kSlots + 4 * NT + 1];
    __shared__ int first_bad[3][D];  // the first key with +infinity, -infinity, NaN in an element
    __shared__ int any_bad, failed;
    __shared__ uint32_t issued;  // copies of keys and values
    auto wait = [&](uint32_t bar, uint32_t parity) { return barrier_wait(bar, parity, &failed); };
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t tiles = (shared_address(dynamic) + 1023) / 1024 * 1024;
    auto q_tile = [&](uint32_t i) { return tiles + i * L::kTileBytes; };
    auto slot = [&](uint32_t s) { return tiles + (NT + s) * L::kTileBytes; };
    const uint32_t bar0 = shared_address(bars);
    auto q_full = [&](uint32_t i) { return bar0 + 8 * i; };
    auto full = [&](uint32_t s) { return bar0 + 8 * (2 + s); };
    auto empty = [&](uint32_t s) { return bar0 + 8 * (2 + kSlots + s); };
    auto raw = [&](uint32_t s) { return bar0 + 8 * (2 + 2 * kSlots + s); };  // values that are to be cleaned
    auto clean = [&](uint32_t s) { return bar0 + 8 * (2 + 3 * kSlots + s); };
    auto s_full = [&](uint32_t i) { return bar0 + 8 * (2 + 4 * kSlots + i); };
    auto p_full = [&](uint32_t i, uint32_t half) { return bar0 + 8 * (2 + 4 * kSlots + NT + 2 * i + half); };
    auto o_full = [&](uint32_t i) { return bar0 + 8 * (2 + 4 * kSlots + 3 * NT + i); };
    const uint32_t products_done = bar0 + 8 * (2 + 4 * kSlots + 4 * NT);  // where a wait has run out

    // the last sequence first, and in each the last tile first: of causal ones the longest; all heads of a tile in turn
    const uint32_t per = p.pairs ? p.heads / 2 : p.heads;
    const uint32_t kRows = p.pairs ? kTile : NT * kTile, next_row = p.pairs ? 0 : kTile;  // from a tile of queries to the next
    const uint32_t piece = blockIdx.x / per, which = blockIdx.x - piece * per, h = p.pairs ? 2 * which : which, kh = p.group_div.div(h);
    auto count = [&](uint32_t i) {
        uint32_t first, n;
        rows_of(p.starts, p.sequences - 1 - i, p.tokens, first, n);
        return (uint64_t)(n + kRows - 1) / kRows;
    };
    const Found f = find(p.sequences, piece, count, buf, &found);
    if (!f.any) return;
    const uint32_t seq = p.sequences - 1 - f.i;
    uint32_t q_first, n, k_first, m;
    rows_of(p.starts, seq, p.tokens, q_first, n);
    rows_of(p.k_starts, seq, p.k_tokens, k_first, m);
    const uint32_t row0 = ((n + kRows - 1) / kRows - 1 - (uint32_t)(piece - f.first)) * kRows;
    const int ahead = (int)m - (int)n;  // a query sees keys up to its own index plus this
    // tiles of keys that tile i of the queries sees
    uint32_t steps[2] = {0, 0}, most = 0;
#pragma unroll
    for (uint32_t i = 0; i < NT; ++i) {
        const uint32_t lo = row0 + i * next_row;
        if (lo >= n) continue;
        const int seen = p.causal ? max(0, min((int)m, (int)min(lo + kTile, n) + ahead)) : (int)m;
        steps[i] = ((uint32_t)seen + kTile - 1) / kTile;
        most = max(most, steps[i]);
    }
    // the first tile of keys that some row does not see whole
    const uint32_t partial = p.causal ? (uint32_t)max(0, min((int)m, (int)row0 + ahead + 1)) / kTile : m / kTile;

    if (warp == 0) tensor_alloc(shared_address(&tensor_base), 512);
    if (threadIdx.x == 32) {
        for (uint32_t i = 0; i < 2; ++i) barrier_init(q_full(i), 1);
        for (uint32_t s = 0; s < kSlots; ++s) barrier_init(full(s), 1), barrier_init(empty(s), 1), barrier_init(raw(s), 1), barrier_init(clean(s), 2);
        for (uint32_t i = 0; i < NT; ++i)
            barrier_init(s_full(i), 1), barrier_init(p_full(i, 0), 4), barrier_init(p_full(i, 1), 4), barrier_init(o_full(i), 1);
        barrier_init(products_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        any_bad = failed = 0;
        issued = 0;
    }
    for (uint32_t e = threadIdx.x; e < 3 * D; e += kThreads) (&first_bad[0][0])[e] = 0x7FFFFFFF;
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tensor = tensor_base;

    if (warp >= 8) {
        registers_down<88>();
        if (warp == 8) {  // copies
            auto load = [&](uint32_t to, uint32_t bar, const CUtensorMap* map, bool token_last, uint32_t token, uint32_t head) {
                barrier_expect(bar, L::kTileBytes);
                for (uint32_t x = 0; x < D / 64; ++x)
                    copy_tile(to + x * L::kRowTile, map, bar, (int)(x * 64), (int)(token_last ? head : token), (int)(token_last ? token : head));
            };
            if (elected()) for (uint32_t item = 0; item < 2 * most; ++item) {
                const uint32_t j = item / 2, kv = item % 2, s = item % kSlots, use = item / kSlots;
                if (use && !wait(empty(s), (use - 1) & 1)) break;
                if (item == 0 && steps[0]) load(q_tile(0), q_full(0), &maps.q, maps.tokens_last & 1, q_first + row0, h);
                load(slot(s), kv && j >= partial ? raw(s) : full(s), kv ? &maps.v : &maps.k, maps.tokens_last >> (1 + kv) & 1,
                     k_first + j * kTile, kh);
                if (NT == 2 && item == 0 && steps[1]) load(q_tile(1), q_full(1), &maps.q, maps.tokens_last & 1, q_first + row0 + next_row, h + p.pairs);
                issued = item + 1;
            }
            __syncwarp();
        } else if (warp == 9) {  // products
            constexpr uint32_t kScore = product_descriptor(kBf16, kTile, kTile, false), kValue = product_descriptor(kBf16, kTile, D, true);
            auto scores = [&](uint32_t i, uint32_t j) {
                const uint64_t k = tile_descriptor(slot(2 * j % kSlots), 1024, 16), q = tile_descriptor(q_tile(i), 1024, 16);
#pragma unroll
                for (uint32_t d = 0; d < D / 16; ++d) {
                    const uint32_t off = (d / 4 * L::kRowTile + d % 4 * 32) / 16;
                    product(tensor + kScores + i * kTile, q + off, k + off, kScore, d > 0);
                }
                product_commit(s_full(i));
            };
            if (most) wait(full(0), 0);
            for (uint32_t i = 0; i < NT; ++i) {
                if (!steps[i]) continue;
                wait(q_full(i), 0);
                __syncwarp();
                if (elected()) scores(i, 0);
            }
            __syncwarp();
            if (most && elected()) product_commit(empty(0));
            for (uint32_t j = 0; j < most; ++j) {
                const uint32_t s = (2 * j + 1) % kSlots;
                if (j < partial) wait(full(s), (2 * j + 1) / kSlots & 1);
                else wait(clean(s), (j - partial) / L::kAgain & 1);
                if (j + 1 < most) wait(full((2 * j + 2) % kSlots), (2 * j + 2) / kSlots & 1);
                const uint64_t v = tile_descriptor(slot(s), 1024, L::kRowTile);
#pragma unroll
                for (uint32_t i = 0; i < NT; ++i) {
                    if (j >= steps[i]) continue;
#pragma unroll
                    for (uint32_t half = 0; half < 2; ++half) {
                        wait(p_full(i, half), j & 1);
                        __syncwarp();
                        tensor_fence_after();
                        if (elected()) {
#pragma unroll
                            for (uint32_t d = half * 4; d < half * 4 + 4; ++d)
                                product(tensor + kOutput + i * D, tensor + kScores + i * kTile + d * 8, v + d * (2048 / 16), kValue, j > 0 || d > 0);
                            if (half && j + 1 == steps[i]) product_commit(o_full(i));
                            if (half && (i + 1 == NT || j >= steps[NT - 1])) product_commit(empty(s));
                            if (half && j + 1 < steps[i]) scores(i, j + 1);
                        }
                    }
                }
                __syncwarp();
                if (j + 1 < most && elected()) product_commit(empty((2 * j + 2) % kSlots));
            }
        } else if (warp >= 10) {  // values
            for (uint32_t j = partial; j < most; ++j) {
                const uint32_t s = (2 * j + 1) % kSlots, rows = min(kTile, m - j * kTile);
                wait(raw(s), (j - partial) / L::kAgain & 1);
                constexpr uint32_t kUnits = 8;  // of 16 bytes, eight elements, on their way
                for (uint32_t e0 = threadIdx.x - 320; e0 < kTile * (D / 8); e0 += 64 * kUnits) {
                    uint4 w[kUnits];
                    uint32_t at[kUnits];
#pragma unroll
                    for (uint32_t u = 0; u < kUnits; ++u) {
                        const uint32_t e = e0 + 64 * u, r = e / (D / 8), c = e % (D / 8);
                        at[u] = slot(s) + c / 8 * L::kRowTile + r * 128 + (c % 8 ^ r % 8) * 16;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[u].x), "=r"(w[u].y), "=r"(w[u].z), "=r"(w[u].w) : "r"(at[u]));
                    }
#pragma unroll
                    for (uint32_t u = 0; u < kUnits; ++u) {
                        const uint32_t e = e0 + 64 * u, r = e / (D / 8), c = e % (D / 8);
                        if (r < rows && all_finite<T>(w[u])) continue;
                        uint32_t v[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
                        for (uint32_t x = 0; x < 8 && r < rows; ++x) {
                            const uint32_t bits = v[x / 2] >> (x % 2 * 16) & 0xFFFFu;
                            constexpr uint32_t kTop = kBf16 ? 0x7F80u : 0x7C00u;
                            if ((bits & kTop) != kTop) continue;
                            v[x / 2] &= x % 2 ? 0xFFFFu : 0xFFFF0000u;
                            const int kind = (bits & 0x7FFFu) != kTop ? 2 : bits >> 15;
                            atomicMin(&first_bad[kind][c * 8 + x], (int)(j * kTile + r));
                            any_bad = 1;
                        }
                        if (r >= rows) v[0] = v[1] = v[2] = v[3] = 0;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at[u]), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                    }
                }
                fence_async();
                __syncwarp();
                if (lane == 0) barrier_arrive(clean(s));
            }
        }
        __syncwarp();
    } else {
        registers_up<208>();
        const uint32_t i = warp / 4, row = row0 + i * next_row + threadIdx.x % kTile;  // threads 128 i .. of tile i
        const uint32_t lanes = (warp % 4 * 32) << 16;
        const uint32_t output = tensor + lanes + kOutput + i * D;
        const uint32_t my_steps = i < NT ? steps[i] : 0;
        const int limit = min((int)m - 1, p.causal ? (int)row + ahead : (int)m - 1);  // the last key that this row sees
        const int least = min((int)m - 1, p.causal ? (int)(row0 + i * next_row) + ahead : (int)m - 1);
        float top = -INFINITY, sum = 0.0f;  // top: what the weights so far refer to
        const uint32_t scores = tensor + lanes + kScores + i * kTile;
        for (uint32_t j = 0; j < my_steps; ++j) {
            wait(s_full(i), j & 1);
            __syncwarp();
            tensor_fence_after();
            float s[kTile];
#pragma unroll
            for (int c = 0; c < (int)kTile; c += 32) tensor_load32(scores + c, s, c);
            tensor_wait_load();
            const int last = limit - (int)(j * kTile);
            if (least - (int)(j * kTile) < (int)kTile - 1) {
#pragma unroll
                for (int c = 0; c < (int)kTile; ++c)
                    if (c > last) s[c] = -INFINITY;
            }
            // a NaN among the scores stays: it is not for the polynomial to show it
            float most4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < (int)kTile - 4; c += 8)
#pragma unroll
                for (int d = 0; d < 4; ++d) most4[d] = max3(most4[d], s[c + d], s[c + 4 + d]);
#pragma unroll
            for (int d = 0; d < 4; ++d) most4[d] = max3(most4[d], s[kTile - 4 + d], most4[d]);
            const float now = max3(max3(most4[0], most4[1], most4[2]), most4[3], most4[3]);
            if (j == 0 || now != now) top = now;
            if (j) {
                const bool grown = (now - top) * p.scale > kLazy;  // from -infinity too; not where both are
                if (__any_sync(~0u, grown)) {
                    const float factor = grown ? exp2_fast((top - now) * p.scale) : 1.0f;
                    if (grown) top = now;
                    sum *= factor;
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        tensor_load32(output + c, o, 0);
                        tensor_wait_load();
#pragma unroll
                        for (int d = 0; d < 32; ++d) o[d] *= factor;
                        tensor_store32(output + c, o, 0);
                    }
                }
            }
            const float from = top == -INFINITY ? 0.0f : fmaf(-top, p.scale, kLifted);
            float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            const float2 scale2 = make_float2(p.scale, p.scale), from2 = make_float2(from, from);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[kHalf / 2];
#pragma unroll
                for (int c = 0; c < (int)kHalf; c += 2) {
                    const float2 x = __ffma2_rn(make_float2(s[half * kHalf + c], s[half * kHalf + c + 1]), scale2, from2);
                    const float2 y = c / 2 % 8 < kPolynomial ? exp2_polynomial<T>(x) : make_float2(exp2_fast(x.x), exp2_fast(x.y));
                    part[c / 2 % 2] = __fadd2_rn(part[c / 2 % 2], y);
                    w[c / 2] = pack2<T>(y.x, y.y);
                }
                tensor_store32(scores + half * (kHalf / 2), w, 0);
                tensor_wait_store();
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(p_full(i, half));
            }
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
        }
        if (my_steps) wait(o_full(i), 0);
        if (partial < most) wait(clean((2 * most - 1) % kSlots), (most - 1 - partial) / L::kAgain & 1);  // what was noted is there
        __syncwarp();
        tensor_fence_after();
        const bool mine = i < NT && row < n;
        T* out = static_cast<T*>(p.out) + (uint64_t)(q_first + row) * p.os[0] + (h + (p.pairs ? i : 0)) * p.os[1];
        const float inverse = failed ? NAN : limit < 0 ? 0.0f : 1.0f / sum;
        if (i < NT) {
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                float o[32] = {};
                __syncwarp();
                if (my_steps) {
                    tensor_load32(output + c, o, 0);
                    tensor_wait_load();
                }
                if (!mine) continue;
                const bool extra = any_bad != 0;
#pragma unroll
                for (int d = 0; d < 32; ++d) {
                    o[d] = limit < 0 ? 0.0f : o[d] * inverse;
                    if (extra) {
                        if (first_bad[0][c + d] <= limit) o[d] += INFINITY;
                        if (first_bad[1][c + d] <= limit) o[d] -= INFINITY;
                        if (first_bad[2][c + d] <= limit) o[d] = NAN;
                    }
                }
#pragma unroll
                for (int d = 0; d < 32; d += 8) {
                    if (c + d >= (int)p.head) break;
                    Few<T, 8> y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y.set2(e, o[d + 2 * e], o[d + 2 * e + 1]);
                    *reinterpret_cast<uint4*>(out + c + d) = make_uint4(y.w[0], y.w[1], y.w[2], y.w[3]);
                }
            }
        }
    }
    tensor_fence_before();
    __syncthreads();
    if (failed) {
        // no copy and no product outlasts the block: the last copy of each slot, the queries' and all products (again for some
        // seconds at most)
        auto drain = [](uint32_t bar, uint32_t parity) {
            for (uint32_t i = 0; i < 1u << 20 && !barrier_try(bar, parity); ++i) {}
        };
        if (warp == 8 && elected()) {
            for (uint32_t item = issued - min(issued, kSlots); item < issued; ++item) {
                // the barrier that the copy was issued on, and how often it was used before
                const uint32_t s = item % kSlots, j = item / 2;
                if (item % 2 && j >= partial) drain(raw(s), (j - partial) / L::kAgain & 1);
                else drain(full(s), item / kSlots & 1);
            }
            for (uint32_t i = 0; i < NT; ++i)
                if (issued && steps[i]) drain(q_full(i), 0);
        }
        if (warp == 9 && elected()) {
            product_commit(products_done);
            drain(products_done, 0);
        }
        if (threadIdx.x == 0) waits_gave_up = 1;
        __syncthreads();
    }
    if (warp == 0) {
        tensor_fence_after();
        tensor_free(tensor, 512);
    }
}

// The driver's encoder of tiled copies, which the runtime finds.
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                            CUtensorMapFloatOOBfill);
Encode encoder() {
    static const Encode found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result) != cudaSuccess ||
            result != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return (Encode) nullptr;
        }
        return reinterpret_cast<Encode>(f);
    }();
    return found;
}

// Heads [tokens, heads, head] by tiles of 128 tokens and 64 elements; false: not with these strides.
bool encode(CUtensorMap* map, bool* tokens_last, int dtype, const void* data, uint64_t tokens, uint64_t heads, uint32_t head,
            const uint64_t (&s)[2]) {
    // a stride that no coordinate multiplies counts for nothing
    const uint64_t token = tokens > 1 ? s[0] : std::max<uint64_t>(s[1], head) * heads, hs = heads > 1 ? s[1] : head;
    if (reinterpret_cast<uintptr_t>(data) % 16 || !token || !hs || token % 8 || hs % 8 || token >> 38 || hs >> 38) return false;
    *tokens_last = token >= hs;
    const bool last = *tokens_last;
    const cuuint64_t dims[3] = {head, last ? heads : tokens, last ? tokens : heads};
    const cuuint64_t strides[2] = {2 * (last ? hs : token), 2 * (last ? token : hs)};
    const cuuint32_t box[3] = {64, last ? 1u : kTile, last ? kTile : 1u}, ones[3] = {1, 1, 1};
    return encoder()(map, dtype == MTXC_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                     const_cast<void*>(data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the tensor cores take the call; fills the maps.
bool prepare_maps(int dtype, const mtxc_prompt_attention_args* a, const Prompt& p, Maps* maps) {
    if (dtype == MTXC_FLOAT || a->head_dim % 8 || !(p.scale > 0.0f && p.scale < INFINITY) || !a->k_tokens || !encoder()) return false;
    if (reinterpret_cast<uintptr_t>(a->out) % 16 || a->out_strides[0] % 8 || a->out_strides[1] % 8) return false;
    bool last[3];
    if (!encode(&maps->q, &last[0], dtype, a->q, a->tokens, a->heads, a->head_dim, a->q_strides) ||
        !encode(&maps->k, &last[1], dtype, a->k, a->k_tokens, a->kv_heads, a->head_dim, a->k_strides) ||
        !encode(&maps->v, &last[2], dtype, a->v, a->k_tokens, a->kv_heads, a->head_dim, a->v_strides))
        return false;
    maps->tokens_last = last[0] | last[1] << 1 | last[2] << 2;
    return true;
}

template <typename T, int D, int NT>
int launch(const mtxc_prompt_attention_args* a, const Maps& maps, const Prompt& p) {
    using L = Layout<D, NT>;
    // the same limit in every call: calls from several threads do not undo each other's
    cudaError_t err = cudaFuncSetAttribute(prompt_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes);
    if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
    // as many tiles as the sequences can have: one each may be part filled
    const uint64_t tiles = a->tokens / (p.pairs ? kTile : NT * kTile) + std::min(a->sequences, a->tokens);
    const uint64_t per = p.pairs ? a->heads / 2 : a->heads;
    if (tiles * per >> 31) return fail(MTXC_ERR_SHAPE, "mtxc_prompt_attention: too many tiles of queries and heads");
    prompt_kernel<T, D, NT><<<(unsigned)(tiles * per), kThreads, L::kBytes, ctx().stream()>>>(maps, p);
    return check_launch("prompt_kernel");
}

}  // namespace
}  // namespace mtxc

using namespace mtxc;

extern "C" int mtxc_waits_gave_up(int* gave_up) {
    if (!gave_up) return fail(MTXC_ERR_INVALID_ARGUMENT, "mtxc_waits_gave_up: null pointer");
    if (int rc = require_init()) return rc;
    const int none = 0;
    cudaStream_t st = ctx().stream();
    cudaError_t err = cudaMemcpyFromSymbolAsync(gave_up, waits_gave_up, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (err == cudaSuccess) err = cudaStreamSynchronize(st);
    if (err == cudaSuccess && *gave_up) err = cudaMemcpyToSymbolAsync(waits_gave_up, &none, sizeof none, 0, cudaMemcpyHostToDevice, st);
    if (err == cudaSuccess) err = cudaStreamSynchronize(st);
    return err == cudaSuccess ? MTXC_OK : cuda_fail(err, "mtxc_waits_gave_up");
}

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
    if (a->out == a->k || a->out == a->v) return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": an output over keys or values");
    if (int rc = laid_alike(who, a->out, a->out_strides, a->q, a->q_strides, {a->tokens, a->heads})) return rc;
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
        if constexpr (!std::is_same_v<T, float>) {
            Maps maps;
            if (prepare_maps(dtype, a, p, &maps)) {
                // two heads that share keys see the same of them: no step has one tile of queries only
                p.pairs = p.head <= 128 && p.group % 2 == 0;
                rc = p.head <= 64 ? launch<T, 64, 2>(a, maps, p) : p.head <= 128 ? launch<T, 128, 2>(a, maps, p) : launch<T, 256, 1>(a, maps, p);
                return;
            }
        }
        rc = launch_any<T>(a, p);
    });
    return rc;
}
