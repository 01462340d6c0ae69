// Attention of one new token of each sequence over a paged cache, for sm_100a.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m a running maximum
//
// The keys and values are read once: bound by HBM.  The work -- tiles of keys for each key head and each 16 of its query
// heads, of all sequences one after another -- is shared out evenly over a fixed number of workers (warps; blocks of the
// kernel for any head), whatever the lengths are, which only the device knows.  A unit (sequence, heads) that lies within one
// worker is written there; of one that workers share, each leaves its sums and maxima in the workspace, and a second launch
// joins them in order.
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
    uint32_t batch, heads, kv_heads, group, groups, units, head, max_pages, tile, workers;  // groups: of 16 query heads
    FastDiv groups_div;
    const void* q;
    void* out;
    uint64_t qs[2], os[2];
    const int* table;
    uint64_t table_stride;
    const int* lengths;
    float scale;      // times log2(e)
    bool vector;      // the kernel of 16-byte units
    float* partial;   // [2 * workers][rows][pitch]: sums; at pitch - 4 their maximum, the sum of weights and (in 8 bits) its maximum
    uint32_t rows;    // of a unit
    uint32_t pitch;   // a multiple of four
};

__device__ __forceinline__ uint32_t length_of(const Decode& d, uint32_t b) {
    const int n = d.lengths[b];
    return n < 0 ? 0u : (uint32_t)min((unsigned long long)n, (unsigned long long)d.max_pages * d.cache.page_size);
}
__device__ __forceinline__ uint32_t tiles_of(const Decode& d, uint32_t b) { return (length_of(d, b) + d.tile - 1) / d.tile; }

// The workers that share the work: each has some.
__device__ __forceinline__ uint64_t sharing(const Decode& d, uint64_t work) { return min(work, (uint64_t)d.workers); }

// Where a worker leaves its part of a unit: one that it begins (and another worker ends), or one that was begun before.
__device__ __forceinline__ float* part_of(const Decode& d, uint64_t worker, bool begins) {
    return d.partial + (2 * worker + begins) * d.rows * d.pitch;
}

// The page and slot of key j of sequence b; false: the table names no page of the cache.
__device__ __forceinline__ bool place_of(const Decode& d, uint32_t b, uint32_t j, uint32_t& page, uint32_t& slot) {
    uint32_t i;
    d.cache.page_div.divmod(j, i, slot);
    page = (uint32_t)d.table[b * d.table_stride + i];
    return page < d.cache.pages;
}

// Rows of a unit: query heads first .. first + count - 1.
__device__ __forceinline__ uint32_t rows_of(const Decode& d, uint32_t unit, uint32_t& head, uint32_t& first) {
    head = d.groups_div.div(unit);
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
    let_next_start();
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
        float* const part = part_of(d, blockIdx.x, tile0 == 0);
        if (column < d.head) {
#pragma unroll
            for (uint32_t i = 0; i < kRows; ++i) {
                const uint32_t r = row0 + i * row_step;
                if (r < rows) {
                    if (whole) {
                        const float o = row_max[r] == -INFINITY ? 0.0f : acc[i] / row_sum[r];
                        static_cast<T*>(d.out)[b * d.os[0] + (first + r) * d.os[1] + column] = from_float<T>(o);
                    } else {
                        float* const p = part + r * d.pitch;
                        p[column] = acc[i];
                        if (column == 0) p[d.pitch - 4] = row_max[r], p[d.pitch - 3] = row_sum[r];
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

// ------------------------------------------------------------------------------------------
// Half types, and caches in 8 bits under half queries, by 16-byte units.
//
// A warp works by itself: it copies the keys and values of its tile (16 of a half type, 32 of 8 bits) into a ring of its own
// in shared memory, up to kStages of them (192 KB an SM in flight and in use), and multiplies them on the tensor cores: 16
// keys are the rows and 8 or 16 queries (those that a unit lacks are zeros) the columns of K Q', 16 elements of the head are
// the rows of V' P'.  Warp-wide products, since the keys pass once and HBM bounds them (the tensor pipe is busy for 15 %):
// tcgen05's tiles of 128 rows would be filled by waiting for 128 keys.  (With the queries as 16 rows, half of them zeros for a
// group of 8, both took twice the products, registers and exponentials: 228 us for [4 x 91k] e4m3.)  There is no barrier between
// warps, and the copies run on across the borders of units and sequences.  The page numbers of a tile are loaded one tile before
// its copies are issued.
//
// Over plain caches a weight is two operands, what 16 bits hold of it and what that leaves: 16 or 22 bits for a second product.
// The result is then as far from 64 bits as its own rounding (relative 0.0017 in bfloat16, with one operand 0.0021), for 1.5 % of
// the time (235 us for 232).  Over 8 bits, where the issue of instructions counts, weights are float16 (2.1e-4, of which 2.0e-4
// are the result's rounding).
//
// Measured, heads of 128, 32 over 8: 64 sequences of 1,024 to 8,192 tokens bf16 224 us in a few calls, 5.6 TB/s (0.85 of the copy
// figure), 235 back to back for a second, under the power limit; 4 of 16,384 to 131,072 in 8 bits under 56 heads f16 172 us, 5.4
// TB/s, and 195.  Bound by HBM and, at the end, by the SMs that get less of it than others: equal shares of 8 bits ended 157 to
// 191 us after the start.  In 8 bits 8 warps with three tiles took 195 us in a few calls (bound by each warp's latency) where 12
// with two took 168.
//
// In 8 bits the bytes become float16, which holds them exactly, beside queries as float16 with their largest element between
// 2^15 and 2^16 (their rows' powers of two, like the keys' scales, come back into the scores): float16 ones keep every bit,
// bfloat16 ones theirs down to 2^-32 of the largest.  The values' scales 2^e go into the weights that meet them:
// those are 2^(s + e - m) with m the running maximum of s + e, at most 1 whatever the scales are.  The weights of the
// denominator are 2^(s - m') with a maximum m' of their own: m lies up to 96 from it, and 2^(s - m) would lose or overflow
// the sum.  A row of values that is all zeros (its scale is 2^0, whatever its neighbours have) does not lift m: the rows are
// looked through in the tiles that lift it.  Both together 2 % of the time ([4 x 91k]: 191 -> 194 us).
//
// float16 weights are taken 2^15 times: the largest is 2^15 (65,504 is the type's last), and what is rounded to multiples of
// 2^-24 is the part of them below 2^-29 of it.  Without, a key with nearly all the weight rounded 131,071 others of 2^-25.2 to
// nothing, and those are the output where its value is 0.  It costs nothing: the factor is in the exponent.
// ------------------------------------------------------------------------------------------
// Warps of a block, one block an SM, and tiles of a warp's ring: what 227 KB hold.
constexpr uint32_t warps_of(uint32_t steps, bool small) { return steps > 8 ? 4 : small ? 12 : 8; }
constexpr int stages_of(uint32_t steps, bool small) { return steps > 8 || !small ? 3 : 2; }
uint32_t steps_of(uint32_t head) {  // of 16 elements, as the kernel is built for
    for (uint32_t s : {4u, 5u, 6u, 8u, 12u})
        if (head <= 16 * s) return s;
    return 16;
}

template <int STEPS, bool SMALL>
struct Ring {
    static constexpr uint32_t kKeys = SMALL ? 32 : 16;
    static constexpr uint32_t kUnits = SMALL ? STEPS : 2 * STEPS;     // 16-byte units of a row
    static constexpr uint32_t kPitch = (kUnits | 1) * 16;             // an odd number of them: rows in different banks
    static constexpr uint32_t kSide = kKeys * kPitch, kStage = 2 * kSide;
    static constexpr int kStages = stages_of(STEPS, SMALL);
    static constexpr uint32_t kWarp = kStages * (kStage + 128);       // the last: which keys count, and their exponents
    static constexpr uint32_t kBytes = warps_of(STEPS, SMALL) * kWarp;
};

__device__ __forceinline__ void matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void matrices_turned(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements over a warp, its columns made rows.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    Few<T, 4> f;
    f.set2(0, a, b);
    return f.w[0];
}
// Two weights as two parts of T each, the first one rounded down from a little less: a weight that is not 0 has no part of 0, nor
// a negative one, with which an infinite value would become NaN.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& first, uint32_t& second) {
    constexpr float kLess = 1.0f - 1.0f / 8192;
    float2 kept;
    if constexpr (std::is_same_v<T, __half>) {
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(first) : "f"(b * kLess), "f"(a * kLess));
        kept = __half22float2(*reinterpret_cast<const __half2*>(&first));
    } else {
        first = __byte_perm(__float_as_uint(a * kLess), __float_as_uint(b * kLess), 0x7632);
        kept = make_float2(__uint_as_float(first << 16), __uint_as_float(first & 0xFFFF0000u));
    }
    second = pack2<T>(a - kept.x, b - kept.y);
}
__device__ __forceinline__ uint32_t halves_of(uint32_t bytes) {  // two bytes of e4m3 as two float16
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)bytes, __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float power(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A place in the stream of tiles.
struct Place {
    uint32_t b, unit, tile, tiles, length;
    __device__ __forceinline__ void next(const Decode& d) {  // there is one
        if (++tile < tiles) return;
        tile = 0;
        if (++unit < d.units) return;
        unit = 0;
        do {
            ++b;
            length = length_of(d, b);
            tiles = (length + d.tile - 1) / d.tile;
        } while (tiles == 0);
    }
};

template <typename T, int STEPS, bool SMALL, int COLUMNS>  // COLUMNS: of queries, in eights
__global__ void __launch_bounds__(warps_of(STEPS, SMALL) * 32, 1) decode_units_kernel(const Decode d) {
    using R = Ring<STEPS, SMALL>;
    using M = std::conditional_t<SMALL, __half, T>;  // the products' type
    constexpr uint32_t kKeys = R::kKeys, kTiles = kKeys / 16;
    constexpr int kStages = R::kStages;
    constexpr float kLifted = std::is_same_v<M, __half> ? 15.0f : 0.0f;  // the largest weight is 2^kLifted
    extern __shared__ uint4 smem4[];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem4) + warp * R::kWarp;
    uint32_t* const notes = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(smem4) + warp * R::kWarp + kStages * R::kStage);
    let_next_start();
    auto count = [&](uint32_t b) { return (uint64_t)tiles_of(d, b) * d.units; };
    const Counts counts = warp_counts(d.batch, count);
    const uint64_t work = counts.total, workers = sharing(d, work);
    const uint64_t worker = (uint64_t)warp * gridDim.x + blockIdx.x;  // little work: one warp of each block first
    if (worker >= workers) return;
    uint64_t left = work * (worker + 1) / workers - work * worker / workers;
    Place now;
    {
        const uint64_t first = work * worker / workers;
        const Found f = warp_find(d.batch, first, counts, count);
        now.b = f.i;
        now.length = length_of(d, f.i);
        now.tiles = (now.length + kKeys - 1) / kKeys;
        now.unit = (uint32_t)((first - f.first) / now.tiles);
        now.tile = (uint32_t)((first - f.first) - (uint64_t)now.unit * now.tiles);
    }
    // elements that the heads lack stay zeros: no copy reaches them
    const uint32_t units = d.head * (SMALL ? 1 : 2) / 16;  // of a row that are copied
    for (uint32_t i = lane; units < R::kUnits && i < kStages * R::kStage / 16; i += 32)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i * 16), "r"(0) : "memory");
    __syncwarp();

    // the tile to be copied next: its page, slot and head (a lane a key), and what is left to look at
    Place ahead = now;
    uint64_t unseen = left;
    uint32_t page = ~0u, slot = 0, head = 0;
    auto look = [&]() {
        page = ~0u;
        if (unseen == 0) return;
        --unseen;
        const uint32_t key = ahead.tile * kKeys + lane;
        head = d.groups_div.div(ahead.unit);
        if (lane < kKeys && key < ahead.length) {
            uint32_t i;
            d.cache.page_div.divmod(key, i, slot);
            page = (uint32_t)d.table[ahead.b * d.table_stride + i];
        }
        if (unseen) ahead.next(d);
    };
    uint32_t note = 0, note_to = 0;  // on its way to stage note_to
    auto copy = [&](uint32_t stage) {
        const bool ok = page < d.cache.pages;
        uint64_t from[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const CacheSide& c = d.cache.side[k];
            from[k] = ok ? (page * c.s[0] + slot * c.s[1] + head * c.s[2]) * (SMALL ? 1 : 2) : ~0ull;
        }
        notes[note_to * 32 + lane] = note;  // that of the tile before has come
        note = ok;
        if constexpr (SMALL)
            if (ok) {
                const CacheSide &c = d.cache.side[0], &v = d.cache.side[1];
                const int8_t key = c.exponents[page * c.es[0] + slot * c.es[1] + head * c.es[2]];
                const int8_t value = v.exponents[page * v.es[0] + slot * v.es[1] + head * v.es[2]];
                note = 1u | (uint32_t)(uint8_t)key << 8 | (uint32_t)(uint8_t)value << 16;
            }
        note_to = stage;
        // lanes side by side along a row, and rows in turn
        const uint32_t to = ring + stage * R::kStage;
#pragma unroll
        for (uint32_t e = 0; e < kKeys * R::kUnits; e += 32) {
            const uint32_t i = e + lane, row = i / R::kUnits, unit = i - row * R::kUnits;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint64_t at = __shfl_sync(~0u, from[k], row);
                const void* src = static_cast<const uint8_t*>(d.cache.side[k].data) + (at == ~0ull ? 0 : at + unit * 16);
                if (unit < units)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * R::kSide + row * R::kPitch + unit * 16), "l"(src),
                                 "r"(at == ~0ull ? 0 : 16)
                                 : "memory");
            }
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    look();
    for (uint32_t s = 0; s + 1 < kStages; ++s) {
        copy(s);
        commit();
        look();
    }

    auto among = [](float x) {  // the largest of the lanes of a column
#pragma unroll
        for (int m = 4; m < 32; m *= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, m));
        return x;
    };
    uint32_t stage = 0;
    while (left) {
        // a unit, as far as this worker has it
        uint32_t h, first;
        const uint32_t rows = rows_of(d, now.unit, h, first), b = now.b, tile0 = now.tile, tiles = now.tiles;
        uint32_t q[STEPS][COLUMNS][2];
        float factor[COLUMNS][2];  // of this thread's columns 2 t, 2 t + 1
        {
            // column g of the second operand: elements 2 t, 2 t + 1 and 8 further (of 8 bits: 4 t .. 4 t + 3, as a thread finds
            // four bytes of a key side by side)
            const T* base = static_cast<const T*>(d.q) + b * d.qs[0] + first * d.qs[1];
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n) {
                const uint32_t row = g + 8 * n;
                const T* x = base + row * d.qs[1];
                factor[n][0] = factor[n][1] = d.scale;
                if constexpr (!SMALL) {
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t c = 16 * s + 8 * e + 2 * t;
                            q[s][n][e] = row < rows && c < d.head ? pack2<T>(to_float(x[c]), to_float(x[c + 1])) : 0u;
                        }
                } else {
                    uint32_t most = 0;
                    float v[STEPS][4];
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t c = 16 * s + 4 * t + e;
                            v[s][e] = row < rows && c < d.head ? to_float(x[c]) : 0.0f;
                            const uint32_t bits = __float_as_uint(v[s][e]) & 0x7FFFFFFFu;
                            most = max(most, bits < 0x7F800000u ? bits : 0u);
                        }
                    most = max(most, __shfl_xor_sync(~0u, most, 1));
                    most = max(most, __shfl_xor_sync(~0u, most, 2));
                    const int e = most ? max(-126, (int)(most >> 23) - 127 - 15) : 0;  // at most 112
                    const float down = power_of_two(-e), up = power_of_two(e);
#pragma unroll
                    for (int i = 0; i < 2; ++i) factor[n][i] *= __shfl_sync(~0u, up, 4 * (2 * t + i));
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i) q[s][n][i] = pack2<__half>(v[s][2 * i] * down, v[s][2 * i + 1] * down);
                }
            }
        }
        // top: what the weights refer to, kLifted below the largest (SMALL: with their values' scales); peak: what those of the
        // denominator do, the largest (SMALL: of this thread's own keys until the end)
        float o[STEPS][COLUMNS][4], top[COLUMNS][2], peak[COLUMNS][2], sum[COLUMNS][2];
#pragma unroll
        for (int n = 0; n < COLUMNS; ++n) {
            top[n][0] = top[n][1] = peak[n][0] = peak[n][1] = kLowest, sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
        }
        bool any = false;  // key counts, were its score -infinity
        bool ends, done;   // done: with the unit's last tile
        do {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            // this tile has come; the one after those on their way goes where the last one was
            copy(stage == 0 ? kStages - 1 : stage - 1);
            commit();
            look();
            const uint32_t keys = ring + stage * R::kStage, values = keys + R::kSide;
            float s[kTiles][COLUMNS][4];  // keys g, g + 8 of 16 x columns 2 t, 2 t + 1
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                for (int n = 0; n < COLUMNS; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
                uint32_t r[4];
                if constexpr (!SMALL) {
                    matrices(r, keys + lane % 16 * R::kPitch + (2 * c + lane / 16) * 16);
#pragma unroll
                    for (int n = 0; n < COLUMNS; ++n) multiply<M>(s[0][n], r, q[c][n][0], q[c][n][1]);
                } else {
                    matrices(r, keys + lane * R::kPitch + c * 16);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a[4] = {halves_of(r[2 * i] & 0xFFFFu), halves_of(r[2 * i + 1] & 0xFFFFu),
                                               halves_of(r[2 * i] >> 16), halves_of(r[2 * i + 1] >> 16)};
#pragma unroll
                        for (int n = 0; n < COLUMNS; ++n) multiply<M>(s[i][n], a, q[c][n][0], q[c][n][1]);
                    }
                }
            }
            // scores in powers of two
            const uint32_t mine = notes[stage * 32 + lane], counting = __ballot_sync(~0u, mine & 1);
            any = any || counting;
            float most[COLUMNS][2], highest[COLUMNS][2], shift[kTiles][2];  // with and without shift: the values' scales
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) most[n][e] = -INFINITY, highest[n][e] = SMALL ? peak[n][e] : -INFINITY;
#pragma unroll
            for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t key = 16 * i + 8 * r + g;
                    const bool counts = counting >> key & 1;
                    float scale = 1.0f;
                    shift[i][r] = 0.0f;
                    if constexpr (SMALL) {
                        const uint32_t x = __shfl_sync(~0u, mine, key);
                        scale = power_of_two((int8_t)(x >> 8 & 0xFFu));
                        shift[i][r] = (float)(int8_t)(x >> 16 & 0xFFu);
                    }
#pragma unroll
                    for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& x = s[i][n][2 * r + e];
                            x = counts ? x * (factor[n][e] * scale) : -INFINITY;
                            highest[n][e] = fmaxf(highest[n][e], x);
                            if (SMALL) most[n][e] = fmaxf(most[n][e], x + shift[i][r]);
                        }
                }
            bool grown = false;
            float old[COLUMNS][2];
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    old[n][e] = top[n][e];
                    top[n][e] = fmaxf(top[n][e], among(SMALL ? most[n][e] : highest[n][e]) - kLifted);
                    grown = grown || top[n][e] != old[n][e];
                    if (SMALL) {
                        sum[n][e] *= power(peak[n][e] - highest[n][e]);
                        peak[n][e] = highest[n][e];
                    }
                }
            if (__any_sync(~0u, grown)) {
                if constexpr (SMALL) {
                    uint32_t any = 0;  // of this lane's key: a value that is not 0
#pragma unroll
                    for (uint32_t u = 0; u < R::kUnits; ++u) {
                        uint4 x;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(values + lane * R::kPitch + u * 16) : "memory");
                        any |= (x.x | x.y | x.z | x.w) & 0x7F7F7F7Fu;
                    }
                    const uint32_t zeros = __ballot_sync(~0u, any == 0) & counting;
                    if (zeros) {
#pragma unroll
                        for (int n = 0; n < COLUMNS; ++n) most[n][0] = most[n][1] = -INFINITY;
#pragma unroll
                        for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                if (zeros >> (16 * i + 8 * r + g) & 1) shift[i][r] = -INFINITY;
#pragma unroll
                                for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) most[n][e] = fmaxf(most[n][e], s[i][n][2 * r + e] + shift[i][r]);
                            }
#pragma unroll
                        for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) top[n][e] = fmaxf(old[n][e], among(most[n][e]) - kLifted);
                    }
                }
#pragma unroll
                for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float by = top[n][e] == old[n][e] ? 1.0f : power(old[n][e] - top[n][e]);
                        if (!SMALL) sum[n][e] *= by;
#pragma unroll
                        for (int i = 0; i < STEPS; ++i) o[i][n][e] *= by, o[i][n][2 + e] *= by;
                    }
            }
            uint32_t w[kTiles][COLUMNS][2], rest[COLUMNS][2];  // rest: the second parts
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n) {
#pragma unroll
                for (uint32_t i = 0; i < kTiles; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float v[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x = s[i][n][2 * r + e];
                            v[e] = power((SMALL ? x + shift[i][r] : x) - top[n][e]);
                            sum[n][e] += SMALL ? power(x - peak[n][e]) : v[e];
                        }
                        if constexpr (SMALL) w[i][n][r] = turned(pack2<M>(v[0], v[1]));
                        else {
                            uint32_t first, second;
                            split2<M>(v[0], v[1], first, second);
                            w[i][n][r] = turned(first), rest[n][r] = turned(second);
                        }
                    }
            }
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
                uint32_t r[4];
                if constexpr (!SMALL) {
                    matrices_turned(r, values + (lane / 16 * 8 + lane % 8) * R::kPitch + (2 * c + lane / 8 % 2) * 16);
#pragma unroll
                    for (int n = 0; n < COLUMNS; ++n) {
                        multiply<M>(o[c][n], r, w[0][n][0], w[0][n][1]);
                        multiply<M>(o[c][n], r, rest[n][0], rest[n][1]);
                    }
                } else {
                    // a register has two elements of two keys: keys together, and the even elements are rows 0 to 7, the odd
                    // ones rows 8 to 15
                    matrices_turned(r, values + lane * R::kPitch + c * 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r[i] = __byte_perm(r[i], 0, 0x3120);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a[4] = {halves_of(r[2 * i] & 0xFFFFu), halves_of(r[2 * i] >> 16), halves_of(r[2 * i + 1] & 0xFFFFu),
                                               halves_of(r[2 * i + 1] >> 16)};
#pragma unroll
                        for (int n = 0; n < COLUMNS; ++n) multiply<M>(o[c][n], a, w[i][n][0], w[i][n][1]);
                    }
                }
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
            done = now.tile + 1 == tiles;
            ends = --left == 0 || done;
            if (left) now.next(d);
        } while (!ends);
        // the end of the unit, or of this worker's part of it
        const bool whole = tile0 == 0 && done;
#pragma unroll
        for (int n = 0; n < COLUMNS; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (SMALL) {
                    const float high = peak[n][e];
                    peak[n][e] = among(high);
                    sum[n][e] *= power(high - peak[n][e]);
                } else peak[n][e] = top[n][e];
#pragma unroll
                for (int m = 4; m < 32; m *= 2) sum[n][e] += __shfl_xor_sync(~0u, sum[n][e], m);
                const uint32_t row = 8 * n + 2 * t + e;
                if (row >= rows) continue;
                const float by = whole ? (any ? 1.0f / sum[n][e] : 0.0f) : 1.0f;
                const float back = SMALL && whole ? exp2f(top[n][e] - peak[n][e]) : 1.0f;  // not in `by`: both may be far from 1
                T* const out = static_cast<T*>(d.out) + b * d.os[0] + (first + row) * d.os[1];
                float* const part = part_of(d, worker, tile0 == 0) + row * d.pitch;
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t c = 16 * i + (SMALL ? 2 * g + r : 8 * r + g);
                        if (c >= d.head) continue;
                        if (whole) out[c] = from_float<T>(o[i][n][2 * r + e] * by * back);
                        else part[c] = o[i][n][2 * r + e];
                    }
                if (!whole && g == 0) {
                    part[d.pitch - 4] = any || SMALL ? top[n][e] : -INFINITY;
                    part[d.pitch - 3] = sum[n][e];
                    part[d.pitch - 2] = any ? peak[n][e] : -INFINITY;
                }
            }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, bool SMALL, int STEPS>
int launch_steps(const Decode& d) {
    using R = Ring<STEPS, SMALL>;
    auto kernel = d.rows <= 8 ? decode_units_kernel<T, STEPS, SMALL, 1> : decode_units_kernel<T, STEPS, SMALL, 2>;
    // the same limit in every call: calls from several threads do not undo each other's
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)R::kBytes);
    if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
    kernel<<<ctx().sm_count, warps_of(STEPS, SMALL) * 32, R::kBytes, ctx().stream()>>>(d);
    return check_launch("decode_units_kernel");
}

template <typename T, bool SMALL>
int launch_units(const Decode& d) {
    switch (steps_of(d.head)) {
        case 4: return launch_steps<T, SMALL, 4>(d);
        case 5: return launch_steps<T, SMALL, 5>(d);
        case 6: return launch_steps<T, SMALL, 6>(d);
        case 8: return launch_steps<T, SMALL, 8>(d);
        case 12: return launch_steps<T, SMALL, 12>(d);
        default: return launch_steps<T, SMALL, 16>(d);
    }
}

// Joins the parts of the units that workers share: block (unit, sequence), or, where there are few (FEW), (query head,
// sequence); warps take parts in turn, a lane four columns (and four more 128 further).  A sequence without keys gets zeros here.
// APART: the parts' sums and their denominators refer to maxima of their own.
template <typename T, bool FEW, bool APART>
__global__ void __launch_bounds__(FEW ? 512 : 128) decode_join_kernel(const Decode d) {
    constexpr uint32_t kJoinThreads = FEW ? 512 : 128;
    constexpr uint32_t kWarps = kJoinThreads / 32;
    __shared__ uint64_t buf[kWarps];
    __shared__ float factors[kJoinThreads], wide[kWarps], wide_peak[kWarps];
    __shared__ float4 sums[kWarps][kMaxHead / 4];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t b = blockIdx.y, tiles = tiles_of(d, b);
    uint32_t unit = blockIdx.x, row0 = 0;
    if (FEW) {
        const uint32_t h = blockIdx.x / d.group, in = blockIdx.x - h * d.group;
        unit = h * d.groups + in / kRows, row0 = in % kRows;
    }
    uint32_t h, query;
    const uint32_t rows = rows_of(d, unit, h, query), row1 = FEW ? row0 + 1 : rows;
    auto before = [&](uint32_t i) { return (uint64_t)tiles_of(d, i) * d.units; };
    auto behind = [&](uint32_t i) { return (uint64_t)tiles_of(d, b + 1 + i) * d.units; };
    const uint64_t start = total_of(b, before, buf), work = start + (uint64_t)tiles * d.units + total_of(d.batch - b - 1, behind, buf);
    wait_for_previous();  // every block: what follows in the stream follows the first kernel too
    T* const base_out = static_cast<T*>(d.out) + b * d.os[0] + query * d.os[1];
    if (tiles == 0) {
        for (uint32_t row = row0; row < row1; ++row)
            for (uint32_t c = threadIdx.x; c < d.head; c += kJoinThreads) base_out[row * d.os[1] + c] = from_float<T>(0.0f);
        return;
    }
    const uint64_t first = start + (uint64_t)unit * tiles, workers = sharing(d, work);
    const uint32_t c0 = (uint32_t)(((first + 1) * workers - 1) / work), c1 = (uint32_t)(((first + tiles) * workers - 1) / work);
    if (c0 == c1) return;
    for (uint32_t row = row0; row < row1; ++row) {
        T* const out = base_out + row * d.os[1];
        auto part = [&](uint32_t c) { return part_of(d, c, c == c0) + row * d.pitch; };
        const uint32_t quads = d.pitch / 4 - 1;
        float top = -INFINITY, peak = -INFINITY, sum = 0.0f;
        float4 acc[kMaxHead / 128] = {};
        for (uint32_t base = c0; base <= c1; base += kJoinThreads) {
            // the sums so far follow the maximum, as in the kernels before
            const uint32_t n = min(kJoinThreads, c1 + 1 - base);
            float m = -INFINITY, l = 0.0f, high = -INFINITY;
            if (threadIdx.x < n) {
                const float4 mlh = *reinterpret_cast<const float4*>(part(base + threadIdx.x) + d.pitch - 4);
                m = mlh.x, l = mlh.y, high = APART ? mlh.z : mlh.x;
            }
            // the first parts of each warp are on their way before it is known what they count (few rows: 14.7 -> 10.7 us for one
            // sequence of 1,500 tokens; many rows have next to none, and the registers would cost blocks)
            constexpr uint32_t kFirst = FEW ? 6 : 0;
            float4 parts[kMaxHead / 128][kFirst + 1];
#pragma unroll
            for (uint32_t k = 0; k < kMaxHead / 128; ++k)
#pragma unroll
                for (uint32_t i = 0; i < kFirst; ++i)
                    if (warp + i * kWarps < n && lane + 32 * k < quads)
                        parts[k][i] = reinterpret_cast<const float4*>(part(base + warp + i * kWarps))[lane + 32 * k];
            float now = m, now_peak = high;
#pragma unroll
            for (int x = 16; x; x /= 2) {
                now = fmaxf(now, __shfl_xor_sync(~0u, now, x));
                if (APART) now_peak = fmaxf(now_peak, __shfl_xor_sync(~0u, now_peak, x));
            }
            __syncthreads();
            if (lane == 0) wide[warp] = now, wide_peak[warp] = now_peak;
            __syncthreads();
            now = top, now_peak = peak;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                now = fmaxf(now, wide[w]);
                if (APART) now_peak = fmaxf(now_peak, wide_peak[w]);
            }
            const float by = top == now ? 1.0f : exp2f(top - now);
            top = now;
            const float factor = m == top ? 1.0f : exp2f(m - top);
            if (APART) {
                sum = sum * (peak == now_peak ? 1.0f : exp2f(peak - now_peak)) + l * (high == now_peak ? 1.0f : exp2f(high - now_peak));
                peak = now_peak;
            } else sum = sum * by + l * factor;
            factors[threadIdx.x] = factor;
            __syncthreads();
#pragma unroll
            for (uint32_t k = 0; k < kMaxHead / 128; ++k) {
                const uint32_t quad = lane + 32 * k;
                if (quad >= quads) continue;
                float4 a = acc[k];
                a.x *= by, a.y *= by, a.z *= by, a.w *= by;
                auto add = [&](const float4& v, float f) {
                    a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
                };
#pragma unroll
                for (uint32_t i = 0; i < kFirst; ++i)
                    if (warp + i * kWarps < n) add(parts[k][i], factors[warp + i * kWarps]);
#pragma unroll 4
                for (uint32_t i = warp + kFirst * kWarps; i < n; i += kWarps) add(reinterpret_cast<const float4*>(part(base + i))[quad], factors[i]);
                acc[k] = a;
            }
        }
#pragma unroll
        for (int m = 16; m; m /= 2) sum += __shfl_xor_sync(~0u, sum, m);
        __syncthreads();
        if (lane == 0) wide[warp] = sum;
#pragma unroll
        for (uint32_t k = 0; k < kMaxHead / 128; ++k)
            if (lane + 32 * k < quads) sums[warp][lane + 32 * k] = acc[k];
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) sum += wide[w];
        for (uint32_t c = threadIdx.x; c < d.head; c += kJoinThreads) {
            float o = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) o += reinterpret_cast<const float*>(sums[w])[c];
            o /= sum;  // first: the other factor may be far from 1
            if (APART) o *= exp2f(top - peak);
            out[c] = from_float<T>((APART ? peak : top) == -INFINITY ? 0.0f : o);
        }
        __syncthreads();  // before the next row's
    }
}

// Its start, and the sums over the lengths, behind the first kernel's work.
template <typename T, bool APART>
int launch_join(const Decode& d) {
    // few rows have many parts each, many units few or none: there the blocks are small enough to start beside the first
    // kernel's (one sequence of 1,500 tokens, 32 heads: 15 us with 512 threads, 20 with 128; 256 of 500: 178 and 117, and 113 by units)
    const bool few = (uint64_t)d.heads * d.batch <= 4u * ctx().sm_count;
    const cudaError_t err = few ? launch_next(decode_join_kernel<T, true, APART>, dim3(d.heads, d.batch), 512, ctx().stream(), d)
                                : launch_next(decode_join_kernel<T, false, APART>, dim3(d.units, d.batch), 128, ctx().stream(), d);
    return err == cudaSuccess ? check_launch("decode_join_kernel") : cuda_fail(err, "decode_join_kernel");
}

// Whether the kernel of 16-byte units takes the call.
bool by_units(const Decode& d, int dtype, const mtxc_decode_attention_args* a) {
    const bool small = a->cache.dtype == MTXC_FLOAT8_E4M3;
    const uint64_t unit = small ? 16 : 8;
    if (dtype == MTXC_FLOAT || d.head % unit) return false;
    for (int k = 0; k < 2; ++k) {
        if (reinterpret_cast<uintptr_t>(a->cache.data[k]) % 16) return false;
        for (int i = 0; i < 3; ++i)
            if (a->cache.strides[k][i] % unit) return false;
    }
    return true;
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
    d.groups_div = FastDiv(std::max(1u, d.groups));
    d.rows = std::min(kRows, std::max(1u, d.group));
    d.pitch = (d.head + 3) / 4 * 4 + 4;
    d.vector = by_units(d, dtype, a);
    d.tile = d.vector ? (a->cache.dtype == MTXC_FLOAT8_E4M3 ? 32 : 16) : kAnyTile;
    d.workers = ctx().sm_count * (d.vector ? warps_of(steps_of(d.head), a->cache.dtype == MTXC_FLOAT8_E4M3) : 2u);
    return MTXC_OK;
}

size_t partial_bytes(const Decode& d) { return ((size_t)2 * d.workers * d.rows * d.pitch * sizeof(float) + 255) / 256 * 256; }

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
    if (a->out == a->cache.data[0] || a->out == a->cache.data[1])
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": an output over the cache");
    if (int rc = laid_alike(who, a->out, a->out_strides, a->q, a->q_strides, {a->batch, a->heads})) return rc;
    const size_t bytes = partial_bytes(d);
    d.partial = static_cast<float*>(a->workspace ? a->workspace : ctx().workspace);
    if (reinterpret_cast<uintptr_t>(a->workspace) % 256)
        return fail(MTXC_ERR_INVALID_ARGUMENT, who + ": the workspace must be aligned to 256 bytes");
    if (bytes > (a->workspace ? a->workspace_bytes : ctx().workspace_bytes))
        return fail(MTXC_ERR_WORKSPACE, who + ": the partial sums need " + std::to_string(bytes) + " bytes of workspace");
    const bool small = a->cache.dtype == MTXC_FLOAT8_E4M3;
    int rc = MTXC_OK;
    dispatch_float(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if constexpr (!std::is_same_v<T, float>) {
            if (d.vector) {
                rc = small ? launch_units<T, true>(d) : launch_units<T, false>(d);
                if (rc) return;
                rc = small ? launch_join<T, true>(d) : launch_join<T, false>(d);
                return;
            }
        }
        const size_t smem = sizeof(float) * (kRows * d.head + 2 * kAnyTile * (d.head + 1) + kRows * kAnyTile);
        constexpr int kMost = sizeof(float) * (kRows * kMaxHead + 2 * kAnyTile * (kMaxHead + 1) + kRows * kAnyTile);
        auto kernel = small ? decode_any_kernel<T, true> : decode_any_kernel<T, false>;
        // the same limit in every call: calls from several threads do not undo each other's
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (err != cudaSuccess) {
            rc = cuda_fail(err, "cudaFuncSetAttribute");
            return;
        }
        kernel<<<d.workers, kAnyThreads, smem, ctx().stream()>>>(d);
        if ((rc = check_launch("decode_any_kernel"))) return;
        rc = launch_join<T, false>(d);
    });
    return rc;
}
