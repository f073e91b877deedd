// Grouped-query attention over a cache held in 4 bits (q4_cache.cuh): the mathematics that all its kernels share, and the one for blocks of a few rows (up to 16 a kv head at heads of 128)
// and for the head widths that q4_prompt.cuh does not take.  q4_step.cuh: up to four rows.
//
// out_r = sum_j p_rj v_j, p_rj = exp(s_rj - m_r) / l_r, s_rj = scale q_r . k_j.  A cached value is d_jb (c - 8) with one scale d per slot j and block b of 32
// dimensions, so   q_r . k_j = sum_b d_jb sum_{i in b} q_ri (c_ji - 8)   and   out_r = sum_j (p_rj d_jb) (c_ji - 8):
// both are products with codes, which f16 holds exactly.  The other factor, q_ri or p_rj d_jb, is an fp32 number that enters as two f16 numbers, 22 bits;
// the matrix instructions (mma.sync m16n8k16 with fp32 sums, a block is K = 32) add the products, and d_jb multiplies a block's sum in fp32.  Nothing is
// rounded to fewer than 22 bits, and the error is that of fp32 arithmetic.
//   scores   A = codes [16 slots][16 dimensions], two ldmatrix'd words a lane and block
//   output   A = codes^T [16 dimensions][16 slots], from the transposing ldmatrix
// The scores come out slot by row and the weights go in row by slot: movmatrix turns 8 x 8 of them.  Weights are scaled by a power of two so
// that the largest |d| seen so far, times the largest weight, is below 2^14: both digits stay in f16's normal range over 2^20 and more.  The matrix
// instructions cut their sums off towards zero (measured: 1 + 1.5 * 2^-24, a thousand times, is 1), which a long chain would add up to a
// bias, so a tile's output sums start at zero and join the running ones by a rounded addition; and codes enter with their offset taken off
// wherever a sum would otherwise begin far from zero.
//
// A warp works for itself: rows of queries (kRows of them) against tiles of 32 slots, which lane 0 fetches by bulk copies into the warp's own
// ring; the softmax is the running-maximum form.  The warps of a CTA take different rows or different tiles (row_warps), CTAs take
// different rows, runs of slots (gridDim.x) and kv heads; what several warps have of one row is merged in shared memory, what several
// CTAs have by a second launch.
// What bounds it: instructions, not memory: unpacking and the matrix instructions of a tile, which no row of the block can do without.  12 rows of 8 kv heads of 128:
// 20 us at 500 slots, 25.5 at 4003, 73 at 60000 (a byte read once would be 11 us there).  Steps of more than four rows come here too, as three launches: 28 / 4 and 64 / 8 heads of 128 take 14.8
// and 15.9 us at 1000 slots, 18.6 and 21.3 at 8000.  So do prompts of other widths, whose tiles every warp fetches for itself: 512 tokens into an empty cache 58 us with 12 / 4 heads of 96,
// 108 with 16 / 4 of 256.
#pragma once
#include <type_traits>

#include "q4_cache.cuh"

namespace zk {

constexpr uint32_t kQ4Tile = 32;             // slots of a tile

// How a warp's rows lie on the eight columns of a product.
enum Q4Columns : int {
    kQ4Digits = 0,       // four rows, a column a digit: half the products of the next for up to four rows (a step of a model with groups of four; q4_step.cuh)
    kQ4Rows8 = 1,        // eight rows, the digits one after the other
    kQ4Rows16 = 2,       // sixteen rows: the unpacked codes serve two products
    kQ4Prompt = 3        // none of these: the tensor cores proper (q4_prompt.cuh)
};
__host__ __device__ constexpr int q4_rows(int columns) { return columns == kQ4Digits ? 4 : columns == kQ4Rows8 ? 8 : 16; }
__host__ __device__ constexpr int q4_warps(int columns) { return columns == kQ4Digits ? 8 : 4; }
constexpr int kQ4Stages = 2;                 // tiles of a warp's ring: three were no faster, and take an SM's shared memory

struct Q4Attend {
    Q4Cache cache;
    Q4Rotation turn;
    const float* q;            // rows q_ld apart
    const int* position;
    const int* filled;
    const float* weight_in;    // [kv_heads][slots]
    float* weight_out;         // or null
    float* out;                // [tokens][heads * head_dim]
    float* part_out;           // workspace [kv_heads][splits][rows][head_dim]: sums of a run of slots, relative to its own maximum
    float* part_stats;         // workspace [kv_heads][splits][rows][2]: that maximum (of scores in units of log 2) and the sum of weights
    float* scores;             // workspace [kv_heads][rows][slots], or null: the scores are not kept
    float* stats;              // workspace [kv_heads][rows]: maximum + log2 of the sum, or null
    uint4* queries;            // workspace [kv_heads][row tiles of eight][blocks][2][32 lanes]: the rows as the products take them
    float* factors;            // workspace [kv_heads][padded rows]: what makes scores of their products
    uint32_t tokens, heads, group;      // group = heads / kv_heads; a kv head has tokens * group rows, row = token * group + head of the group
    uint32_t splits, row_warps;
    uint32_t run_tile;         // slots of a tile that runs are counted in
    uint32_t padded;           // rows, rounded up to a whole number of what a warp takes
    const float* k;            // rows kv_ld apart
    const float* v;
    float* k_held;             // or null
    float* v_held;
    size_t q_ld, kv_ld;
    float scale;
    int* error_word;
};

// The runs of slots the CTAs of a row take: the same arithmetic where they are merged.
struct Q4Runs {
    uint32_t tiles, per, active;
};
__device__ __forceinline__ Q4Runs q4_runs(uint32_t slots_seen, uint32_t splits, uint32_t key_warps, uint32_t tile) {
    Q4Runs r;
    r.tiles = (slots_seen + tile - 1) / tile;
    r.per = max((r.tiles + splits - 1) / splits, key_warps);
    r.active = (r.tiles + r.per - 1) / r.per;
    return r;
}

// d = a * b + c
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float low, float high) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// The upper eleven bits of a number: what f16 holds of it without rounding.
__device__ __forceinline__ float upper_digit(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }
// Codes in the low (high) nibbles of two halves, less eight.
__device__ __forceinline__ uint32_t signed_low(uint32_t x) {
    const uint32_t v = (x & 0x000f000fu) | 0x64006400u;
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0xe408e408u));                         // 1024 + c - 1032
    return r;
}
__device__ __forceinline__ uint32_t signed_high(uint32_t x) {
    const uint32_t v = (x & 0x00f000f0u) | 0x64006400u;
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0x2c002c00u), "r"(0xd480d480u));   // (1024 + 16 c) / 16 - 72
    return r;
}
// a += b, two at a time
__device__ __forceinline__ void add_pairs(float (&a)[4], const float (&b)[4]) {
    asm("{ .reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;\n\t"
        "mov.b64 x, {%2, %3}; mov.b64 y, {%6, %7}; add.rn.f32x2 x, x, y; mov.b64 {%2, %3}, x; }"
        : "+f"(a[0]), "+f"(a[1]), "+f"(a[2]), "+f"(a[3]) : "f"(b[0]), "f"(b[1]), "f"(b[2]), "f"(b[3]));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Four slots' scales of all blocks, kept as they are until they are used.
template <int kBlocks>
struct Q4Scales {
    uint32_t pair[4][(kBlocks + 1) / 2];
    // slots at, at + 8, at + 16, at + 24
    __device__ __forceinline__ void load(const __half* s, uint32_t at) {
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            const __half* from = s + (at + 8 * o) * kBlocks;
            if constexpr (kBlocks % 4 == 0) {
#pragma unroll
                for (int b = 0; b < kBlocks / 4; ++b) {
                    const uint2 two = reinterpret_cast<const uint2*>(from)[b];
                    pair[o][2 * b] = two.x;
                    pair[o][2 * b + 1] = two.y;
                }
            } else if constexpr (kBlocks % 2 == 0) {
#pragma unroll
                for (int b = 0; b < kBlocks / 2; ++b) pair[o][b] = reinterpret_cast<const uint32_t*>(from)[b];
            } else {
#pragma unroll
                for (int b = 0; b < kBlocks; b += 2)
                    pair[o][b / 2] = __half_as_ushort(from[b]) | (b + 1 < kBlocks ? static_cast<uint32_t>(__half_as_ushort(from[b + 1])) << 16 : 0u);
            }
        }
    }
    __device__ __forceinline__ float of(int o, int block) const {
        const __half2 two = *reinterpret_cast<const __half2*>(&pair[o][block / 2]);
        return block % 2 ? __high2float(two) : __low2float(two);
    }
    // the largest magnitude among the scales of slot `at` alone, as f16 bits
    static __device__ __forceinline__ uint32_t largest(const __half* s, uint32_t at) {
        const __half* from = s + at * kBlocks;
        if constexpr (kBlocks % 2 == 0) {
            uint32_t top = 0;
#pragma unroll
            for (int b = 0; b < kBlocks / 2; ++b) top = __vmaxu2(top, reinterpret_cast<const uint32_t*>(from)[b] & 0x7fff7fffu);
            return max(top & 0xffffu, top >> 16);
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) top = max(top, __half_as_ushort(from[b]) & 0x7fffu);
            return top;
        }
    }
};

template <int kBlocks>
__host__ __device__ constexpr uint32_t q4_stage_bytes() { return kQ4Tile * kBlocks * 36; }         // 16 + 16 code bytes and 2 + 2 of scales a slot and block
// Dynamic shared memory of q4_attend_kernel: the warps' rings, then the rows of queries as the products take them.
template <int kBlocks, int kColumns>
__host__ __device__ constexpr uint32_t q4_attend_smem(uint32_t row_warps) {
    return q4_warps(kColumns) * kQ4Stages * q4_stage_bytes<kBlocks>() + row_warps * (kColumns == kQ4Rows16 ? 4 : 2) * kBlocks * 512;
}

// What makes scores (in units of log 2) of the products of a row that is 2^(13 - e) as large.  Never zero, as it would be for a row of zeros or a very small scale: a masked score, minus
// infinity, times zero is not a number.  The products' sums are below 2^45, so that with 2^-126 instead every score is zero to more than 32 bits of its exponential.
constexpr float kQ4LeastFactor = 1.17549435e-38f;             // 2^-126
__device__ __forceinline__ float q4_row_factor(float scale, int e) {
    const int units = e - 13;                // in two steps, for it may be beyond what one power of two can be
    return fmaxf(fabsf(scale) * 1.4426950408889634f * power_of_two(units / 2) * power_of_two(units - units / 2), kQ4LeastFactor);
}

// A warp turns one row of queries into the products' second operand.  A lane's words of a block are its dimensions 4t, 4t+2 | 16+4t, 16+4t+2 (low and high nibbles of
// bytes 4t and 4t+2) and 4t+1, 4t+3 | 17+4t, 19+4t, of the lane's column; kDigits: columns 2r and 2r + 1 are row r's digits; else
// a column is a row and the digits are two such sets.  The row, times a power of two, has its largest value in [2^13, 2^14).  Returns the row's factor, which makes scores
// (in units of log 2) of the products.
template <int kBlocks, bool kDigits>
__device__ __forceinline__ float q4_lay_row(const float (&x)[kBlocks], uint4* to, uint32_t row, float scale, uint32_t lane) {
    float top = 0.0f;
#pragma unroll
    for (int g = 0; g < kBlocks; ++g) top = fmaxf(top, fabsf(x[g]));
    const uint32_t size = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    const int e = max(static_cast<int>(size >> 23) - 127, -114);
    const float up = scale < 0.0f ? -power_of_two(13 - e) : power_of_two(13 - e);
    const uint32_t part = lane >> 4, t = (lane & 15u) >> 2, step = lane & 1u, half = (lane >> 1) & 1u, word = 2 * step + part;
    __half* const halves = reinterpret_cast<__half*>(to);
#pragma unroll
    for (int g = 0; g < kBlocks; ++g) {
        const float y = x[g] * up, upper = upper_digit(y);
        const __half first = __float2half_rn(upper), other = __float2half_rn(y - upper);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const uint32_t column = kDigits ? 2 * row + d : row & 7u;
            const size_t at = kDigits ? g * 32 + column * 4 + t : ((static_cast<size_t>(row >> 3) * kBlocks + g) * 2 + d) * 32 + column * 4 + t;
            halves[(at * 4 + word) * 2 + half] = d ? other : first;
        }
    }
    return q4_row_factor(scale, e);
}

// A lane's value of a block (0 .. kBlocks - 1 of the key, then of the value) of new token t, the key's rotated.
template <int kBlocks>
__device__ __forceinline__ float q4_new_value(const Q4Attend& p, uint32_t h, uint32_t t, uint32_t item, size_t turned, uint32_t lane) {
    const size_t head_at = t * p.kv_ld + static_cast<size_t>(h) * kBlocks * 32;
    return item >= kBlocks ? __ldcg(p.v + head_at + (item - kBlocks) * 32 + lane) : q4_rotated(p.k + head_at, item * 32 + lane, p.turn, turned);
}
// A warp quantises such a block into its slot.  Lanes 0 .. 15 return the block's bytes.
template <int kBlocks>
__device__ __forceinline__ uint8_t q4_append_block(const Q4Attend& p, float x, uint32_t h, uint32_t t, uint32_t item, uint32_t filled, uint32_t lane, __half& scale) {
    const bool is_value = item >= kBlocks;
    const uint32_t block = is_value ? item - kBlocks : item, slot = filled + t;
    const Q4Quantised q = q4_quantise(x, lane);
    const uint32_t high = __shfl_down_sync(0xffffffffu, q.code, 16);
    const uint8_t byte = static_cast<uint8_t>(q.code | high << 4);
    if (lane < 16) (is_value ? p.cache.v_codes : p.cache.k_codes)[q4_codes_at(h, slot, block, kBlocks, p.cache.slots) + lane] = byte;
    if (lane == 0) (is_value ? p.cache.v_scales : p.cache.k_scales)[q4_scale_at(h, slot, block, kBlocks, p.cache.slots)] = q.scale;
    float* held = is_value ? p.v_held : p.k_held;
    if (held) held[(static_cast<size_t>(t) * p.cache.kv_heads + h) * kBlocks * 32 + block * 32 + lane] = (static_cast<float>(q.code) - 8.0f) * __half2float(q.scale);
    scale = q.scale;
    return byte;
}

// New keys (rotated) and values into the slots behind *filled, where nothing else is to be prepared: four lanes a block, a lane has eight values, which are a word of its
// codes.  512 tokens of 8 kv heads of 128 values: 8.8 us launch after launch (a lane a value, which rotates
// every pair twice and quantises through the warp: 14).
constexpr uint32_t kQ4AppendThreads = 256;
template <int kBlocks>
__global__ void __launch_bounds__(kQ4AppendThreads) q4_append_kernel(const __grid_constant__ Q4Attend p) {
    const uint32_t items = p.tokens * p.cache.kv_heads * 2 * kBlocks, item = blockIdx.x * (kQ4AppendThreads / 4) + threadIdx.x / 4, mine = min(item, items - 1), j = threadIdx.x & 3u;
    const uint32_t piece = mine % (2 * kBlocks), h = mine / (2 * kBlocks) % p.cache.kv_heads, t = mine / (2 * kBlocks) / p.cache.kv_heads;
    const bool is_value = piece >= kBlocks;
    const uint32_t block = is_value ? piece - kBlocks : piece;
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicExch(p.error_word, kErrBadPosition);
        return;
    }
    Q4Rotation turn = p.turn;
    if (is_value) turn.pairs = 0;
    const float* const from = is_value ? p.v : p.k;
    float x[8];
    q4_rotated_eight(x, from + t * p.kv_ld + static_cast<size_t>(h) * kBlocks * 32, block * 32 + 4 * j, turn, static_cast<size_t>(position) + t, q4_rotates_fours(from, p.kv_ld, kBlocks * 32, turn));
    uint32_t top = 0, first = 0xffffffffu;                    // the largest magnitude; its first place, above the sign there
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if ((__float_as_uint(x[e]) & 0x7fffffffu) == top) first = min(first, (4 * j + (e & 3) + (e >> 2) * 16) * 2 + (__float_as_uint(x[e]) >> 31));
    first = min(first, __shfl_xor_sync(0xffffffffu, first, 1));
    first = min(first, __shfl_xor_sync(0xffffffffu, first, 2));
    if (item >= items) return;
    const __half scale = q4_scale_of(__uint_as_float(top | (first & 1u) << 31));
    const float d = __half2float(scale), inverse = __frcp_rn(d);
    uint32_t word = 0, code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        code[e] = q4_code_of(x[e], d, inverse);
        word |= code[e] << (8 * (e & 3) + 4 * (e >> 2));
    }
    const uint32_t slot = static_cast<uint32_t>(filled) + t;
    reinterpret_cast<uint32_t*>((is_value ? p.cache.v_codes : p.cache.k_codes) + q4_codes_at(h, slot, block, kBlocks, p.cache.slots))[j] = word;
    if (j == 0) (is_value ? p.cache.v_scales : p.cache.k_scales)[q4_scale_at(h, slot, block, kBlocks, p.cache.slots)] = scale;
    float* held = is_value ? p.v_held : p.k_held;
    if (held) {
        held += (static_cast<size_t>(t) * p.cache.kv_heads + h) * kBlocks * 32 + block * 32 + 4 * j;
#pragma unroll
        for (int e = 0; e < 8; ++e) held[(e & 3) + (e >> 2) * 16] = (static_cast<float>(code[e]) - 8.0f) * d;
    }
}

// What a block's attention begins with: the new tokens' keys (rotated) and values go into the slots behind *filled, and their queries (rotated) are laid out
// for the products.  grid = (tokens, kv_heads); a warp takes a block of the key or the value, or a row of queries.
constexpr uint32_t kQ4PrepareWarps = 16;
template <int kBlocks>
__global__ void __launch_bounds__(kQ4PrepareWarps * 32) q4_prepare_kernel(const __grid_constant__ Q4Attend p) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, t = blockIdx.x, h = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) {
        if (threadIdx.x == 0 && t == 0 && h == 0) atomicExch(p.error_word, kErrBadPosition);
        return;
    }
    const size_t turned = static_cast<size_t>(position) + t;
    const uint32_t rows = p.tokens * p.group, last = t + 1 == p.tokens ? p.padded - rows : 0u;       // the last token's CTA clears the rows that pad a tile
    for (uint32_t item = warp; item < 2 * kBlocks + p.group + last; item += warps) {
        if (item < 2 * kBlocks) {
            __half ignored;
            q4_append_block<kBlocks>(p, q4_new_value<kBlocks>(p, h, t, item, turned, lane), h, t, item, static_cast<uint32_t>(filled), lane, ignored);
            continue;
        }
        const uint32_t j = item - 2 * kBlocks, row = t * p.group + j;
        float x[kBlocks] = {};
        if (j < p.group) {
            const float* from = p.q + t * p.q_ld + static_cast<size_t>(h * p.group + j) * kBlocks * 32;
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) x[g] = q4_rotated(from, g * 32 + lane, p.turn, turned);
        }
        const float factor = q4_lay_row<kBlocks, false>(x, p.queries + static_cast<size_t>(h) * p.padded * kBlocks * 8, row, p.scale, lane);
        if (lane == 0) p.factors[static_cast<size_t>(h) * p.padded + row] = factor;
    }
}

// grid = (splits, CTAs for the rows, kv_heads); the rows that see most slots come first.
template <int kBlocks, int kColumns>
__global__ void __launch_bounds__(q4_warps(kColumns) * 32, kBlocks > 4 ? 1 : 3) q4_attend_kernel(const __grid_constant__ Q4Attend p) {
    constexpr int kWarps = q4_warps(kColumns), kStages = kQ4Stages, kRows = q4_rows(kColumns), kDim = kBlocks * 32, kTiles = kColumns == kQ4Rows16 ? 2 : 1;
    constexpr uint32_t kStage = q4_stage_bytes<kBlocks>(), kCodes = kQ4Tile * kBlocks * 16, kScales = kQ4Tile * kBlocks * 2;
    extern __shared__ __align__(128) uint8_t q4_smem[];
    __shared__ uint64_t landed[kWarps][kStages], queries_landed;
    __shared__ float row_max[kWarps][16], row_sum[kWarps][16], row_unit[kWarps];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = lane & 3u, h = blockIdx.z;
    const uint32_t key_warps = kWarps / p.row_warps, row_warp = warp % p.row_warps, key_warp = warp / p.row_warps;
    const uint32_t rows = p.tokens * p.group, cta_rows = p.row_warps * kRows;
    const uint32_t cta_first = (gridDim.y - 1 - blockIdx.y) * cta_rows, first = cta_first + row_warp * kRows;
    uint4* const queries = reinterpret_cast<uint4*>(q4_smem + kWarps * kStages * kStage);
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&landed[warp][s], 1);
        if (warp == 0) mbar_init(&queries_landed, 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;      // the append has said so
    const uint32_t filled = filled_in, real_rows = min(cta_rows, rows - cta_first);
    const uint32_t seen = filled + (cta_first + real_rows - 1) / p.group + 1;           // slots of the CTA's last token
    const Q4Runs runs = q4_runs(seen, p.splits, key_warps, kQ4Tile);
    const uint32_t begin = blockIdx.x * runs.per, end = min(runs.tiles, begin + runs.per);
    if (begin >= end) return;                                                            // nobody counts on this run

    // lane 0 keeps the ring filled
    uint8_t* ring = q4_smem + warp * kStages * kStage;
    const size_t head_slots = static_cast<size_t>(h) * p.cache.slots;
    auto fetch = [&](uint32_t tile, int stage) {
        const size_t slot = head_slots + static_cast<size_t>(tile) * kQ4Tile;
        uint8_t* to = ring + stage * kStage;
        mbar_arrive_expect_tx(&landed[warp][stage], kStage);
        bulk_g2s(to, p.cache.k_codes + slot * (kBlocks * 16), kCodes, &landed[warp][stage]);
        bulk_g2s(to + 2 * kCodes, p.cache.k_scales + slot * kBlocks, kScales, &landed[warp][stage]);
        bulk_g2s(to + kCodes, p.cache.v_codes + slot * (kBlocks * 16), kCodes, &landed[warp][stage]);
        bulk_g2s(to + 2 * kCodes + kScales, p.cache.v_scales + slot * kBlocks, kScales, &landed[warp][stage]);
    };
    const uint32_t mine = begin + key_warp < end && first < rows ? (end - begin - key_warp + key_warps - 1) / key_warps : 0u;      // tiles of this warp
    if (lane == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");       // the stores of the launch before come ahead of the copies
        if (warp == 0) {
            const uint32_t bytes = min(cta_rows, p.padded - cta_first) * kBlocks * 128;
            mbar_arrive_expect_tx(&queries_landed, bytes);
            bulk_g2s(queries, p.queries + (static_cast<size_t>(h) * p.padded + cta_first) * kBlocks * 8, bytes, &queries_landed);
        }
        for (uint32_t i = 0; i < min(mine, static_cast<uint32_t>(kStages)); ++i) fetch(begin + key_warp + i * key_warps, i);
    }
    const uint4* const my_queries = queries + row_warp * kTiles * kBlocks * 64;
    // of the lane's rows: the last slot each sees, and what makes scores of its products
    uint32_t last_seen[kTiles][2], least = 0xffffffffu;
    float factor[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t r = 8 * n + 2 * t + c;
            last_seen[n][c] = filled + min(first + r, rows - 1) / p.group;
            least = min(least, last_seen[n][c]);
            factor[n][c] = __ldcg(p.factors + static_cast<size_t>(h) * p.padded + min(first + r, p.padded - 1));
        }
    least = __reduce_min_sync(0xffffffffu, least);
    bool failed = !__all_sync(0xffffffffu, mbar_wait(&queries_landed, 0));
    if (failed && lane == 0) atomicExch(p.error_word, kErrFullWaitTimeout);

    float acc[kTiles][2 * kBlocks][4];
    float m[kTiles][2], l[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * kBlocks; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][i][j] = 0.0f;
    }
    // Weights times 2^(kFull - unit) times their slot's d are below 2^14: d is below 2^unit and a weight at most 2^kSlack.
    constexpr float kSlack = 8.0f;
    constexpr int kFull = 6, kHeadroom = 14;            // f16's exponent field less 14: the power of two above a scale
    int unit = -32;
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};

    // A tile; kWhole: every row sees every slot of it.
    auto work = [&](const uint8_t* stage, uint32_t slot0, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        const uint32_t a = lane >> 2;                     // the lane's slots are a, a + 8, a + 16, a + 24
        const __half* k_scales = reinterpret_cast<const __half*>(stage + 2 * kCodes);
        const __half* v_scales = k_scales + kQ4Tile * kBlocks;
        const uint32_t matrix = ((lane >> 3) * kBlocks * 8 + (lane & 7u)) * 16;
        float s[2][kTiles][4] = {};                       // [half of the tile][..][slot a of the half, columns 2t, 2t+1; slot a + 8]
        {
            Q4Scales<kBlocks> d;
            d.load(k_scales, a);
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
                uint32_t w[4];
                ldmatrix_x4(w, smem_u32(stage) + matrix + g * 128);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t u = w[2 * half], v = w[2 * half + 1], x = u >> 8, y = v >> 8;
                    const float da = d.of(2 * half, g), db = d.of(2 * half + 1, g);
                    const uint32_t even[4] = {signed_low(u), signed_low(v), signed_high(u), signed_high(v)};
                    const uint32_t odd[4] = {signed_low(x), signed_low(y), signed_high(x), signed_high(y)};
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const uint4 upper = my_queries[(n * kBlocks + g) * 64 + lane], lower = my_queries[(n * kBlocks + g) * 64 + 32 + lane];
                        float c[4];
                        mma_f16(c, even, lower.x, lower.y, zero);
                        mma_f16(c, odd, lower.z, lower.w, c);
                        mma_f16(c, even, upper.x, upper.y, c);
                        mma_f16(c, odd, upper.z, upper.w, c);
                        s[half][n][0] = fmaf(da, c[0], s[half][n][0]);
                        s[half][n][1] = fmaf(da, c[1], s[half][n][1]);
                        s[half][n][2] = fmaf(db, c[2], s[half][n][2]);
                        s[half][n][3] = fmaf(db, c[3], s[half][n][3]);
                    }
                }
            }
        }
        auto hidden = [&](int half, int n, int j) { return !kWhole && slot0 + 16 * half + 8 * (j / 2) + a > last_seen[n][j & 1]; };
        // the largest scale of a value that any row sees, as a power of two
        const uint32_t top = __reduce_max_sync(0xffffffffu, kWhole || slot0 + lane < seen ? Q4Scales<kBlocks>::largest(v_scales, lane) : 0u);
        const int new_unit = max(unit, min(static_cast<int>(top >> 10), 30) - kHeadroom);
        bool moved = new_unit != unit;
        float next[kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            if constexpr (!kWhole) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[half][n][j] = hidden(half, n, j) ? -INFINITY : s[half][n][j];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = fmaxf(fmaxf(s[0][n][c], s[0][n][2 + c]), fmaxf(s[1][n][c], s[1][n][2 + c]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) * factor[n][c];
                next[n][c] = x > m[n][c] + kSlack ? x : m[n][c];      // a maximum that is little larger leaves the weights above one, and the sums as they are
                moved |= next[n][c] != m[n][c];
            }
        }
        if (p.scores) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t row = first + 8 * n + 2 * t + c;
                    if (row >= rows) continue;
                    float* to = p.scores + (static_cast<size_t>(h) * rows + row) * p.cache.slots + slot0 + a;
#pragma unroll
                    for (int half = 0; half < 2; ++half) { to[16 * half] = s[half][n][c] * factor[n][c]; to[16 * half + 8] = s[half][n][2 + c] * factor[n][c]; }
                }
        }
        if (__any_sync(0xffffffffu, moved)) {
            const float of_unit = unit == -32 ? 0.0f : power_of_two(unit - new_unit);
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float corr = m[n][c] == -INFINITY ? 0.0f : exp2_fast(m[n][c] - next[n][c]);
                    l[n][c] *= corr;
                    m[n][c] = next[n][c];
#pragma unroll
                    for (int j = 0; j < 2 * kBlocks; ++j) {
                        acc[n][j][c] *= corr * of_unit;
                        acc[n][j][2 + c] *= corr * of_unit;
                    }
                }
            unit = new_unit;
        }
        const float up = power_of_two(kFull - unit);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float by = factor[n][j & 1], from = m[n][j & 1] == -INFINITY ? 0.0f : m[n][j & 1];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float w = exp2_fast(fmaf(s[half][n][j], by, -from));
                    l[n][j & 1] += w;
                    s[half][n][j] = w * up;
                }
            }
        Q4Scales<kBlocks> d;
        d.load(v_scales, a);
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            uint32_t w[4];
            ldmatrix_x4_trans(w, smem_u32(stage) + kCodes + matrix + g * 128);
            uint32_t even[2][4], odd[2][4];               // dimensions 2r and 16 + 2r, 2r + 1 and 17 + 2r of the block, r the lane's row
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t u = w[2 * half], v = w[2 * half + 1], x = u >> 8, y = v >> 8;
                even[half][0] = signed_low(u); even[half][1] = signed_high(u); even[half][2] = signed_low(v); even[half][3] = signed_high(v);
                odd[half][0] = signed_low(x); odd[half][1] = signed_high(x); odd[half][2] = signed_low(y); odd[half][3] = signed_high(y);
            }
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float sum[2][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // a slot that is not seen may hold anything
                    auto weight = [&](int j) { return hidden(half, n, j) ? 0.0f : s[half][n][j] * d.of(2 * half + j / 2, g); };
                    const float w0 = weight(0), w1 = weight(1), w2 = weight(2), w3 = weight(3);
                    const float h0 = upper_digit(w0), h1 = upper_digit(w1), h2 = upper_digit(w2), h3 = upper_digit(w3);
                    const uint32_t b0 = transposed(pack_f16(h0, h1)), b1 = transposed(pack_f16(h2, h3));
                    const uint32_t c0 = transposed(pack_f16(w0 - h0, w1 - h1)), c1 = transposed(pack_f16(w2 - h2, w3 - h3));
                    mma_f16(sum[0], even[half], b0, b1, half ? static_cast<const float (&)[4]>(sum[0]) : zero);
                    mma_f16(sum[1], odd[half], b0, b1, half ? static_cast<const float (&)[4]>(sum[1]) : zero);
                    mma_f16(sum[0], even[half], c0, c1, sum[0]);
                    mma_f16(sum[1], odd[half], c0, c1, sum[1]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) add_pairs(acc[n][2 * g + i], sum[i]);
            }
        }
    };

    int stage = 0;
    uint32_t phase = 0;
    for (uint32_t i = 0; i < mine; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait(&landed[warp][stage], phase))) {
            // the copies that are under way land (or are given up) before the ring is used for anything else
            if (lane == 0) {
                atomicExch(p.error_word, kErrFullWaitTimeout);
                for (uint32_t j = i; j < min(mine, i + kStages); ++j) mbar_wait(&landed[warp][j % kStages], (j / kStages) & 1u);
            }
            __syncwarp();
            failed = true;
            break;
        }
        const uint32_t tile = begin + key_warp + i * key_warps, slot0 = tile * kQ4Tile;
        if (slot0 + kQ4Tile - 1 <= least) work(ring + stage * kStage, slot0, std::true_type{});
        else work(ring + stage * kStage, slot0, std::false_type{});
        __syncwarp();                       // everybody is done with the stage
        if (lane == 0 && i + kStages < mine) fetch(tile + kStages * key_warps, stage);
        if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
        }
    }

    // the warp's sums into its ring's memory, [row][dimension]
    float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
            const uint32_t r = 8 * n + 2 * t + c;
            if (lane < 4) { row_max[warp][r] = m[n][c]; row_sum[warp][r] = failed ? NAN : l[n][c]; }
        }
#pragma unroll
        for (int g = 0; g < kBlocks; ++g)
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const uint32_t e = g * 32 + 2 * (lane >> 2) + odd;
                const float (&c)[4] = acc[n][2 * g + odd];
                sums[(8 * n + 2 * t) * kDim + e] = c[0];
                sums[(8 * n + 2 * t + 1) * kDim + e] = c[1];
                sums[(8 * n + 2 * t) * kDim + e + 16] = c[2];
                sums[(8 * n + 2 * t + 1) * kDim + e + 16] = c[3];
            }
    }
    if (lane == 0) row_unit[warp] = unit == -32 ? 0.0f : power_of_two(unit - kFull);
    __syncthreads();
    // the key warps' shares of a row
    const bool alone = p.splits == 1;
    for (uint32_t i = threadIdx.x; i < real_rows * kDim; i += kWarps * 32) {
        const uint32_t r = i / kDim, e = i % kDim, rw = r / kRows, at = r % kRows, row = cta_first + r;
        float top = row_max[rw][at];
        for (uint32_t k = 1; k < key_warps; ++k) top = fmaxf(top, row_max[k * p.row_warps + rw][at]);
        float sum = 0.0f, o = 0.0f;
        for (uint32_t k = 0; k < key_warps; ++k) {
            const uint32_t w = k * p.row_warps + rw;
            const float its = row_max[w][at], by = its == -INFINITY ? 0.0f : exp2_fast(its - top);
            const float share = reinterpret_cast<const float*>(q4_smem + w * kStages * kStage)[at * kDim + e];
            sum += by * row_sum[w][at];
            o += its == -INFINITY ? 0.0f : by * row_unit[w] * share;
        }
        if (alone) {
            const uint32_t token = row / p.group, head = h * p.group + row % p.group;
            p.out[(static_cast<size_t>(token) * p.heads + head) * kDim + e] = o / sum;
            if (e == 0) {
                if (!(sum > 0.0f) || !(sum < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
                if (p.stats) p.stats[static_cast<size_t>(h) * rows + row] = top + log2f(sum);
                if (p.scores) reinterpret_cast<float2*>(p.part_stats)[static_cast<size_t>(h) * rows + row] = make_float2(top, sum);
            }
        } else {
            const size_t part = (static_cast<size_t>(h) * p.splits + blockIdx.x) * rows + row;
            p.part_out[part * kDim + e] = o;
            if (e == 0) { p.part_stats[2 * part] = top; p.part_stats[2 * part + 1] = sum; }
        }
    }
}

// What the CTAs of a launch leave: the first `join_ctas` CTAs of a kv head put the runs of its rows together, the others add up what the slots received (512 each),
// where scores were kept.  Neither waits for the other: a row's maximum and sum over its runs are formed where they are needed.
//   rows     `parts` warps a row, each with every so-manieth run, all of their loads in flight at once (a step's time here is round trips)
//   slots    a thread a slot
// The rows of one CTA of the launch before (cta_rows of them) have their number of runs from its arithmetic.  grid = (join_ctas + CTAs for slots, kv_heads).
constexpr uint32_t kQ4FinishWarps = 16, kQ4FinishRuns = 3, kQ4KeptRows = 32;      // runs of a warp at a time; rows whose scores are kept
struct Q4Whole {
    float top, sum;
};
// A row's maximum and sum over all of its runs, in every lane.
__device__ __forceinline__ Q4Whole q4_whole(const float2* stats, uint32_t active, uint32_t rows, uint32_t lane) {
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t s = lane; s < active; s += 32) {
        const float2 its = __ldcg(stats + static_cast<size_t>(s) * rows);
        const float next = fmaxf(top, its.x);
        // a run without a maximum has no sum, or that of scores that are not numbers
        sum = (next == -INFINITY ? sum : sum * exp2_fast(top - next)) + (its.x == -INFINITY ? its.y : exp2_fast(its.x - next) * its.y);
        top = next;
    }
    const float own = top;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    sum = own == -INFINITY ? sum : sum * exp2_fast(own - top);      // a NaN stays, whatever the maxima are
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return Q4Whole{top, sum};
}

__global__ void __launch_bounds__(kQ4FinishWarps * 32) q4_finish_kernel(const __grid_constant__ Q4Attend p, uint32_t cta_rows, uint32_t key_warps, uint32_t parts, uint32_t join_ctas) {
    __shared__ float4 share[kQ4FinishWarps][64];
    __shared__ float whole[kQ4KeptRows];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, part = warp % parts, h = blockIdx.y, rows = p.tokens * p.group, quads = p.cache.blocks * 8;
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;
    const uint32_t filled = filled_in;
    auto runs_of = [&](uint32_t row) { return q4_runs(filled + (min(rows, (row / cta_rows + 1) * cta_rows) - 1) / p.group + 1, p.splits, key_warps, p.run_tile).active; };
    auto stats_of = [&](uint32_t row) { return reinterpret_cast<const float2*>(p.part_stats) + static_cast<size_t>(h) * p.splits * rows + row; };
    if (blockIdx.x >= join_ctas) {
        const uint32_t slot = (blockIdx.x - join_ctas) * kQ4FinishWarps * 32 + threadIdx.x, seen = filled + p.tokens;
        if (slot - threadIdx.x >= seen) return;
        for (uint32_t row = warp; row < rows; row += kQ4FinishWarps) {
            const Q4Whole w = q4_whole(stats_of(row), runs_of(row), rows, lane);
            if (lane == 0) whole[row] = w.top + log2f(w.sum);
        }
        const size_t at = static_cast<size_t>(h) * p.cache.slots + slot;
        const float before = slot < filled ? p.weight_in[at] : 0.0f;
        __syncthreads();
        if (slot >= seen) return;
        float sum = 0.0f;
#pragma unroll 4
        for (uint32_t r = slot < filled ? 0u : (slot - filled) * p.group; r < rows; ++r)
            sum += exp2_fast(__ldcg(p.scores + (static_cast<size_t>(h) * rows + r) * p.cache.slots + slot) - whole[r]);
        p.weight_out[at] = sum + before;
        return;
    }
    const uint32_t row = blockIdx.x * (kQ4FinishWarps / parts) + warp / parts;
    const bool mine = row < rows;
    Q4Whole w{};
    if (mine) {
        const uint32_t active = runs_of(row);
        const float2* stats = stats_of(row);
        const float4* from = reinterpret_cast<const float4*>(p.part_out) + (static_cast<size_t>(h) * p.splits * rows + row) * quads;
        float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        // a warp's first runs are asked for before anything is known of the maxima
        auto ask = [&](float4 (&x)[kQ4FinishRuns][2], float (&its)[kQ4FinishRuns], uint32_t s0) {
#pragma unroll
            for (uint32_t i = 0; i < kQ4FinishRuns; ++i) {
                const uint32_t s = s0 + i * parts;
                its[i] = s < active ? __ldcg(stats + static_cast<size_t>(s) * rows).x : -INFINITY;
#pragma unroll
                for (uint32_t q = 0; q < 2; ++q)
                    x[i][q] = s < active && lane + 32 * q < quads ? __ldcg(from + static_cast<size_t>(s) * rows * quads + lane + 32 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        float4 x[kQ4FinishRuns][2];
        float its[kQ4FinishRuns];
        ask(x, its, part);
        w = q4_whole(stats, active, rows, lane);
        for (uint32_t s0 = part; s0 < active; s0 += kQ4FinishRuns * parts) {
            if (s0 != part) ask(x, its, s0);
#pragma unroll
            for (uint32_t i = 0; i < kQ4FinishRuns; ++i) {
                const float by = its[i] == -INFINITY ? 0.0f : exp2_fast(its[i] - w.top);
#pragma unroll
                for (uint32_t q = 0; q < 2; ++q) { o[q].x += by * x[i][q].x; o[q].y += by * x[i][q].y; o[q].z += by * x[i][q].z; o[q].w += by * x[i][q].w; }
            }
        }
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) share[warp][lane + 32 * q] = o[q];
    }
    __syncthreads();
    if (part || !mine) return;
    const uint32_t token = row / p.group, head = h * p.group + row % p.group;
    for (uint32_t q = lane; q < quads; q += 32) {
        float4 o = share[warp][q];
        for (uint32_t i = 1; i < parts; ++i) { const float4 x = share[warp + i][q]; o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w; }
        float* to = p.out + ((static_cast<size_t>(token) * p.heads + head) * quads + q) * 4;
        to[0] = o.x / w.sum; to[1] = o.y / w.sum; to[2] = o.z / w.sum; to[3] = o.w / w.sum;
    }
    if (lane == 0) {
        if (!(w.sum > 0.0f) || !(w.sum < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
        if (p.stats) p.stats[static_cast<size_t>(h) * rows + row] = w.top + log2f(w.sum);
    }
}

// What the slots received in a block of many rows: the scores are formed once more, now that the rows' sums are known.  A warp takes 32
// slots, its unpacked codes in registers; tiles of eight rows, as q4_attend_kernel left them, pass through shared memory for the CTA's
// eight warps.  A cluster's eight CTAs share the rows, and their sums meet in rank 0.  grid = (8, runs of 256 slots, kv_heads).
constexpr int kReceivedWarps = 8, kReceivedCtas = 8, kReceivedStages = 3;
constexpr uint32_t kReceivedSlots = kReceivedWarps * 32;
template <int kBlocks>
__global__ void __cluster_dims__(kReceivedCtas, 1, 1) __launch_bounds__(kReceivedWarps * 32, kBlocks > 4 ? 1 : 2) q4_received_again_kernel(const __grid_constant__ Q4Attend p) {
    namespace cg = cooperative_groups;
    constexpr uint32_t kTile = kBlocks * 64;                            // quads of eight rows
    extern __shared__ __align__(16) uint4 tiles[];                      // [kReceivedStages][kTile]
    __shared__ float share[kReceivedSlots];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = lane & 3u, rank = cluster.block_rank(), h = blockIdx.z;
    const uint32_t rows = p.tokens * p.group, row_tiles = (rows + 7) / 8, cta_slot = blockIdx.y * kReceivedSlots, slot0 = cta_slot + 32 * warp;
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;
    const uint32_t filled = filled_in, seen = filled + p.tokens;
    if (cta_slot >= seen) return;                                       // all of the cluster's CTAs
    // the slots' codes and scales; slots behind the last token are another's or nobody's: zeros
    uint32_t w[4][kBlocks];
    float d[4][kBlocks];
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        const uint32_t slot = slot0 + 8 * o + (lane >> 2);
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            w[o][g] = slot < seen ? __ldcg(reinterpret_cast<const uint32_t*>(p.cache.k_codes + q4_codes_at(h, slot, g, kBlocks, p.cache.slots)) + t) : 0u;
            d[o][g] = slot < seen ? __half2float(__ldcg(p.cache.k_scales + q4_scale_at(h, slot, g, kBlocks, p.cache.slots))) : 0.0f;
        }
    }
    // the row tiles that see the CTA's first slot, dealt out to the cluster's CTAs
    const uint32_t first_tile = cta_slot < filled ? 0u : (cta_slot - filled) * p.group / 8;
    const uint4* from = p.queries + static_cast<size_t>(h) * (p.padded / 8) * kTile;
    auto fetch = [&](uint32_t tile, int stage) {
        for (uint32_t i = threadIdx.x; i < kTile; i += kReceivedWarps * 32) copy16_or_zero(smem_u32(tiles + stage * kTile + i), from + static_cast<size_t>(tile) * kTile + i, true);
    };
    const uint32_t count = first_tile + rank < row_tiles ? (row_tiles - first_tile - rank + kReceivedCtas - 1) / kReceivedCtas : 0u;
    for (int s = 0; s < kReceivedStages - 1; ++s) {
        if (static_cast<uint32_t>(s) < count) fetch(first_tile + rank + s * kReceivedCtas, s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum[4] = {};
    for (uint32_t i = 0; i < count; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kReceivedStages - 2) : "memory");
        __syncthreads();
        if (i + kReceivedStages - 1 < count) fetch(first_tile + rank + (i + kReceivedStages - 1) * kReceivedCtas, (i + kReceivedStages - 1) % kReceivedStages);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t row0 = (first_tile + rank + i * kReceivedCtas) * 8;
        if (slot0 > filled + min(row0 + 7, rows - 1) / p.group) continue;          // none of the tile's rows sees any of the warp's slots
        const uint4* rows_at = tiles + i % kReceivedStages * kTile + lane;
        float whole[2], factor[2];
        uint32_t last_seen[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t row = row0 + 2 * t + c;
            const size_t at = static_cast<size_t>(h) * rows + min(row, rows - 1);
            whole[c] = row < rows ? __ldcg(p.stats + at) : INFINITY;
            factor[c] = __ldcg(p.factors + static_cast<size_t>(h) * p.padded + min(row, rows - 1));
            last_seen[c] = filled + min(row, rows - 1) / p.group;
        }
        float s[2][4] = {};
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            const uint4 upper = rows_at[g * 64], lower = rows_at[g * 64 + 32];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t u = w[2 * half][g], v = w[2 * half + 1][g], x = u >> 8, y = v >> 8;
                const uint32_t even[4] = {signed_low(u), signed_low(v), signed_high(u), signed_high(v)};
                const uint32_t odd[4] = {signed_low(x), signed_low(y), signed_high(x), signed_high(y)};
                float c[4];
                mma_f16(c, even, lower.x, lower.y, zero);
                mma_f16(c, odd, lower.z, lower.w, c);
                mma_f16(c, even, upper.x, upper.y, c);
                mma_f16(c, odd, upper.z, upper.w, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[half][j] = fmaf(d[2 * half + j / 2][g], c[j], s[half][j]);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (slot0 + 16 * half + 8 * (j / 2) + (lane >> 2) <= last_seen[j & 1]) sum[2 * half + j / 2] += exp2_fast(s[half][j] * factor[j & 1] - whole[j & 1]);
    }
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        sum[o] += __shfl_xor_sync(0xffffffffu, sum[o], 1);
        sum[o] += __shfl_xor_sync(0xffffffffu, sum[o], 2);
        if (t == 0) share[32 * warp + 8 * o + (lane >> 2)] = sum[o];
    }
    cluster.sync();
    const uint32_t slot = cta_slot + threadIdx.x;
    if (rank == 0 && slot < seen) {
        float x = 0.0f;
        for (uint32_t r = 0; r < kReceivedCtas; ++r) x += cluster.map_shared_rank(share, r)[threadIdx.x];
        const size_t at = static_cast<size_t>(h) * p.cache.slots + slot;
        p.weight_out[at] = x + (slot < filled ? p.weight_in[at] : 0.0f);
    }
    cluster.sync();
}

}  // namespace zk
