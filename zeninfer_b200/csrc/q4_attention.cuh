// Grouped-query attention over a cache held in 4 bits (q4_cache.cuh): one kernel for a step, a block of drafted tokens and a prompt.
//
// out_r = sum_j p_rj v_j, p_rj = exp(s_rj - m_r) / l_r, s_rj = scale q_r . k_j.  A cached value is d_jb (c - 8) with one scale d per slot j and block b of 32
// dimensions, so   q_r . k_j = sum_b d_jb sum_{i in b} q_ri (c_ji - 8)   and   out_r = sum_j (p_rj d_jb) (c_ji - 8):
// both are products with codes, which f16 holds exactly.  The other factor, q_ri or p_rj d_jb, is an fp32 number that enters as two f16 numbers, 22 bits;
// the matrix instructions (mma.sync m16n8k16 with fp32 sums, a block is K = 32) add the products, and d_jb multiplies a block's sum in fp32.  Nothing is
// rounded to fewer than 22 bits, and the error is that of fp32 arithmetic.
//   scores   A = codes [16 slots][16 dimensions], taken from the packed word by one AND each: the low and the high nibble are the f16 subnormals
//            code * 2^-24 and code * 2^-20 (the q beside the high ones is 2^-4 as large); the sums begin at -8 sum q
//   output   A = codes^T [16 dimensions][16 slots], from the transposing ldmatrix, as c - 8 (an OR with 1024's exponent and a subtraction): sums that begin
//            at an offset of 8 sum p would lose what the average of many values leaves
// The scores come out slot by row and the weights go in row by slot: movmatrix turns 8 x 8 of them.  Weights are scaled by a power of two so
// that the largest |d| seen so far, times a weight of 1, is 2^14: both digits stay in f16's normal range over 2^28.
//
// A warp works for itself: rows of queries (kRows of them) against tiles of 32 slots, which lane 0 fetches by bulk copies into the warp's own
// ring; the softmax is the running-maximum form.  The warps of a CTA take different rows or different tiles (row_warps), CTAs take
// different rows, runs of slots (gridDim.x) and kv heads; what several warps have of one row is merged in shared memory, what several
// CTAs have by a second launch.
#pragma once
#include "q4_cache.cuh"

namespace zk {

constexpr uint32_t kQ4Tile = 32;             // slots of a tile
constexpr int kQ4Stages = 3;                 // tiles of a warp's ring

// How a warp's rows lie on the eight columns of a product.
enum Q4Columns : int {
    kQ4Digits = 0,       // four rows, a column a digit: half the products of the next for up to four rows (a step of a model with groups of four)
    kQ4Rows8 = 1,        // eight rows, the digits one after the other
    kQ4Rows16 = 2        // sixteen rows: the unpacked codes serve two products
};
__host__ __device__ constexpr int q4_rows(int columns) { return columns == kQ4Digits ? 4 : columns == kQ4Rows8 ? 8 : 16; }
__host__ __device__ constexpr int q4_warps(int columns) { return columns == kQ4Digits ? 8 : 4; }

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
    uint4* queries;            // workspace [kv_heads][row tiles of eight][Q4Query::kQuads][32 lanes]: the rows as the products take them, or null
    uint32_t tokens, heads, group;      // group = heads / kv_heads; a kv head has tokens * group rows, row = token * group + head of the group
    uint32_t splits, row_warps;
    size_t q_ld;
    float scale;
    int* error_word;
};

// The runs of slots the CTAs of a row take: the same arithmetic where they are merged.
struct Q4Runs {
    uint32_t tiles, per, active;
};
__device__ __forceinline__ Q4Runs q4_runs(uint32_t slots_seen, uint32_t splits, uint32_t key_warps) {
    Q4Runs r;
    r.tiles = (slots_seen + kQ4Tile - 1) / kQ4Tile;
    r.per = max((r.tiles + splits - 1) / splits, key_warps);
    r.active = (r.tiles + r.per - 1) / r.per;
    return r;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x2(uint32_t (&r)[2], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t (&r)[2], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(address) : "memory");
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
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// A slot's scales.
template <int kBlocks>
__device__ __forceinline__ void load_scales(float (&d)[kBlocks], const __half* s) {
    if constexpr (kBlocks % 2 == 0) {
#pragma unroll
        for (int b = 0; b < kBlocks; b += 2) {
            const float2 two = __half22float2(*reinterpret_cast<const __half2*>(s + b));
            d[b] = two.x;
            d[b + 1] = two.y;
        }
    } else {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) d[b] = __half2float(s[b]);
    }
}

// Rows of queries as the product's second operand, and what their scores are multiplied by.
template <int kBlocks, int kColumns>
struct Q4Query {
    static constexpr int kTiles = kColumns == kQ4Rows16 ? 2 : 1, kDigitSteps = kColumns == kQ4Digits ? 1 : 2;
    uint32_t b[kTiles][kBlocks][kDigitSteps][4];      // [..][digit][step 0: low, high nibbles; step 1: low, high]
    float start[kTiles][kBlocks][2];                  // -8 sum q of the lane's two columns, in the products' units
    float factor[kTiles][2];                          // scale * log2(e) / the products' units, of the lane's two columns' rows

    // A tile of eight rows as quads of words, a lane's own: kept by one kernel, taken by another.
    static constexpr int kQuads = (kBlocks * 10 + 2 + 3) / 4;
    __device__ __forceinline__ void keep(uint4* to, int n, uint32_t lane) const {
        uint32_t w[4 * kQuads];
#pragma unroll
        for (int i = 0; i < 4 * kQuads; ++i) w[i] = i < 8 * kBlocks ? b[n][i / 8][i / 4 % kDigitSteps][i % 4] : i < 10 * kBlocks ? __float_as_uint(start[n][(i - 8 * kBlocks) / 2][i % 2]) : i < 10 * kBlocks + 2 ? __float_as_uint(factor[n][i % 2]) : 0u;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) to[i * 32 + lane] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __device__ __forceinline__ void take(const uint4* from, uint32_t lane) {
        uint32_t w[4 * kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const uint4 four = from[i * 32 + lane];
            w[4 * i] = four.x; w[4 * i + 1] = four.y; w[4 * i + 2] = four.z; w[4 * i + 3] = four.w;
        }
#pragma unroll
        for (int i = 0; i < 10 * kBlocks + 2; ++i) {
            if (i < 8 * kBlocks) b[0][i / 8][i / 4 % kDigitSteps][i % 4] = w[i];
            else if (i < 10 * kBlocks) start[0][(i - 8 * kBlocks) / 2][i % 2] = __uint_as_float(w[i]);
            else factor[0][i % 2] = __uint_as_float(w[i]);
        }
    }

    // rows: fp32 [..][kBlocks * 32] in shared memory, the warp's first; count: how many are real
    __device__ __forceinline__ void load(const float* rows, uint32_t count, uint32_t pitch, float scale, uint32_t lane) {
        const uint32_t column = lane >> 2, t = lane & 3u;
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            const uint32_t row = kColumns == kQ4Digits ? column >> 1 : 8 * n + column;
            float4 low[kBlocks], high[kBlocks];
            float top = 0.0f;
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
                low[g] = high[g] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (row < count) {
                    low[g] = *reinterpret_cast<const float4*>(rows + row * pitch + g * 32 + 4 * t);
                    high[g] = *reinterpret_cast<const float4*>(rows + row * pitch + g * 32 + 16 + 4 * t);
                }
                for (float x : {low[g].x, low[g].y, low[g].z, low[g].w, high[g].x, high[g].y, high[g].z, high[g].w}) top = fmaxf(top, fabsf(x));
            }
            uint32_t size = __float_as_uint(top);
            size = max(size, __shfl_xor_sync(0xffffffffu, size, 1));
            size = max(size, __shfl_xor_sync(0xffffffffu, size, 2));
            // the row times a power of two has its largest value in [2^13, 2^14)
            const int e = max(static_cast<int>(size >> 23) - 127, -114);
            const float up = power_of_two(13 - e);
            const float mine = ldexpf(scale * 1.4426950408889634f, 24 + e - 13);
            const bool second = kColumns == kQ4Digits && (column & 1u);          // this column is the lower digit
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
                float sum = 0.0f;
                auto digits = [&](int step, int part, float x, float y, float unit) {
                    x *= up;
                    y *= up;
                    const float xh = upper_digit(x), yh = upper_digit(y);
                    const uint32_t first_digit = pack_f16(xh * unit, yh * unit), other = pack_f16((x - xh) * unit, (y - yh) * unit);
                    if (kColumns == kQ4Digits) b[n][g][0][2 * step + part] = second ? other : first_digit;
                    else { b[n][g][0][2 * step + part] = first_digit; b[n][g][kDigitSteps - 1][2 * step + part] = other; }
                    // what the digits as rounded stand for
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&first_digit)), l = __half22float2(*reinterpret_cast<const __half2*>(&other));
                    const float of_first = (h.x + h.y) / unit, of_other = (l.x + l.y) / unit;
                    sum += kColumns == kQ4Digits ? (second ? of_other : of_first) : of_first + of_other;
                };
                digits(0, 0, low[g].x, low[g].z, 1.0f);
                digits(0, 1, high[g].x, high[g].z, 0.0625f);
                digits(1, 0, low[g].y, low[g].w, 1.0f);
                digits(1, 1, high[g].y, high[g].w, 0.0625f);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= -8.0f * 5.9604644775390625e-8f;                           // 2^-24
                start[n][g][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                start[n][g][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
            factor[n][0] = __shfl_sync(0xffffffffu, mine, 8 * t);
            factor[n][1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
        }
    }

    // Scores, in units of log 2, of 16 slots whose codes begin at `codes` (two octets) with the lane's two slots' scales: s[n][0..1] are
    // slot lane / 4 and the lane's two columns, s[n][2..3] slot lane / 4 + 8.  kQ4Digits: s[0][0] and s[0][2] are row lane % 4, the others nothing.
    __device__ __forceinline__ void scores(float (&s)[kTiles][4], uint32_t codes, const float (&da)[kBlocks], const float (&db)[kBlocks], uint32_t lane) const {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
        const uint32_t at = codes + ((lane >> 3) & 1u) * kBlocks * 128 + (lane & 7u) * 16;
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            uint32_t w[2];
            ldmatrix_x2(w, at + g * 128);
            const uint32_t x = w[0] >> 8, y = w[1] >> 8;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float c[4] = {start[n][g][0], start[n][g][1], start[n][g][0], start[n][g][1]};
#pragma unroll
                for (int d = 0; d < kDigitSteps; ++d) {
                    mma_f16(c, w[0] & 0x000f000fu, w[1] & 0x000f000fu, w[0] & 0x00f000f0u, w[1] & 0x00f000f0u, b[n][g][d][0], b[n][g][d][1]);
                    mma_f16(c, x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, b[n][g][d][2], b[n][g][d][3]);
                }
                if (kColumns == kQ4Digits) {
                    s[n][0] = fmaf(da[g], c[0] + c[1], s[n][0]);
                    s[n][2] = fmaf(db[g], c[2] + c[3], s[n][2]);
                } else {
                    s[n][0] = fmaf(da[g], c[0], s[n][0]);
                    s[n][1] = fmaf(da[g], c[1], s[n][1]);
                    s[n][2] = fmaf(db[g], c[2], s[n][2]);
                    s[n][3] = fmaf(db[g], c[3], s[n][3]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] *= factor[n][i & 1];
    }
};

template <int kBlocks>
__host__ __device__ constexpr uint32_t q4_stage_bytes() { return kQ4Tile * kBlocks * 36; }         // 16 + 16 code bytes and 2 + 2 of scales a slot and block
__host__ __device__ constexpr uint32_t q4_query_pitch(int blocks) { return blocks * 32 + 4; }      // floats; rows four banks apart
// Dynamic shared memory of q4_attend_kernel: the warps' rings, then the rows of queries.
template <int kBlocks, int kColumns>
__host__ __device__ constexpr uint32_t q4_attend_smem(uint32_t row_warps) {
    return q4_warps(kColumns) * kQ4Stages * q4_stage_bytes<kBlocks>() + row_warps * q4_rows(kColumns) * q4_query_pitch(kBlocks) * 4;
}

// grid = (splits, CTAs for the rows, kv_heads); the rows that see most slots come first.
template <int kBlocks, int kColumns>
__global__ void __launch_bounds__(q4_warps(kColumns) * 32) q4_attend_kernel(const __grid_constant__ Q4Attend p) {
    constexpr int kWarps = q4_warps(kColumns), kRows = q4_rows(kColumns), kDim = kBlocks * 32;
    using Query = Q4Query<kBlocks, kColumns>;
    constexpr int kTiles = Query::kTiles;
    constexpr uint32_t kStage = q4_stage_bytes<kBlocks>(), kCodes = kQ4Tile * kBlocks * 16, kScales = kQ4Tile * kBlocks * 2;
    extern __shared__ __align__(128) uint8_t q4_smem[];
    __shared__ uint64_t landed[kWarps][kQ4Stages];
    __shared__ float row_max[kWarps][16], row_sum[kWarps][16], row_unit[kWarps];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = lane & 3u, h = blockIdx.z;
    const uint32_t key_warps = kWarps / p.row_warps, row_warp = warp % p.row_warps, key_warp = warp / p.row_warps;
    const uint32_t rows = p.tokens * p.group, cta_rows = p.row_warps * kRows;
    const uint32_t cta_first = (gridDim.y - 1 - blockIdx.y) * cta_rows, first = cta_first + row_warp * kRows;
    float* queries = reinterpret_cast<float*>(q4_smem + kWarps * kQ4Stages * kStage);
    constexpr uint32_t kPitch = q4_query_pitch(kBlocks);
    if (lane == 0)
        for (int s = 0; s < kQ4Stages; ++s) mbar_init(&landed[warp][s], 1);
    if (lane == 0) mbar_fence_init();
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;      // the append has said so
    const uint32_t filled = filled_in, real_rows = min(cta_rows, rows - cta_first);
    const uint32_t seen = filled + (cta_first + real_rows - 1) / p.group + 1;           // slots of the CTA's last token
    const Q4Runs runs = q4_runs(seen, p.splits, key_warps);
    const uint32_t begin = blockIdx.x * runs.per, end = min(runs.tiles, begin + runs.per);
    if (begin >= end) return;                                                            // nobody counts on this run
    __syncwarp();

    // lane 0 keeps the ring filled
    uint8_t* ring = q4_smem + warp * kQ4Stages * kStage;
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
    const uint32_t mine = begin + key_warp < end ? (end - begin - key_warp + key_warps - 1) / key_warps : 0u;      // tiles of this warp
    if (lane == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");       // the append's stores come before the copies
        for (uint32_t i = 0; i < min(mine, static_cast<uint32_t>(kQ4Stages)); ++i) fetch(begin + key_warp + i * key_warps, i);
    }
    // the CTA's rows, rotated
    for (uint32_t i = threadIdx.x; i < real_rows * kDim; i += kWarps * 32) {
        const uint32_t r = i / kDim, e = i % kDim, row = cta_first + r, token = row / p.group, head = h * p.group + row % p.group;
        queries[r * kPitch + e] = q4_rotated(p.q + token * p.q_ld + static_cast<size_t>(head) * kDim, e, p.turn, static_cast<size_t>(position) + token);
    }
    __syncthreads();
    Query query;
    query.load(queries + row_warp * kRows * kPitch, first < rows ? min(static_cast<uint32_t>(kRows), rows - first) : 0u, kPitch, p.scale, lane);
    if constexpr (kColumns != kQ4Digits) {
        if (p.queries && key_warp == 0 && blockIdx.x == 0)
            for (int n = 0; n < kTiles; ++n)
                if (first + 8 * n < rows) query.keep(p.queries + (static_cast<size_t>(h) * ((rows + 7) / 8) + first / 8 + n) * Query::kQuads * 32, n, lane);
    }
    // the last slot each of the lane's rows sees
    uint32_t last_seen[kTiles][2], least = 0xffffffffu;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t row = first + (kColumns == kQ4Digits ? t : 8 * n + 2 * t + c);
            last_seen[n][c] = filled + min(row, rows - 1) / p.group;
            least = min(least, last_seen[n][c]);
        }
    least = __reduce_min_sync(0xffffffffu, least);

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
    int unit = -32;                       // the weights' power of two is 14 - unit
    bool failed = false;
    for (uint32_t i = 0; i < mine; ++i) {
        const int stage = i % kQ4Stages;
        if (!__all_sync(0xffffffffu, mbar_wait(&landed[warp][stage], (i / kQ4Stages) & 1u))) {
            // the copies that are under way land (or are given up) before the ring is used for anything else
            if (lane == 0) {
                atomicExch(p.error_word, kErrFullWaitTimeout);
                for (uint32_t j = i; j < min(mine, i + kQ4Stages); ++j) mbar_wait(&landed[warp][j % kQ4Stages], (j / kQ4Stages) & 1u);
            }
            __syncwarp();
            failed = true;
            break;
        }
        const uint32_t tile = begin + key_warp + i * key_warps, slot0 = tile * kQ4Tile;
        const uint32_t k_codes = smem_u32(ring + stage * kStage), v_codes = k_codes + kCodes;
        const __half* k_scales = reinterpret_cast<const __half*>(ring + stage * kStage + 2 * kCodes);
        const __half* v_scales = k_scales + kQ4Tile * kBlocks;
        const bool whole = slot0 + kQ4Tile - 1 <= least;           // every row sees every slot of the tile
        float s[2][kTiles][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t a = 16 * half + (lane >> 2), b = a + 8;
            float da[kBlocks], db[kBlocks];
            load_scales<kBlocks>(da, k_scales + a * kBlocks);
            load_scales<kBlocks>(db, k_scales + b * kBlocks);
            query.scores(s[half], k_codes + half * 2 * kBlocks * 128, da, db, lane);
            if (!whole) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (slot0 + a > last_seen[n][c]) s[half][n][c] = -INFINITY;
                        if (slot0 + b > last_seen[n][c]) s[half][n][2 + c] = -INFINITY;
                    }
            }
            if (p.scores) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int c = 0; c < (kColumns == kQ4Digits ? 1 : 2); ++c) {
                        const uint32_t row = first + (kColumns == kQ4Digits ? t : 8 * n + 2 * t + c);
                        if (row >= rows) continue;
                        float* to = p.scores + (static_cast<size_t>(h) * rows + row) * p.cache.slots + slot0;
                        to[a] = s[half][n][c];
                        to[b] = s[half][n][2 + c];
                    }
            }
        }
        // the largest scale of a value that any row sees, as a power of two
        uint32_t top = 0;
#pragma unroll
        for (int g = 0; g < kBlocks; ++g)
            if (slot0 + lane < seen) top = max(top, static_cast<uint32_t>(__half_as_ushort(v_scales[lane * kBlocks + g])) & 0x7fffu);
        top = __reduce_max_sync(0xffffffffu, top);
        const int new_unit = max(unit, min(static_cast<int>(top >> 10), 30) - 14);
        // the new maxima
        float corr[kTiles][2];
        bool moved = new_unit != unit;
        const float of_unit = unit == -32 ? 0.0f : power_of_two(unit - new_unit);
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = fmaxf(fmaxf(s[0][n][c], s[0][n][2 + c]), fmaxf(s[1][n][c], s[1][n][2 + c]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                const float next = fmaxf(m[n][c], x);
                moved |= next != m[n][c];
                corr[n][c] = m[n][c] == -INFINITY ? 0.0f : exp2_fast(m[n][c] - next);
                m[n][c] = next;
                if (kColumns == kQ4Digits) { corr[n][1] = corr[n][0]; m[n][1] = m[n][0]; break; }
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    l[n][c] *= corr[n][c];
                    const float by = corr[n][c] * of_unit;
#pragma unroll
                    for (int j = 0; j < 2 * kBlocks; ++j) {
                        acc[n][j][c] *= by;
                        acc[n][j][2 + c] *= by;
                    }
                }
            unit = new_unit;
        }
        const float up = power_of_two(14 - unit);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t a = 16 * half + (lane >> 2), b = a + 8;
            float w[kTiles][4];
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = s[half][n][j], top_of = m[n][j & 1];
                    w[n][j] = x == -INFINITY ? 0.0f : exp2_fast(x - top_of);
                    l[n][j & 1] += w[n][j];
                    if (kColumns == kQ4Digits) { if (j & 1) w[n][j] = 0.0f; }
                }
            float da[kBlocks], db[kBlocks];
            load_scales<kBlocks>(da, v_scales + a * kBlocks);
            load_scales<kBlocks>(db, v_scales + b * kBlocks);
            const uint32_t at = v_codes + (2 * half + ((lane >> 3) & 1u)) * kBlocks * 128 + (lane & 7u) * 16;
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
                uint32_t v[2];
                ldmatrix_x2_trans(v, at + g * 128);
                const uint32_t x = v[0] >> 8, y = v[1] >> 8;
                const uint32_t a00 = signed_low(v[0]), a01 = signed_high(v[0]), a02 = signed_low(v[1]), a03 = signed_high(v[1]);
                const uint32_t a10 = signed_low(x), a11 = signed_high(x), a12 = signed_low(y), a13 = signed_high(y);
                const float ua = da[g] * up, ub = db[g] * up;
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    // a slot that is not seen may hold anything
                    auto weight = [&](int j, float u) { return !whole && slot0 + (j < 2 ? a : b) > last_seen[n][j & 1] ? 0.0f : w[n][j] * u; };
                    if (kColumns == kQ4Digits) {
                        const float wa = weight(0, ua), wb = weight(2, ub), ha = upper_digit(wa), hb = upper_digit(wb);
                        const uint32_t b0 = transposed(pack_f16(ha, wa - ha)), b1 = transposed(pack_f16(hb, wb - hb));
                        mma_f16(acc[n][2 * g], a00, a01, a02, a03, b0, b1);
                        mma_f16(acc[n][2 * g + 1], a10, a11, a12, a13, b0, b1);
                    } else {
                        const float w0 = weight(0, ua), w1 = weight(1, ua), w2 = weight(2, ub), w3 = weight(3, ub);
                        const float h0 = upper_digit(w0), h1 = upper_digit(w1), h2 = upper_digit(w2), h3 = upper_digit(w3);
                        const uint32_t b0 = transposed(pack_f16(h0, h1)), b1 = transposed(pack_f16(h2, h3));
                        const uint32_t c0 = transposed(pack_f16(w0 - h0, w1 - h1)), c1 = transposed(pack_f16(w2 - h2, w3 - h3));
                        mma_f16(acc[n][2 * g], a00, a01, a02, a03, b0, b1);
                        mma_f16(acc[n][2 * g + 1], a10, a11, a12, a13, b0, b1);
                        mma_f16(acc[n][2 * g], a00, a01, a02, a03, c0, c1);
                        mma_f16(acc[n][2 * g + 1], a10, a11, a12, a13, c0, c1);
                    }
                }
            }
        }
        __syncwarp();                       // everybody is done with the stage
        if (lane == 0 && i + kQ4Stages < mine) fetch(tile + kQ4Stages * key_warps, stage);
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
            const uint32_t r = kColumns == kQ4Digits ? t : 8 * n + 2 * t + c;
            if (lane < 4 && !(kColumns == kQ4Digits && c)) { row_max[warp][r] = m[n][c]; row_sum[warp][r] = failed ? NAN : l[n][c]; }
        }
#pragma unroll
        for (int g = 0; g < kBlocks; ++g)
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const uint32_t e = g * 32 + 2 * (lane >> 2) + odd;
                const float (&c)[4] = acc[n][2 * g + odd];
                if (kColumns == kQ4Digits) {
                    sums[t * kDim + e] = c[0] + c[1];
                    sums[t * kDim + e + 16] = c[2] + c[3];
                } else {
                    sums[(8 * n + 2 * t) * kDim + e] = c[0];
                    sums[(8 * n + 2 * t + 1) * kDim + e] = c[1];
                    sums[(8 * n + 2 * t) * kDim + e + 16] = c[2];
                    sums[(8 * n + 2 * t + 1) * kDim + e + 16] = c[3];
                }
            }
    }
    if (lane == 0) row_unit[warp] = unit == -32 ? 0.0f : power_of_two(unit - 14);
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
            const float share = reinterpret_cast<const float*>(q4_smem + w * kQ4Stages * kStage)[at * kDim + e];
            sum += by * row_sum[w][at];
            o += its == -INFINITY ? 0.0f : by * row_unit[w] * share;
        }
        if (alone) {
            const uint32_t token = row / p.group, head = h * p.group + row % p.group;
            p.out[(static_cast<size_t>(token) * p.heads + head) * kDim + e] = o / sum;
            if (e == 0) {
                if (!(sum > 0.0f) || !(sum < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
                if (p.stats) p.stats[static_cast<size_t>(h) * rows + row] = top + log2f(sum);
            }
        } else {
            const size_t part = (static_cast<size_t>(h) * p.splits + blockIdx.x) * rows + row;
            p.part_out[part * kDim + e] = o;
            if (e == 0) { p.part_stats[2 * part] = top; p.part_stats[2 * part + 1] = sum; }
        }
    }
}

// The runs of a row put together: grid = (rows, kv_heads), a thread a dimension.  Rows are those of one CTA of the launch before
// (cta_rows of them), whose arithmetic gives the number of runs.
__global__ void __launch_bounds__(256) q4_join_kernel(const __grid_constant__ Q4Attend p, uint32_t cta_rows, uint32_t key_warps) {
    const uint32_t row = blockIdx.x, h = blockIdx.y, rows = p.tokens * p.group, dim = p.cache.blocks * 32;
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;
    const uint32_t last_row = min(rows, (row / cta_rows + 1) * cta_rows) - 1;
    const uint32_t active = q4_runs(static_cast<uint32_t>(filled) + last_row / p.group + 1, p.splits, key_warps).active;
    const size_t first = static_cast<size_t>(h) * p.splits * rows + row;
    // every warp has all the runs' maxima and sums, a run a lane, and the runs' outputs are asked for eight at a time: two round trips
    const uint32_t lane = threadIdx.x & 31u;
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t s = lane; s < active; s += 32) top = fmaxf(top, __ldcg(p.part_stats + 2 * (first + static_cast<size_t>(s) * rows)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float o = 0.0f;
    for (uint32_t s0 = 0; s0 < active; s0 += 32) {
        float by = 0.0f;
        if (s0 + lane < active) {
            const float2 its = __ldcg(reinterpret_cast<const float2*>(p.part_stats) + first + static_cast<size_t>(s0 + lane) * rows);
            by = its.x == -INFINITY ? 0.0f : exp2_fast(its.x - top);
            sum += by * its.y;
        }
        const uint32_t count = min(32u, active - s0);
        const float* from = p.part_out + (first + static_cast<size_t>(s0) * rows) * dim + threadIdx.x;
        const size_t step = static_cast<size_t>(rows) * dim;
#pragma unroll 8
        for (uint32_t s = 0; s < count; ++s) o += __shfl_sync(0xffffffffu, by, s) * __ldcg(from + s * step);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const uint32_t token = row / p.group, head = h * p.group + row % p.group;
    p.out[(static_cast<size_t>(token) * p.heads + head) * dim + threadIdx.x] = o / sum;
    if (threadIdx.x == 0) {
        if (!(sum > 0.0f) || !(sum < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
        if (p.stats) p.stats[static_cast<size_t>(h) * rows + row] = top + log2f(sum);
    }
}

// What the slots received, from kept scores: a thread a slot.
__global__ void __launch_bounds__(256) q4_received_kernel(const __grid_constant__ Q4Attend p) {
    const uint32_t slot = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, rows = p.tokens * p.group;
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions) || slot >= static_cast<uint32_t>(filled) + p.tokens) return;
    float sum = 0.0f;
    for (uint32_t r = slot < static_cast<uint32_t>(filled) ? 0u : (slot - filled) * p.group; r < rows; ++r) {
        const size_t row = static_cast<size_t>(h) * rows + r;
        sum += exp2_fast(__ldcg(p.scores + row * p.cache.slots + slot) - __ldcg(p.stats + row));
    }
    const size_t at = static_cast<size_t>(h) * p.cache.slots + slot;
    p.weight_out[at] = sum + (slot < static_cast<uint32_t>(filled) ? p.weight_in[at] : 0.0f);
}

// What the slots received in a block of many rows: the scores are formed once more, now that the rows' sums are known.  A warp takes 32
// slots, its unpacked codes in registers; tiles of eight rows, as q4_attend_kernel left them, pass through shared memory for the CTA's
// eight warps.  A cluster's eight CTAs share the rows, and their sums meet in rank 0.  grid = (8, runs of 256 slots, kv_heads).
constexpr int kReceivedWarps = 8, kReceivedCtas = 8, kReceivedStages = 3;
constexpr uint32_t kReceivedSlots = kReceivedWarps * 32;
template <int kBlocks>
__global__ void __cluster_dims__(kReceivedCtas, 1, 1) __launch_bounds__(kReceivedWarps * 32) q4_received_again_kernel(const __grid_constant__ Q4Attend p) {
    namespace cg = cooperative_groups;
    using Query = Q4Query<kBlocks, kQ4Rows8>;
    constexpr int kQuads = Query::kQuads;
    extern __shared__ __align__(16) uint4 tiles[];                      // [kReceivedStages][kQuads * 32]
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
    // the slots' codes, unpacked, and scales; slots behind the last token are another's or nobody's: zeros
    uint32_t w[2][kBlocks][2];
    float da[2][kBlocks], db[2][kBlocks];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t a = slot0 + 16 * half + (lane >> 2);
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t slot = a + 8 * e;
                const bool real = slot < seen;
                w[half][g][e] = real ? __ldcg(reinterpret_cast<const uint32_t*>(p.cache.k_codes + q4_codes_at(h, slot, g, kBlocks, p.cache.slots)) + t) : 0u;
                const float d = real ? __half2float(__ldcg(p.cache.k_scales + q4_scale_at(h, slot, g, kBlocks, p.cache.slots))) : 0.0f;
                if (e) db[half][g] = d; else da[half][g] = d;
            }
        }
    }
    // the row tiles that see the CTA's first slot, dealt out to the cluster's CTAs
    const uint32_t first_tile = cta_slot < filled ? 0u : (cta_slot - filled) * p.group / 8;
    const uint4* from = p.queries + static_cast<size_t>(h) * row_tiles * kQuads * 32;
    auto fetch = [&](uint32_t tile, int stage) {
        for (uint32_t i = threadIdx.x; i < kQuads * 32; i += kReceivedWarps * 32)
            copy16_or_zero(smem_u32(tiles + stage * kQuads * 32 + i), from + static_cast<size_t>(tile) * kQuads * 32 + i, true);
    };
    const uint32_t count = first_tile + rank < row_tiles ? (row_tiles - first_tile - rank + kReceivedCtas - 1) / kReceivedCtas : 0u;
    for (int s = 0; s < kReceivedStages - 1; ++s) {
        if (static_cast<uint32_t>(s) < count) fetch(first_tile + rank + s * kReceivedCtas, s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    float sum[2][2] = {};
    for (uint32_t i = 0; i < count; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kReceivedStages - 2) : "memory");
        __syncthreads();
        if (i + kReceivedStages - 1 < count) fetch(first_tile + rank + (i + kReceivedStages - 1) * kReceivedCtas, (i + kReceivedStages - 1) % kReceivedStages);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t row0 = (first_tile + rank + i * kReceivedCtas) * 8;
        if (slot0 > filled + min(row0 + 7, rows - 1) / p.group) continue;          // none of the tile's rows sees any of the warp's slots
        Query query;
        query.take(tiles + i % kReceivedStages * kQuads * 32, lane);
        float whole[2];
        uint32_t last_seen[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t row = row0 + 2 * t + c;
            whole[c] = row < rows ? __ldcg(p.stats + static_cast<size_t>(h) * rows + row) : INFINITY;
            last_seen[c] = filled + min(row, rows - 1) / p.group;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float s[4] = {};
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
                float c[4] = {query.start[0][g][0], query.start[0][g][1], query.start[0][g][0], query.start[0][g][1]};
                const uint32_t u = w[half][g][0], v = w[half][g][1], x = u >> 8, y = v >> 8;
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    mma_f16(c, u & 0x000f000fu, v & 0x000f000fu, u & 0x00f000f0u, v & 0x00f000f0u, query.b[0][g][d][0], query.b[0][g][d][1]);
                    mma_f16(c, x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, query.b[0][g][d][2], query.b[0][g][d][3]);
                }
                s[0] = fmaf(da[half][g], c[0], s[0]);
                s[1] = fmaf(da[half][g], c[1], s[1]);
                s[2] = fmaf(db[half][g], c[2], s[2]);
                s[3] = fmaf(db[half][g], c[3], s[3]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t slot = slot0 + 16 * half + 8 * (j / 2) + (lane >> 2);
                if (slot <= last_seen[j & 1]) sum[half][j / 2] += exp2_fast(s[j] * query.factor[0][j & 1] - whole[j & 1]);
            }
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = sum[half][e];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            if (t == 0) share[32 * warp + 16 * half + 8 * e + (lane >> 2)] = x;
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
