// A key/value cache held in 4 bits: its layout, the quantisation of new keys and values, and the eviction of slots.
//
// 32 consecutive values of a head are a block, as in Q4_0: an f16 scale d and codes 0 .. 15, value = d * (code - 8).  The codes of eight
// slots' equal blocks are 128 consecutive bytes ([slots / 8][blocks][8][16]): what a warp fetches as one 8 x 16-byte matrix has no bank
// conflicts, and a run of slots is one piece of memory that a bulk copy takes.
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "zk_ptx.cuh"

namespace zk {

constexpr uint32_t kQ4Block = 32, kQ4MaxBlocks = 8;      // values of a block; blocks of a head (head_dim <= 256)

struct Q4Cache {
    uint8_t* k_codes;
    uint8_t* v_codes;
    __half* k_scales;
    __half* v_scales;
    uint32_t kv_heads, blocks, slots;      // blocks = head_dim / 32
};

// Byte offset of a block's 16 code bytes, and index of its scale.
__host__ __device__ __forceinline__ size_t q4_codes_at(uint32_t kv_head, uint32_t slot, uint32_t block, uint32_t blocks, uint32_t slots) {
    return (((static_cast<size_t>(kv_head) * (slots >> 3) + (slot >> 3)) * blocks + block) * 8 + (slot & 7)) * 16;
}
__host__ __device__ __forceinline__ size_t q4_scale_at(uint32_t kv_head, uint32_t slot, uint32_t block, uint32_t blocks, uint32_t slots) {
    return (static_cast<size_t>(kv_head) * slots + slot) * blocks + block;
}

// Whether `tokens` slots behind *filled are in the cache, and the rows of the tables exist.
__device__ __forceinline__ bool q4_places_ok(int filled, int position, uint32_t tokens, uint32_t slots, uint32_t pairs, uint32_t positions) {
    return filled >= 0 && static_cast<uint64_t>(filled) + tokens <= slots && (!pairs || (position >= 0 && static_cast<uint64_t>(position) + tokens <= positions));
}

struct Q4Rotation {
    const float* cos_t;       // [positions][pairs]
    const float* sin_t;
    uint32_t pairs, positions;
    uint32_t adjacent;
};

// Dimension `e` of a head vector, to be rotated by the tables' row: what is asked for without knowing the row, and the rest.  Every product and
// sum is rounded on its own, so that a key turns out the same in every kernel that forms it.
struct Q4Raw {
    float mine, other;
};
__device__ __forceinline__ uint32_t q4_partner(uint32_t e, const Q4Rotation& r) { return r.adjacent ? e ^ 1u : e < r.pairs ? e + r.pairs : e - r.pairs; }
__device__ __forceinline__ Q4Raw q4_raw(const float* head, uint32_t e, const Q4Rotation& r) {
    return Q4Raw{__ldcg(head + e), e < 2 * r.pairs ? __ldcg(head + q4_partner(e, r)) : 0.0f};
}
__device__ __forceinline__ float q4_rotated(const Q4Raw& x, uint32_t e, const Q4Rotation& r, size_t row) {
    if (e >= 2 * r.pairs) return x.mine;
    const uint32_t pair = r.adjacent ? e >> 1 : e < r.pairs ? e : e - r.pairs;
    const bool low = r.adjacent ? !(e & 1u) : e < r.pairs;
    const float c = __ldg(r.cos_t + row * r.pairs + pair), s = __ldg(r.sin_t + row * r.pairs + pair);
    return low ? __fsub_rn(__fmul_rn(x.mine, c), __fmul_rn(x.other, s)) : __fadd_rn(__fmul_rn(x.other, s), __fmul_rn(x.mine, c));
}
__device__ __forceinline__ float q4_rotated(const float* head, uint32_t e, const Q4Rotation& r, size_t row) { return q4_rotated(q4_raw(head, e, r), e, r, row); }

// Eight dimensions of a head vector, rotated: at .. at + 3 and at + 16 .. at + 19.  Four at a time where the whole head turns and everything is aligned, else one by one; the
// operations are q4_rotated's.
__device__ __forceinline__ bool q4_rotates_fours(const float* q, size_t q_ld, uint32_t dim, const Q4Rotation& r) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(q) | (q_ld * 4) | (r.pairs ? reinterpret_cast<uintptr_t>(r.cos_t) | reinterpret_cast<uintptr_t>(r.sin_t) : 0);
    return all % 16 == 0 && (!r.pairs || 2 * r.pairs == dim);
}
// kTurn: 0 not at all, 1 adjacent pairs, 2 pairs a half apart; for those that go four at a time.
template <int kTurn>
__device__ __forceinline__ void q4_rotated_fours(float (&x)[8], const float* head, uint32_t at, const Q4Rotation& r, size_t row) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const uint32_t e = at + 16 * part;
        const float4 mine = __ldcg(reinterpret_cast<const float4*>(head + e));
        float* y = x + 4 * part;
        if constexpr (kTurn == 0) {
            y[0] = mine.x; y[1] = mine.y; y[2] = mine.z; y[3] = mine.w;
        } else if constexpr (kTurn == 1) {
            const float* const cos_t = r.cos_t + row * r.pairs + e / 2;
            const float* const sin_t = r.sin_t + row * r.pairs + e / 2;
            const float2 c = __ldg(reinterpret_cast<const float2*>(cos_t)), s = __ldg(reinterpret_cast<const float2*>(sin_t));
            y[0] = __fsub_rn(__fmul_rn(mine.x, c.x), __fmul_rn(mine.y, s.x)); y[1] = __fadd_rn(__fmul_rn(mine.x, s.x), __fmul_rn(mine.y, c.x));
            y[2] = __fsub_rn(__fmul_rn(mine.z, c.y), __fmul_rn(mine.w, s.y)); y[3] = __fadd_rn(__fmul_rn(mine.z, s.y), __fmul_rn(mine.w, c.y));
        } else {
            const bool low = e < r.pairs;
            const uint32_t pair = low ? e : e - r.pairs;
            const float4 its = __ldcg(reinterpret_cast<const float4*>(head + (low ? e + r.pairs : pair)));
            const float* const cos_t = r.cos_t + row * r.pairs + pair;
            const float* const sin_t = r.sin_t + row * r.pairs + pair;
            const float4 c = __ldg(reinterpret_cast<const float4*>(cos_t)), s = __ldg(reinterpret_cast<const float4*>(sin_t));
            auto turned = [&](float a, float b, float cc, float ss) { return low ? __fsub_rn(__fmul_rn(a, cc), __fmul_rn(b, ss)) : __fadd_rn(__fmul_rn(b, ss), __fmul_rn(a, cc)); };
            y[0] = turned(mine.x, its.x, c.x, s.x); y[1] = turned(mine.y, its.y, c.y, s.y); y[2] = turned(mine.z, its.z, c.z, s.z); y[3] = turned(mine.w, its.w, c.w, s.w);
        }
    }
}
__device__ __forceinline__ void q4_rotated_eight(float (&x)[8], const float* head, uint32_t at, const Q4Rotation& r, size_t row, bool fours) {
    if (!fours) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = q4_rotated(head, at + (e & 3) + (e >> 2) * 16, r, row);
    } else if (!r.pairs) {
        q4_rotated_fours<0>(x, head, at, r, row);
    } else if (r.adjacent) {
        q4_rotated_fours<1>(x, head, at, r, row);
    } else {
        q4_rotated_fours<2>(x, head, at, r, row);
    }
}

// The quantisation of a block: the scale is that of the first value of largest magnitude, `at`, and the code the integer
// nearest to x / d + 8.  The choice is exact: x / d >= c - 8.5 is x >= (c - 8.5) d for positive d, a product of five bits and eleven
// that fp32 holds, so the estimate by a rounded reciprocal, off by one at most, is put right by two comparisons.
__device__ __forceinline__ __half q4_scale_of(float at) {
    if ((__float_as_uint(at) & 0x7fffffffu) >= 0x7f800000u) return __ushort_as_half(static_cast<unsigned short>(0x7e00u));      // an infinity or a NaN among the values: the block reads as NaN
    return __float2half_rn(fminf(fmaxf(at * -0.125f, -65504.0f), 65504.0f));
}
// d: the scale as fp32, inverse: __frcp_rn(d)
__device__ __forceinline__ uint32_t q4_code_of(float x, float d, float inverse) {
    if (!(fabsf(d) > 0.0f)) return 8;      // zero, or NaN
    const float guess = fminf(fmaxf(floorf(fmaf(x, inverse, 8.5f)), -1.0f), 16.0f);
    auto reaches = [&](float c) { const float border = (c - 8.5f) * d; return d > 0.0f ? x >= border : x <= border; };
    float c = guess;
    if (!reaches(c)) c -= 1.0f;
    else if (reaches(c + 1.0f)) c += 1.0f;
    return static_cast<uint32_t>(fminf(fmaxf(c, 0.0f), 15.0f));
}

// A warp quantises a block, a value a lane: the scale, and the lane's code.
struct Q4Quantised {
    __half scale;
    uint32_t code;
};
__device__ __forceinline__ Q4Quantised q4_quantise(float x, uint32_t lane) {
    const uint32_t size = __float_as_uint(x) & 0x7fffffffu;
    const uint32_t top = __reduce_max_sync(0xffffffffu, size);
    Q4Quantised r;
    r.scale = q4_scale_of(__shfl_sync(0xffffffffu, x, __ffs(__ballot_sync(0xffffffffu, size == top)) - 1));
    const float d = __half2float(r.scale);
    r.code = q4_code_of(x, d, __frcp_rn(d));
    return r;
}

// ---- eviction ----------------------------------------------------------------------------------------------------------------
//
// A cluster of eight CTAs takes a kv head.  Up to kEvictSolo slots every CTA chooses for itself, for an exchange costs more than the work it saves; above, each
// has a run of the slots, each warp a run of the CTA's.  The weight of the last slot that stays is found by a radix select over order-preserving keys, three
// passes of 11, 11 and 10 bits.  In a cluster every CTA reads the others' sums of 32 bins, and then the bins of the one sum that has the border (distributed shared memory gives some ten
// bytes a clock: reading all bins of all CTAs took 7000 clocks a pass); bins and sums have two places in turn, so that a pass is one barrier of the cluster.  Then every warp counts what stays of its run, and a prefix over CTAs and
// warps gives each kept slot its place: the choice and the order are the same in every run.
//   into another cache   a CTA moves the places it knows: an eighth of them, or what stays of its own run
//   in place             all move together in rounds, all of a round read before any of it is written: a slot never moves up, so what a round overwrites lies in front of what
//                        later rounds read
// What bounds it: the chain of three select passes, counting and listing, and the moved bytes (pieces of 16 bytes out of lines of 128) for large caches; round trips and barriers
// for small ones.  8 kv heads of 128: 76 of 1100 dropped in 8.2 us, 57309 of 65501 in 27 us (the bytes alone: 3.3).
// In place, with a list in global memory and two cluster barriers a round: 76 of 1100 in 10.5 us, 512 of 4096 in 14.2, 2048 of 8192 in 21, 57309 of 65501 in 31.
constexpr int kEvictThreads = 1024, kEvictCtas = 8, kEvictPieces = 4, kEvictHeld = 8;      // pieces of a thread in a round; weights of a thread in registers
constexpr uint32_t kEvictBins = 2048, kEvictSolo = kEvictThreads * kEvictHeld, kEvictListed = 8192;      // places a CTA lists in shared memory

struct Q4Evict {
    Q4Cache from, to;
    const float* weight;       // [kv_heads][from.slots]
    float* weight_to;          // [kv_heads][to.slots]
    const int* filled;
    int* kept;                 // [kv_heads][keep], or null
    int* list;                 // workspace [kv_heads][from.slots]: the slot at every rank
    uint32_t keep, keep_first, keep_last;
    int* error_word;
};

// Larger for larger weights; the zeros are equal, NaN is the least.
__device__ __forceinline__ uint32_t evict_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__global__ void __cluster_dims__(kEvictCtas, 1, 1) __launch_bounds__(kEvictThreads) q4_evict_kernel(const __grid_constant__ Q4Evict p) {
    namespace cg = cooperative_groups;
    extern __shared__ int own_list[];                      // [kEvictListed]: the slots at the places this CTA moves
    __shared__ uint32_t hists[2][kEvictBins];
    __shared__ __align__(8) uint32_t groups[2][kEvictBins / 32];
    __shared__ uint32_t warp_more[32], warp_ties[32];      // a warp's slots above the border, and at it
    __shared__ uint32_t s_bin, s_left, s_before, s_ties_before;
    __shared__ uint32_t cta_more, cta_ties;                // read by the other CTAs
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), h = blockIdx.y;
    pdl_launch_dependents();
    for (uint32_t i = tid; i < 2 * kEvictBins; i += kEvictThreads) hists[0][i] = 0;
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    if (filled < 0 || static_cast<uint32_t>(filled) > p.from.slots) {      // the same for every CTA of the grid
        if (tid == 0 && rank == 0 && h == 0) atomicExch(p.error_word, kErrBadPosition);
        return;
    }
    const uint32_t n = filled, keep = min(n, p.keep);
    const float* weight = p.weight + static_cast<size_t>(h) * p.from.slots;
    int* list = p.list + static_cast<size_t>(h) * p.from.slots;
    // slots [low, high) compete for `wanted` places; all others stay
    const bool all = n <= p.keep, in_place = p.to.k_codes == p.from.k_codes, solo = n <= kEvictSolo;
    const uint32_t low = all ? n : p.keep_first, high = all ? n : n - p.keep_last, wanted = all ? 0u : keep - p.keep_first - p.keep_last;
    const uint32_t ctas = solo ? 1u : kEvictCtas, me = solo ? 0u : rank;
    const uint32_t per_warp = ((n + ctas * 32 - 1) / (ctas * 32) + 31) & ~31u;
    const uint32_t begin = min(n, (me * 32 + warp) * per_warp), end = min(n, begin + per_warp), turns = per_warp / 32;
    float held[kEvictHeld];                 // slot begin + 32 j + lane
#pragma unroll
    for (uint32_t j = 0; j < kEvictHeld; ++j) held[j] = j < turns && begin + 32 * j + lane < end ? __ldcg(weight + begin + 32 * j + lane) : 0.0f;
    // every slot of the warp's run: the first ones from registers
    auto each = [&](auto run) {
#pragma unroll
        for (uint32_t j = 0; j < kEvictHeld; ++j) if (j < turns) run(begin + 32 * j + lane, held[j]);
#pragma unroll 4
        for (uint32_t j = kEvictHeld; j < turns; ++j) {
            const uint32_t i = begin + 32 * j + lane;
            run(i, i < end ? __ldcg(weight + i) : 0.0f);
        }
    };
    auto lanes_upto = [&](uint32_t mine) {                 // the sum of a warp's `mine` up to and with this lane's
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, mine, o);
            if (static_cast<int>(lane) >= o) mine += v;
        }
        return mine;
    };

    // the wanted-th largest key among the competing slots, and how many that equal it stay
    uint32_t border = 0xffffffffu, ties_wanted = 0;
    if (wanted) {
        uint32_t prefix = 0, remaining = wanted, mask = 0;
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t digits = pass == 2 ? 1023u : 2047u;
            uint32_t* const hist = hists[pass & 1];
            __syncthreads();
            each([&](uint32_t i, float w) {
                const uint32_t key = evict_key(w);
                if (i < end && i >= low && i < high && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & digits], 1u);
            });
            if (solo) {
                __syncthreads();
                // thread t looks after bins 2047 - 2 t and 2046 - 2 t, from the largest down
                const uint2 two = reinterpret_cast<const uint2*>(hist)[kEvictThreads - 1 - tid];
                const uint32_t mine = two.x + two.y;
                uint32_t upto = lanes_upto(mine);
                if (lane == 31) warp_more[warp] = upto;
                __syncthreads();
                upto += __reduce_add_sync(0xffffffffu, lane < warp ? warp_more[lane] : 0u);
                if (upto >= remaining && upto - mine < remaining) {
                    const uint32_t left = remaining - (upto - mine);
                    s_bin = kEvictBins - 1 - 2 * tid - (two.y >= left ? 0u : 1u);
                    s_left = two.y >= left ? left : left - two.y;
                }
            } else {
                __syncthreads();
                const uint32_t first = __reduce_add_sync(0xffffffffu, hist[64 * warp + lane]), second = __reduce_add_sync(0xffffffffu, hist[64 * warp + 32 + lane]);
                if (lane == 0) { groups[pass & 1][2 * warp] = first; groups[pass & 1][2 * warp + 1] = second; }
                cluster.sync();
                if (warp == 0) {      // from the largest down: a lane has two groups, then a bin of the one with the border
                    uint32_t x = 0, y = 0;
#pragma unroll
                    for (uint32_t r = 0; r < kEvictCtas; ++r) {
                        const uint2 two = reinterpret_cast<const uint2*>(cluster.map_shared_rank(groups[pass & 1], r))[31 - lane];
                        x += two.x;
                        y += two.y;
                    }
                    uint32_t upto = lanes_upto(x + y), before = upto - x - y;
                    const int owner = __ffs(__ballot_sync(0xffffffffu, upto >= remaining)) - 1;      // there is one: as many compete as are wanted
                    const uint32_t upper = before + y >= remaining;                // the lane's larger group has it
                    const uint32_t group = __shfl_sync(0xffffffffu, 2 * (31 - lane) + upper, owner), left = remaining - __shfl_sync(0xffffffffu, upper ? before : before + y, owner);
                    uint32_t mine = 0;
#pragma unroll
                    for (uint32_t r = 0; r < kEvictCtas; ++r) mine += cluster.map_shared_rank(hist, r)[32 * group + 31 - lane];
                    upto = lanes_upto(mine);
                    if (upto >= left && upto - mine < left) { s_bin = 32 * group + 31 - lane; s_left = left - (upto - mine); }
                }
            }
            __syncthreads();
            prefix |= s_bin << shift;
            remaining = s_left;
            mask |= digits << shift;
            if (pass == 1) for (uint32_t i = tid; i < kEvictBins; i += kEvictThreads) hists[0][i] = 0;      // which nobody reads behind this pass's barrier
        }
        border = prefix;
        ties_wanted = remaining;
    }
    // what stays of every warp's run
    uint32_t more = 0, ties = 0;
    each([&](uint32_t i, float w) {
        const bool real = i < end, competes = i >= low && i < high;
        const uint32_t key = evict_key(w);
        more += real && (!competes || (wanted && key > border));
        ties += real && competes && wanted && key == border;
    });
    more = __reduce_add_sync(0xffffffffu, more);
    ties = __reduce_add_sync(0xffffffffu, ties);
    __syncthreads();
    if (lane == 0) { warp_more[warp] = more; warp_ties[warp] = ties; }
    if (tid == 0) s_before = s_ties_before = 0;
    __syncthreads();
    if (!solo) {
        if (warp == 0) {
            const uint32_t m = __reduce_add_sync(0xffffffffu, warp_more[lane]), t = __reduce_add_sync(0xffffffffu, warp_ties[lane]);
            if (lane == 0) { cta_more = m; cta_ties = t; }
        }
        cluster.sync();
        if (warp == 0) {
            const uint32_t m = __reduce_add_sync(0xffffffffu, lane < rank ? *cluster.map_shared_rank(&cta_more, lane) : 0u);
            const uint32_t t = __reduce_add_sync(0xffffffffu, lane < rank ? *cluster.map_shared_rank(&cta_ties, lane) : 0u);
            if (lane == 0) { s_before = m; s_ties_before = t; }
        }
        cluster.sync();                                    // behind it no CTA reads another's shared memory
    }
    // the places this CTA moves into another cache
    const uint32_t share = ((keep + kEvictCtas - 1) / kEvictCtas + 7) & ~7u;
    const uint32_t first_place = solo ? min(keep, rank * share) : s_before + min(s_ties_before, ties_wanted);
    const uint32_t end_place = solo ? min(keep, first_place + share) : s_before + cta_more + min(s_ties_before + cta_ties, ties_wanted);
    const bool listed = !in_place && end_place - first_place <= kEvictListed;
    uint32_t before = s_before + __reduce_add_sync(0xffffffffu, lane < warp ? warp_more[lane] : 0u), ties_before = s_ties_before + __reduce_add_sync(0xffffffffu, lane < warp ? warp_ties[lane] : 0u);
    each([&](uint32_t i, float w) {
        const bool real = i < end, competes = i >= low && i < high;
        const uint32_t key = evict_key(w);
        const bool above = real && (!competes || (wanted && key > border)), tie = real && competes && wanted && key == border;
        const uint32_t below = (1u << lane) - 1u, aboves = __ballot_sync(0xffffffffu, above), tied = __ballot_sync(0xffffffffu, tie);
        const uint32_t tie_rank = ties_before + __popc(tied & below);
        if (above || (tie && tie_rank < ties_wanted)) {
            const uint32_t place = before + __popc(aboves & below) + min(tie_rank, ties_wanted);
            const bool mine = place >= first_place && place < end_place;
            if (listed) { if (mine) own_list[place - first_place] = static_cast<int>(i); }
            else if (!solo || rank == 0) list[place] = static_cast<int>(i);
            if (solo ? mine : true) {
                if (p.kept) p.kept[static_cast<size_t>(h) * p.keep + place] = static_cast<int>(i);
                if (!in_place) p.weight_to[static_cast<size_t>(h) * p.to.slots + place] = w;
            }
        }
        before += __popc(aboves);
        ties_before += __popc(tied);
    });
    if (!listed && (in_place || solo)) cluster.sync();     // the list is whole
    else __syncthreads();                                  // the CTA's part of it

    // the move: a kept slot is 2 * blocks pieces of 16 code bytes, and beside them its scales (and in place its weight).  Eight neighbouring threads take
    // one piece of eight neighbouring places, which are written as one line.
    const uint32_t blocks = p.from.blocks, pieces = 2 * blocks, movers = in_place ? kEvictCtas : 1u, mover = in_place ? rank : 0u;
    const uint32_t a_round = movers * kEvictThreads * kEvictPieces / (8 * pieces) * 8, from_place = in_place ? 0u : first_place & ~7u, to_place = in_place ? keep : end_place;
    for (uint32_t first = from_place; first < to_place; first += a_round) {
        uint4 code[kEvictPieces];
        __half scale[kEvictPieces];
        float w[kEvictPieces];
        uint32_t place[kEvictPieces], piece[kEvictPieces];
        bool mine[kEvictPieces];
#pragma unroll
        for (int u = 0; u < kEvictPieces; ++u) {
            const uint32_t i = (u * movers + mover) * kEvictThreads + tid;
            piece[u] = (i >> 3) % pieces;
            place[u] = first + i / (8 * pieces) * 8 + (i & 7u);
            mine[u] = i < a_round * pieces && place[u] < to_place && (in_place || place[u] >= first_place);
            if (!mine[u]) continue;
            const bool value = piece[u] >= blocks;
            const uint32_t block = value ? piece[u] - blocks : piece[u], slot = static_cast<uint32_t>(listed ? own_list[place[u] - first_place] : __ldcg(list + place[u]));
            code[u] = __ldcg(reinterpret_cast<const uint4*>((value ? p.from.v_codes : p.from.k_codes) + q4_codes_at(h, slot, block, blocks, p.from.slots)));
            scale[u] = __ldcg((value ? p.from.v_scales : p.from.k_scales) + q4_scale_at(h, slot, block, blocks, p.from.slots));
            if (in_place && piece[u] == 0) w[u] = __ldcg(weight + slot);
        }
        if (in_place) cluster.sync();
#pragma unroll
        for (int u = 0; u < kEvictPieces; ++u) {
            if (!mine[u]) continue;
            const bool value = piece[u] >= blocks;
            const uint32_t block = value ? piece[u] - blocks : piece[u];
            *reinterpret_cast<uint4*>((value ? p.to.v_codes : p.to.k_codes) + q4_codes_at(h, place[u], block, blocks, p.to.slots)) = code[u];
            (value ? p.to.v_scales : p.to.k_scales)[q4_scale_at(h, place[u], block, blocks, p.to.slots)] = scale[u];
            if (in_place && piece[u] == 0) p.weight_to[static_cast<size_t>(h) * p.to.slots + place[u]] = w[u];
        }
        if (in_place) cluster.sync();
    }
}

}  // namespace zk
