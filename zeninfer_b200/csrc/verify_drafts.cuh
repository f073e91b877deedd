// Drafted tokens against the model's own filtered distributions (the sampled form of a speculative block).
//
// A drafted token x of distribution q is accepted with probability min(1, p(x) / q(x)) and otherwise replaced by a draw from max(p - q, 0): the
// outcome is distributed as p.  p is what sample_pick.cuh draws from, of one row of logits: e_i = exp((v_i - max) / T) in double over the finite
// ones, cut to the top_k highest, then to the shortest run of the most likely whose share reaches top_p.
//
// A cluster takes a row and a CTA a run of the vocabulary, its logits and exponentials in shared memory.  Every row decides its own draft AND draws its
// own replacement, as if all drafts before it had been accepted, so that nothing waits for a decision: the rows run side by side, and one warp
// puts their answers together in a second launch.
//
// The cuts (top_k over counts, top_p over masses) look for the entry, in descending order, at which a sum of weights is reached.  The range of values is divided into
// 1024 equal bins, which spreads logits far better than the bits of their keys do (eight bits of a key put most of a row into five bins, and
// its threads queued up there: 290 us for 9 rows of 128256); the bin of the border is divided again while it holds more than a list
// takes, and the entries of the list are compared with each other, equal values by id.  A mass is an integer, the exponential's 2^-51ths of the
// row's sum rounded up, added in three limbs of 17 bits by 32-bit atomics: its sums do not depend on the order in which threads add to a bin.  Sums of exponentials are
// added in a fixed order.
// What bounds it: passes over the CTA's 16 entries a thread (load, exponentials, histogram, cut, two sums: 2 to 7 thousand cycles each) and cluster barriers of some 1500: three without a cut,
// six with top-p, ten with both, and two for each division behind a cut's first.
// 9 rows of 128256, top-p: 31.3 us, 5 rows, top-k 40 and top-p: 32 to 33 us, 3 rows of 32000, no cut: 11.1 us; clusters of 16 CTAs took 63, 47 and 10.4, for eight of them fit the GPU at a time.
#pragma once
#include <cooperative_groups.h>

#include <cstdint>

#include "sample_key.cuh"
#include "zk_ptx.cuh"

namespace zk {

constexpr int kVerifyThreads = 1024, kVerifyLimbs = 3, kVerifyLimbBits = 17, kVerifyMine = 256, kVerifyAll = 1024;
constexpr uint32_t kVerifyBins = 1024, kVerifyRun = 16384;          // entries a CTA takes at most
constexpr double kVerifyUnit = 2251799813685248.0;                  // 2^51: the mass of a whole row

struct VerifyEntry {
    unsigned long long weight;
    float value;
    uint32_t id;
};
// Dynamic shared memory: exponentials and logits of the CTA's run, the bins' limbs, the CTA's and the row's entries at the border.
__host__ __device__ constexpr uint32_t verify_smem_bytes(uint32_t per_cta) { return per_cta * 12 + kVerifyLimbs * kVerifyBins * 4 + (kVerifyMine + kVerifyAll) * 16; }

struct VerifyParams {
    const float* logits;       // rows logits_ld apart
    size_t logits_ld;
    uint32_t vocab, drafts, per_cta;
    const long long* tokens;
    const int* q_ids;          // [drafts][kSampleMaxCandidates], or null: the drafts are certain
    const double* q_probs;
    const int* q_count;
    const double* uniforms;
    double temperature;
    uint32_t top_k;
    float top_p;
    long long* out;
    int* accepted;
    double* probs;             // or null
    long long* draws;          // workspace [drafts + 1]: the token a row would go on with
    int* fits;                 // workspace [drafts + 1]: whether the row's draft is accepted
    int* error_word;
};

// What a CTA hands to the others, by the exchange it belongs to: a field is written for one of them only, so a reader needs no barrier behind it.
struct VerifyShare {
    double reference, sum;             // the value its exponentials are relative to, and their sum
    double kept, left;                 // the sum of what a cut left; of max(p - q, 0), both in the row's units
    double left_again;
    unsigned long long ties, each;
    uint32_t top_key, low_key, finite;
    uint32_t listed, bin_high, bin_low, any_each;
};

// The least integer that is not below e * unit, 0 <= e * unit <= 2^51: what is left of 2^52 + e * unit in its lower bits.  Upwards, so that masses which reach a share exactly (three
// of six equal ones the half) reach it in integers too.
__device__ __forceinline__ unsigned long long mass_of(double e, double unit) { return static_cast<unsigned long long>(__double_as_longlong(__fma_ru(e, unit, 4503599627370496.0))) & 0xfffffffffffffull; }

// e^y for y <= 0, given 2^(j / 64) for j = 0 .. 63: y = n ln 2 / 64 + r with |r| < 0.0055, whose series up to r^5 / 120 leaves out less than 2^-54.  About half of the double-precision
// instructions of exp.
constexpr uint32_t kVerifyPowers = 64;
__device__ __forceinline__ double verify_exp(double y, const double* powers) {
    if (y < -700.0) return exp(y);
    constexpr double kRound = 6755399441055744.0;             // 1.5 * 2^52: a sum with it has the nearest whole number in its lower bits
    constexpr double kUpper = 0x1.62e42ffp-7, kRest = -0x1.718432a1b0e26p-41;                // ln 2 / 64 = kUpper + kRest; n * kUpper is exact
    const double shifted = fma(y, 92.33248261689366, kRound), n = shifted - kRound;          // 64 / ln 2
    const int whole = __double2loint(shifted);
    const double r = fma(-n, kRest, fma(-n, kUpper, y));
    const double s = fma(r, fma(r, fma(r, fma(r, 1.0 / 120.0, 1.0 / 24.0), 1.0 / 6.0), 0.5), 1.0);
    const double of = powers[whole & 63], e = fma(of, r * s, of);
    return __hiloint2double(__double2hiint(e) + ((whole >> 6) << 20), __double2loint(e));
}

template <int kCtas>
__global__ void __launch_bounds__(kVerifyThreads) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t verify_smem[];
    __shared__ VerifyShare share;
    __shared__ double warp_sum[32], s_q;
    __shared__ unsigned long long s_left;
    __shared__ uint32_t warp_high[32], warp_low[32], warp_count[32], s_bin, s_mine, s_high, s_low, s_count, s_before, s_fits;
    __shared__ double s_sum, s_ahead, s_scale, powers[kVerifyPowers];
    __shared__ unsigned long long groups[32];          // totals of 32 bins each
    __shared__ int s_last;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), row = blockIdx.y;
    double* e = reinterpret_cast<double*>(verify_smem);                      // [per_cta]
    float* v = reinterpret_cast<float*>(e + p.per_cta);                      // [per_cta], per_cta a multiple of four
    uint32_t* limbs = reinterpret_cast<uint32_t*>(v + p.per_cta);            // [kVerifyLimbs][kVerifyBins], then the bins' totals
    unsigned long long* totals = reinterpret_cast<unsigned long long*>(limbs);
    VerifyEntry* own_list = reinterpret_cast<VerifyEntry*>(limbs + kVerifyLimbs * kVerifyBins);
    VerifyEntry* all_list = own_list + kVerifyMine;
    const uint32_t base = rank * p.per_cta;
    const uint32_t whole_run = base < p.vocab ? min(p.per_cta, p.vocab - base) : 0u;
    uint32_t n = whole_run;                            // entries left in it
    // a thread's run of consecutive entries, for sums in order of id (an odd number of them: no two lanes of a warp on one bank)
    const uint32_t per_thread = ((p.per_cta + kVerifyThreads - 1) / kVerifyThreads) | 1u;
    uint32_t begin = min(n, tid * per_thread), end = min(n, begin + per_thread);
    pdl_launch_dependents();
    if (tid < kVerifyPowers) powers[tid] = exp2(tid / 64.0);
    pdl_wait();
    if (rank == 0 && tid == 0) p.draws[row] = -1;      // ahead of the barriers that the draw comes behind
    const float* logits = p.logits + row * p.logits_ld + base;
    const bool is_draft = row < p.drafts;
    long long token = is_draft ? __ldcg(p.tokens + row) : -1;
    if (is_draft && (token < 0 || token >= static_cast<long long>(p.vocab))) {
        if (rank == 0 && tid == 0) atomicExch(p.error_word, kErrBadToken);
        token = -1;
    }
    const bool has_token = token >= 0 && token / p.per_cta == rank;
    // What the CTAs hand over is read by warp 0, lane r from CTA r, and told to the others: a request of every warp for the same word costs as much as its own.
    auto its = [&](uint32_t r) { return cluster.map_shared_rank(&share, r); };
    const bool reads = warp == 0 && lane < kCtas;
    auto value_of = [](uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); };
    // a CTA's sum, in every thread: of threads and warps in order
    auto cta_sum = [&](double mine) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_down_sync(0xffffffffu, mine, o);
        __syncthreads();
        if (lane == 0) warp_sum[warp] = mine;
        __syncthreads();
        double s = warp_sum[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    // the largest and the smallest key and the number of entries of a CTA, in every thread
    auto cta_range = [&](uint32_t& high, uint32_t& low, uint32_t& count) {
        high = __reduce_max_sync(0xffffffffu, high);
        low = __reduce_min_sync(0xffffffffu, low);
        count = __reduce_add_sync(0xffffffffu, count);
        __syncthreads();
        if (lane == 0) { warp_high[warp] = high; warp_low[warp] = low; warp_count[warp] = count; }
        __syncthreads();
        high = __reduce_max_sync(0xffffffffu, warp_high[lane]);
        low = __reduce_min_sync(0xffffffffu, warp_low[lane]);
        count = __reduce_add_sync(0xffffffffu, warp_count[lane]);
    };

    // the logits, the largest and smallest of the finite ones and how many there are
    uint32_t top = 0, low = 0xffffffffu, finite = 0;
    auto take = [&](uint32_t i, float x) {
        x += 0.0f;                                      // the zeros are equal
        const uint32_t key = sample_key(x);
        v[i] = x;
        top = max(top, key);
        if (key) low = min(low, key);
        finite += key != 0u;
    };
    if (reinterpret_cast<uintptr_t>(logits) % 16 == 0) {
#pragma unroll 4
        for (uint32_t i = 4 * tid; i + 3 < n; i += 4 * kVerifyThreads) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(logits + i));
            take(i, x.x); take(i + 1, x.y); take(i + 2, x.z); take(i + 3, x.w);
        }
        if (const uint32_t i = (n & ~3u) + tid; i < n) take(i, __ldcg(logits + i));
    } else {
#pragma unroll 4
        for (uint32_t i = tid; i < n; i += kVerifyThreads) take(i, __ldcg(logits + i));
    }
    cta_range(top, low, finite);
    const bool greedy = p.temperature == 0.0;
    const uint32_t top_k = greedy ? 1u : p.top_k;
    const double temperature = greedy ? 1.0 : p.temperature, per_unit = 1.0 / temperature;

    auto drop = [&](uint32_t i) { v[i] = NAN; e[i] = 0.0; };
    // Once few entries are left they close ranks, an entry a thread; their places in the run are kept behind the values.  The order, by which equal values are told apart, stays.
    uint32_t* const places = reinterpret_cast<uint32_t*>(v + p.per_cta) - kVerifyAll;
    bool few = false;
    auto close_ranks = [&]() {
        if (p.per_cta < 2 * kVerifyAll) return;
        uint32_t left = 0;
        for (uint32_t i = begin; i < end; ++i) left += sample_key(v[i]) != 0u;
        uint32_t at = left;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, at, o);
            if (static_cast<int>(lane) >= o) at += x;
        }
        __syncthreads();
        if (lane == 31) warp_count[warp] = at;
        __syncthreads();
        at += __reduce_add_sync(0xffffffffu, lane < warp ? warp_count[lane] : 0u) - left;
        const uint32_t all = __reduce_add_sync(0xffffffffu, warp_count[lane]);
        if (all > kVerifyAll) return;
        for (uint32_t i = begin; i < end; ++i) if (sample_key(v[i])) all_list[at++] = VerifyEntry{0, v[i], i};
        __syncthreads();
        n = all;
        if (tid < n) { v[tid] = all_list[tid].value; places[tid] = all_list[tid].id; }
        begin = min(n, tid);
        end = min(n, tid + 1);
        few = true;
        __syncthreads();
    };
    // where the run's entry `local` is now, or -1
    auto place_of = [&](uint32_t local) {
        if (!few) return static_cast<int>(local);
        uint32_t low_end = 0, high_end = n;
        while (low_end < high_end) {
            const uint32_t mid = (low_end + high_end) / 2;
            if (places[mid] < local) low_end = mid + 1;
            else high_end = mid;
        }
        return low_end < n && places[low_end] == local ? static_cast<int>(low_end) : -1;
    };
    // Of the entries that equal `border` all behind the first `ties` (in order of id) go, and so do all below it.
    auto cut_ties = [&](uint32_t border, unsigned long long ties) {
        uint32_t equal = 0;
        for (uint32_t i = begin; i < end; ++i) equal += sample_key(v[i]) == border;
        uint32_t upto = equal;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (static_cast<int>(lane) >= o) upto += x;
        }
        if (lane == 31) warp_count[warp] = upto;
        __syncthreads();
        uint32_t before = upto - equal;
        for (uint32_t w = 0; w < warp; ++w) before += warp_count[w];
        if (tid == kVerifyThreads - 1) share.ties = before + equal;
        cluster.sync();
        unsigned long long seen = before;
        for (uint32_t r = 0; r < rank; ++r) seen += its(r)->ties;
        cluster.sync();
        for (uint32_t i = begin; i < end; ++i) {
            const uint32_t key = sample_key(v[i]);
            if (key < border || (key == border && seen++ >= ties)) drop(i);
        }
        __syncthreads();
    };
    // Leaves the shortest run of entries, in descending order (equal values: the lowest ids), whose weights reach `wanted` > 0, at least one.
    // weigh(i): an entry's weight.  high, low: keys that no entry which takes part is beyond.
    auto cut = [&](unsigned long long wanted, auto weigh, uint32_t high, uint32_t low) {
        double v_low = fmax(static_cast<double>(value_of(low)), static_cast<double>(value_of(high)) - 64.0 * temperature);      // far below, nothing is worth bins of its own
        for (;;) {
            if (high == low) {         // equal values: so many of them as are wanted, each of the same weight
                unsigned long long each = 0;
                if (tid == 0) share.any_each = 0;
                __syncthreads();
                for (uint32_t i = tid; i < n; i += kVerifyThreads) if (sample_key(v[i]) == high) each = weigh(i);
                if (each) { share.each = each; share.any_each = 1; }
                cluster.sync();
                for (int r = 0; r < kCtas; ++r) if (its(r)->any_each) each = its(r)->each;
                cluster.sync();
                each = max(each, 1ull);
                cut_ties(high, (wanted + each - 1) / each);
                return;
            }
            // 1024 bins from the top down; in 32 bits (of halves, which do not overflow) where the range allows it: either way a larger value has no larger bin
            const double v_high = value_of(high), per = kVerifyBins / (v_high - v_low);
            const float half_high = 0.5f * value_of(high), per_half = static_cast<float>(2.0 * per);
            const bool narrow = !(per_half > 1e-30f && per_half < 1e30f);
            auto bin_of = [&](float x) {
                return narrow ? static_cast<uint32_t>(fmin((v_high - static_cast<double>(x)) * per, kVerifyBins - 1.0)) : static_cast<uint32_t>(fminf((half_high - 0.5f * x) * per_half, kVerifyBins - 1.0f));
            };
            for (uint32_t i = tid; i < kVerifyLimbs * kVerifyBins; i += kVerifyThreads) limbs[i] = 0;
            if (tid == 0) { s_bin = 0xffffffffu; s_mine = 0; }
            __syncthreads();
            uint32_t bins[kVerifyRun / kVerifyThreads / 2];   // of the thread's entries, two a word; kVerifyBins: it goes whatever the border is, kNone: it stays, or is gone
            constexpr uint32_t kNone = 0xffff;
#pragma unroll
            for (uint32_t j = 0; j < kVerifyRun / kVerifyThreads; ++j) {
                const uint32_t i = tid + j * kVerifyThreads;
                uint32_t bin = kNone;
                if (i < n) {
                    const float x = v[i];
                    const uint32_t key = sample_key(x);
                    if (key && key < low) bin = kVerifyBins;
                    else if (key && key <= high) {
                        const unsigned long long w = weigh(i);
                        bin = bin_of(x);
#pragma unroll
                        for (int k = 0; k < kVerifyLimbs; ++k) {
                            uint32_t limb = static_cast<uint32_t>(w >> (k * kVerifyLimbBits));
                            if (k + 1 < kVerifyLimbs) limb &= (1u << kVerifyLimbBits) - 1u;          // an entry may be all of the row: 2^51
                            if (limb) atomicAdd(limbs + k * kVerifyBins + bin, limb);
                        }
                    }
                }
                bins[j / 2] = j % 2 ? bins[j / 2] | bin << 16 : bin;
            }
            __syncthreads();
            unsigned long long mine = 0;
#pragma unroll
            for (int k = 0; k < kVerifyLimbs; ++k) mine += static_cast<unsigned long long>(limbs[k * kVerifyBins + tid]) << (k * kVerifyLimbBits);
            __syncthreads();
            totals[tid] = mine;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
            if (lane == 0) groups[warp] = mine;
            cluster.sync();
            // the border among the row's groups of 32 bins, and then among the bins of one: distributed shared memory gives some ten bytes a clock, so few are read
            if (warp == 0) {
                auto reached = [&](unsigned long long sum, unsigned long long from, unsigned long long& left) {      // the lane at which sums reach `from`, or 32; what is left there
                    unsigned long long upto = sum;
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
                        if (static_cast<int>(lane) >= o) upto += x;
                    }
                    const int at = __ffs(__ballot_sync(0xffffffffu, upto >= from)) - 1;
                    left = from - __shfl_sync(0xffffffffu, upto - sum, at & 31);
                    return at < 0 ? 32 : at;
                };
                unsigned long long sum = 0, left = 0;
#pragma unroll
                for (int r = 0; r < kCtas; ++r) sum += cluster.map_shared_rank(groups, r)[lane];
                const int group = reached(sum, wanted, left);
                if (group < 32) {
                    sum = 0;
#pragma unroll
                    for (int r = 0; r < kCtas; ++r) sum += cluster.map_shared_rank(totals, r)[32 * group + lane];
                    const int at = reached(sum, left, left);
                    if (lane == 0) { s_bin = 32 * group + at; s_left = left; }
                }
            }
            __syncthreads();
            const uint32_t border = s_bin;                  // none: rounding left the whole short of what is wanted, and everything stays
            if (border != 0xffffffffu) wanted = s_left;
            // what lies below the border goes; the entries of its bin are listed, and counted on where there are too many
            uint32_t bin_high = 0, bin_low = 0xffffffffu, unused = 0;
#pragma unroll
            for (uint32_t j = 0; j < kVerifyRun / kVerifyThreads; ++j) {
                const uint32_t i = tid + j * kVerifyThreads, bin = j % 2 ? bins[j / 2] >> 16 : bins[j / 2] & 0xffffu;
                if (bin == kNone) continue;
                if (bin == border) {
                    const float x = v[i];
                    const uint32_t key = sample_key(x);
                    bin_high = max(bin_high, key);
                    bin_low = min(bin_low, key);
                    const uint32_t at = atomicAdd(&s_mine, 1u);
                    if (at < kVerifyMine) own_list[at] = VerifyEntry{weigh(i), x, base + i};
                } else if (bin > border || bin == kVerifyBins) {
                    drop(i);
                }
            }
            cta_range(bin_high, bin_low, unused);
            if (tid == 0) { share.listed = s_mine; share.bin_high = bin_high; share.bin_low = bin_low; }
            cluster.sync();
            if (border == 0xffffffffu) return;
            if (warp == 0) {
                const uint32_t listed = reads ? its(lane)->listed : 0u;
                bin_high = __reduce_max_sync(0xffffffffu, reads ? its(lane)->bin_high : 0u);
                bin_low = __reduce_min_sync(0xffffffffu, reads ? its(lane)->bin_low : 0xffffffffu);
                const uint32_t all = __reduce_add_sync(0xffffffffu, listed), ahead = __reduce_add_sync(0xffffffffu, lane < rank ? listed : 0u);
                const bool fit = __all_sync(0xffffffffu, listed <= kVerifyMine);
                if (lane == 0) { s_count = all; s_before = ahead; s_fits = fit; s_high = bin_high; s_low = bin_low; }
            }
            __syncthreads();
            const uint32_t count = s_count, before_mine = s_before;
            const bool fits = s_fits;
            if (!fits || count > kVerifyAll) {
                high = s_high;
                low = s_low;
                v_low = value_of(low);
                continue;
            }
            for (uint32_t r = warp; r < kCtas; r += 32) {      // a warp a CTA: its entries behind those of the CTAs before
                uint32_t at = 0;
                const uint32_t listed = lane < kCtas ? its(lane)->listed : 0u;
                at = __reduce_add_sync(0xffffffffu, lane < r ? listed : 0u);
                const uint32_t theirs = __shfl_sync(0xffffffffu, listed, r);
                for (uint32_t i = lane; i < theirs; i += 32) all_list[at + i] = cluster.map_shared_rank(own_list, r)[i];
            }
            __syncthreads();
            // a warp decides an entry of the CTA's: it stays when what comes before it does not reach what is wanted
            for (uint32_t i = warp; i < s_mine; i += 32) {
                const VerifyEntry me = all_list[before_mine + i];
                unsigned long long sum = 0;
                for (uint32_t j = lane; j < count; j += 32) {
                    const VerifyEntry other = all_list[j];
                    if (other.value > me.value || (other.value == me.value && other.id < me.id)) sum += other.weight;
                }
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0 && sum >= wanted) drop(me.id - base);
            }
            __syncthreads();
            return;
        }
    };

    double reference = value_of(top);              // what the CTA's exponentials are relative to; without an entry, anything
    if (!top) reference = -INFINITY;
    if (top_k && top_k < p.vocab) {
        if (tid == 0) { share.top_key = top; share.low_key = low; share.finite = finite; }
        cluster.sync();
        if (warp == 0) {
            const uint32_t high = __reduce_max_sync(0xffffffffu, reads ? its(lane)->top_key : 0u), lowest = __reduce_min_sync(0xffffffffu, reads ? its(lane)->low_key : 0xffffffffu);
            const uint32_t all = __reduce_add_sync(0xffffffffu, reads ? its(lane)->finite : 0u);
            if (lane == 0) { s_high = high; s_low = lowest; s_count = all; }
        }
        cluster.sync();                            // the fields are written again below
        const uint32_t row_top = s_high, row_low = s_low, row_finite = s_count;
        __syncthreads();
        if (top_k < row_finite) {
            cut(top_k, [](uint32_t) { return 1ull; }, row_top, row_low);
            close_ranks();
        }
    }
    // exponentials relative to the CTA's own largest value: no one waits for the row's
    double mine = 0.0;
#pragma unroll 4
    for (uint32_t i = begin; i < end; ++i) {
        const float x = v[i];
        const double w = sample_key(x) ? verify_exp((static_cast<double>(x) - reference) * per_unit, powers) : 0.0;
        e[i] = w;
        mine += w;
    }
    mine = cta_sum(mine);
    if (tid == 0) { share.reference = reference; share.sum = mine; share.top_key = top; share.low_key = low; share.finite = finite; }
    cluster.sync();
    if (warp == 0) {
        // what a CTA's exponentials count in the row
        const double theirs = reads ? its(lane)->reference : -INFINITY;
        double highest = theirs;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) highest = fmax(highest, __shfl_xor_sync(0xffffffffu, highest, o));
        const double factor = theirs == -INFINITY ? 0.0 : exp((theirs - highest) * per_unit);
        double all = reads ? factor * its(lane)->sum : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        const uint32_t high = __reduce_max_sync(0xffffffffu, reads ? its(lane)->top_key : 0u), lowest = __reduce_min_sync(0xffffffffu, reads ? its(lane)->low_key : 0xffffffffu);
        const uint32_t count = __reduce_add_sync(0xffffffffu, reads ? its(lane)->finite : 0u);
        if (lane == rank) s_scale = factor;
        if (lane == 0) { s_sum = all; s_high = high; s_low = lowest; s_count = count; }
    }
    __syncthreads();
    const double whole = s_sum, scale = s_scale;
    const uint32_t row_top = s_high, row_low = s_low, row_finite = s_count;
    if (!row_finite) {
        if (rank == 0 && tid == 0) {
            p.draws[row] = -1;
            p.fits[row] = 0;
            if (is_draft && p.probs) p.probs[row] = 0.0;
        }
        cluster.sync();                            // nobody leaves while its shared memory is read
        return;
    }

    double kept = whole;                           // the sum that makes probabilities of exponentials
    if (!greedy && p.top_p > 0.0f && p.top_p < 1.0f) {
        const double unit = kVerifyUnit * (scale / whole);
        cut(max(1ll, __double2ll_ru(static_cast<double>(p.top_p) * kVerifyUnit)), [&](uint32_t i) { return mass_of(e[i], unit); }, row_top, row_low);
        mine = 0.0;
#pragma unroll 4
        for (uint32_t i = begin; i < end; ++i) mine += e[i];
        mine = cta_sum(mine);
        if (tid == 0) share.kept = mine * scale;
        cluster.sync();
        if (warp == 0) {
            double all = reads ? its(lane)->kept : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            if (lane == 0) s_sum = all;
        }
        __syncthreads();
        kept = s_sum;
    }
    // The CTA that has the draft decides, and e becomes p - q where a draft may be replaced, both in the CTA's units
    const uint32_t entries = is_draft && p.q_ids ? static_cast<uint32_t>(min(max(__ldcg(p.q_count + row), 0), static_cast<int>(kSampleMaxCandidates))) : 0u;
    const size_t list = static_cast<size_t>(row) * kSampleMaxCandidates;
    const double of_one = kept / scale;            // a probability of 1
    if (tid == 0) s_q = 0.0;
    __syncthreads();
    if (has_token) {
        for (uint32_t j = tid; j < entries; j += kVerifyThreads)
            if (__ldcg(p.q_ids + list + j) == token) s_q = __ldcg(p.q_probs + list + j);
        __syncthreads();
        if (tid == 0) {
            const int at = place_of(static_cast<uint32_t>(token) - base);
            const double mine_p = at < 0 ? 0.0 : e[at] * scale / kept, q = p.q_ids ? s_q : 1.0;
            p.fits[row] = __ldcg(p.uniforms + row) * q < mine_p;
            if (p.probs) p.probs[row] = mine_p;
            if (!p.q_ids && at >= 0) e[at] = fmax(e[at] - of_one, 0.0);
        }
    } else if (is_draft && token < 0 && rank == 0 && tid == 0) {
        p.fits[row] = 0;
        if (p.probs) p.probs[row] = 0.0;
    }
    __syncthreads();
    for (uint32_t j = tid; j < entries; j += kVerifyThreads) {
        const int id = __ldcg(p.q_ids + list + j);
        if (id < 0 || static_cast<uint32_t>(id) < base || static_cast<uint32_t>(id) - base >= whole_run) continue;
        if (const int at = place_of(static_cast<uint32_t>(id) - base); at >= 0) e[at] = fmax(e[at] - __ldcg(p.q_probs + list + j) * of_one, 0.0);
    }
    __syncthreads();
    // The draw: the first entry with a share whose cumulative sum, in order of id, reaches u of the whole.  A thread's sums begin at what lies before its run.  A CTA's end is the next
    // one's beginning, formed by the same two rounded operations on both sides (no multiply-add, which rounds once), and it grows from CTA to CTA: one of them has the goal between its ends.
    double mine_left, before, cta_left;
    auto scan = [&]() {
        mine_left = 0.0;
#pragma unroll 4
        for (uint32_t i = begin; i < end; ++i) mine_left += e[i];
        double upto = mine_left;
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, upto, o);
            if (static_cast<int>(lane) >= o) upto += x;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        double warps = 0.0, all = 0.0;
        for (uint32_t w = 0; w < 32; ++w) {
            if (w == warp) warps = all;
            all += warp_sum[w];
        }
        const double lanes = __shfl_up_sync(0xffffffffu, upto, 1);
        before = warps + (lane ? lanes : 0.0);
        mine_left = warps + upto;                   // where the run ends
        cta_left = __dmul_rn(all, scale);
    };
    scan();
    if (tid == 0) share.left = cta_left;
    cluster.sync();
    // the CTAs' shares, added in order
    auto shares = [&](bool again) {
        if (warp == 0) {
            const double theirs = reads ? (again ? its(lane)->left_again : its(lane)->left) : 0.0;
            double sum = 0.0, mine_ahead = 0.0;
#pragma unroll
            for (int r = 0; r < kCtas; ++r) {
                if (r == static_cast<int>(rank)) mine_ahead = sum;
                sum += __shfl_sync(0xffffffffu, theirs, r);
            }
            const uint32_t any = __ballot_sync(0xffffffffu, theirs > 0.0);
            if (lane == 0) { s_sum = sum; s_ahead = mine_ahead; s_last = 31 - __clz(any); }
        }
        __syncthreads();
    };
    shares(false);
    double all = s_sum, ahead = s_ahead;
    if (!(all > 0.0)) {                             // nothing is left: p itself, formed anew
        __syncthreads();
        for (uint32_t i = begin; i < end; ++i) {
            const float x = v[i];
            e[i] = sample_key(x) ? verify_exp((static_cast<double>(x) - reference) * per_unit, powers) : 0.0;
        }
        scan();
        if (tid == 0) share.left_again = cta_left;
        cluster.sync();
        shares(true);
        all = s_sum;
        ahead = s_ahead;
    }
    const int last_with_any = s_last;
    // the product's rounding error decides where a sum equals it
    const double u = __ldcg(p.uniforms + p.drafts), goal = u * all, goal_rest = fma(u, all, -goal);
    auto at_goal = [&](double x) { return x > 0.0 && (x > goal || (x == goal && goal_rest <= 0.0)); };
    auto reached = [&](double local) { return at_goal(__dadd_rn(ahead, __dmul_rn(local, scale))); };
    // the ends of threads' runs grow up to rounding; the first that has reached the goal is looked for
    uint32_t first = reached(mine_left) ? tid : 0xffffffffu, none = 0, counted = 0;
    cta_range(none, first, counted);
    // not before this CTA, and before the next one; where rounding left the row's last sum short, the last CTA with a share
    if (!at_goal(ahead) && (at_goal(__dadd_rn(ahead, cta_left)) || static_cast<int>(rank) == last_with_any)) {
        if (first == 0xffffffffu) first = kVerifyThreads - 1;          // rounding left the last sum short: the last entry with a share
        // from the thread's run on backwards until there is an entry with a share (its own run has one but for rounding)
        if (tid == first) {
            double run = before;
            int found = -1;
            for (uint32_t i = begin; i < end; ++i) {
                if (!(e[i] * scale > 0.0)) continue;
                run += e[i];
                found = static_cast<int>(i);
                if (reached(run)) break;
            }
            for (int i = static_cast<int>(begin) - 1; found < 0 && i >= 0; --i) if (e[i] * scale > 0.0) found = i;
            for (uint32_t i = end; found < 0 && i < n; ++i) if (e[i] * scale > 0.0) found = static_cast<int>(i);
            for (uint32_t i = 0; found < 0 && i < n; ++i) if (e[i] > 0.0) found = static_cast<int>(i);      // shares that only their sum keeps from vanishing
            if (found >= 0) p.draws[row] = static_cast<long long>(base) + (few ? static_cast<int>(places[found]) : found);
        }
    }
    cluster.sync();                                  // nobody leaves while its shared memory is read
}

// The rows' answers put together: one warp.
__global__ void __launch_bounds__(32) verify_answer_kernel(const __grid_constant__ VerifyParams p) {
    pdl_launch_dependents();
    pdl_wait();
    uint32_t accepted = 0;
    for (uint32_t first = 0; first < p.drafts; first += 32) {
        const uint32_t i = first + threadIdx.x;
        const uint32_t fit = __ballot_sync(0xffffffffu, i < p.drafts && __ldcg(p.fits + i));
        accepted += fit == 0xffffffffu ? 32u : static_cast<uint32_t>(__ffs(~fit) - 1);
        if (fit != 0xffffffffu) break;
    }
    for (uint32_t i = threadIdx.x; i <= p.drafts; i += 32) p.out[i] = i < accepted ? __ldcg(p.tokens + i) : i == accepted ? __ldcg(p.draws + i) : -1ll;
    if (threadIdx.x == 0) *p.accepted = static_cast<int>(accepted);
}

}  // namespace zk
