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
// row's sum, added in three limbs of 17 bits by 32-bit atomics: its sums do not depend on the order in which threads add to a bin.  Sums of exponentials are
// added in a fixed order.
// What bounds it: the double-precision instructions of exp, and a dozen cluster barriers.
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

// What a CTA hands to the others.
struct VerifyShare {
    double sum;
    unsigned long long ties;
    uint32_t top_key, low_key, count;
};

template <int kCtas>
__global__ void __launch_bounds__(kVerifyThreads) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t verify_smem[];
    __shared__ VerifyShare share;
    __shared__ double warp_sum[32], s_q;
    __shared__ unsigned long long warp_total[32], s_left;
    __shared__ uint32_t warp_count[32], s_bin, s_mine;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), row = blockIdx.y;
    double* e = reinterpret_cast<double*>(verify_smem);                      // [per_cta]
    float* v = reinterpret_cast<float*>(e + p.per_cta);                      // [per_cta], per_cta a multiple of four
    uint32_t* limbs = reinterpret_cast<uint32_t*>(v + p.per_cta);            // [kVerifyLimbs][kVerifyBins]
    VerifyEntry* own_list = reinterpret_cast<VerifyEntry*>(limbs + kVerifyLimbs * kVerifyBins);
    VerifyEntry* all_list = own_list + kVerifyMine;
    const uint32_t base = rank * p.per_cta, n = base < p.vocab ? min(p.per_cta, p.vocab - base) : 0u;
    // a thread's run of consecutive entries, for sums in order of id (an odd number of them: no two lanes of a warp on one bank)
    const uint32_t per_thread = ((p.per_cta + kVerifyThreads - 1) / kVerifyThreads) | 1u, begin = min(n, tid * per_thread), end = min(n, begin + per_thread);
    pdl_launch_dependents();
    pdl_wait();
    const float* logits = p.logits + row * p.logits_ld + base;
    const bool is_draft = row < p.drafts;
    long long token = is_draft ? __ldcg(p.tokens + row) : -1;
    if (is_draft && (token < 0 || token >= static_cast<long long>(p.vocab))) {
        if (rank == 0 && tid == 0) atomicExch(p.error_word, kErrBadToken);
        token = -1;
    }

    // sums over the cluster, the same in every CTA: of a double a thread, in the order of threads and CTAs
    auto cluster_sum = [&](double mine) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_down_sync(0xffffffffu, mine, o);
        if (lane == 0) warp_sum[warp] = mine;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int w = 0; w < 32; ++w) s += warp_sum[w];
            share.sum = s;
        }
        cluster.sync();
        double s = 0.0;
        for (int r = 0; r < kCtas; ++r) s += cluster.map_shared_rank(&share, r)->sum;
        cluster.sync();
        return s;
    };

    // the logits, the largest of the finite ones and how many there are
    uint32_t top = 0, finite = 0;
    for (uint32_t i = tid; i < n; i += kVerifyThreads) {
        const float x = __ldcg(logits + i) + 0.0f;      // the zeros are equal
        const uint32_t key = sample_key(x);
        v[i] = x;
        top = max(top, key);
        finite += key != 0u;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    finite = __reduce_add_sync(0xffffffffu, finite);
    if (tid == 0) { share.top_key = 0; share.count = 0; }
    __syncthreads();
    if (lane == 0) { atomicMax(&share.top_key, top); atomicAdd(&share.count, finite); }
    cluster.sync();
    top = 0;
    finite = 0;
    for (int r = 0; r < kCtas; ++r) { top = max(top, cluster.map_shared_rank(&share, r)->top_key); finite += cluster.map_shared_rank(&share, r)->count; }
    cluster.sync();
    if (!finite) {
        if (rank == 0 && tid == 0) {
            p.draws[row] = -1;
            p.fits[row] = 0;
            if (is_draft && p.probs) p.probs[row] = 0.0;
        }
        return;
    }
    const double highest = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
    auto drop = [&](uint32_t i, bool with_exponentials) {
        v[i] = NAN;
        if (with_exponentials) e[i] = 0.0;
    };
    // the largest and the smallest key of the entries that take part, over the cluster
    auto key_range = [&](uint32_t& high, uint32_t& low) {
        high = __reduce_max_sync(0xffffffffu, high);
        low = __reduce_min_sync(0xffffffffu, low);
        if (tid == 0) { share.top_key = 0; share.low_key = 0xffffffffu; }
        __syncthreads();
        if (lane == 0) { atomicMax(&share.top_key, high); atomicMin(&share.low_key, low); }
        cluster.sync();
        for (int r = 0; r < kCtas; ++r) { high = max(high, cluster.map_shared_rank(&share, r)->top_key); low = min(low, cluster.map_shared_rank(&share, r)->low_key); }
        cluster.sync();
    };
    auto value_of = [](uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); };
    // Of the entries that equal `border` all behind the first `ties` (in order of id) go, and so do all below it.
    auto cut_ties = [&](uint32_t border, unsigned long long ties, bool with_exponentials) {
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
        for (uint32_t r = 0; r < rank; ++r) seen += cluster.map_shared_rank(&share, r)->ties;
        cluster.sync();
        for (uint32_t i = begin; i < end; ++i) {
            const uint32_t key = sample_key(v[i]);
            if (key < border || (key == border && seen++ >= ties)) drop(i, with_exponentials);
        }
        __syncthreads();
    };
    // Leaves the shortest run of entries, in descending order (equal values: the lowest ids), whose weights reach `wanted` > 0, at least one.
    // weigh(i): an entry's weight.  low: no entry that takes part is below it.
    auto cut = [&](unsigned long long wanted, auto weigh, uint32_t low, double reach, bool with_exponentials) {
        uint32_t high = top;
        double v_low = fmax(static_cast<double>(value_of(low)), highest - reach);       // far below, nothing is worth bins of its own
        for (;;) {
            if (high == low) {         // equal values: so many of them as are wanted, each of the same weight
                if (tid == 0) share.count = 0;
                __syncthreads();
                unsigned long long each = 0;
                for (uint32_t i = tid; i < n; i += kVerifyThreads) if (sample_key(v[i]) == high) each = weigh(i);
                if (each) atomicExch(&s_left, each);
                if (each && !share.count) share.count = 1;
                cluster.sync();
                for (int r = 0; r < kCtas; ++r) if (cluster.map_shared_rank(&share, r)->count) each = *cluster.map_shared_rank(&s_left, r);
                cluster.sync();
                each = max(each, 1ull);
                cut_ties(high, (wanted + each - 1) / each, with_exponentials);
                return;
            }
            const double v_high = value_of(high), per = kVerifyBins / (v_high - v_low);
            auto bin_of = [&](float x) { return static_cast<uint32_t>(fmin((v_high - static_cast<double>(x)) * per, kVerifyBins - 1.0)); };
            for (uint32_t i = tid; i < kVerifyLimbs * kVerifyBins; i += kVerifyThreads) limbs[i] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += kVerifyThreads) {
                const uint32_t key = sample_key(v[i]);
                if (!key || key > high || key < low) continue;
                const unsigned long long w = weigh(i);
                const uint32_t bin = bin_of(v[i]);
#pragma unroll
                for (int k = 0; k < kVerifyLimbs; ++k) {
                    uint32_t limb = static_cast<uint32_t>(w >> (k * kVerifyLimbBits));
                    if (k + 1 < kVerifyLimbs) limb &= (1u << kVerifyLimbBits) - 1u;          // an entry may be all of the row: 2^51
                    if (limb) atomicAdd(limbs + k * kVerifyBins + bin, limb);
                }
            }
            cluster.sync();
            // thread j has bin j of the whole row
            unsigned long long mine = 0;
            for (int r = 0; r < kCtas; ++r) {
                const uint32_t* its = cluster.map_shared_rank(limbs, r) + tid;
#pragma unroll
                for (int k = 0; k < kVerifyLimbs; ++k) mine += static_cast<unsigned long long>(its[k * kVerifyBins]) << (k * kVerifyLimbBits);
            }
            unsigned long long upto = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
                if (static_cast<int>(lane) >= o) upto += x;
            }
            if (lane == 31) warp_total[warp] = upto;
            if (tid == 0) { s_bin = 0xffffffffu; s_left = wanted; s_mine = 0; }
            __syncthreads();
            unsigned long long before = 0;
            for (uint32_t w = 0; w < warp; ++w) before += warp_total[w];
            upto += before;
            if (upto >= wanted && upto - mine < wanted) { s_bin = tid; s_left = wanted - (upto - mine); }        // one thread at most
            cluster.sync();                                                                                       // and everybody has read the limbs
            if (s_bin == 0xffffffffu) {      // rounding left the whole short of what is wanted: everything stays
                for (uint32_t i = tid; i < n; i += kVerifyThreads) if (sample_key(v[i]) < low) drop(i, with_exponentials);
                cluster.sync();
                return;
            }
            const uint32_t border = s_bin;
            wanted = s_left;
            // what lies below the border goes; the entries of its bin are listed, and counted on where there are too many
            uint32_t bin_high = 0, bin_low = 0xffffffffu;
            for (uint32_t i = tid; i < n; i += kVerifyThreads) {
                const uint32_t key = sample_key(v[i]);
                if (!key || key > high) continue;
                const uint32_t bin = key < low ? kVerifyBins : bin_of(v[i]);
                if (bin > border) drop(i, with_exponentials);
                if (bin != border) continue;
                bin_high = max(bin_high, key);
                bin_low = min(bin_low, key);
                const uint32_t at = atomicAdd(&s_mine, 1u);
                if (at < kVerifyMine) own_list[at] = VerifyEntry{weigh(i), v[i], base + i};
            }
            __syncthreads();
            if (tid == 0) share.count = s_mine;
            cluster.sync();
            uint32_t count = 0, before_mine = 0;
            bool fits = true;
            for (uint32_t r = 0; r < kCtas; ++r) {
                const uint32_t its = cluster.map_shared_rank(&share, r)->count;
                fits &= its <= kVerifyMine;
                if (r < rank) before_mine += its;
                count += its;
            }
            if (!fits || count > kVerifyAll) {
                cluster.sync();
                key_range(bin_high, bin_low);
                high = bin_high;
                low = bin_low;
                v_low = value_of(low);
                continue;
            }
            for (uint32_t r = 0, at = 0; r < kCtas; ++r) {
                const uint32_t its = cluster.map_shared_rank(&share, r)->count;
                if (tid < its) all_list[at + tid] = cluster.map_shared_rank(own_list, r)[tid];
                at += its;
            }
            cluster.sync();
            // a warp decides an entry of the CTA's: it stays when what comes before it does not reach what is wanted
            for (uint32_t i = warp; i < s_mine; i += 32) {
                const VerifyEntry me = all_list[before_mine + i];
                unsigned long long sum = 0;
                for (uint32_t j = lane; j < count; j += 32) {
                    const VerifyEntry its = all_list[j];
                    if (its.value > me.value || (its.value == me.value && its.id < me.id)) sum += its.weight;
                }
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0 && sum >= wanted) drop(me.id - base, with_exponentials);
            }
            __syncthreads();
            return;
        }
    };

    const bool greedy = p.temperature == 0.0;
    const uint32_t top_k = greedy ? 1u : p.top_k;
    const double temperature = greedy ? 1.0 : p.temperature;
    // the smallest key of a row is asked for once, by its first cut
    uint32_t least = 0xffffffffu;
    auto least_key = [&]() {
        for (uint32_t i = tid; i < n; i += kVerifyThreads) {
            const uint32_t key = sample_key(v[i]);
            if (key) least = min(least, key);
        }
        uint32_t ignored = 0;
        key_range(ignored, least);
        return least;
    };
    if (top_k && top_k < finite) cut(top_k, [](uint32_t) { return 1ull; }, least_key(), 64.0 * temperature, false);
    double mine = 0.0;
    for (uint32_t i = begin; i < end; ++i) {
        const float x = v[i];
        const double w = sample_key(x) ? exp((static_cast<double>(x) - highest) / temperature) : 0.0;
        e[i] = w;
        mine += w;
    }
    double sum = cluster_sum(mine);
    if (!greedy && p.top_p > 0.0f && p.top_p < 1.0f) {
        const double unit = kVerifyUnit / sum;
        least = 0xffffffffu;
        cut(max(1ll, __double2ll_ru(static_cast<double>(p.top_p) * kVerifyUnit)), [&](uint32_t i) { return static_cast<unsigned long long>(__double2ll_rn(e[i] * unit)); }, least_key(),
            64.0 * temperature, true);
        mine = 0.0;
        for (uint32_t i = begin; i < end; ++i) mine += e[i];
        sum = cluster_sum(mine);
    }
    // e becomes p, then p - q
    for (uint32_t i = begin; i < end; ++i) e[i] /= sum;
    if (tid == 0) s_q = 0.0;
    __syncthreads();
    const uint32_t entries = is_draft && p.q_ids ? static_cast<uint32_t>(min(max(__ldcg(p.q_count + row), 0), static_cast<int>(kSampleMaxCandidates))) : 0u;
    const size_t list = static_cast<size_t>(row) * kSampleMaxCandidates;
    if (is_draft && token >= 0 && token / p.per_cta == rank) {       // the CTA that has the draft decides
        if (p.q_ids) {
            for (uint32_t j = tid; j < entries; j += kVerifyThreads)
                if (__ldcg(p.q_ids + list + j) == token) s_q = __ldcg(p.q_probs + list + j);
            __syncthreads();
        }
        if (tid == 0) {
            const double mine_p = e[token - base], q = p.q_ids ? s_q : 1.0;
            p.fits[row] = __ldcg(p.uniforms + row) * q < mine_p;
            if (p.probs) p.probs[row] = mine_p;
        }
        __syncthreads();
    } else if (is_draft && token < 0 && rank == 0 && tid == 0) {
        p.fits[row] = 0;
        if (p.probs) p.probs[row] = 0.0;
    }
    // what is left, and whether anything is: a copy of p is not kept, a row with nothing left is formed anew
    double left = 0.0;
    if (is_draft) {
        if (p.q_ids) {
            for (uint32_t j = tid; j < entries; j += kVerifyThreads) {
                const int id = __ldcg(p.q_ids + list + j);
                if (id >= 0 && static_cast<uint32_t>(id) >= base && static_cast<uint32_t>(id) - base < n) e[id - base] = fmax(e[id - base] - __ldcg(p.q_probs + list + j), 0.0);
            }
        } else if (tid == 0 && token >= 0 && token / p.per_cta == rank) {
            e[token - base] = fmax(e[token - base] - 1.0, 0.0);
        }
        __syncthreads();
    }
    for (uint32_t i = begin; i < end; ++i) left += e[i];
    double whole = cluster_sum(left);
    if (!(whole > 0.0)) {
        left = 0.0;
        for (uint32_t i = begin; i < end; ++i) {
            const float x = v[i];
            e[i] = sample_key(x) ? exp((static_cast<double>(x) - highest) / temperature) / sum : 0.0;
            left += e[i];
        }
        __syncthreads();
        whole = cluster_sum(left);
    }
    // the draw: the first entry with a share whose cumulative sum, in order of id, reaches u of the whole; where rounding leaves the last
    // sum short of it, the last such entry
    double upto = left;
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, upto, o);
        if (static_cast<int>(lane) >= o) upto += x;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    double before = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) before = 0.0;
    double warps = 0.0;
    for (uint32_t w = 0; w < warp; ++w) warps += warp_sum[w];
    if (tid == kVerifyThreads - 1) share.sum = warps + upto;
    cluster.sync();
    double ctas = 0.0, all = 0.0;
    for (int r = 0; r < kCtas; ++r) {
        const double s = cluster.map_shared_rank(&share, r)->sum;
        if (r < static_cast<int>(rank)) ctas += s;
        all += s;
    }
    const double goal = __ldcg(p.uniforms + p.drafts) * all;
    double run = ctas + (warps + before);
    int found = 0x7fffffff, last = -1;
    for (uint32_t i = begin; i < end; ++i) {
        if (e[i] <= 0.0) continue;
        run += e[i];
        last = static_cast<int>(base + i);
        if (run >= goal) { found = last; break; }
    }
    found = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(found)));
    last = __reduce_max_sync(0xffffffffu, last);
    if (tid == 0) { share.top_key = 0x7fffffffu; share.count = 0; }
    __syncthreads();
    if (lane == 0) { atomicMin(&share.top_key, static_cast<uint32_t>(found)); atomicMax(&share.count, static_cast<uint32_t>(last + 1)); }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        uint32_t first = 0x7fffffffu, end_of = 0;
        for (int r = 0; r < kCtas; ++r) {
            first = min(first, cluster.map_shared_rank(&share, r)->top_key);
            end_of = max(end_of, cluster.map_shared_rank(&share, r)->count);
        }
        p.draws[row] = first != 0x7fffffffu ? static_cast<long long>(first) : static_cast<long long>(end_of) - 1;
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
