// Drafted tokens against the model's own filtered distributions (the sampled form of a speculative block).
//
// A drafted token x of distribution q is accepted with probability min(1, p(x) / q(x)) and otherwise replaced by a draw from max(p - q, 0): the
// outcome is distributed as p.  p is what sample_pick.cuh draws from, of one row of logits: e_i = exp((v_i - max) / T) in double over the finite
// ones, cut to the top_k highest, then to the shortest run of the most likely whose share reaches top_p.
//
// A cluster takes a row and a CTA a run of the vocabulary, its logits and exponentials in shared memory.  Every row decides its own draft AND draws its
// own replacement, as if all drafts before it had been accepted, so that nothing waits for a decision: the rows run side by side, and one warp
// puts their answers together in a second launch.  The cuts are radix selects over order-preserving keys, four passes of eight bits: top_k over
// counts, top_p over masses.  A mass is an integer, the exponential times 2^62 / sum, so that its sums do not depend on the order in which
// threads add to a bin; sums of exponentials are added in a fixed order.
// What bounds it: about thirty double-precision instructions an entry for exp, and a dozen cluster barriers.
#pragma once
#include <cooperative_groups.h>

#include <cstdint>

#include "sample_key.cuh"
#include "zk_ptx.cuh"

namespace zk {

constexpr int kVerifyThreads = 1024;
constexpr double kVerifyUnit = 4611686018427387904.0;      // 2^62: the mass of a whole row

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
    uint32_t hist[256];
    unsigned long long mass[256];
    double sum;
    unsigned long long ties;
    uint32_t top_key, count;
};

template <int kCtas>
__global__ void __launch_bounds__(kVerifyThreads) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t verify_smem[];
    __shared__ VerifyShare share;
    __shared__ unsigned long long total[256];
    __shared__ double warp_sum[32], s_q;
    __shared__ uint32_t warp_count[32];
    __shared__ uint32_t s_prefix;
    __shared__ unsigned long long s_left;
    __shared__ int s_winner;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = cluster.block_rank(), row = blockIdx.y;
    double* e = reinterpret_cast<double*>(verify_smem);                      // [per_cta]
    float* v = reinterpret_cast<float*>(e + p.per_cta);                      // [per_cta]
    const uint32_t base = rank * p.per_cta, n = base < p.vocab ? min(p.per_cta, p.vocab - base) : 0u;
    // a thread's run of consecutive entries, for sums in order of id
    const uint32_t per_thread = (p.per_cta + kVerifyThreads - 1) / kVerifyThreads, begin = min(n, tid * per_thread), end = min(n, begin + per_thread);
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

    // The first entries in descending order whose weight reaches `wanted`: their last key, and the weight of those that equal it which is
    // still wanted.  weigh(i): an entry's weight, 0 for one that does not take part.
    uint32_t border = 0;
    auto select = [&](unsigned long long wanted, auto weigh) {
        if (tid == 0) { s_prefix = 0; s_left = wanted; }
        uint32_t mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) share.mass[tid] = 0;
            __syncthreads();
            const uint32_t prefix = s_prefix;
            for (uint32_t i = tid; i < n; i += kVerifyThreads) {
                const uint32_t key = sample_key(v[i]);
                const unsigned long long w = key && (key & mask) == prefix ? weigh(i) : 0ull;
                if (w) atomicAdd(&share.mass[(key >> shift) & 255u], w);
            }
            cluster.sync();
            if (tid < 256) {
                unsigned long long sum = 0;
                for (int r = 0; r < kCtas; ++r) sum += cluster.map_shared_rank(&share, r)->mass[tid];
                total[tid] = sum;
            }
            cluster.sync();
            if (warp == 0) {
                unsigned long long mine = 0;
                for (int j = 0; j < 8; ++j) mine += total[255 - 8 * lane - j];
                unsigned long long upto = mine;
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (static_cast<int>(lane) >= o) upto += x;
                }
                const unsigned long long left = s_left;
                uint32_t reached = __ballot_sync(0xffffffffu, upto >= left);
                // rounding may leave the whole a hair short of what is wanted: then the last bin that has any
                const uint32_t any = __ballot_sync(0xffffffffu, mine != 0ull);
                const int at = reached ? __ffs(reached) - 1 : 31 - __clz(any);
                if (static_cast<int>(lane) == at) {
                    unsigned long long rest = left - (upto - mine);
                    int bin = 255 - 8 * static_cast<int>(lane), last = bin;
                    for (int j = 0; j < 8; ++j, --bin) {
                        if (!total[bin]) continue;
                        last = bin;
                        if (total[bin] >= rest) break;
                        rest -= total[bin];
                    }
                    if (total[last] < rest || !reached) rest = total[last];
                    s_prefix = prefix | static_cast<uint32_t>(last) << shift;
                    s_left = rest;
                }
            }
            __syncthreads();
            mask |= 255u << shift;
        }
        border = s_prefix;
        const unsigned long long left = s_left;
        __syncthreads();
        return left;
    };
    // Entries that equal the border's key and come behind the first `ties` of them (in order of id) go: their value becomes NaN, the exponential 0;
    // so do all below the border.
    auto cut = [&](unsigned long long ties, bool with_exponentials) {
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
            if (key < border || (key == border && seen++ >= ties)) {
                v[i] = NAN;
                if (with_exponentials) e[i] = 0.0;
            }
        }
        __syncthreads();
    };

    const bool greedy = p.temperature == 0.0;
    const uint32_t top_k = greedy ? 1u : p.top_k;
    const double temperature = greedy ? 1.0 : p.temperature;
    if (top_k && top_k < finite) cut(select(top_k, [](uint32_t) { return 1ull; }), false);
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
        auto weigh = [&](uint32_t i) { return static_cast<unsigned long long>(__double2ll_rn(e[i] * unit)); };
        const unsigned long long wanted = max(1ll, __double2ll_ru(static_cast<double>(p.top_p) * kVerifyUnit));
        const unsigned long long rest = select(wanted, weigh);
        const float at = __uint_as_float(border & 0x80000000u ? border & 0x7fffffffu : ~border);
        const unsigned long long each = max(1ll, __double2ll_rn(exp((static_cast<double>(at) - highest) / temperature) * unit));
        cut((rest + each - 1) / each, true);
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
    if (tid == 0) s_winner = 0x7fffffff;
    __syncthreads();
    double before = upto - left;                    // replaced below by sums in a fixed order
    before = __shfl_up_sync(0xffffffffu, upto, 1);
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
