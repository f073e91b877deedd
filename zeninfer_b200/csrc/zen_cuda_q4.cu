// C-ABI of the 4-bit key/value cache and of the check of drafted tokens (include/zen_cuda.h): argument checks and launches.
#include "../../include/zen_cuda.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <unordered_map>

#include "host_state.h"
#include "q4_attention.cuh"
#include "q4_cache.cuh"
#include "q4_prompt.cuh"
#include "q4_received.cuh"
#include "q4_step.cuh"
#include "verify_drafts.cuh"

namespace zk_host {
bool set_q4_wait_budget(long long cycles) { return cudaMemcpyToSymbol(zk::g_wait_budget_cycles, &cycles, sizeof cycles) == cudaSuccess; }
}  // namespace zk_host

namespace {

using zk_host::Entry;

template <typename... KArgs, typename... Args>
cudaError_t launch(const Entry& e, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, unsigned cluster, Args... args) {
    if (smem > 24 * 1024 || cluster > 8) {      // without an opt-in a block has 48 KB, what it declares statically among them
        static std::unordered_map<const void*, size_t> allowed;      // what the kernels of this signature may use so far; under the Entry's lock
        auto at = allowed.find(reinterpret_cast<const void*>(kernel));
        if (at == allowed.end() || smem > at->second) {
            cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (r == cudaSuccess && cluster > 8) r = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (r != cudaSuccess) return r;
            allowed[reinterpret_cast<const void*>(kernel)] = smem;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = e.stream;
    cudaLaunchAttribute attr[2]{};
    unsigned count = 0;
    if (e.pdl) {
        attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[count++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster) {
        attr[count].id = cudaLaunchAttributeClusterDimension;
        attr[count].val.clusterDim.x = cluster;
        attr[count].val.clusterDim.y = attr[count].val.clusterDim.z = 1;
        ++count;
    }
    cfg.attrs = attr;
    cfg.numAttrs = count;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

uint32_t u32(size_t v) { return static_cast<uint32_t>(v); }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

bool cache_ok(const zen_cuda_q4_cache* c) {
    return c && c->k_codes && c->v_codes && c->k_scales && c->v_scales && aligned16(c->k_codes) && aligned16(c->v_codes) && aligned16(c->k_scales) && aligned16(c->v_scales) &&
           c->kv_heads && c->kv_heads <= 65535 && c->head_dim && c->head_dim % zk::kQ4Block == 0 && c->head_dim <= zk::kQ4Block * zk::kQ4MaxBlocks && c->slots &&
           c->slots % 32 == 0 && c->slots <= 0x40000000u;
}
zk::Q4Cache device_form(const zen_cuda_q4_cache& c) {
    return zk::Q4Cache{c.k_codes, c.v_codes, reinterpret_cast<__half*>(c.k_scales), reinterpret_cast<__half*>(c.v_scales), c.kv_heads, c.head_dim / zk::kQ4Block, c.slots};
}

constexpr size_t kSms = 148, kWaveCtas = 2 * kSms;
// 128 slots a CTA of q4_received.cuh up to one CTA an SM, 256 above: a tile of rows out of L2 then serves both (8192 slots of 8 kv heads: 111 us, 131 with 128).
constexpr size_t kReceivedSingle = kSms;
constexpr size_t kOneRun = 8, kOneRunRows = 1024;      // tiles of a cache that q4_prompt.cuh does not split for more than so many rows of all kv heads
// Above so many rows of a kv head: q4_prompt.cuh, whose time hardly depends on them.  Heads of 128, 12 rows: 39 us by q4_attention.cuh and 50 by q4_prompt.cuh at 20000 slots, 20 rows:
// 56 and 50 (31 and 26 at 4003); heads of 64, 17 rows: 56 and 68, 24 rows: 23.4 and 23.2.
constexpr size_t prompt_rows(size_t blocks) { return blocks == 2 ? 24 : 16; }

// How a call is cut up, from its sizes alone: how many slots are filled is known on the device only.
struct AttentionPlan {
    int columns{};
    uint32_t rows{}, padded{}, row_warps{}, cta_rows{}, row_ctas{}, splits{}, key_warps{}, cluster{}, run_tile{zk::kQ4Tile};
    bool keep_scores{};
    size_t part_out{}, part_stats{}, scores{}, stats{}, queries{}, factors{}, bytes{};      // offsets into the workspace, and its size; 0: not a call
};
AttentionPlan attention_plan(const zen_cuda_q4_attention* a, size_t tokens) {
    AttentionPlan n;
    if (!a || !cache_ok(&a->cache) || !a->heads || a->heads % a->cache.kv_heads || a->heads > 65535 || !tokens || tokens > a->cache.slots) return n;
    const size_t kv_heads = a->cache.kv_heads, rows = tokens * (a->heads / kv_heads), blocks = a->cache.head_dim / zk::kQ4Block, tiles = a->cache.slots / zk::kQ4Tile;
    if (tokens * a->heads > 0x1fffffffu / blocks) return n;      // what a launch counts in 32 bits
    n.columns = rows <= 4 ? zk::kQ4Digits : rows <= 8 || blocks > 4 ? zk::kQ4Rows8 : zk::kQ4Rows16;
    if ((blocks == 2 || blocks == 4) && rows > prompt_rows(blocks)) {
        const size_t row_tiles = (rows + zk::kQpRows - 1) / zk::kQpRows, key_tiles = (a->cache.slots + zk::kQpKeys - 1) / zk::kQpKeys;
        if (row_tiles > 65535) return n;
        n.columns = zk::kQ4Prompt;
        n.rows = u32(rows); n.cta_rows = zk::kQpRows; n.row_ctas = u32(row_tiles); n.padded = u32(row_tiles * zk::kQpRows); n.key_warps = 1; n.run_tile = zk::kQpKeys;
        // runs side by side until every SM has its CTA; a few tiles of many rows are one run, for joining many rows costs more than that saves (333 tokens of 16 heads, 7 tiles:
        // 34.4 us in one run, 37.5 in three; but 3 tokens of 32 heads, 8 tiles: 25.2 us in one, 18.0 in eight)
        n.splits = key_tiles <= kOneRun && rows * kv_heads > kOneRunRows ? 1u : u32(std::max<size_t>(1, std::min(kSms / (row_tiles * kv_heads), key_tiles)));
        n.keep_scores = a->weight_out && rows <= zk::kQ4KeptRows;
        size_t at = 0;
        auto take = [&](size_t bytes) { const size_t mine = at; at += up16(bytes); return mine; };
        if (n.splits > 1) n.part_out = take(kv_heads * n.splits * rows * a->cache.head_dim * sizeof(float));
        if (n.splits > 1 || n.keep_scores) n.part_stats = take(kv_heads * n.splits * rows * 2 * sizeof(float));
        if (n.keep_scores) n.scores = take(kv_heads * rows * a->cache.slots * sizeof(float));
        else if (a->weight_out) {
            n.stats = take(kv_heads * rows * sizeof(float));
            n.queries = take(kv_heads * row_tiles * 2 * zk::kQpRows * a->cache.head_dim * sizeof(uint16_t));
            n.factors = take(kv_heads * n.padded * sizeof(float));
        }
        n.bytes = std::max<size_t>(at, 16);
        return n;
    }
    const size_t per_warp = zk::q4_rows(n.columns), warps = zk::q4_warps(n.columns);
    size_t row_warps = 1;
    while (row_warps < warps && row_warps * per_warp < rows) row_warps *= 2;
    const size_t cta_rows = row_warps * per_warp, row_ctas = (rows + cta_rows - 1) / cta_rows;
    if (row_ctas > 65535) return n;
    if (a->weight_out && rows > zk::kQ4KeptRows && (a->cache.slots + zk::kReceivedSlots - 1) / zk::kReceivedSlots > 65535) return n;      // CTAs of the launch that adds them up, along y
    n.rows = u32(rows); n.padded = u32((rows + per_warp - 1) / per_warp * per_warp); n.row_warps = u32(row_warps); n.cta_rows = u32(cta_rows); n.row_ctas = u32(row_ctas);
    n.key_warps = u32(warps / row_warps);
    // runs of slots side by side until every SM has its CTAs, no run shorter than a tile a warp
    n.splits = u32(std::max<size_t>(1, std::min(kWaveCtas / (row_ctas * kv_heads), tiles / n.key_warps)));
    n.keep_scores = a->weight_out && rows <= zk::kQ4KeptRows;
    if (n.columns == zk::kQ4Digits && tiles <= 8 * n.key_warps * zk::kQ4ClusterTiles) {
        n.cluster = 1;
        while (n.cluster < 8 && n.cluster * n.key_warps < tiles) n.cluster *= 2;
        n.splits = n.cluster;
        n.bytes = 16;                 // what the call needs stays in shared memory
        return n;
    }
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t mine = at; at += up16(bytes); return mine; };
    if (n.splits > 1 || n.columns == zk::kQ4Digits) n.part_out = take(kv_heads * n.splits * rows * a->cache.head_dim * sizeof(float));
    if (n.splits > 1 || n.columns == zk::kQ4Digits || n.keep_scores) n.part_stats = take(kv_heads * n.splits * rows * 2 * sizeof(float));
    if (n.columns != zk::kQ4Digits) {
        n.queries = take(kv_heads * n.padded * blocks * 8 * sizeof(uint4));
        n.factors = take(kv_heads * n.padded * sizeof(float));
    }
    if (n.keep_scores) n.scores = take(kv_heads * rows * a->cache.slots * sizeof(float));
    else if (a->weight_out) n.stats = take(kv_heads * rows * sizeof(float));
    n.bytes = at;
    return n;
}

template <typename Run>
cudaError_t by_blocks(uint32_t blocks, Run run) {
    switch (blocks) {
    case 1: return run(std::integral_constant<int, 1>{});
    case 2: return run(std::integral_constant<int, 2>{});
    case 3: return run(std::integral_constant<int, 3>{});
    case 4: return run(std::integral_constant<int, 4>{});
    case 5: return run(std::integral_constant<int, 5>{});
    case 6: return run(std::integral_constant<int, 6>{});
    case 7: return run(std::integral_constant<int, 7>{});
    default: return run(std::integral_constant<int, 8>{});
    }
}

template <typename Run>
cudaError_t by_prompt_blocks(uint32_t blocks, Run run) { return blocks == 2 ? run(std::integral_constant<int, 2>{}) : run(std::integral_constant<int, 4>{}); }

struct Span {
    uintptr_t begin, end;
};
bool apart(const Span& a, const Span& b) { return a.end <= b.begin || b.end <= a.begin; }
Span span_of(const void* p, size_t bytes) { return Span{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes}; }

size_t verify_room(const zen_cuda_draft_check* c) {
    if (!c || !c->vocab || c->vocab > ZEN_CUDA_VERIFY_MAX_VOCAB || c->drafts > ZEN_CUDA_VERIFY_MAX_DRAFTS) return 0;
    return up16((size_t(c->drafts) + 1) * (sizeof(long long) + sizeof(int)));
}

}  // namespace

extern "C" {

size_t zen_cuda_q4_attention_workspace_bytes(const zen_cuda_q4_attention* a, size_t tokens) { return attention_plan(a, tokens).bytes; }

int zen_cuda_dev_q4_attention(const zen_cuda_q4_attention* a, const float* d_q, const float* d_k, const float* d_v, size_t tokens, float* d_out,
                              void* stream) {
    Entry e(stream);
    const AttentionPlan plan = attention_plan(a, tokens);
    if (!plan.bytes) return e.fail("dev_q4_attention: bad arguments (head_dim a multiple of 32 up to 256, slots a multiple of 32, heads a multiple of kv_heads, 1 .. slots tokens)");
    const size_t q_row = size_t(a->heads) * a->cache.head_dim, kv_row = size_t(a->cache.kv_heads) * a->cache.head_dim;
    if (!d_q || !d_k || !d_v || !d_out || !a->filled || (a->q_ld && a->q_ld < q_row) || (a->kv_ld && a->kv_ld < kv_row) || !std::isfinite(a->scale))
        return e.fail("dev_q4_attention: bad arguments (rows)");
    if (a->pairs && (a->pairs > a->cache.head_dim / 2 || !a->cos_t || !a->sin_t || !a->position || !a->positions)) return e.fail("dev_q4_attention: bad arguments (rotation)");
    if (!a->weight_in != !a->weight_out) return e.fail("dev_q4_attention: weight_in and weight_out go together");
    if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < plan.bytes) return e.fail("dev_q4_attention: the workspace is missing, not 16-byte aligned or too small");
    if (!e.ok) return 0;
    const zk::Q4Rotation turn{a->cos_t, a->sin_t, a->pairs, a->positions, a->adjacent ? 1u : 0u};
    const zk::Q4Cache cache = device_form(a->cache);
    uint8_t* room = static_cast<uint8_t*>(a->workspace);
    auto part = [&](size_t at) { return reinterpret_cast<float*>(room + at); };
    const bool digits = plan.columns == zk::kQ4Digits;
    zk::Q4Attend p{};
    p.cache = cache; p.turn = turn; p.q = d_q; p.k = d_k; p.v = d_v; p.k_held = a->k_held; p.v_held = a->v_held;
    p.position = a->position; p.filled = a->filled; p.weight_in = a->weight_in; p.weight_out = a->weight_out; p.out = d_out;
    p.tokens = u32(tokens); p.heads = a->heads; p.group = a->heads / cache.kv_heads; p.splits = plan.splits; p.row_warps = plan.row_warps; p.padded = plan.padded; p.run_tile = plan.run_tile;
    p.q_ld = a->q_ld ? a->q_ld : q_row; p.kv_ld = a->kv_ld ? a->kv_ld : kv_row; p.scale = a->scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(a->cache.head_dim)) : a->scale;
    p.error_word = e.d_error;
    if (plan.cluster) {
        return e.leave(by_blocks(cache.blocks, [&](auto blocks) {
            constexpr int kBlocks = decltype(blocks)::value;
            return launch(e, zk::q4_step_kernel<kBlocks, true>, dim3(plan.cluster, 1, cache.kv_heads), dim3(zk::kQ4StepWarps * 32), zk::q4_step_smem<kBlocks>(a->weight_out), plan.cluster, p);
        }), "dev_q4_attention");
    }
    p.part_out = part(plan.part_out); p.part_stats = part(plan.part_stats);
    if (plan.keep_scores) p.scores = part(plan.scores);
    else if (a->weight_out) p.stats = part(plan.stats);
    const bool prompt = plan.columns == zk::kQ4Prompt;
    if (prompt) {
        if (p.stats) { p.queries = reinterpret_cast<uint4*>(room + plan.queries); p.factors = part(plan.factors); }
        const size_t items = tokens * cache.kv_heads * 2 * cache.blocks, a_cta = zk::kQ4AppendThreads / 4;
        const cudaError_t r = by_prompt_blocks(cache.blocks, [&](auto blocks) {
            constexpr int kBlocks = decltype(blocks)::value;
            const cudaError_t appended = launch(e, zk::q4_append_kernel<kBlocks>, dim3(u32((items + a_cta - 1) / a_cta)), dim3(zk::kQ4AppendThreads), 0, 0, p);
            return appended != cudaSuccess ? appended : launch(e, zk::q4_prompt_kernel<kBlocks>, dim3(plan.splits, plan.row_ctas, cache.kv_heads), dim3(zk::kQpThreads), zk::q4_prompt_smem<kBlocks>(), 0, p);
        });
        if (!e.leave(r, "dev_q4_attention")) return 0;
    } else if (!digits) {
        p.queries = reinterpret_cast<uint4*>(room + plan.queries); p.factors = part(plan.factors);
        const cudaError_t r = by_blocks(cache.blocks, [&](auto blocks) {
            return launch(e, zk::q4_prepare_kernel<decltype(blocks)::value>, dim3(u32(tokens), cache.kv_heads), dim3(32 * std::min<uint32_t>(zk::kQ4PrepareWarps, 2 * cache.blocks + p.group)), 0, 0, p);
        });
        if (!e.leave(r, "dev_q4_attention: new slots")) return 0;
    }
    auto attend = [&](auto blocks, auto columns) {
        constexpr int kBlocks = decltype(blocks)::value, kColumns = decltype(columns)::value;
        return launch(e, zk::q4_attend_kernel<kBlocks, kColumns>, dim3(plan.splits, plan.row_ctas, cache.kv_heads), dim3(zk::q4_warps(kColumns) * 32), zk::q4_attend_smem<kBlocks, kColumns>(plan.row_warps), 0, p);
    };
    const cudaError_t r = prompt ? cudaSuccess : by_blocks(cache.blocks, [&](auto blocks) {
        constexpr int kBlocks = decltype(blocks)::value;
        if (digits) return launch(e, zk::q4_step_kernel<kBlocks, false>, dim3(plan.splits, 1, cache.kv_heads), dim3(zk::kQ4StepWarps * 32), zk::q4_step_smem<kBlocks>(false), 0, p);
        if constexpr (kBlocks <= 4) {
            if (plan.columns == zk::kQ4Rows16) return attend(blocks, std::integral_constant<int, zk::kQ4Rows16>{});
        }
        return attend(blocks, std::integral_constant<int, zk::kQ4Rows8>{});
    });
    if (!e.leave(r, "dev_q4_attention")) return 0;
    const bool join = plan.splits > 1 || digits;
    if (join || plan.keep_scores) {
        uint32_t parts = 1;      // warps of a row, while all of them are on the SMs at once: 5328 rows of three runs take 10 us with one, 21 with four
        while (parts < zk::kQ4FinishWarps && parts < plan.splits && size_t(plan.rows) * cache.kv_heads * parts * 2 <= kSms * 64) parts *= 2;
        const uint32_t a_cta = zk::kQ4FinishWarps / parts, join_ctas = join ? (plan.rows + a_cta - 1) / a_cta : 0;
        const uint32_t slot_ctas = plan.keep_scores ? (cache.slots + zk::kQ4FinishWarps * 32 - 1) / (zk::kQ4FinishWarps * 32) : 0;
        if (!e.leave(launch(e, zk::q4_finish_kernel, dim3(join_ctas + slot_ctas, cache.kv_heads), dim3(zk::kQ4FinishWarps * 32), 0, 0, p, plan.cta_rows, plan.key_warps, parts, join_ctas),
                     "dev_q4_attention: finish"))
            return 0;
    }
    if (!a->weight_out || plan.keep_scores) return 1;
    if (prompt) {
        const uint32_t tiles = (cache.slots + zk::kQrSlots - 1) / zk::kQrSlots, sets = size_t(tiles) * cache.kv_heads > kReceivedSingle ? zk::kQrSets : 1;
        return e.leave(by_prompt_blocks(cache.blocks, [&](auto blocks) {
            constexpr int kBlocks = decltype(blocks)::value;
            return launch(e, zk::q4_received_kernel<kBlocks>, dim3((tiles + sets - 1) / sets, cache.kv_heads), dim3(zk::kQrThreads), zk::q4_received_smem<kBlocks>(sets), 0, p, sets);
        }), "dev_q4_attention: weights");
    }
    return e.leave(by_blocks(cache.blocks, [&](auto blocks) {
        constexpr int kBlocks = decltype(blocks)::value;
        return launch(e, zk::q4_received_again_kernel<kBlocks>, dim3(zk::kReceivedCtas, (cache.slots + zk::kReceivedSlots - 1) / zk::kReceivedSlots, cache.kv_heads), dim3(zk::kReceivedWarps * 32),
                      zk::kReceivedStages * kBlocks * 64 * sizeof(uint4), 0, p);
    }), "dev_q4_attention: weights");
}

size_t zen_cuda_q4_cache_evict_workspace_bytes(const zen_cuda_q4_cache* from) {
    return cache_ok(from) ? size_t(from->kv_heads) * from->slots * sizeof(int) : 0;
}

int zen_cuda_dev_q4_cache_evict(const zen_cuda_q4_cache* from, const float* weight, const int32_t* filled, const zen_cuda_q4_cache* to, float* weight_to, size_t keep,
                                size_t keep_first, size_t keep_last, int32_t* kept, void* workspace, size_t workspace_bytes, void* stream) {
    Entry e(stream);
    if (!cache_ok(from) || !cache_ok(to) || from->kv_heads != to->kv_heads || from->head_dim != to->head_dim) return e.fail("dev_q4_cache_evict: bad arguments (caches)");
    if (!weight || !weight_to || !filled || !keep || keep > to->slots || keep_first > keep || keep_last > keep - keep_first)
        return e.fail("dev_q4_cache_evict: bad arguments (1 <= keep <= slots, keep_first + keep_last <= keep)");
    if (!workspace || !aligned16(workspace) || workspace_bytes < zen_cuda_q4_cache_evict_workspace_bytes(from))
        return e.fail("dev_q4_cache_evict: the workspace is missing, not 16-byte aligned or too small");
    const bool in_place = from->k_codes == to->k_codes && from->v_codes == to->v_codes && from->k_scales == to->k_scales && from->v_scales == to->v_scales &&
                          weight == weight_to && from->slots == to->slots;
    if (!in_place) {      // nothing that is read may be something that is written
        auto spans = [](const zen_cuda_q4_cache& c, const float* w, Span* s) {
            const size_t cells = size_t(c.kv_heads) * c.slots;
            s[0] = span_of(c.k_codes, cells * (c.head_dim / 2)); s[1] = span_of(c.v_codes, cells * (c.head_dim / 2));
            s[2] = span_of(c.k_scales, cells * (c.head_dim / 16)); s[3] = span_of(c.v_scales, cells * (c.head_dim / 16));
            s[4] = span_of(w, cells * sizeof(float));
        };
        Span read[5], written[5];
        spans(*from, weight, read);
        spans(*to, weight_to, written);
        for (const Span& r : read)
            for (const Span& w : written)
                if (!apart(r, w)) return e.fail("dev_q4_cache_evict: the two caches are neither the same nor apart");
    }
    if (!e.ok) return 0;
    const zk::Q4Evict p{device_form(*from), device_form(*to), weight, weight_to, filled, kept, static_cast<int*>(workspace), u32(keep), u32(keep_first), u32(keep_last), e.d_error};
    return e.leave(launch(e, zk::q4_evict_kernel, dim3(zk::kEvictCtas, from->kv_heads), dim3(zk::kEvictThreads), zk::kEvictListed * sizeof(int), 0, p), "dev_q4_cache_evict");
}

size_t zen_cuda_verify_drafts_workspace_bytes(const zen_cuda_draft_check* c) { return verify_room(c); }

int zen_cuda_dev_verify_drafts(const zen_cuda_draft_check* c, void* stream) {
    Entry e(stream);
    const size_t room = verify_room(c);
    if (!room) return e.fail("dev_verify_drafts: bad arguments (1 .. ZEN_CUDA_VERIFY_MAX_VOCAB entries, at most ZEN_CUDA_VERIFY_MAX_DRAFTS drafts)");
    if (!c->logits || c->logits_ld < c->vocab || (c->drafts && !c->tokens) || !c->uniforms || !c->out || !c->accepted || !c->q_ids != !c->q_probs || !c->q_ids != !c->q_count)
        return e.fail("dev_verify_drafts: bad arguments");
    if (!(c->temperature >= 0.0f) || !std::isfinite(c->temperature) || std::isnan(c->top_p)) return e.fail("dev_verify_drafts: the temperature is finite and not negative");
    if (!c->workspace || !aligned16(c->workspace) || c->workspace_bytes < room) return e.fail("dev_verify_drafts: the workspace is missing, not 16-byte aligned or too small");
    if (!e.ok) return 0;
    const uint32_t rows = c->drafts + 1;
    zk::VerifyParams p{};
    p.logits = c->logits; p.logits_ld = c->logits_ld; p.vocab = c->vocab; p.drafts = c->drafts;
    p.tokens = reinterpret_cast<const long long*>(c->tokens); p.q_ids = c->q_ids; p.q_probs = c->q_probs; p.q_count = c->q_count; p.uniforms = c->uniforms;
    p.temperature = c->temperature; p.top_k = c->top_k; p.top_p = c->top_p;
    p.out = reinterpret_cast<long long*>(c->out); p.accepted = c->accepted; p.probs = c->probs;
    p.draws = static_cast<long long*>(c->workspace); p.fits = reinterpret_cast<int*>(p.draws + rows); p.error_word = e.d_error;
    auto run = [&](auto ctas) {
        constexpr int kCtas = decltype(ctas)::value;
        p.per_cta = (c->vocab + kCtas - 1) / kCtas;
        p.per_cta = (p.per_cta + 3) & ~3u;
        return launch(e, zk::verify_rows_kernel<kCtas>, dim3(kCtas, rows), dim3(zk::kVerifyThreads), zk::verify_smem_bytes(p.per_cta), kCtas, p);
    };
    static_assert(ZEN_CUDA_VERIFY_MAX_VOCAB == 16 * zk::kVerifyRun, "what sixteen CTAs take");
    // sixteen CTAs a row where a run of eight would not fit shared memory
    const cudaError_t r = c->vocab > 8 * zk::kVerifyRun ? run(std::integral_constant<int, 16>{}) : run(std::integral_constant<int, 8>{});
    if (!e.leave(r, "dev_verify_drafts")) return 0;
    return e.leave(launch(e, zk::verify_answer_kernel, dim3(1), dim3(32), 0, 0, p), "dev_verify_drafts: answer");
}

}  // extern "C"
