// The bookkeeping of a speculative decoding step on gfx950: what a tree of drafted tokens needs
// besides its attention and its sampler. All lengths and choices stay on the device, so that a
// step can be captured into a graph.
//
// The tree: node i has the parent parents[i], -1 for a root; a parent comes before its children. A
// node whose parent is neither -1 nor an earlier node is unused, and so are its descendants.
#include "common.hpp"

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);

constexpr int kTreeMax = EFM_DRAFT_TREE_MAX_NODES;

// A node's ancestors are its own bit and those of its parent's set. Pointer doubling: after round r
// a node's word holds its 2^r nearest ancestors and `up` the next one, so a tree of depth D takes
// ceil(log2(D + 1)) rounds. A workgroup makes one 64-node column of the masks.
__global__ __launch_bounds__(kTreeMax) void draft_tree_plan_kernel(int n, const int32_t* parents, uint32_t kv_len,
                                                                   const uint32_t* d_kv_len, int32_t pos_offset, uint64_t* mask,
                                                                   int32_t* positions, int32_t position_stride) {
    __shared__ uint64_t s_set[2][kTreeMax];   // of this round and the last, so that a round has one barrier
    __shared__ int s_up[2][kTreeMax];
    __shared__ int s_depth[2][kTreeMax];   // ancestors in the set; unused nodes: negative
    const int i = threadIdx.x, word = blockIdx.x, words = gridDim.x;
    constexpr int kUnused = -(1 << 20);   // stays negative however many are added up
    const uint32_t len = d_kv_len != nullptr ? d_kv_len[0] : kv_len;
    const int p = i < n ? parents[i] : -1;
    const bool ok = p >= -1 && p < i && len >= (uint32_t)n;
    uint64_t set = i / 64 == word ? 1ull << (i % 64) : 0ull;
    int up = ok ? p : -1, depth = !ok ? kUnused : p >= 0 ? 1 : 0;
    for (int b = 0;; b ^= 1) {
        s_set[b][i] = set, s_up[b][i] = up, s_depth[b][i] = depth;
        if (!__syncthreads_or(up >= 0)) break;
        if (up >= 0) {
            set |= s_set[b][up];
            depth = max(depth + s_depth[b][up], kUnused);
            up = s_up[b][up];
        }
    }
    if (i >= n) return;
    if (mask != nullptr) mask[(size_t)i * words + word] = depth < 0 ? 0ull : set;
    if (positions != nullptr && word == 0) {
        const int pos = (int)((len >= (uint32_t)n ? len - (uint32_t)n : 0u) + (uint32_t)pos_offset + (uint32_t)max(depth, 0));
        for (int r = 0; r < 3; ++r) positions[(size_t)r * position_stride + i] = pos;
    }
}

// Every node looks for the parent that accepts it; what is left of the walk is a chain of LDS reads,
// one for each accepted node.
__global__ __launch_bounds__(kTreeMax) void draft_tree_accept_kernel(int n, const int32_t* parents, const int32_t* draft,
                                                                     const int32_t* target, const uint32_t* d_kv_len,
                                                                     uint32_t next_nodes, uint32_t* d_kv_len_out, int32_t* commit,
                                                                     int32_t* tokens) {
    __shared__ int s_next[kTreeMax];
    __shared__ int s_target[kTreeMax];
    __shared__ int s_path[kTreeMax];
    __shared__ int s_count;
    const int i = threadIdx.x;
    const uint32_t len = d_kv_len[0];
    int p = -1, d = -1;
    if (i < n) {
        p = parents[i];
        d = draft[i];
        s_target[i] = target[i];
    }
    s_next[i] = kTreeMax;
    __syncthreads();
    if (p >= 0 && p < i && d >= 0 && s_target[p] == d) atomicMin(&s_next[p], i);
    __syncthreads();
    if (i == 0) {
        int count = 0;
        if (len >= (uint32_t)n)
            for (int at = 0; at < kTreeMax; at = s_next[at]) s_path[count++] = at;   // a node's next is behind it
        s_count = count;
        commit[0] = len >= (uint32_t)n ? (int32_t)(len - (uint32_t)n) : 0;
        commit[1] = count;
        d_kv_len_out[0] = len >= (uint32_t)n ? len - (uint32_t)n + (uint32_t)count + next_nodes : len;
    }
    __syncthreads();
    if (i >= n) return;
    const bool on = i < s_count;
    commit[2 + i] = on ? s_path[i] : -1;
    if (tokens != nullptr) tokens[i] = on ? s_target[s_path[i]] : -1;
}

// Row base + path[i] of every layer's K and V goes to row base + i. A thread moves the same 16 bytes of all rows, in
// order; path[i] >= i and the path rises, so that no row is written before it is read. A path that does not rise so ends
// there. A wave holds 64 of the path's nodes, and its loads of 8 rows go out together: what bounds it is the chain of
// launch, path, rows and stores (28 layers of 4 heads of 128: 6.2 -> 3.4 us; the walk's one workgroup takes 2.0).
__global__ __launch_bounds__(kWave) void draft_tree_move_kernel(uint16_t* k, uint16_t* v, int64_t layer_stride, int64_t k_sn, int64_t k_sh,
                                                                int64_t v_sn, int64_t v_sh, int hd, int chunks, uint32_t max_rows, int n,
                                                                const int32_t* commit) {
    typedef uint32_t vec_t __attribute__((ext_vector_type(4)));
    constexpr int B = 8;   // rows under way
    const int lane = threadIdx.x, c = min((int)(blockIdx.x * kWave) + lane, chunks - 1);   // the last chunk again past the end
    int path = lane < n ? commit[2 + lane] : 0;
    const uint32_t base = (uint32_t)commit[0];
    int count = min(commit[1], n);
    if ((uint64_t)base + (uint64_t)n > max_rows) return;
    const bool is_v = blockIdx.z != 0;
    const int64_t sn = is_v ? v_sn : k_sn;
    const int head = c * 8 / hd;
    uint16_t* const at = (is_v ? v : k) + (int64_t)blockIdx.y * layer_stride + (int64_t)base * sn + head * (is_v ? v_sh : k_sh) + c * 8 % hd;
    int last = -1;
    for (int g = 0; g < count; g += kWave) {
        if (g > 0) path = g + lane < n ? commit[2 + g + lane] : 0;
        int before = __shfl_up(path, 1, kWave);
        before = lane == 0 ? last : before;
        const uint64_t ends = __ballot(!(path > before && path < n));
        if (ends != 0) count = min(count, g + __builtin_ctzll(ends));
        last = __builtin_amdgcn_readlane(path, kWave - 1);
        const int rows = min(count - g, kWave);
        for (int i0 = 0; i0 < rows; i0 += B) {
            vec_t x[B];
#pragma unroll
            for (int j = 0; j < B; ++j) x[j] = *reinterpret_cast<const vec_t*>(at + (int64_t)__builtin_amdgcn_readlane(path, min(i0 + j, rows - 1)) * sn);
#pragma unroll
            for (int j = 0; j < B; ++j) asm volatile("" : "+v"(x[j]));   // all of them before the first store
#pragma unroll
            for (int j = 0; j < B; ++j)
                if (i0 + j < rows && __builtin_amdgcn_readlane(path, i0 + j) != g + i0 + j)
                    *reinterpret_cast<vec_t*>(at + (int64_t)(g + i0 + j) * sn) = x[j];
        }
    }
}

static int tree_nodes_ok(const char* who, uint32_t nodes) {
    if (nodes == 0) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: a tree has a node at least", who);
    if (nodes > (uint32_t)kTreeMax) return set_error(EFM_ERR_UNSUPPORTED, "%s: %u nodes, %d at most", who, nodes, kTreeMax);
    return EFM_OK;
}

static bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

}  // namespace efm

using namespace efm;

extern "C" int efm_draft_tree_plan(uint32_t nodes, const int32_t* parents, uint32_t kv_len, const uint32_t* d_kv_len,
                                   int32_t pos_offset, uint64_t* mask, int32_t* positions, int32_t position_stride,
                                   hipStream_t stream) {
    const int rc = tree_nodes_ok("draft_tree_plan", nodes);
    if (rc) return rc;
    if (!parents || (!mask && !positions)) return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_plan: null pointer");
    if (misaligned(parents, 4) || misaligned(d_kv_len, 4) || misaligned(mask, 8) || misaligned(positions, 4))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_plan: misaligned pointer");
    if (d_kv_len == nullptr && kv_len < nodes)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_plan: kv_len %u below the %u nodes", kv_len, nodes);
    if (positions != nullptr && position_stride < (int32_t)nodes)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_plan: position_stride %d below the %u nodes", position_stride, nodes);
    const int threads = ((int)nodes + kWave - 1) / kWave * kWave;
    hipLaunchKernelGGL(draft_tree_plan_kernel, dim3(threads / 64), dim3(threads), 0, stream, (int)nodes, parents, kv_len, d_kv_len,
                       pos_offset, mask, positions, position_stride);
    return check_launch("draft_tree_plan");
}

extern "C" int efm_draft_tree_accept(uint32_t nodes, const int32_t* parents, const int32_t* draft_tokens,
                                     const int32_t* target_tokens, const uint32_t* d_kv_len, uint32_t next_nodes,
                                     uint32_t* d_kv_len_out, int32_t* commit, int32_t* tokens_out, hipStream_t stream) {
    const int rc = tree_nodes_ok("draft_tree_accept", nodes);
    if (rc) return rc;
    if (!parents || !draft_tokens || !target_tokens || !d_kv_len || !d_kv_len_out || !commit)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_accept: null pointer");
    if (misaligned(parents, 4) || misaligned(draft_tokens, 4) || misaligned(target_tokens, 4) || misaligned(d_kv_len, 4) ||
        misaligned(d_kv_len_out, 4) || misaligned(commit, 4) || misaligned(tokens_out, 4))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_accept: misaligned pointer");
    if (next_nodes > (uint32_t)kTreeMax)
        return set_error(EFM_ERR_UNSUPPORTED, "draft_tree_accept: %u next nodes, %d at most", next_nodes, kTreeMax);
    const int threads = ((int)nodes + kWave - 1) / kWave * kWave;
    hipLaunchKernelGGL(draft_tree_accept_kernel, dim3(1), dim3(threads), 0, stream, (int)nodes, parents, draft_tokens, target_tokens,
                       d_kv_len, next_nodes, d_kv_len_out, commit, tokens_out);
    return check_launch("draft_tree_accept");
}

extern "C" int efm_draft_tree_move_kv(const efm_attention_ctx* ctx, uint32_t layers, int64_t layer_stride, void* k_cache, void* v_cache,
                                      uint32_t max_rows, uint32_t nodes, const int32_t* commit, hipStream_t stream) {
    int rc = validate_attention_ctx(ctx, "draft_tree_move_kv");
    if (rc) return rc;
    rc = tree_nodes_ok("draft_tree_move_kv", nodes);
    if (rc) return rc;
    if (!k_cache || !v_cache || !commit) return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_move_kv: null pointer");
    if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(commit, 4))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_move_kv: misaligned pointer");
    if (layer_stride < 0 || (layer_stride == 0 && layers > 1))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_move_kv: layer_stride %lld", (long long)layer_stride);
    if (layer_stride % 8 != 0)
        return set_error(EFM_ERR_UNSUPPORTED, "draft_tree_move_kv: layer_stride must be a multiple of 8 elements");
    if (max_rows < nodes)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "draft_tree_move_kv: %u nodes in a cache of %u rows", nodes, max_rows);
    if (layers > 4096u || ctx->num_kv_heads > 4096u)   // a grid stays below 2^32 threads
        return set_error(EFM_ERR_UNSUPPORTED, "draft_tree_move_kv: %u layers of %u KV heads", layers, ctx->num_kv_heads);
    if (layers == 0) return EFM_OK;
    const int hd = (int)ctx->head_dim, chunks = (int)ctx->num_kv_heads * hd / 8;
    const int64_t row = (int64_t)ctx->num_kv_heads * hd;
    hipLaunchKernelGGL(draft_tree_move_kernel, dim3((chunks + kWave - 1) / kWave, layers, 2), dim3(kWave), 0, stream, static_cast<uint16_t*>(k_cache),
                       static_cast<uint16_t*>(v_cache), layer_stride, ctx->k_stride_n ? (int64_t)ctx->k_stride_n : row,
                       ctx->k_stride_h ? (int64_t)ctx->k_stride_h : hd, ctx->kv_stride_n ? (int64_t)ctx->kv_stride_n : row,
                       ctx->kv_stride_h ? (int64_t)ctx->kv_stride_h : hd, hd, chunks, max_rows, (int)nodes, commit);
    return check_launch("draft_tree_move_kv");
}
