// ragged_attention.hip -- attention over a batch of requests of different
// lengths for gfx950: over a paged KV cache (a chunk of new tokens each,
// single tokens included) and over whole packed prompts.
//
// Rows are tokens: q [T, QH, D], request i owning rows offsets[i] ..
// offsets[i + 1].  Its query j has position first + j, first = context_i -
// n_i (paged) or 0 (packed), and sees the keys 0 .. first + j:
//   out = sum_k p_k v_k / sum_k p_k,  p_k = e^(scale q.k - max).
// Query head h reads KV head h / (QH / KVH).  The lengths live on the device
// only, so a recorded call follows them from replay to replay; the host knows
// bounds (rows, requests, the longest query and key range).
//
// What the device finds wrong stays inside the call: row ranges are clamped to
// the rows there are, a query that sees a key of a page outside the pool, and
// every query of a request whose context passes max_context, comes out as NaN;
// a query that sees no key (position below 0) as zeros.  Rows of no request
// are not written.
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <cmath>

namespace rl {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct RaggedParams {
    const uint32_t* offsets;  // [sequences + 1]
    const uint32_t* context;  // [sequences] (paged)
    const uint32_t* table;    // [sequences, max_blocks] (paged)
    uint32_t sequences;
    uint32_t tokens;
    uint32_t q_heads;
    uint32_t kv_heads;
    uint32_t group;  // query heads per KV head
    uint32_t head_dim;
    uint32_t max_queries;
    uint32_t max_context;
    uint32_t max_blocks;
    uint32_t pages;
    uint32_t shift;  // log2 of the page size
    uint64_t q_token, q_head;  // strides in elements
    uint64_t k_token, k_head;  // (packed)
    uint64_t v_token, v_head;
    float scale;
    float scale_log2;  // scale * log2(e)
};

// Request i as the device finds it.
struct Request {
    uint32_t begin;  // first row
    uint32_t n;      // rows
    uint32_t keys;
    int64_t first;  // position of the first row
    bool bad;       // more keys than max_context
};

template <bool PAGED>
__device__ inline Request load_request(const RaggedParams& p, uint32_t i) {
    Request r;
    r.begin = min(p.offsets[i], p.tokens);
    const uint32_t end = min(p.offsets[i + 1], p.tokens);
    r.n = end > r.begin ? min(end - r.begin, p.max_queries) : 0u;
    const uint32_t ctx = PAGED ? p.context[i] : r.n;
    r.bad = PAGED && ctx > p.max_context;
    r.keys = PAGED ? min(ctx, p.max_context) : ctx;
    r.first = int64_t(r.keys) - r.n;
    return r;
}

// The request that owns row t: the last one whose first row is not past it.
__device__ inline uint32_t find_request(const RaggedParams& p, uint32_t t) {
    uint32_t lo = 0, hi = p.sequences;  // offsets[lo] <= t < offsets[hi], as far as they ascend
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (p.offsets[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Element offset of a key's K row (with stride and head of K) or V row; kNoRow
// for a key of a page outside the pool.
constexpr uint64_t kNoRow = ~uint64_t(0);
template <bool PAGED>
__device__ inline uint64_t key_row(const RaggedParams& p, uint32_t request, uint32_t begin,
                                   uint32_t key, uint32_t kv_head, uint64_t token_stride,
                                   uint64_t head_stride) {
    if constexpr (PAGED) {
        const uint32_t page = p.table[uint64_t(request) * p.max_blocks + (key >> p.shift)];
        if (page >= p.pages) return kNoRow;
        const uint64_t row = ((uint64_t(page) * p.kv_heads + kv_head) << p.shift) +
                             (key & ((1u << p.shift) - 1));
        return row * p.head_dim;
    } else {
        return uint64_t(begin + key) * token_stride + kv_head * head_stride;
    }
}

// ------------------------------------------------- one wave per query row
//
// Any head size up to 512, any strides and alignment: keys 256 at a time, a
// lane's four dot products in order, the probabilities through LDS, lanes =
// output elements for the values.  Bound by the vector ALUs and by key rows
// read lane by lane.
template <typename T, int DT, bool PAGED>
__global__ __launch_bounds__(64) void k_ragged_rows(const T* __restrict__ q,
                                                    const T* __restrict__ k,
                                                    const T* __restrict__ v, T* __restrict__ out,
                                                    RaggedParams p) {
    constexpr int KEYS = 256;
    __shared__ float qs[64 * DT];
    __shared__ float ps[KEYS];
    __shared__ uint64_t vrow[KEYS];
    const uint32_t lane = threadIdx.x;
    const uint32_t t = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads;
    const uint32_t i = find_request(p, t);
    const Request r = load_request<PAGED>(p, i);
    if (t < r.begin || t - r.begin >= r.n) return;
    const uint32_t D = p.head_dim, kv_head = head / p.group;
    const int64_t position = r.first + (t - r.begin);
    const uint32_t key_end = position < 0 ? 0u : uint32_t(position) + 1;
#pragma unroll
    for (int e = 0; e < DT; ++e) {
        const uint32_t d = lane + 64 * e;
        qs[d] = d < D ? to_float(q[t * p.q_token + head * p.q_head + d]) : 0.0f;
    }
    __syncthreads();

    float o[DT], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < DT; ++e) o[e] = 0.0f;
    for (uint32_t base = 0; base < key_end; base += KEYS) {
        float s[KEYS / 64], mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < KEYS / 64; ++c) {
            const uint32_t key = base + lane + 64 * c;
            s[c] = -INFINITY;
            if (key < key_end) {
                const uint64_t row =
                    key_row<PAGED>(p, i, r.begin, key, kv_head, p.k_token, p.k_head);
                vrow[lane + 64 * c] =
                    key_row<PAGED>(p, i, r.begin, key, kv_head, p.v_token, p.v_head);
                if (row == kNoRow) {
                    s[c] = NAN;
                } else {
                    float dot = 0.0f;
                    for (uint32_t d = 0; d < D; ++d) dot += qs[d] * to_float(k[row + d]);
                    s[c] = dot * p.scale;
                }
            }
            mx = fmaxf(mx, s[c]);
        }
        const float m_new = fmaxf(m, wave_max_dpp(mx));
        const float shift = m_new == -INFINITY ? 0.0f : m_new;  // only masked or -inf scores yet
        const float alpha = exp_fast(m - shift);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < KEYS / 64; ++c) {
            const float e = exp_fast(s[c] - shift);
            ps[lane + 64 * c] = e;
            l += e;
        }
#pragma unroll
        for (int e = 0; e < DT; ++e) o[e] *= alpha;
        __syncthreads();
        const uint32_t n = min(uint32_t(KEYS), key_end - base);
        for (uint32_t j = 0; j < n; ++j) {
            const float pj = ps[j];
            const uint64_t row = vrow[j];
#pragma unroll
            for (int e = 0; e < DT; ++e) {
                const uint32_t d = lane + 64 * e;
                if (d < D) o[e] += pj * (row == kNoRow ? 0.0f : to_float(v[row + d]));
            }
        }
        __syncthreads();
    }
    l = wave_sum_dpp(l);
    const float inv = r.bad ? NAN : key_end == 0 ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < DT; ++e) {
        const uint32_t d = lane + 64 * e;
        if (d < D)
            out[(uint64_t(t) * p.q_heads + head) * D + d] = from_float<T>(o[e] * inv);
    }
}

// -------------------------------------------------------------- workspace

constexpr uint64_t kWorkspaceAlign = 256;

uint64_t workspace_bytes(const rl_context* ctx, uint64_t sequences, uint64_t tokens,
                         uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim) {
    (void)ctx, (void)sequences, (void)tokens, (void)q_heads, (void)kv_heads, (void)head_dim;
    return kWorkspaceAlign;
}

// ------------------------------------------------------------- validation

// Checks shared by both attentions, the rows' part.
rl_status check_batch(uint64_t sequences, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads,
                      uint64_t head_dim, uint64_t max_queries, float scale) {
    if (sequences == 0 || tokens == 0 || q_heads == 0 || head_dim == 0 || max_queries == 0)
        return fail(RL_ERR_INVALID_SHAPE, "attention dimensions must be greater than zero");
    if (kv_heads == 0 || q_heads % kv_heads != 0)
        return fail(RL_ERR_MODEL_FORMAT, "Q heads %llu must be divisible by non-zero KV heads %llu",
                    (unsigned long long)q_heads, (unsigned long long)kv_heads);
    if (sequences >= UINT32_MAX || tokens > UINT32_MAX || q_heads > UINT32_MAX ||
        max_queries > UINT32_MAX || tokens > UINT32_MAX / q_heads)
        return fail(RL_ERR_INVALID_SHAPE, "attention row count exceeds u32");
    if (head_dim > 512)
        return fail(RL_ERR_INVALID_SHAPE, "attention head size %llu exceeds 512",
                    (unsigned long long)head_dim);
    if (!(scale > 0.0f) || scale == INFINITY)
        return fail(RL_ERR_INVALID_SHAPE, "attention scale must be positive and finite, got %g",
                    double(scale));
    return RL_OK;
}

template <typename T, bool PAGED>
void launch_rows(rl_context* ctx, const T* q, const T* k, const T* v, T* out,
                 const RaggedParams& p) {
    const dim3 grid(p.tokens * p.q_heads), block(64);
    if (p.head_dim <= 64)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 1, PAGED>), grid, block, q, k, v, out, p);
    else if (p.head_dim <= 128)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 2, PAGED>), grid, block, q, k, v, out, p);
    else if (p.head_dim <= 256)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 4, PAGED>), grid, block, q, k, v, out, p);
    else
        RL_LAUNCH(ctx, (k_ragged_rows<T, 8, PAGED>), grid, block, q, k, v, out, p);
}

template <typename T>
rl_status packed_entry(rl_context* ctx, const char* name, const rl_buffer* q,
                       const uint64_t* q_dims, const uint64_t* q_strides, const rl_buffer* k,
                       const uint64_t* k_dims, const uint64_t* k_strides, const rl_buffer* v,
                       const uint64_t* v_dims, const uint64_t* v_strides,
                       const rl_buffer* offsets, uint64_t sequences, uint64_t max_queries,
                       float scale, const rl_buffer* out) {
    constexpr uint64_t es = sizeof(T);
    if (rl_status st = check_token_view("query", q, q_dims, q_strides, es)) return st;
    if (rl_status st = check_token_view("key", k, k_dims, k_strides, es)) return st;
    if (rl_status st = check_token_view("value", v, v_dims, v_strides, es)) return st;
    const uint64_t tokens = q_dims[0], q_heads = q_dims[1], kv_heads = k_dims[1], D = q_dims[2];
    if (k_dims[0] != tokens || k_dims[2] != D) return fail_shape_mismatch(q_dims, 3, k_dims, 3);
    for (int d = 0; d < 3; ++d)
        if (v_dims[d] != k_dims[d]) return fail_shape_mismatch(k_dims, 3, v_dims, 3);
    if (rl_status st = check_batch(sequences, tokens, q_heads, kv_heads, D, max_queries, scale))
        return st;
    if (rl_status st = check_u32("offsets", offsets, sequences + 1)) return st;
    if (rl_status st = check_output(out, tokens * q_heads * D, es, "packed attention")) return st;
    if (rl_status st = require_context(ctx)) return st;
    if (rl_status st = activate(ctx)) return st;

    RaggedParams p{};
    p.offsets = static_cast<const uint32_t*>(offsets->data);
    p.sequences = uint32_t(sequences);
    p.tokens = uint32_t(tokens);
    p.q_heads = uint32_t(q_heads);
    p.kv_heads = uint32_t(kv_heads);
    p.group = uint32_t(q_heads / kv_heads);
    p.head_dim = uint32_t(D);
    p.max_queries = uint32_t(max_queries);
    p.max_context = p.max_queries;
    p.q_token = q_strides[0];
    p.q_head = q_strides[1];
    p.k_token = k_strides[0];
    p.k_head = k_strides[1];
    p.v_token = v_strides[0];
    p.v_head = v_strides[1];
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    launch_rows<T, false>(ctx, static_cast<const T*>(q->data), static_cast<const T*>(k->data),
                          static_cast<const T*>(v->data), static_cast<T*>(out->data), p);
    return after_launch(ctx, name);
}

template <typename T>
rl_status paged_entry(rl_context* ctx, const char* name, const rl_buffer* q,
                      const rl_buffer* k_pages, const rl_buffer* v_pages, const rl_buffer* table,
                      const rl_buffer* offsets, const rl_buffer* context, uint64_t sequences,
                      uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                      uint64_t pages, uint64_t page_size, uint64_t max_blocks,
                      uint64_t max_queries, uint64_t max_context, float scale,
                      const rl_buffer* workspace, const rl_buffer* out) {
    constexpr uint64_t es = sizeof(T);
    if (rl_status st =
            check_batch(sequences, tokens, q_heads, kv_heads, head_dim, max_queries, scale))
        return st;
    if (rl_status st = check_pages(pages, page_size)) return st;
    if (max_blocks == 0 || max_context == 0)
        return fail(RL_ERR_INVALID_SHAPE, "attention dimensions must be greater than zero");
    if (max_blocks > UINT32_MAX || max_context >= UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "attention key range exceeds u32");
    if (max_context > max_blocks * page_size)
        return fail(RL_ERR_INVALID_SHAPE,
                    "a context of %llu exceeds a table row of %llu pages of %llu positions",
                    (unsigned long long)max_context, (unsigned long long)max_blocks,
                    (unsigned long long)page_size);
    if (rl_status st = check_buffer(q, "query")) return st;
    const uint64_t numel = tokens * q_heads * head_dim;
    if (q->byte_len != q->len * es)
        return fail(RL_ERR_UNSUPPORTED_DTYPE, "query buffer is not %s", es == 4 ? "F32" : "F16");
    if (q->len != numel)
        return fail(RL_ERR_INVALID_SHAPE, "query buffer has %llu elements, expected %llu",
                    (unsigned long long)q->len, (unsigned long long)numel);
    if (rl_status st = check_pool("key pages", k_pages, pages, kv_heads, page_size, head_dim, es))
        return st;
    if (rl_status st = check_pool("value pages", v_pages, pages, kv_heads, page_size, head_dim, es))
        return st;
    if (rl_status st = check_u32("block table", table, sequences * max_blocks)) return st;
    if (rl_status st = check_u32("offsets", offsets, sequences + 1)) return st;
    if (rl_status st = check_u32("context lengths", context, sequences)) return st;
    if (rl_status st = check_output(out, numel, es, "paged attention")) return st;
    if (rl_status st = check_buffer(workspace, "workspace")) return st;
    if (rl_status st = require_context(ctx)) return st;
    const uint64_t need = workspace_bytes(ctx, sequences, tokens, q_heads, kv_heads, head_dim);
    if (ctx->workspaces.count(workspace->data) == 0)
        return fail(RL_ERR_INVALID_ARGUMENT,
                    "the workspace is not one of rl_paged_attention_workspace on this context");
    if (ctx->workspaces[workspace->data] < need)
        return fail(RL_ERR_INVALID_SHAPE, "workspace has %llu bytes, expected %llu",
                    (unsigned long long)ctx->workspaces[workspace->data],
                    (unsigned long long)need);
    if (rl_status st = activate(ctx)) return st;

    RaggedParams p{};
    p.offsets = static_cast<const uint32_t*>(offsets->data);
    p.context = static_cast<const uint32_t*>(context->data);
    p.table = static_cast<const uint32_t*>(table->data);
    p.sequences = uint32_t(sequences);
    p.tokens = uint32_t(tokens);
    p.q_heads = uint32_t(q_heads);
    p.kv_heads = uint32_t(kv_heads);
    p.group = uint32_t(q_heads / kv_heads);
    p.head_dim = uint32_t(head_dim);
    p.max_queries = uint32_t(max_queries);
    p.max_context = uint32_t(max_context);
    p.max_blocks = uint32_t(max_blocks);
    p.pages = uint32_t(pages);
    p.shift = log2_of(page_size);
    p.q_token = q_heads * head_dim;
    p.q_head = head_dim;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    launch_rows<T, true>(ctx, static_cast<const T*>(q->data),
                         static_cast<const T*>(k_pages->data),
                         static_cast<const T*>(v_pages->data), static_cast<T*>(out->data), p);
    return after_launch(ctx, name);
}

rl_status workspace_entry(rl_context* ctx, uint64_t sequences, uint64_t tokens, uint64_t q_heads,
                          uint64_t kv_heads, uint64_t head_dim, rl_buffer* out) {
    if (out == nullptr) return fail(RL_ERR_INVALID_ARGUMENT, "output buffer pointer is null");
    *out = rl_buffer{nullptr, 0, 0};
    if (rl_status st = check_batch(sequences, tokens, q_heads, kv_heads, head_dim, 1, 1.0f))
        return st;
    if (rl_status st = require_context(ctx)) return st;
    if (ctx->capturing)
        return fail(RL_ERR_DEVICE, "a workspace cannot be made while recording a graph");
    const uint64_t bytes = workspace_bytes(ctx, sequences, tokens, q_heads, kv_heads, head_dim);
    rl_buffer made{nullptr, 0, 0};
    if (rl_status st = rl_buffer_empty(ctx, bytes, 1, &made)) return st;
    const hipError_t err = hipMemsetAsync(made.data, 0, bytes, ctx->stream);
    if (err != hipSuccess) {
        rl_buffer_release(ctx, &made);
        return fail(RL_ERR_DEVICE, "workspace: %s", hipGetErrorString(err));
    }
    ctx->workspaces[made.data] = bytes;
    *out = made;
    return RL_OK;
}

}  // namespace
}  // namespace rl

using namespace rl;

extern "C" {

rl_status rl_paged_attention_workspace(rl_context* ctx, uint64_t sequences, uint64_t tokens,
                                       uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                                       rl_buffer* out) {
    return guarded([&] {
        return workspace_entry(ctx, sequences, tokens, q_heads, kv_heads, head_dim, out);
    });
}

rl_status rl_paged_attention_f32(rl_context* ctx, const rl_buffer* q, const rl_buffer* k_pages,
                                 const rl_buffer* v_pages, const rl_buffer* block_table,
                                 const rl_buffer* offsets, const rl_buffer* context,
                                 uint64_t sequences, uint64_t tokens, uint64_t q_heads,
                                 uint64_t kv_heads, uint64_t head_dim, uint64_t pages,
                                 uint64_t page_size, uint64_t max_blocks, uint64_t max_queries,
                                 uint64_t max_context, float scale, const rl_buffer* workspace,
                                 const rl_buffer* out) {
    return guarded([&] {
        return paged_entry<float>(ctx, "paged_attention_f32", q, k_pages, v_pages, block_table,
                                  offsets, context, sequences, tokens, q_heads, kv_heads, head_dim,
                                  pages, page_size, max_blocks, max_queries, max_context, scale,
                                  workspace, out);
    });
}

rl_status rl_paged_attention_f16(rl_context* ctx, const rl_buffer* q, const rl_buffer* k_pages,
                                 const rl_buffer* v_pages, const rl_buffer* block_table,
                                 const rl_buffer* offsets, const rl_buffer* context,
                                 uint64_t sequences, uint64_t tokens, uint64_t q_heads,
                                 uint64_t kv_heads, uint64_t head_dim, uint64_t pages,
                                 uint64_t page_size, uint64_t max_blocks, uint64_t max_queries,
                                 uint64_t max_context, float scale, const rl_buffer* workspace,
                                 const rl_buffer* out) {
    return guarded([&] {
        return paged_entry<half_t>(ctx, "paged_attention_f16", q, k_pages, v_pages, block_table,
                                   offsets, context, sequences, tokens, q_heads, kv_heads,
                                   head_dim, pages, page_size, max_blocks, max_queries,
                                   max_context, scale, workspace, out);
    });
}

rl_status rl_packed_attention_f32(rl_context* ctx, const rl_buffer* q, const uint64_t* q_dims,
                                  const uint64_t* q_strides, const rl_buffer* k,
                                  const uint64_t* k_dims, const uint64_t* k_strides,
                                  const rl_buffer* v, const uint64_t* v_dims,
                                  const uint64_t* v_strides, const rl_buffer* offsets,
                                  uint64_t sequences, uint64_t max_queries, float scale,
                                  const rl_buffer* out) {
    return guarded([&] {
        return packed_entry<float>(ctx, "packed_attention_f32", q, q_dims, q_strides, k, k_dims,
                                   k_strides, v, v_dims, v_strides, offsets, sequences,
                                   max_queries, scale, out);
    });
}

rl_status rl_packed_attention_f16(rl_context* ctx, const rl_buffer* q, const uint64_t* q_dims,
                                  const uint64_t* q_strides, const rl_buffer* k,
                                  const uint64_t* k_dims, const uint64_t* k_strides,
                                  const rl_buffer* v, const uint64_t* v_dims,
                                  const uint64_t* v_strides, const rl_buffer* offsets,
                                  uint64_t sequences, uint64_t max_queries, float scale,
                                  const rl_buffer* out) {
    return guarded([&] {
        return packed_entry<half_t>(ctx, "packed_attention_f16", q, q_dims, q_strides, k, k_dims,
                                    k_strides, v, v_dims, v_strides, offsets, sequences,
                                    max_queries, scale, out);
    });
}

}  // extern "C"
