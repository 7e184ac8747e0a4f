// paged.hip -- a KV cache in pages for gfx950: the plan of a step (block
// tables, slots and positions from the requests' lengths) and the append
// (RoPE of Q and K, K and V to their slots).
//
// A page holds page_size positions of every KV head, [pages, KVH, page_size,
// D]: within a page each head's rows are contiguous, as in the [1, KVH,
// max_seq, D] cache of one sequence.  Request i's position p lives in page
// table[i, p / page_size], row p % page_size; slot = page * page_size + row.
// page_size is a power of two, so both are a shift and a mask.
#include "common.hpp"
#include "ragged.hpp"

#include <algorithm>

#pragma clang fp contract(off)

namespace rl {
namespace {

// ------------------------------------------------------------------- plan
//
// With c_i cached and n_i new tokens, page size P and B entries a table row:
//   o_i = sum_{j < i} n_j,  have_i = min(ceil(c_i / P), B),
//   need_i = min(ceil((c_i + n_i) / P), B) - have_i,  f_i = sum_{j < i} need_j,
//   table[i, have_i + k] = free[f_i + k] for k < need_i,
//   token o_i + j: position c_i + j.
// One launch: every workgroup scans the lengths (two sums, saturating at
// 2^32 - 1, which keeps them associative) in chunks of kPlanThreads requests
// and serves its own share of the requests and of the tokens, so that no
// workgroup waits for another's sums; the rescan reads 8 bytes a request out
// of L2.  Tokens find their request by a binary search in LDS.  The first
// position of a new page is always a new token's: that token writes the
// table entry.  Every other read of the table is of an entry that the plan
// does not write.  Bound by latency: two dependent reads (lengths, then
// table or free list) and the scan's two barriers: 3.3 us for 48 requests of one
// token, 4.5 for 480 with 49 thousand tokens (a call 5.3; 8.5 with a workgroup for
// 8192 tokens instead of 1024).
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PlanParams {
    uint32_t sequences;
    uint32_t tokens;
    uint32_t max_blocks;
    uint32_t free_pages;
    uint32_t pages;
    uint32_t shift;         // log2 of the page size
    uint32_t token_share;   // tokens and requests of a workgroup
    uint32_t request_share;
};

__device__ inline uint32_t add_sat(uint32_t a, uint32_t b) {
    return __builtin_elementwise_add_sat(a, b);
}

// Inclusive sum over the wave, saturating: within rows of 16 lanes, then
// each row's last lane into the rows after it.
__device__ inline uint32_t wave_scan_sat(uint32_t v) {
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xF, 0xF, false)));
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xF, 0xF, false)));
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xF, 0xF, false)));
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xF, 0xF, false)));
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xA, 0xF, false)));
    v = add_sat(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xC, 0xF, false)));
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(
    const uint32_t* __restrict__ cached, const uint32_t* __restrict__ fresh,
    const uint32_t* __restrict__ free_pages, uint32_t* table, uint32_t* __restrict__ offsets,
    uint32_t* __restrict__ context, uint32_t* __restrict__ slots, uint32_t* __restrict__ positions,
    uint32_t* __restrict__ taken, PlanParams p) {
    __shared__ uint32_t first_token[kPlanThreads];
    __shared__ uint32_t first_page[kPlanThreads];
    __shared__ uint32_t had[kPlanThreads];
    __shared__ uint32_t sums[2][kPlanWaves];
    const uint32_t t = threadIdx.x, wave = t / 64, lane = t % 64;
    const uint64_t token0 = uint64_t(blockIdx.x) * p.token_share;
    const uint64_t token_end = min(uint64_t(p.tokens), token0 + p.token_share);
    const uint64_t mine0 = uint64_t(blockIdx.x) * p.request_share;
    const uint64_t mine_end = min(uint64_t(p.sequences), mine0 + p.request_share);
    const uint64_t page_mask = (uint64_t(1) << p.shift) - 1;
    uint32_t tokens_before = 0, pages_before = 0;  // of the chunks before
    uint64_t next = token0;                        // first token not yet served

    for (uint64_t base = 0; base < p.sequences; base += kPlanThreads) {
        const uint64_t i = base + t;
        const bool live = i < p.sequences;
        const uint32_t c = live ? cached[i] : 0, n = live ? fresh[i] : 0;
        const uint64_t have = min((uint64_t(c) + page_mask) >> p.shift, uint64_t(p.max_blocks));
        const uint64_t whole =
            min((uint64_t(c) + n + page_mask) >> p.shift, uint64_t(p.max_blocks));
        const uint32_t need = uint32_t(whole - have);
        const uint32_t n_sum = wave_scan_sat(n), need_sum = wave_scan_sat(need);
        if (lane == 63) {
            sums[0][wave] = n_sum;
            sums[1][wave] = need_sum;
        }
        __syncthreads();
        uint32_t before = tokens_before, page_before = pages_before;
#pragma unroll
        for (uint32_t w = 0; w < kPlanWaves; ++w) {
            const uint32_t a = sums[0][w], b = sums[1][w];
            before = w < wave ? add_sat(before, a) : before;
            page_before = w < wave ? add_sat(page_before, b) : page_before;
            tokens_before = add_sat(tokens_before, a);
            pages_before = add_sat(pages_before, b);
        }
        // exclusive sums: the wave's inclusive ones from the lane before
        const uint32_t n_ex = uint32_t(__shfl_up(int(n_sum), 1, 64));
        const uint32_t need_ex = uint32_t(__shfl_up(int(need_sum), 1, 64));
        before = add_sat(before, lane ? n_ex : 0u);
        page_before = add_sat(page_before, lane ? need_ex : 0u);
        first_token[t] = before;
        first_page[t] = page_before;
        had[t] = c;
        if (live && i >= mine0 && i < mine_end) {
            offsets[i] = before;
            context[i] = add_sat(c, n);
        }
        __syncthreads();
        const uint64_t served = min(token_end, uint64_t(tokens_before));
        for (uint64_t tok = next + t; tok < served; tok += kPlanThreads) {
            // the last request of the chunk whose first token is not past it
            uint32_t at = 0;
#pragma unroll
            for (uint32_t step = kPlanThreads / 2; step != 0; step /= 2)
                at = first_token[at + step] <= tok ? at + step : at;
            const uint64_t row = base + at;
            const uint64_t pos = uint64_t(had[at]) + (tok - first_token[at]);
            const uint64_t block = pos >> p.shift;
            const uint64_t had_blocks = (uint64_t(had[at]) + page_mask) >> p.shift;
            uint32_t page = RL_NO_PAGE;
            if (block < p.max_blocks) {
                if (block < had_blocks) {
                    page = table[row * p.max_blocks + block];
                } else {
                    const uint64_t take = uint64_t(first_page[at]) + (block - had_blocks);
                    if (take < p.free_pages) page = free_pages[take];
                    if ((pos & page_mask) == 0) table[row * p.max_blocks + block] = page;
                }
            }
            const bool held = page < p.pages;
            slots[tok] = held ? (page << p.shift) + uint32_t(pos & page_mask) : RL_NO_SLOT;
            positions[tok] = held ? uint32_t(pos) : 0u;
        }
        next = max(next, served);
        __syncthreads();  // the chunk's sums may be replaced
        if (next >= token_end && base + kPlanThreads >= mine_end && blockIdx.x != 0) break;
    }
    // tokens behind the last request's
    for (uint64_t tok = next + t; tok < token_end; tok += kPlanThreads) {
        slots[tok] = RL_NO_SLOT;
        positions[tok] = 0;
    }
    if (blockIdx.x == 0 && t == 0) {  // has scanned every chunk
        offsets[p.sequences] = tokens_before;
        taken[0] = pages_before;
    }
}

// ------------------------------------------------------------------ append
//
// Per token t with position p and slot s, pairs (a, b) = (x[i], x[i + D/2]):
// (a cos - b sin, b cos + a sin) for Q into q_out and for K into row s of its
// pages, V copied to row s; each product and sum rounded by itself, as
// rl_rope_* does.  A thread holds N pairs' cos and sin (f32, 2 N values) and
// turns them for `kHeads` heads of its token, so that the tables (L2) cost
// 2 / kHeads times the bytes of an f16 row.  Lanes run along a row, then over
// heads: whole rows on consecutive lanes.  Bound by HBM: 35.2 us for 8223 tokens
// of 32/8 heads of 128 in f16 (206 MB, 5.9 TB/s; a plain copy of as much runs at
// 4.9), by its launch below some hundred tokens.
struct RowsView {
    uint64_t token_stride;
    uint64_t head_stride;
};

struct AppendParams {
    RowsView q, k, v;
    FastDiv packs;       // packs of N pairs in a row
    FastDiv head_steps;  // threads over the heads of one token
    uint32_t items;
    uint32_t q_heads;
    uint32_t kv_heads;
    uint32_t half_dim;
    uint32_t table_rows;
    uint32_t shift;
    uint64_t slots;  // of the whole pool
};

template <typename T, int N, int kHeads, bool STREAM_IN, bool STREAM_OUT>
__global__ __launch_bounds__(256) void k_paged_append(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const float* __restrict__ cos_table, const float* __restrict__ sin_table,
    const uint32_t* __restrict__ positions, const uint32_t* __restrict__ slots,
    T* __restrict__ q_out, T* __restrict__ k_pages, T* __restrict__ v_pages, AppendParams p) {
    typedef typename VecOf<T, N>::type V;
    typedef typename VecOf<float, N>::type VF;
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    if (item >= p.items) return;
    uint32_t rest, pack, token, step;
    p.packs.divmod(item, rest, pack);
    p.head_steps.divmod(rest, token, step);
    const uint32_t pair = pack * N;
    const uint32_t rotated = p.q_heads + p.kv_heads;
    const uint32_t heads = rotated + p.kv_heads;

    // every load before the first use: rows, then the token's place
    V a[kHeads], b[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const uint32_t head = step + uint32_t(j) * p.head_steps.divisor;
        if (head >= heads) continue;
        const T* src =
            head < p.q_heads ? q + token * p.q.token_stride + head * p.q.head_stride
            : head < rotated
                ? k + token * p.k.token_stride + (head - p.q_heads) * p.k.head_stride
                : v + token * p.v.token_stride + (head - rotated) * p.v.head_stride;
        const V* first = reinterpret_cast<const V*>(src + pair);
        const V* second = reinterpret_cast<const V*>(src + p.half_dim + pair);
        a[j] = STREAM_IN ? load_stream(first) : *first;
        b[j] = STREAM_IN ? load_stream(second) : *second;
    }
    const uint32_t position = positions[token], slot = slots[token];
    if (slot >= p.slots || position >= p.table_rows) return;
    const uint64_t t = uint64_t(position) * p.half_dim + pair;
    const VF c = *reinterpret_cast<const VF*>(cos_table + t);
    const VF s = *reinterpret_cast<const VF*>(sin_table + t);
    const uint32_t dim = 2 * p.half_dim;
    const uint64_t page = slot >> p.shift, row = slot & ((1u << p.shift) - 1);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const uint32_t head = step + uint32_t(j) * p.head_steps.divisor;
        if (head >= heads) continue;
        T* dst;
        if (head < p.q_heads) {
            dst = q_out + (uint64_t(token) * p.q_heads + head) * dim;
        } else {
            const bool is_k = head < rotated;
            const uint32_t kv = head - (is_k ? p.q_heads : rotated);
            dst = (is_k ? k_pages : v_pages) + (((page * p.kv_heads + kv) << p.shift) + row) * dim;
        }
        V x = a[j], y = b[j];
        if (head < rotated) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float first = to_float(a[j][e]), second = to_float(b[j][e]);
                x[e] = from_float<T>(first * c[e] - second * s[e]);
                y[e] = from_float<T>(second * c[e] + first * s[e]);
            }
        }
        V* first = reinterpret_cast<V*>(dst + pair);
        V* second = reinterpret_cast<V*>(dst + p.half_dim + pair);
        if constexpr (STREAM_OUT) {
            store_stream(first, x);
            store_stream(second, y);
        } else {
            *first = x;
            *second = y;
        }
    }
}

// ------------------------------------------------------------- validation

// A [tokens, heads, D] view (unit innermost stride) inside its buffer.
rl_status check_rows_view(const char* what, const rl_buffer* b, const uint64_t* dims,
                          const uint64_t* strides, uint64_t es) {
    if (rl_status st = check_buffer(b, what)) return st;
    if (dims == nullptr || strides == nullptr)
        return fail(RL_ERR_INVALID_ARGUMENT, "dims or strides is null");
    if (b->byte_len != b->len * es)
        return fail(RL_ERR_UNSUPPORTED_DTYPE, "%s buffer is not %s", what,
                    es == 4 ? "F32" : "F16");
    return RL_OK;
}

}  // namespace

rl_status check_token_view(const char* what, const rl_buffer* b, const uint64_t* dims,
                           const uint64_t* strides, uint64_t es) {
    if (rl_status st = check_rows_view(what, b, dims, strides, es)) return st;
    for (int d = 0; d < 3; ++d)
        if (dims[d] == 0)
            return fail(RL_ERR_INVALID_SHAPE, "shape dimensions must be greater than zero");
    if (strides[2] != 1)
        return fail(RL_ERR_NON_CONTIGUOUS, "%s rows need a unit innermost stride, got %llu", what,
                    (unsigned long long)strides[2]);
    unsigned __int128 last = 0;  // below 2^64 before each sum, so none wraps
    for (int d = 0; d < 3; ++d) {
        last += (unsigned __int128)(dims[d] - 1) * strides[d];
        if (last >= b->len)
            return fail(RL_ERR_INVALID_SHAPE,
                        "%s view reaches past the end of its %llu-element buffer", what,
                        (unsigned long long)b->len);
    }
    return RL_OK;
}

rl_status check_u32(const char* what, const rl_buffer* b, uint64_t len) {
    if (rl_status st = check_buffer(b, what)) return st;
    if (b->byte_len != b->len * sizeof(uint32_t))
        return fail(RL_ERR_UNSUPPORTED_DTYPE, "%s buffer is not U32", what);
    if (b->len != len)
        return fail(RL_ERR_INVALID_SHAPE, "%s buffer has %llu elements, expected %llu", what,
                    (unsigned long long)b->len, (unsigned long long)len);
    return RL_OK;
}

rl_status check_pages(uint64_t pages, uint64_t page_size) {
    if (pages == 0) return fail(RL_ERR_INVALID_SHAPE, "the page count must be greater than zero");
    if (page_size == 0 || (page_size & (page_size - 1)) != 0)
        return fail(RL_ERR_INVALID_SHAPE, "the page size must be a power of two, got %llu",
                    (unsigned long long)page_size);
    if (pages > UINT32_MAX || page_size > UINT32_MAX || pages * page_size > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "%llu pages of %llu positions exceed the u32 slots",
                    (unsigned long long)pages, (unsigned long long)page_size);
    return RL_OK;
}

rl_status check_pool(const char* what, const rl_buffer* b, uint64_t pages, uint64_t kv_heads,
                     uint64_t page_size, uint64_t head_dim, uint64_t es) {
    if (rl_status st = check_buffer(b, what)) return st;
    if (b->byte_len != b->len * es)
        return fail(RL_ERR_UNSUPPORTED_DTYPE, "%s buffer is not %s", what,
                    es == 4 ? "F32" : "F16");
    const unsigned __int128 want =
        (unsigned __int128)(pages * page_size) * ((unsigned __int128)kv_heads * head_dim);
    if (want != b->len)
        return fail(RL_ERR_INVALID_SHAPE,
                    "%s buffer has %llu elements, expected [%llu, %llu, %llu, %llu]", what,
                    (unsigned long long)b->len, (unsigned long long)pages,
                    (unsigned long long)kv_heads, (unsigned long long)page_size,
                    (unsigned long long)head_dim);
    return RL_OK;
}

uint32_t log2_of(uint64_t power) { return 63 - uint32_t(__builtin_clzll(power)); }

namespace {

rl_status plan_entry(rl_context* ctx, const rl_buffer* cached, const rl_buffer* fresh,
                     uint64_t sequences, const rl_buffer* free_pages, const rl_buffer* table,
                     uint64_t max_blocks, uint64_t pages, uint64_t page_size,
                     const rl_buffer* offsets, const rl_buffer* context, uint64_t tokens,
                     const rl_buffer* slots, const rl_buffer* positions, const rl_buffer* taken) {
    if (sequences == 0 || max_blocks == 0 || tokens == 0)
        return fail(RL_ERR_INVALID_SHAPE, "plan dimensions must be greater than zero");
    if (sequences >= UINT32_MAX || max_blocks > UINT32_MAX || tokens > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "plan dimension exceeds u32");
    if (rl_status st = check_pages(pages, page_size)) return st;
    if (rl_status st = check_u32("cached lengths", cached, sequences)) return st;
    if (rl_status st = check_u32("new lengths", fresh, sequences)) return st;
    if (rl_status st = check_buffer(free_pages, "free pages")) return st;
    if (rl_status st = check_u32("free pages", free_pages, free_pages->len)) return st;
    if (free_pages->len > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "plan dimension exceeds u32");
    if (rl_status st = check_u32("block table", table, sequences * max_blocks)) return st;
    if (rl_status st = check_u32("offsets", offsets, sequences + 1)) return st;
    if (rl_status st = check_u32("context lengths", context, sequences)) return st;
    if (rl_status st = check_u32("slots", slots, tokens)) return st;
    if (rl_status st = check_u32("positions", positions, tokens)) return st;
    if (rl_status st = check_u32("taken", taken, 1)) return st;
    if (rl_status st = require_context(ctx)) return st;
    if (rl_status st = activate(ctx)) return st;

    PlanParams p{};
    p.sequences = uint32_t(sequences);
    p.tokens = uint32_t(tokens);
    p.max_blocks = uint32_t(max_blocks);
    p.free_pages = uint32_t(free_pages->len);
    p.pages = uint32_t(pages);
    p.shift = log2_of(page_size);
    // a token a thread while that is at most two workgroups a CU
    const uint64_t groups = std::min<uint64_t>(
        ceil_div(std::max(tokens, sequences), kPlanThreads), 2 * uint64_t(ctx->num_cus));
    p.token_share = uint32_t(ceil_div(tokens, groups));
    p.request_share = uint32_t(ceil_div(sequences, groups));
    const auto u32 = [](const rl_buffer* b) { return static_cast<uint32_t*>(b->data); };
    RL_LAUNCH(ctx, k_paged_plan, dim3(unsigned(groups)), dim3(kPlanThreads), u32(cached),
              u32(fresh), u32(free_pages), u32(table), u32(offsets), u32(context), u32(slots),
              u32(positions), u32(taken), p);
    return after_launch(ctx, "paged_plan");
}

constexpr uint64_t kStreamRows = uint64_t(88) << 20;

template <typename T, int N>
void launch_append(rl_context* ctx, uint64_t tokens, uint64_t heads, AppendParams p, const T* q,
                   const T* k, const T* v, const float* cos_table, const float* sin_table,
                   const uint32_t* positions, const uint32_t* slots, T* q_out, T* k_pages,
                   T* v_pages) {
    const uint64_t packs = p.half_dim / N;
    p.packs = FastDiv(uint32_t(packs));
    // Few items: a thread a head, so that there are enough of them.  Many: four
    // heads a thread and streamed stores; from kStreamRows of rows on, more than the
    // MALL keeps beside what is written, streamed loads too, with two heads a thread.
    // One MI355X, 32/8 heads of 128 in f16, a thread a head / four / two and streamed
    // loads: 543 tokens 5.8 / 5.9 us; 1055, 6.9 / 5.9; 2079 (26 MB of rows) 10.7 / 9.6
    // / 10.7, 10.3 with four and plain stores; 5663 (70 MB) - / 21.9 / 25.2; 8223 (101
    // MB) - / 37.2 / 35.2, 44.3 with four and plain stores.  Other heads: 15/5 of 64 in f16,
    // 4127 tokens 7.3 / 6.0 / 7.2, 24607 (79 MB) 34.1 / 29.4 / 33.2, 34847 (112 MB) 45.5 /
    // 43.4 / 45.3; 32/8 of 128 in f32, 543 tokens 6.7 / 5.9 / 6.1, 2079 (51 MB) 21.4 / 16.5 /
    // 18.5, 4127 (101 MB) 41.2 / 35.6 / 34.4, 6175 (152 MB) 58.5 / 54.4 / 50.4; 9/3 of 64
    // in f32, 8223 (32 MB) 12.7 / 11.1 / 12.2, 30751 (118 MB) 47.5 / 44.2 / 41.0.
    const bool many = tokens * heads * packs >= uint64_t(ctx->num_cus) * 1024;
    const bool stream = many && tokens * heads * 2 * p.half_dim * sizeof(T) >= kStreamRows;
    const uint64_t steps = ceil_div(heads, stream ? 2 : many ? 4 : 1);
    p.head_steps = FastDiv(uint32_t(steps));
    p.items = uint32_t(tokens * steps * packs);
    const dim3 grid(unsigned(ceil_div(p.items, 256))), block(256);
#define RL_APPEND(HEADS, IN, OUT)                                                             \
    RL_LAUNCH(ctx, (k_paged_append<T, N, HEADS, IN, OUT>), grid, block, q, k, v, cos_table,   \
              sin_table, positions, slots, q_out, k_pages, v_pages, p)
    if (stream) RL_APPEND(2, true, true);
    else if (many) RL_APPEND(4, false, true);
    else RL_APPEND(1, false, false);
#undef RL_APPEND
}

template <typename T>
rl_status append_entry(rl_context* ctx, const char* name, const rl_buffer* q_src,
                       const uint64_t* q_dims, const uint64_t* q_strides, const rl_buffer* k_src,
                       const uint64_t* k_dims, const uint64_t* k_strides, const rl_buffer* v_src,
                       const uint64_t* v_dims, const uint64_t* v_strides,
                       const rl_buffer* cos_table, const rl_buffer* sin_table,
                       uint64_t table_rows, const rl_buffer* positions, const rl_buffer* slots,
                       const rl_buffer* q_out, const rl_buffer* k_pages, const rl_buffer* v_pages,
                       uint64_t pages, uint64_t page_size) {
    constexpr uint64_t es = sizeof(T);
    if (rl_status st = check_token_view("query", q_src, q_dims, q_strides, es)) return st;
    if (rl_status st = check_token_view("key", k_src, k_dims, k_strides, es)) return st;
    if (rl_status st = check_token_view("value", v_src, v_dims, v_strides, es)) return st;
    const uint64_t tokens = q_dims[0], q_heads = q_dims[1], kv_heads = k_dims[1], D = q_dims[2];
    if (k_dims[0] != tokens || k_dims[2] != D)
        return fail_shape_mismatch(q_dims, 3, k_dims, 3);
    for (int d = 0; d < 3; ++d)
        if (v_dims[d] != k_dims[d]) return fail_shape_mismatch(k_dims, 3, v_dims, 3);
    if (D % 2 != 0)
        return fail(RL_ERR_INVALID_SHAPE, "RoPE head size must be even, got %llu",
                    (unsigned long long)D);
    const uint64_t most = std::max({tokens, q_heads, kv_heads, D});
    const unsigned __int128 numel =  // does not wrap if each factor is below 2^32
        (unsigned __int128)tokens * D * ((unsigned __int128)q_heads + 2 * kv_heads);
    if (most > UINT32_MAX || numel > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "append element count exceeds u32");
    if (table_rows == 0 || table_rows > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "invalid RoPE table rows %llu",
                    (unsigned long long)table_rows);
    for (const rl_buffer* table : {cos_table, sin_table}) {
        if (rl_status st = check_buffer(table, "RoPE table")) return st;
        if (table->byte_len != table->len * sizeof(float))
            return fail(RL_ERR_UNSUPPORTED_DTYPE, "RoPE tables must be F32");
        if (table->len != table_rows * (D / 2))
            return fail(RL_ERR_INVALID_SHAPE, "RoPE table has %llu elements, expected [%llu, %llu]",
                        (unsigned long long)table->len, (unsigned long long)table_rows,
                        (unsigned long long)(D / 2));
    }
    if (rl_status st = check_u32("positions", positions, tokens)) return st;
    if (rl_status st = check_u32("slots", slots, tokens)) return st;
    if (rl_status st = check_pages(pages, page_size)) return st;
    if (rl_status st = check_output(q_out, tokens * q_heads * D, es, "paged append")) return st;
    if (rl_status st = check_pool("key pages", k_pages, pages, kv_heads, page_size, D, es))
        return st;
    if (rl_status st = check_pool("value pages", v_pages, pages, kv_heads, page_size, D, es))
        return st;
    if (rl_status st = require_context(ctx)) return st;
    if (rl_status st = activate(ctx)) return st;

    AppendParams p{};
    p.q = RowsView{q_strides[0], q_strides[1]};
    p.k = RowsView{k_strides[0], k_strides[1]};
    p.v = RowsView{v_strides[0], v_strides[1]};
    p.q_heads = uint32_t(q_heads);
    p.kv_heads = uint32_t(kv_heads);
    p.half_dim = uint32_t(D / 2);
    p.table_rows = uint32_t(table_rows);
    p.shift = log2_of(page_size);
    p.slots = pages * page_size;
    const uint64_t heads = q_heads + 2 * kv_heads;
    const T* q = static_cast<const T*>(q_src->data);
    const T* k = static_cast<const T*>(k_src->data);
    const T* v = static_cast<const T*>(v_src->data);
    const float* cs = static_cast<const float*>(cos_table->data);
    const float* sn = static_cast<const float*>(sin_table->data);
    const uint32_t* ps = static_cast<const uint32_t*>(positions->data);
    const uint32_t* sl = static_cast<const uint32_t*>(slots->data);
    T* qo = static_cast<T*>(q_out->data);
    T* kp = static_cast<T*>(k_pages->data);
    T* vp = static_cast<T*>(v_pages->data);
    // 16-byte packs where every row and half row lies on their grid, single
    // elements otherwise
    constexpr int N = 16 / int(es);
    bool packed = (D / 2) % N == 0 && aligned_to(cs, 16) && aligned_to(sn, 16);
    for (const void* ptr : {(const void*)q, (const void*)k, (const void*)v, (const void*)qo,
                            (const void*)kp, (const void*)vp})
        packed = packed && aligned_to(ptr, 16);
    for (const RowsView& w : {p.q, p.k, p.v})
        packed = packed && w.token_stride % N == 0 && w.head_stride % N == 0;
    if (packed)
        launch_append<T, N>(ctx, tokens, heads, p, q, k, v, cs, sn, ps, sl, qo, kp, vp);
    else
        launch_append<T, 1>(ctx, tokens, heads, p, q, k, v, cs, sn, ps, sl, qo, kp, vp);
    return after_launch(ctx, name);
}

}  // namespace
}  // namespace rl

using namespace rl;

extern "C" {

rl_status rl_paged_plan(rl_context* ctx, const rl_buffer* cached, const rl_buffer* fresh,
                        uint64_t sequences, const rl_buffer* free_pages,
                        const rl_buffer* block_table, uint64_t max_blocks, uint64_t pages,
                        uint64_t page_size, const rl_buffer* offsets, const rl_buffer* context,
                        uint64_t tokens, const rl_buffer* slots, const rl_buffer* positions,
                        const rl_buffer* taken) {
    return guarded([&] {
        return plan_entry(ctx, cached, fresh, sequences, free_pages, block_table, max_blocks,
                          pages, page_size, offsets, context, tokens, slots, positions, taken);
    });
}

rl_status rl_qkv_rope_paged_append_f32(
    rl_context* ctx, const rl_buffer* q_src, const uint64_t* q_dims, const uint64_t* q_strides,
    const rl_buffer* k_src, const uint64_t* k_dims, const uint64_t* k_strides,
    const rl_buffer* v_src, const uint64_t* v_dims, const uint64_t* v_strides,
    const rl_buffer* cos_table, const rl_buffer* sin_table, uint64_t table_rows,
    const rl_buffer* positions, const rl_buffer* slots, const rl_buffer* q_out,
    const rl_buffer* k_pages, const rl_buffer* v_pages, uint64_t pages, uint64_t page_size) {
    return guarded([&] {
        return append_entry<float>(ctx, "qkv_rope_paged_append_f32", q_src, q_dims, q_strides,
                                   k_src, k_dims, k_strides, v_src, v_dims, v_strides, cos_table,
                                   sin_table, table_rows, positions, slots, q_out, k_pages,
                                   v_pages, pages, page_size);
    });
}

rl_status rl_qkv_rope_paged_append_f16(
    rl_context* ctx, const rl_buffer* q_src, const uint64_t* q_dims, const uint64_t* q_strides,
    const rl_buffer* k_src, const uint64_t* k_dims, const uint64_t* k_strides,
    const rl_buffer* v_src, const uint64_t* v_dims, const uint64_t* v_strides,
    const rl_buffer* cos_table, const rl_buffer* sin_table, uint64_t table_rows,
    const rl_buffer* positions, const rl_buffer* slots, const rl_buffer* q_out,
    const rl_buffer* k_pages, const rl_buffer* v_pages, uint64_t pages, uint64_t page_size) {
    return guarded([&] {
        return append_entry<half_t>(ctx, "qkv_rope_paged_append_f16", q_src, q_dims, q_strides,
                                    k_src, k_dims, k_strides, v_src, v_dims, v_strides, cos_table,
                                    sin_table, table_rows, positions, slots, q_out, k_pages,
                                    v_pages, pages, page_size);
    });
}

}  // extern "C"
