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
#include "mfma_layout.hpp"
#include "ragged.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rl {
namespace {

// Added to the exponent of a probability that is rounded to f16, in the sum as in
// the product, so that it cancels in their quotient: f16's normal range then reaches
// down to 2^-26 of the row's maximum, and what is rounded away below it is at most
// 2^-37 of that a key (2^-25 without: over 100 thousand keys of 2^-27 each beside one
// of weight 1, 7e-4 of the whole).  The largest, kSlack past the maximum, is 2^15,
// below f16's 65504.
constexpr float kRaise = 12.0f;

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
    // Requests of at most this many rows a KV head (tokens times group) belong
    // to the split kernel: it takes those, the others skip them.
    uint32_t small_rows;
    bool longest_first;  // tile kernel: order of the tiles
    // split kernel
    uint32_t slots;        // workgroups a KV head can have running at once
    uint32_t page_bytes;   // of one page, all KV heads
    uint32_t head_bytes;   // of one KV head's rows in a page
    float* part;           // [workgroup][2][16][head size, padded]: unnormalised outputs
    float* part_ml;        // [workgroup][2][16]: (max in log2 units, sum)
    uint32_t* tickets;     // [request][KV head], kTicketStride words apart
};

// Request i as the device finds it.
struct Request {
    uint32_t begin;  // first row
    uint32_t n;      // rows
    uint32_t keys;
    int32_t first;  // position of the first row
    bool bad;       // more keys than max_context
};

template <bool PAGED>
__device__ inline Request load_request(const RaggedParams& p, uint32_t i) {
    Request r;
    r.begin = min(p.offsets[i], p.tokens);
    const uint32_t end = min(p.offsets[i + 1], p.tokens);
    const uint32_t all = end > r.begin ? end - r.begin : 0u;
    r.n = min(all, p.max_queries);
    const uint32_t ctx = PAGED ? p.context[i] : r.n;
    r.bad = PAGED && ctx > p.max_context;
    r.keys = PAGED ? min(ctx, p.max_context) : ctx;
    r.first = PAGED ? int32_t(r.keys) - int32_t(all) : 0;
    return r;
}

// Lane `at`'s request in every lane.
__device__ inline Request request_of_lane(const Request& mine, int at) {
    Request r;
    r.begin = uint32_t(__builtin_amdgcn_readlane(int(mine.begin), at));
    r.n = uint32_t(__builtin_amdgcn_readlane(int(mine.n), at));
    r.keys = uint32_t(__builtin_amdgcn_readlane(int(mine.keys), at));
    r.bad = __builtin_amdgcn_readlane(int(mine.bad), at) != 0;
    r.first = __builtin_amdgcn_readlane(mine.first, at);
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

// One query row by one wave, each product and sum in f32 and only of the keys
// that the row sees: for rows whose output a tile of the kernels below leaves
// non-finite, where 0 * inf and 0 * NaN of keys behind a row, or a page outside
// the pool, may have reached it.  Lane = key for the scores, lane = elements
// lane + 64 e for the values.  Head sizes up to 128, elements aligned to
// themselves.
template <typename T, bool PAGED>
__device__ inline void row_by_wave(const T* __restrict__ q, const T* __restrict__ k,
                                   const T* __restrict__ v, T* __restrict__ out,
                                   const RaggedParams& p, uint32_t request, const Request& r,
                                   uint32_t j, uint32_t head) {
    const uint32_t lane = threadIdx.x % 64, D = p.head_dim, kv_head = head / p.group;
    const T* qrow = q + (r.begin + j) * p.q_token + head * p.q_head;
    const int64_t position = int64_t(r.first) + j;
    const uint32_t key_end = position < 0 ? 0u : uint32_t(position) + 1;
    float o[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    for (uint32_t base = 0; base < key_end; base += 64) {
        const uint32_t n = min(64u, key_end - base);
        const uint32_t key = base + min(lane, n - 1);
        const uint64_t krow =
            key_row<PAGED>(p, request, r.begin, key, kv_head, p.k_token, p.k_head);
        float s = krow == kNoRow ? NAN : 0.0f;
        if (krow != kNoRow) {
            for (uint32_t d = 0; d < D; ++d)
                s = __builtin_fmaf(to_float(qrow[d]), to_float(k[krow + d]), s);
            s *= p.scale;
        }
        if (lane >= n) s = -INFINITY;
        const float m_new = fmaxf(m, wave_max_dpp(s));
        const float shift = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp_fast(m - shift), e = exp_fast(s - shift);
        m = m_new;
        l = l * alpha + e;
        o[0] *= alpha;
        o[1] *= alpha;
        for (uint32_t i = 0; i < n; ++i) {
            const float pi = lane_value(e, int(i));
            const uint64_t vrow =
                key_row<PAGED>(p, request, r.begin, base + i, kv_head, p.v_token, p.v_head);
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
                const uint32_t d = lane + 64 * e2;
                const bool there = vrow != kNoRow && d < D;
                o[e2] += pi * (there ? to_float(v[vrow + d]) : 0.0f);
            }
        }
    }
    l = wave_sum_dpp(l);
    const float inv = r.bad ? NAN : key_end == 0 ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t d = lane + 64 * e;
        if (d < D)
            out[(uint64_t(r.begin + j) * p.q_heads + head) * D + d] = from_float<T>(o[e] * inv);
    }
}

// ------------------------------------------------- one wave per query row
//
// Any head size up to 512, any strides and alignment: keys 256 at a time, a
// lane's four dot products in order, the probabilities through LDS, lanes =
// output elements for the values.  Bound by the vector ALUs and by key rows
// read lane by lane: 47.7 ms for the 8 prompts that the tiles below take 0.35 ms for.
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
    if (t < r.begin || t - r.begin >= r.n || r.n * p.group <= p.small_rows) return;
    const uint32_t D = p.head_dim, kv_head = head / p.group;
    const int64_t position = int64_t(r.first) + (t - r.begin);
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

// ------------------------------------------- few rows per KV head (decode)
//
// The rows of a request that share a KV head (tokens times group, row r = token
// r / group, head r % group) are the 16 columns of one matrix tile, and its
// keys stream past them once: S^T = K Q^T, P = 2^(S scale log2 e - max), O^T +=
// V^T P^T, per wave in its own registers.
//
// Work: every request's keys are cut into units of 4 kKeys (one block of kKeys
// for each of a workgroup's four waves), and all units, request after request,
// dealt out in equal shares to as many workgroups as run at once (two a CU).
// The lengths are only here, so every workgroup finds its share itself, by a
// sum over the requests.  Requests that lie in several shares leave partials,
// which meet by a ticket: the workgroup that finishes last merges them.
//
// The probabilities of f16 enter the second product as the sum of two f16 parts, 22
// bits, which its matrix cores have the time for: with one part the mean error against
// 64 bits was 2.57e-4 of the outputs' for 60 requests of up to 8000 keys, with two 1.77e-4,
// that of the outputs' own rounding, at the same 155 us (head size 32: 39.1 -> 40.5).
//
// Layout: K's operand is its rows as they lie in memory (16 bytes a lane).  V's
// has to come by columns: a lane loads its 4 or 8 columns of eight
// neighbouring rows (f32: of four) and takes the operand of each column across
// those registers (v_perm), so nothing passes through LDS.  Rows of the score
// tiles are keys in the order that leaves a lane the probabilities of exactly
// those eight rows.  A block's registers are refilled as soon as its scores (K)
// and products (V) are through, so the next block's rows are in flight under
// the rest of the work; its page entries are read a block ahead.  Bound by HBM:
// 155 us for 934 MB (60 requests of up to 8000 keys, 32/8 heads of 128 in f16; 6.0
// TB/s, where a plain read runs at 6.2 to 6.4), 75 us for one request of 100,003
// keys (5.5 TB/s); one request of 1536 keys takes 7.3 us, most of it the launch, three
// dependent reads and the hand-over.  Equal shares against each request cut by
// itself: 44 -> 40 us for 64 requests of up to 4000 keys (15/5 heads of 64).
// Registers refilled in place leave two waves a SIMD; three spill (174 -> 243 us).
template <typename T, int DP>
struct SplitShape {
    static constexpr bool kHalf = std::is_same<T, half_t>::value;
    static constexpr int kKeys = kHalf ? 32 : 16;             // keys of a block
    static constexpr int kKTiles = kKeys / 16;
    static constexpr int kKChunks = kHalf ? DP / 32 : DP / 16;  // 16-byte pieces of a K row a lane
    static constexpr int kVRows = kHalf ? 8 : 4;                // neighbouring V rows a lane
    static constexpr int kVSteps = kKeys / (4 * kVRows);
    static constexpr int kVCols = kHalf ? DP / 16 : 4;          // columns of one V load
    static constexpr int kVChunks = kHalf ? 1 : DP / 64;
    static constexpr int kTiles = DP / 16;                      // 16-element tiles of the output
};
typedef half_t hv4 __attribute__((ext_vector_type(4)));

template <typename T, int DP>
struct SplitBlock {
    typedef SplitShape<T, DP> S;
    typedef typename std::conditional<S::kHalf, h8, f32x4>::type KV;
    typedef typename std::conditional<S::kHalf, typename VecOf<half_t, DP / 16>::type,
                                      f32x4>::type VV;
    KV k[S::kKTiles][S::kKChunks];
    VV v[S::kVSteps][S::kVRows][S::kVChunks];
};

constexpr uint32_t kSplitRows = 16;
constexpr int kSplitWaves = 4;
constexpr uint32_t kTicketStride = 64;
constexpr uint64_t kStreamKeyBytes = uint64_t(100) << 20;

// Agent-coherent pairs of floats: written through, and read past, an XCD's L2.
__device__ inline void publish2(float* p, float a, float b) {
    const uint64_t w = uint64_t(__float_as_uint(a)) | uint64_t(__float_as_uint(b)) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), w, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float2 observe2(const float* p) {
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(uint32_t(w)), __uint_as_float(uint32_t(w >> 32)));
}

// A request's units for the split kernel, 0 if it is not one of its own.
__device__ inline uint32_t split_units(const RaggedParams& p, uint32_t i, uint32_t unit_shift,
                                       Request& r) {
    r = load_request<true>(p, min(i, p.sequences - 1));
    if (i >= p.sequences || r.n == 0 || r.n * p.group > p.small_rows) return 0u;
    // no keys to read where every row is zero or NaN: one unit writes them
    const uint32_t units = uint32_t((uint64_t(r.keys) + (1u << unit_shift) - 1) >> unit_shift);
    return r.bad || units == 0 ? 1u : units;
}

__device__ inline uint32_t wave_scan(uint32_t v) {  // inclusive sum
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xF, 0xF, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xF, 0xF, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xF, 0xF, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xF, 0xF, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xA, 0xF, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xC, 0xF, false));
    return v;
}
__device__ inline uint32_t last_lane(uint32_t v) {
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}
__device__ inline uint64_t wide_of_lane(uint64_t v, int at) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), at))) << 32 |
           uint32_t(__builtin_amdgcn_readlane(int(v), at));
}

// FULL: the head size is DP; else it is a smaller multiple of 16 bytes and the
// operands' elements past it are zeros (K, Q) or any row's own (V, whose output
// columns are not stored).
template <int DP>
struct SplitLds {
    float ml[kSplitWaves][kSplitRows][2];
    float o[kSplitWaves][kSplitRows][DP + 4];
    uint32_t odd_rows, ticket;
};
template <typename T, int DP, bool FULL>
__device__ inline void split_rows(const T* __restrict__ q, const T* __restrict__ k,
                                  const T* __restrict__ v, T* __restrict__ out,
                                  const RaggedParams& p, SplitLds<DP>& lds, uint32_t block) {
    typedef SplitShape<T, DP> S;
    typedef SplitBlock<T, DP> Block;
    typedef typename Block::KV KV;
    typedef typename Block::VV VV;
    constexpr bool kHalf = S::kHalf;
    constexpr uint32_t kKeys = S::kKeys;
    constexpr uint32_t kUnit = kSplitWaves * kKeys;
    constexpr uint32_t kUnitShift = __builtin_ctz(kUnit);
    auto& merge_ml = lds.ml;
    auto& merge_o = lds.o;
    uint32_t& odd_rows = lds.odd_rows;
    uint32_t& ticket = lds.ticket;
    const uint32_t hd = FULL ? uint32_t(DP) : p.head_dim;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t lr = lane % 16, g = lane / 16;
    const uint32_t kvh = block % p.kv_heads;
    const uint64_t w = block / p.kv_heads;

    // Every workgroup's share of the units: `per` of them in request order.  The
    // share's requests come in windows of 64, a lane each: `base` is the window's
    // first request, `before` the units of those before it.
    uint32_t base = 0, units_here, upto;
    uint64_t before = 0;
    Request here;
    auto load_window = [&] {
        units_here = split_units(p, base + lane, kUnitShift, here);
        upto = wave_scan(units_here);
    };
    uint64_t total, group_before = 0, group_upto = 0;
    const uint32_t run = (p.sequences + 64 * kSplitWaves - 1) / (64 * kSplitWaves);
    if (p.sequences <= 64) {
        load_window();
        total = last_lane(upto);
    } else {
        // more: each thread sums `run` requests, a lane then four threads' sums (256
        // requests of up to 300 keys, 15/5 heads of 64: 20.8 us, 26.4 where every request
        // was looked for from the first on; 4096: 226 / 1183)
        uint64_t* sums = reinterpret_cast<uint64_t*>(&lds.o[0][0][0]);
        uint64_t sum = 0;
        const uint64_t from = uint64_t(threadIdx.x) * run;
#pragma unroll 4
        for (uint32_t i = 0; i < run; ++i)
            sum += split_units(p, uint32_t(min(from + i, uint64_t(p.sequences))), kUnitShift, here);
        sums[threadIdx.x] = sum;
        __syncthreads();
        uint64_t four = 0;
#pragma unroll
        for (int i = 0; i < kSplitWaves; ++i) four += sums[kSplitWaves * lane + i];
        group_upto = four;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t lower = __shfl_up(group_upto, d, 64);
            group_upto += int(lane) >= d ? lower : 0u;
        }
        group_before = group_upto - four;
        total = wide_of_lane(group_upto, 63);
    }
    const uint64_t per = max(uint64_t(1), (total + p.slots - 1) / p.slots);
    const uint64_t end = min(total, (w + 1) * per);
    // Keys and values that the MALL does not keep between layers or steps anyway
    // are streamed past it (one MI355X: 934 MB 172 / 165 us, 410 MB 83.3 / 79.8, 164
    // MB 38.7 / 37.9; 50 MB 16.5 / 18.4).
    const bool stream = total * kUnit * p.kv_heads * 2 * (hd * sizeof(T)) >= kStreamKeyBytes;
    if (w * per >= end) return;
    if (p.sequences > 64) {  // the share's first window
        const int in = __builtin_ctzll(__ballot(group_upto > w * per));
        base = uint32_t(in) * kSplitWaves * run;
        before = wide_of_lane(group_before, in);
        load_window();
    }
    for (uint64_t at = w * per; at < end;) {
    // the request of unit `at`: the first whose units end past it
    uint64_t past = __ballot(before + upto > at);
    while (past == 0 && base + 64 < p.sequences) {
        before += last_lane(upto);
        base += 64;
        load_window();
        past = __ballot(before + upto > at);
    }
    const int in = past == 0 ? 0 : __builtin_ctzll(past);
    const uint32_t request = base + in;
    const uint32_t units = uint32_t(__builtin_amdgcn_readlane(int(units_here), in));
    const uint64_t first =  // its first unit
        before + uint32_t(__builtin_amdgcn_readlane(int(upto), in)) - units;
    const Request r = request_of_lane(here, in);
    const uint64_t w0 = first / per;  // workgroups w0 .. w0 + n_splits - 1 share the request
    const uint32_t n_splits = uint32_t((first + units - 1) / per - w0) + 1;
    const uint32_t split = uint32_t(w - w0);
    const uint32_t u0 = uint32_t(at - first), u1 = uint32_t(min(uint64_t(units), end - first));
    at = max(at + 1, first + u1);  // (whatever the lengths, an end)
    const uint32_t R = r.n * p.group;
    const uint32_t last = r.keys == 0 ? 0u : r.keys - 1;
    const uint32_t blocks = r.bad ? 0u : (r.keys + kKeys - 1) / kKeys;
    const uint32_t b0 = u0 * kSplitWaves;
    const uint32_t b1 = min(blocks, u1 * kSplitWaves);

    const uint32_t* entries = p.table + uint64_t(request) * p.max_blocks;
    bool bad_page = false;
    auto load_entry = [&](uint32_t blk) {  // of key blk * kKeys + lane
        const uint32_t key = min(blk * kKeys + lane % kKeys, last);
        return entries[key >> p.shift];
    };
    auto checked = [&](uint32_t entry) {  // a page outside the pool: page 0 instead, and noted
        bad_page |= entry >= p.pages;
        return entry < p.pages ? entry : 0u;
    };
    const uint32_t mask = (1u << p.shift) - 1;
    const uint32_t row_bytes = hd * sizeof(T);
    const char* kbase = reinterpret_cast<const char*>(k) + uint64_t(kvh) * p.head_bytes + 16 * g;
    // columns kVCols lr .. of V, those past the head size read the first ones
    const uint32_t col = S::kVCols * lr;
    const char* vbase = reinterpret_cast<const char*>(v) + uint64_t(kvh) * p.head_bytes;
    Block x;
    auto load_keys = [&](auto streamed, uint32_t blk, uint32_t entry) {
        const uint32_t kb = blk * kKeys;
#pragma unroll
        for (int m = 0; m < S::kKTiles; ++m) {
            const uint32_t kk = kHalf ? 32 * (m / 2) + 8 * (lr / 4) + 4 * (m % 2) + lr % 4
                                      : 16 * m + lr;
            const uint32_t key = min(kb + kk, last);
            const uint32_t page = uint32_t(__shfl(int(entry), int(key - kb), 64));
            const char* row = kbase + uint64_t(page) * p.page_bytes + (key & mask) * row_bytes;
#pragma unroll
            for (int c = 0; c < S::kKChunks; ++c) {
                const bool in = FULL || uint32_t(64 * c) + 16 * g < row_bytes;
                const KV* from = reinterpret_cast<const KV*>(row + 64 * c);
                if constexpr (decltype(streamed)::value)
                    x.k[m][c] = in ? load_stream(from) : KV{};
                else
                    x.k[m][c] = in ? *from : KV{};
            }
        }
    };
    auto load_values = [&](auto streamed, uint32_t blk, uint32_t entry) {
        const uint32_t kb = blk * kKeys;
#pragma unroll
        for (int t = 0; t < S::kVSteps; ++t) {
            const uint32_t run = kb + 4 * S::kVRows * t + S::kVRows * g;  // inside one page
            const uint32_t page =
                uint32_t(__shfl(int(entry), int(min(run, last) - kb), 64));
            const char* rows = vbase + uint64_t(page) * p.page_bytes;
#pragma unroll
            for (int e = 0; e < S::kVRows; ++e) {
                const char* row = rows + (min(run + e, last) & mask) * row_bytes;
#pragma unroll
                for (int c = 0; c < S::kVChunks; ++c) {
                    const uint32_t at = col + 64 * c;
                    const VV* from = reinterpret_cast<const VV*>(
                        row + sizeof(T) * (FULL || at < hd ? at : 0u));
                    if constexpr (decltype(streamed)::value)
                        x.v[t][e][c] = load_stream(from);
                    else
                        x.v[t][e][c] = *from;
                }
            }
        }
    };

    // row lr of this KV head: query elements, last key it sees (-1: none)
    const bool row_live = lr < R;
    const uint32_t token = row_live ? lr / p.group : 0u, sub = row_live ? lr % p.group : 0u;
    const int64_t position = int64_t(r.first) + token;
    const int limit = row_live && position >= 0 ? int(min(int64_t(last), position)) : -1;
    const T* qrow = q + (r.begin + token) * p.q_token + (kvh * p.group + sub) * p.q_head;
    KV qf[S::kKChunks];
#pragma unroll
    for (int c = 0; c < S::kKChunks; ++c) {
        const bool in = FULL || uint32_t(64 * c) + 16 * g < row_bytes;
        qf[c] = in ? *reinterpret_cast<const KV*>(reinterpret_cast<const char*>(qrow) + 16 * g +
                                                  64 * c)
                   : KV{};
    }
    f32x4 o[S::kTiles];
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;  // l: this lane's share

    f32x4 s[S::kKTiles];
    auto scores = [&] {
#pragma unroll
        for (int t = 0; t < S::kKTiles; ++t) {
            s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < S::kKChunks; ++c) {
                if constexpr (kHalf) {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[t][c], qf[c], s[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[t][c][e], qf[c][e], s[t],
                                                                    0, 0, 0);
                }
            }
        }
    };
    auto weights = [&](uint32_t blk) {
        // register r of tile t: key blk kKeys + (a constant) + 8 g (f32: 4 g)
        const int seen = limit - int(blk * kKeys) - int(S::kVRows * g);
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < S::kKTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = kHalf ? 32 * (t / 2) + 4 * (t % 2) + e : 16 * t + e;
                s[t][e] = at <= seen ? s[t][e] : -INFINITY;
                mx = fmaxf(mx, s[t][e]);
            }
        mx = rows4_max(mx) * p.scale_log2;
        const float m_new = fmaxf(m, mx);
        const float shift = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - shift);
        const float neg_m = (kHalf ? kRaise : 0.0f) - shift;
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][e] *= alpha;
#pragma unroll
        for (int t = 0; t < S::kKTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], p.scale_log2, neg_m));
    };
    auto values = [&] {
        if constexpr (kHalf) {
#pragma unroll
            for (int t = 0; t < S::kVSteps; ++t) {
                h8 pb, pl;  // high and low parts: 22 bits
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = s[2 * t + e / 4][e % 4];
                    pb[e] = half_t(x);
                    pl[e] = half_t(x - float(pb[e]));
                    l += x;
                }
#pragma unroll
                for (int c = 0; c < S::kTiles; ++c) {
                    h8 va;
#pragma unroll
                    for (int e = 0; e < 8; ++e) va[e] = x.v[t][e][0][c];
                    o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, o[c], 0, 0, 0);
                    o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, o[c], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < S::kVSteps; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    l += s[t][e];
#pragma unroll
                    for (int c = 0; c < S::kTiles; ++c)
                        o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[t][e][c / 4][c % 4],
                                                                    s[t][e], o[c], 0, 0, 0);
                }
        }
    };

    auto walk = [&](auto streamed) {
        uint32_t blk = b0 + wave;
        if (blk >= b1) return;
        uint32_t entry = checked(load_entry(blk));
        load_keys(streamed, blk, entry);
        load_values(streamed, blk, entry);
        uint32_t ahead = load_entry(min(blk + kSplitWaves, b1 - 1));
        for (; blk + kSplitWaves < b1; blk += kSplitWaves) {
            scores();
            entry = checked(ahead);
            ahead = load_entry(min(blk + 2 * kSplitWaves, b1 - 1));
            load_keys(streamed, blk + kSplitWaves, entry);
            weights(blk);
            values();
            load_values(streamed, blk + kSplitWaves, entry);
        }
        scores();
        weights(blk);
        values();
    };
    if (stream)
        walk(std::true_type{});
    else
        walk(std::false_type{});
    l = rows4_sum(l);
    if (__any(bad_page)) l = NAN;  // row_by_wave finds which rows see it

    // the four waves' states -> the range's.  Lane (g, lr), f16: elements
    // kTiles (4 g + e) + c of row lr in o[c][e]; f32: 64 (c / 4) + 4 (4 g + e) + c % 4.
    __syncthreads();  // the share's previous request is through with the LDS
    if (threadIdx.x == 0) odd_rows = 0;
    if (g == 0) {
        merge_ml[wave][lr][0] = m;
        merge_ml[wave][lr][1] = l;
    }
#pragma unroll
    for (int c = 0; c < S::kTiles; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at =
                kHalf ? S::kTiles * (4 * g + e) + c : 64 * (c / 4) + 4 * (4 * g + e) + c % 4;
            merge_o[wave][lr][at] = o[c][e];
        }
    __syncthreads();
    // partials: a workgroup can hold one of a request that began before its share
    // and one of a request that goes on behind it
    const uint64_t slot0 = (uint64_t(kvh) * p.slots + w0) * 2;
    const uint64_t slot = slot0 + 2 * split + (split == 0);
    const uint32_t pairs = hd / 2;
    // row `row`'s output, two elements: stored unless it is not finite
    auto store_row = [&](uint32_t row, uint32_t d, float2 x, float sum) {
        const uint32_t tok = row / p.group;
        const int64_t pos = int64_t(r.first) + tok;
        const float inv = pos < 0 ? 0.0f : 1.0f / sum;
        x.x *= inv;
        x.y *= inv;
        if (r.bad) x = make_float2(NAN, NAN);
        else if (!(fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY)) atomicOr(&odd_rows, 1u << row);
        T* dst = out + d +
                 (uint64_t(r.begin + tok) * p.q_heads + kvh * p.group + row % p.group) * hd;
        dst[0] = from_float<T>(x.x);
        dst[1] = from_float<T>(x.y);
    };
    for (uint32_t i = threadIdx.x; i < R * pairs; i += 64 * kSplitWaves) {
        const uint32_t row = i / pairs, d = 2 * (i % pairs);
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < kSplitWaves; ++x) top = fmaxf(top, merge_ml[x][row][0]);
        const float shift = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int x = 0; x < kSplitWaves; ++x) {
            const float f = __builtin_amdgcn_exp2f(merge_ml[x][row][0] - shift);
            sum += f * merge_ml[x][row][1];
            acc.x += f * merge_o[x][row][d];
            acc.y += f * merge_o[x][row][d + 1];
        }
        if (n_splits == 1) {
            store_row(row, d, acc, sum);
        } else {
            publish2(p.part + (slot * kSplitRows + row) * DP + d, acc.x, acc.y);
            if (d == 0) publish2(p.part_ml + (slot * kSplitRows + row) * 2, top, sum);
        }
    }
    if (n_splits > 1) {
        // Hand-over: every wave's published stores are complete (they are
        // written through to where all XCDs see them, and vmcnt 0 waits for
        // that) before the barrier, and only then is the ticket drawn; the
        // workgroup that draws the last one acquires and reads past its L2.
        // As for the decode of rl_attention_*, the order of the stores and the
        // ticket rests on that wait, not on a release, which would write back
        // the whole L2 in every workgroup.
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        uint32_t* counter = p.tickets + (uint64_t(request) * p.kv_heads + kvh) * kTicketStride;
        if (threadIdx.x == 0)
            ticket = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (ticket != n_splits - 1) continue;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        if (threadIdx.x == 0)  // for the next call
            __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        constexpr uint32_t kChunk = 8;
        for (uint32_t i = threadIdx.x; i < R * pairs; i += 64 * kSplitWaves) {
            const uint32_t row = i / pairs, d = 2 * (i % pairs);
            float top = -INFINITY, sum = 0.0f;
            float2 acc = make_float2(0.0f, 0.0f);
            for (uint32_t s0 = 0; s0 < n_splits; s0 += kChunk) {
                float2 ml[kChunk], ov[kChunk];
#pragma unroll
                for (uint32_t x = 0; x < kChunk; ++x) {
                    const uint32_t n = min(s0 + x, n_splits - 1);
                    const uint64_t from = (slot0 + 2 * n + (n == 0)) * kSplitRows + row;
                    ml[x] = observe2(p.part_ml + from * 2);
                    ov[x] = observe2(p.part + from * DP + d);
                }
                float next = top;
#pragma unroll
                for (uint32_t x = 0; x < kChunk; ++x)
                    if (s0 + x < n_splits) next = fmaxf(next, ml[x].x);
                const float shift = next == -INFINITY ? 0.0f : next;
                const float keep = __builtin_amdgcn_exp2f(top - shift);
                sum *= keep;
                acc.x *= keep;
                acc.y *= keep;
#pragma unroll
                for (uint32_t x = 0; x < kChunk; ++x) {
                    if (s0 + x >= n_splits) continue;
                    const float f = __builtin_amdgcn_exp2f(ml[x].x - shift);
                    sum += f * ml[x].y;
                    acc.x += f * ov[x].x;
                    acc.y += f * ov[x].y;
                }
                top = next;
            }
            store_row(row, d, acc, sum);
        }
    }
    // rows with an output that is not finite once more (after the stores above)
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    uint32_t odd = odd_rows;
    for (uint32_t n = 0; odd != 0; odd &= odd - 1, ++n) {
        if (n % kSplitWaves != wave) continue;
        const uint32_t row = __builtin_ctz(odd);
        row_by_wave<T, true>(q, k, v, out, p, request, r, row / p.group,
                             kvh * p.group + row % p.group);
    }
    }  // the next request of this workgroup's share
}

// -------------------------------------------------- many rows per KV head
//
// A tile is 32 QW of the rows that share a KV head (row r = token r / group,
// head r % group of the KV head's): every K and V block serves all heads of the
// group, and a causal tile is no longer than its 32 QW / group tokens.  QW waves
// of 32 rows times KS shares of the key blocks, merged through LDS at the end.
// S^T = K Q^T leaves each lane one row's scores (32 x 32 tiles), so the running
// max and sum need one exchange between lane halves, and the
// probabilities come out in the operand layout of O^T += V^T P^T, the keys taken
// in perm32 order; V's operand comes by transpose reads out of LDS.
// Head sizes off the multiples of 32 (!FULL) have probabilities of two f16 parts, as
// rl_attention_f16's: 22 bits (one part took 39.2 us where two take 45.2, 10 prompts of up
// to 1600, 32/8 heads of 80, and 115 where they take 149, 8 of up to 3000 with heads of 112).
// K and V go from memory straight to LDS (two stages), each lane fetching 16
// bytes from an address of its own -- its key's row, wherever its page is --
// the page entries read a step ahead.  Keys past the request's last read that
// last row again: nothing outside the request's rows is read, and their scores
// are masked.  Chunk c of row r lies at c ^ lds_swizzle(r).
//
// Tiles are numbered without a sum over the requests: request i's first tile is
// floor(o_i group / TILE) + i, which leaves room for all of its tiles.  Later
// tiles, the longer ones, start first; neighbouring workgroups take
// different KV heads, so that one XCD's workgroups (every eighth) share rows of
// K and V in its L2.
//
// Bound by how little the products and the softmax overlap: every block's barrier
// brings all waves of a workgroup to the same phase, with two or three waves a SIMD.
// Takes 354 to 366 us for 8 prompts of up to 4096 tokens (32/8 heads of 128, 302 GFLOP: 825
// to 850 TFLOP/s, where a large f16 matrix product runs at 1196), the matrix cores busy
// 41 % of the cycles, the vector ALUs 47 %, LDS 21 % without bank conflicts.  Slower:
// the next block's scores beside this one's softmax (356 -> 372 to 391 us), wave
// priorities around the products (no change), 128-key blocks for head size 64 (564 -> 621 us
// for 60 prompts).
template <int QW>
constexpr uint32_t kTileRows = 32 * QW;

// One 16-byte chunk a lane from memory to LDS: lane l's lands at lds + 16 l.
// In assembly so that the compiler's wait counting does not hold the LDS reads
// of the stage in use for a stage being filled; the caller waits for it
// (vmcnt) before the barrier that hands the stage over.
__device__ inline void load_to_lds(const void* from, uint32_t lds) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds), "v"(from)
        : "memory");
}

// Zeros for the chunks of a padded K row.
__device__ __align__(16) const uint32_t zero_chunk[4] = {0, 0, 0, 0};

// A row's running max (log2 units) moves only when a block passes it by more
// than this: probabilities stay below 2^3 (f16: times 2^kRaise), and most blocks skip
// the rescaling.
constexpr float kSlack = 3.0f;

// Tile u's request: the last one whose first tile is not past u (64 candidates
// a step).
__device__ inline uint32_t tiles_before(const RaggedParams& p, uint32_t i, uint32_t rows) {
    return uint32_t(uint64_t(min(p.offsets[i], p.tokens)) * p.group / rows) + i;
}
__device__ inline uint32_t find_tile_request(const RaggedParams& p, uint32_t u, uint32_t rows) {
    const uint32_t lane = threadIdx.x % 64;
    uint32_t lo = 0, hi = p.sequences;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64;
        const uint64_t at = lo + uint64_t(lane) * step;
        const bool ok = at < hi && tiles_before(p, uint32_t(at), rows) <= u;
        const uint64_t found = __ballot(ok);
        const uint32_t k = found == 0 ? 0u : 63u - uint32_t(__builtin_clzll(found));
        lo += k * step;
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Waves a SIMD that the registers have to leave room for: three for head size 128 with
// blocks of 32 keys, else two where two workgroups of four waves fit a CU's LDS.
template <int NT, int QW, int KS, int BN>
constexpr int kTileWaves =
    NT == 4 && QW == 4 && BN == 32 ? 3
    : QW * KS == 4 && 2 * KS * 2 * BN * (NT == 3 ? 128 : 32 * NT) * 2 <= 72 * 1024 ? 2
                                                                                    : 1;

// Up to 64 requests: tile u in the order of the keys that tiles see, most
// first (in steps of a tile's tokens), so that the long ones do not start last.
// Lane i, with request i in `r`, counts its tiles at or past a level; the tile's
// level is the largest that u + 1 tiles reach.  Returns the request, its tile in
// `tile`; `sequences` if there are not that many tiles.
__device__ inline uint32_t find_longest_tile(const RaggedParams& p, const Request& r, uint32_t u,
                                             uint32_t rows, uint32_t& tile) {
    const uint32_t lane = threadIdx.x % 64;
    const bool mine = lane < p.sequences && r.n * p.group > p.small_rows;
    const uint32_t tiles = mine ? (r.n * p.group + rows - 1) / rows : 0u;
    // (bounded, so that levels stay below 2^31)
    const uint32_t low =
        r.first <= 0 ? 0u
                     : uint32_t(min(uint64_t(r.first) * p.group / rows, uint64_t(1) << 29));
    auto reach = [&](uint32_t level) {  // this request's tiles at or past it
        return min(tiles, low + tiles > level ? low + tiles - level : 0u);
    };
    uint32_t lo = 0, hi = 1;  // N(lo) > u >= N(hi) once hi is past all levels
    if (last_lane(wave_scan(tiles)) <= u) return p.sequences;
    while (last_lane(wave_scan(reach(hi))) > u) {
        lo = hi;
        hi *= 2;
    }
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (last_lane(wave_scan(reach(mid))) > u) lo = mid;
        else hi = mid;
    }
    const uint32_t before = last_lane(wave_scan(reach(lo + 1)));
    const uint32_t upto = wave_scan(reach(lo) - reach(lo + 1));
    const int at = __builtin_ctzll(__ballot(upto > u - before));
    // the level's tile of that request: all of its lower ones where it starts past the level
    tile = uint32_t(__builtin_amdgcn_readlane(int(tiles), at)) -
           uint32_t(__builtin_amdgcn_readlane(int(reach(lo)), at)) +
           (u - before - (uint32_t(__builtin_amdgcn_readlane(int(upto), at)) -
                          uint32_t(__builtin_amdgcn_readlane(int(reach(lo) - reach(lo + 1)), at))));
    return uint32_t(at);
}

// A workgroup's request and first row in it; false if it has none.
template <bool PAGED>
__device__ inline bool find_tile(const RaggedParams& p, uint32_t block, uint32_t blocks,
                                 uint32_t tile_rows, uint32_t& request, Request& r,
                                 uint32_t& row0) {
    const uint32_t unit = block / p.kv_heads;
    const uint32_t back = blocks / p.kv_heads - 1 - unit;
    uint32_t tile;
    if (p.sequences <= 64) {  // a request a lane: the lengths are read once
        const uint32_t lane = threadIdx.x % 64;
        const Request mine = load_request<PAGED>(p, min(lane, p.sequences - 1));
        if (p.longest_first) {
            request = find_longest_tile(p, mine, unit, tile_rows, tile);
            if (request >= p.sequences) return false;
        } else {
            const uint32_t first = uint32_t(uint64_t(mine.begin) * p.group / tile_rows) + lane;
            const uint64_t found = __ballot(lane < p.sequences && first <= back);
            if (found == 0) return false;
            request = 63u - uint32_t(__builtin_clzll(found));
            tile = back - uint32_t(__builtin_amdgcn_readlane(int(first), int(request)));
        }
        r = request_of_lane(mine, int(request));
    } else {
        request = find_tile_request(p, back, tile_rows);
        const uint32_t first = tiles_before(p, request, tile_rows);
        if (back < first) return false;
        tile = back - first;
        r = load_request<PAGED>(p, request);
    }
    row0 = tile * tile_rows;
    const uint32_t rows = r.n * p.group;
    return uint64_t(tile) * tile_rows < rows && rows > p.small_rows;
}

// LDS of a tile: two stages of every share's K and V blocks, then the merge.
template <int NT, int QW, int KS, int BN>
struct TileLds {
    static constexpr int kRow = NT == 3 ? 128 : 32 * NT;  // elements of a row
    static constexpr int kStages = 2 * KS * 2 * BN * kRow * 2;
    static constexpr int kMerge = (KS - 1) * QW * 64 * (NT * 16 + 2) * 4;
    unsigned char bytes[kStages > kMerge ? kStages : kMerge];
    uint32_t any_bad;
};
template <int NT, int QW, int KS, int BN, bool PAGED, bool FULL>
__device__ inline void tile_rows(const half_t* __restrict__ q, const half_t* __restrict__ k,
                                 const half_t* __restrict__ v, half_t* __restrict__ out,
                                 const RaggedParams& p, TileLds<NT, QW, KS, BN>& shared,
                                 uint32_t block, uint32_t n_blocks) {
    typedef half_t T;
    constexpr int D = 32 * NT;                    // head size, padded
    constexpr int RD = NT == 3 ? 128 : D;         // elements of an LDS row
    constexpr int CE = 8;                         // elements of a 16-byte chunk
    constexpr int ROW_CHUNKS = RD / CE;
    constexpr int SW = ROW_CHUNKS >= 16 ? 4 : ROW_CHUNKS / 4;  // lds_swizzle's row class
    constexpr int KT = BN / 32;                   // 32-key tiles of a block
    constexpr int DC = D / (2 * CE);              // pairs of chunks of a row (lane halves)
    constexpr int WAVES = QW * KS;
    constexpr int THREADS = 64 * WAVES;
    constexpr uint32_t TILE = kTileRows<QW>;
    constexpr int BLOCK_CHUNKS = BN * ROW_CHUNKS;  // of K, or V
    constexpr int LOADS = BLOCK_CHUNKS * KS / THREADS;  // keys a lane fetches K and V chunks of
    constexpr int BLOCK_BYTES = 16 * BLOCK_CHUNKS;
    constexpr int STAGE_BYTES = KS * 2 * BLOCK_BYTES;
    constexpr int MERGE = NT * 16 + 2;
    static_assert(BLOCK_CHUNKS % 64 == 0 && BLOCK_CHUNKS * KS % THREADS == 0,
                  "a wave's load stays in one block");
    unsigned char* const lds = shared.bytes;
    uint32_t& any_bad = shared.any_bad;

    const uint32_t hd = FULL ? uint32_t(D) : p.head_dim;
    const uint32_t kvh = block % p.kv_heads;
    uint32_t request, row0;
    Request r;
    if (!find_tile<PAGED>(p, block, n_blocks, TILE, request, r, row0)) return;
    const uint32_t rows = r.n * p.group;

    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t qw = wave % QW, share = wave / QW;
    const uint32_t col = lane % 32, hs = lane / 32;
    const uint32_t last = r.keys == 0 ? 0u : r.keys - 1;
    // keys that the tile's last row sees
    auto keys_of = [&](uint32_t row) {  // visible to row `row` of the request
        const int64_t pos = int64_t(r.first) + row / p.group;
        return pos < 0 || r.bad ? 0u : uint32_t(min(int64_t(r.keys), pos + 1));
    };
    const uint32_t keys = keys_of(min(row0 + TILE, rows) - 1);
    const uint32_t blocks = (keys + BN - 1) / BN;
    const uint32_t steps = (blocks + KS - 1) / KS;
    const uint32_t wrow0 = row0 + 32 * qw;  // the wave's first row
    const bool wave_active = wrow0 < rows;
    const uint32_t wave_keys = wave_active ? keys_of(min(wrow0 + 31, rows - 1)) : 0u;
    const uint32_t wave_least = wave_active ? keys_of(wrow0) : 0u;  // its first row's
    const uint32_t row = wrow0 + col;  // this lane's
    const bool row_valid = row < rows;
    const uint32_t token = row_valid ? row / p.group : 0u;
    const uint32_t head = kvh * p.group + (row_valid ? row % p.group : 0u);
    const int limit = row_valid ? int(keys_of(row)) - 1 : -1;  // last key it sees
    if (threadIdx.x == 0) any_bad = 0;

    // what a lane fetches: of key `fetch_key[i]` of its share's block, chunk `ch`
    uint32_t fetch_key[LOADS];
    uint32_t fetch_byte[LOADS];  // of the chunk in its row; ~0u: padding
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        // load i of a wave fills 64 chunks in a row, of one share's block
        const uint32_t all = (i * WAVES + wave) * 64 + lane, c = all % BLOCK_CHUNKS;
        const uint32_t kr = c / ROW_CHUNKS;
        const uint32_t ch = (c % ROW_CHUNKS) ^ lds_swizzle<SW>(kr);
        fetch_key[i] = (all / BLOCK_CHUNKS) * BN + kr;
        fetch_byte[i] = ch * CE < hd ? 16 * ch : ~0u;
    }
    const uint32_t lds_base = uint32_t(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)(lds)));
    const uint32_t* entries = PAGED ? p.table + uint64_t(request) * p.max_blocks : nullptr;
    const uint32_t mask = (1u << p.shift) - 1;
    const char* kbase;
    const char* vbase;
    if constexpr (PAGED) {
        kbase = reinterpret_cast<const char*>(k) + uint64_t(kvh) * p.head_bytes;
        vbase = reinterpret_cast<const char*>(v) + uint64_t(kvh) * p.head_bytes;
    } else {
        kbase = reinterpret_cast<const char*>(k + r.begin * p.k_token + kvh * p.k_head);
        vbase = reinterpret_cast<const char*>(v + r.begin * p.v_token + kvh * p.v_head);
    }
    bool bad_page = false;
    uint32_t entry[LOADS] = {};
    auto load_entries = [&](uint32_t step) {
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                entry[i] = entries[min(step * KS * BN + fetch_key[i], last) >> p.shift];
        }
    };
    auto issue_step = [&](uint32_t step) {
        const uint32_t stage =
            __builtin_amdgcn_readfirstlane(lds_base + (step % 2) * STAGE_BYTES);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t first = (i * WAVES + wave) * 64;  // chunk, over the shares' blocks
            if (step * KS + first / BLOCK_CHUNKS >= blocks) continue;
            const uint32_t key = min(step * KS * BN + fetch_key[i], last);
            uint64_t koff, voff;
            if constexpr (PAGED) {
                const bool in = entry[i] < p.pages;
                bad_page |= !in;
                koff = uint64_t(in ? entry[i] : 0u) * p.page_bytes +
                       (key & mask) * uint32_t(hd * sizeof(T));
                voff = koff;
            } else {
                koff = uint64_t(key) * uint32_t(p.k_token * sizeof(T));
                voff = uint64_t(key) * uint32_t(p.v_token * sizeof(T));
            }
            const char* kp = kbase + koff + fetch_byte[i];
            const char* vp = vbase + voff + fetch_byte[i];
            if (RD > 32 * NT || !FULL) {  // V's padding: not stored, so any finite or not
                const bool pad = fetch_byte[i] == ~0u;
                kp = pad ? reinterpret_cast<const char*>(zero_chunk) : kp;
                vp = pad ? reinterpret_cast<const char*>(zero_chunk) : vp;
            }
            const uint32_t at = stage + 16 * first + first / BLOCK_CHUNKS * BLOCK_BYTES;
            load_to_lds(kp, at);
            load_to_lds(vp, at + BLOCK_BYTES);
        }
    };
    load_entries(0);

    // operands: K chunk 2 c + hs of its key's row; f16: V by transpose reads
    uint32_t koff[DC];
    const uint32_t krow = perm32(col);
#pragma unroll
    for (int c = 0; c < DC; ++c)
        koff[c] = krow * RD * sizeof(T) + 16 * ((2 * c + hs) ^ lds_swizzle<SW>(krow));
    uint32_t voff[2 * NT];
#pragma unroll
    for (int e2 = 0; e2 < 2; ++e2) {
        const uint32_t vr = 8 * (lane / 32) + (lane % 16) / 4 + 4 * e2;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t ch = 2 * ((lane / 16) % 2) + (lane % 4) / 2 + 4 * t;
            voff[e2 * NT + t] = vr * RD * 2 + 16 * (ch ^ lds_swizzle<SW>(vr)) + 8 * (lane % 2);
        }
    }
    h8 qf[DC];
    const T* qrow = q + (r.begin + token) * p.q_token + head * p.q_head + CE * hs;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        const bool in = row_valid && (FULL || uint32_t(2 * CE * c) + CE * hs < hd);
        qf[c] = in ? *reinterpret_cast<const h8*>(qrow + 2 * CE * c) : h8{};
    }
    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // l: this lane's half of the sum

    if (steps > 0) {
        issue_step(0);
        load_entries(1);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (uint32_t step = 0; step < steps; ++step) {
        if (step + 1 < steps) {
            issue_step(step + 1);
            load_entries(step + 2);
        }
        const uint32_t blk = step * KS + share;
        const uint32_t kbase_key = blk * BN;
        const unsigned char* ks = lds + (step % 2) * STAGE_BYTES + share * 2 * BLOCK_BYTES;
        const unsigned char* vs = ks + BLOCK_BYTES;
        if (blk < blocks && kbase_key < wave_keys) {
            f32x16 s[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kt][e] = 0.0f;
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const h8 ka = *reinterpret_cast<const h8*>(
                        ks + kt * 32 * RD * sizeof(T) + koff[c]);
                    s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qf[c], s[kt], 0, 0, 0);
                }
            }
            // register e of tile kt: key kbase_key + 32 kt + 16 (e / 8) + 8 hs + e % 8
            if (kbase_key + BN > wave_least) {
                const int lim = limit - int(kbase_key) - int(8 * hs);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int at = 32 * kt + 16 * (e / 8) + e % 8;
                        if (at > lim) s[kt][e] = -INFINITY;
                    }
            }
            float mx = -INFINITY, my = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    mx = max3(mx, s[kt][e], s[kt][e + 1]);
                    my = max3(my, s[kt][e + 2], s[kt][e + 3]);
                }
            mx = max_halves(fmaxf(mx, my)) * p.scale_log2;
            if (__any(mx > m + kSlack)) {
                const float m_new = fmaxf(m, mx);
                const float alpha = m_new > m ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[t][e] *= alpha;
            }
            const float neg_m = (m == -INFINITY ? 0.0f : -m) + kRaise;
            // the sum adds the same rounded probabilities that the product takes
            const h2 ones = {half_t(1.0f), half_t(1.0f)};
            h8 pb[BN / 16], pl[FULL ? 1 : BN / 16];
#pragma unroll
            for (int c = 0; c < BN / 16; ++c) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(s[c / 2][8 * (c % 2) + e], p.scale_log2, neg_m));
                    pb[c][e] = half_t(x);
                    if constexpr (!FULL) {
                        pl[c][e] = half_t(x - float(pb[c][e]));
                        l += x;
                    }
                }
                if constexpr (FULL) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        l = __builtin_amdgcn_fdot2(h2{pb[c][e], pb[c][e + 1]}, ones, l, false);
                }
            }
#pragma unroll
            for (int c = 0; c < BN / 16; ++c)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const half_t* at = reinterpret_cast<const half_t*>(vs + 16 * c * RD * 2);
                    const h4 lo = lds_read_transposed(at + voff[t] / 2);
                    const h4 hi = lds_read_transposed(at + voff[NT + t] / 2);
                    const h8 va = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    if constexpr (!FULL)
                        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[c], o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pb[c], o[t], 0, 0, 0);
                }
        }
        __builtin_amdgcn_s_waitcnt(0);  // this wave's share of the next stage has landed
        __syncthreads();
    }
    if (PAGED && __any(bad_page) && lane == 0) any_bad = 1;  // read after the barrier below

    if constexpr (KS > 1) {  // shares 1 .. hand their (max, sum, output) to share 0
        float* mg = reinterpret_cast<float*>(lds);
        if (share > 0) {
            float* dst = mg + ((share - 1) * QW * 64 + qw * 64 + lane) * MERGE;
            dst[0] = m;
            dst[1] = l;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) dst[2 + 16 * t + e] = o[t][e];
        }
        __syncthreads();
        if (share != 0) return;
#pragma unroll
        for (int x = 1; x < KS; ++x) {
            const float* src = mg + ((x - 1) * QW * 64 + qw * 64 + lane) * MERGE;
            const float m2 = src[0], top = fmaxf(m, m2);
            const float a1 = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            const float a2 = top > m2 ? __builtin_amdgcn_exp2f(m2 - top) : 1.0f;
            l = l * a1 + src[1] * a2;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[t][e] = o[t][e] * a1 + src[2 + 16 * t + e] * a2;
            m = top;
        }
    } else if (PAGED) {
        __syncthreads();
    }

    const float sum = l + __shfl_xor(l, 32, 64);
    const float inv = limit < 0 ? 0.0f : 1.0f / sum;
    bool odd = PAGED && any_bad != 0;  // row_by_wave finds which rows see the page
    if (row_valid) {
        T* orow = out + (uint64_t(r.begin + token) * p.q_heads + head) * hd;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t d = 32 * t + 8 * g + 4 * hs;
                if (!FULL && d >= hd) continue;
                h4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = limit < 0 ? 0.0f : o[t][4 * g + i] * inv;
                    odd |= !(fabsf(x) < INFINITY);
                    w[i] = r.bad ? half_t(NAN) : half_t(x);
                }
                *reinterpret_cast<h4*>(orow + d) = w;
            }
    }
    if (r.bad) return;
    // rows with an output that is not finite once more, by the whole wave (after
    // its own stores above)
    const uint64_t votes = __ballot(odd && row_valid);
    uint32_t redo = uint32_t(votes | votes >> 32);
    if (redo == 0) return;
    __builtin_amdgcn_s_waitcnt(0);
    for (; redo != 0; redo &= redo - 1) {
        const uint32_t again = wrow0 + __builtin_ctz(redo);
        row_by_wave<T, PAGED>(q, k, v, out, p, request, r, again / p.group,
                              kvh * p.group + again % p.group);
    }
}

// ------------------------------------- many rows per KV head, f32 products
//
// The same tiles with every f32 operand as three bf16 parts (Bf16x3: six of the
// nine products, the rest below 2^-26 of the whole), at a sixth of the bf16 rate
// against a sixteenth for f32 products of the matrix cores (40.8 -> 27.5 us for 5
// prompts of up to 1021 tokens, 9/3 heads of 64; 168 -> 84 for 6 of up to 2000 and
// 90 -> 46 for 7 of up to 1000, 15/5 heads of 64).  Bound by the vector work
// of the splits (51 % of the cycles; matrix cores 24 %) and few waves.  A block is
// 32 keys of one wave, and nothing passes through LDS: K's operand is 32 bytes of a
// key's row a lane; V's comes by columns, so a lane loads its NT elements of eight
// neighbouring rows and splits each column across them.  K's registers are
// refilled once the scores are through, V's after the products.
//
// Queries, probabilities and values are scaled by 2^24 (kPartScale) so that no
// part of theirs falls below bf16's range; of a key only what is below 2^-126
// is lost, which changes a score by less than 2^-59 while query elements are
// below 2^60.  Rows with larger query elements, and rows whose output is not
// finite (infinities, sums of 2^80 and more), are computed again unsplit
// (row_by_wave).
template <int NT, int QW, int KS>
struct TileLdsF32 {
    float merge[KS > 1 ? (KS - 1) * QW * 64 * (NT * 16 + 2) : 1];
    uint32_t any_bad;
};
template <int NT, int QW, int KS, bool PAGED, bool FULL>
__device__ inline void tile_rows_f32(const float* __restrict__ q, const float* __restrict__ k,
                                     const float* __restrict__ v, float* __restrict__ out,
                                     const RaggedParams& p, TileLdsF32<NT, QW, KS>& shared,
                                     uint32_t block, uint32_t n_blocks) {
    constexpr int D = 32 * NT;
    constexpr int DC = D / 16;
    constexpr uint32_t BN = 32;
    constexpr uint32_t TILE = kTileRows<QW>;
    constexpr int MERGE = NT * 16 + 2;
    float* const merge = shared.merge;
    uint32_t& any_bad = shared.any_bad;

    const uint32_t hd = FULL ? uint32_t(D) : p.head_dim;
    const uint32_t kvh = block % p.kv_heads;
    uint32_t request, row0;
    Request r;
    if (!find_tile<PAGED>(p, block, n_blocks, TILE, request, r, row0)) return;
    const uint32_t rows = r.n * p.group;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t lane = threadIdx.x % 64;
    const uint32_t qw = wave % QW, share = wave / QW;
    const uint32_t col = lane % 32, hs = lane / 32;
    const uint32_t last = r.keys == 0 ? 0u : r.keys - 1;
    auto keys_of = [&](uint32_t row) {  // visible to row `row` of the request
        const int64_t pos = int64_t(r.first) + row / p.group;
        return pos < 0 || r.bad ? 0u : uint32_t(min(int64_t(r.keys), pos + 1));
    };
    const uint32_t wrow0 = row0 + 32 * qw;
    const bool wave_active = wrow0 < rows;
    const uint32_t wave_keys = wave_active ? keys_of(min(wrow0 + 31, rows - 1)) : 0u;
    const uint32_t wave_least = wave_active ? keys_of(wrow0) : 0u;
    const uint32_t blocks = (wave_keys + BN - 1) / BN;
    const uint32_t row = wrow0 + col;
    const bool row_valid = row < rows;
    const uint32_t token = row_valid ? row / p.group : 0u;
    const uint32_t head = kvh * p.group + (row_valid ? row % p.group : 0u);
    const int limit = row_valid ? int(keys_of(row)) - 1 : -1;
    if (threadIdx.x == 0) any_bad = 0;

    const uint32_t* entries = PAGED ? p.table + uint64_t(request) * p.max_blocks : nullptr;
    const uint32_t mask = (1u << p.shift) - 1;
    const char* kbase;
    const char* vbase;
    uint32_t k_row_bytes, v_row_bytes;  // between the rows of a page, or of a request
    if constexpr (PAGED) {
        kbase = reinterpret_cast<const char*>(k) + uint64_t(kvh) * p.head_bytes;
        vbase = reinterpret_cast<const char*>(v) + uint64_t(kvh) * p.head_bytes;
        k_row_bytes = v_row_bytes = hd * 4;
    } else {
        kbase = reinterpret_cast<const char*>(k + r.begin * p.k_token + kvh * p.k_head);
        vbase = reinterpret_cast<const char*>(v + r.begin * p.v_token + kvh * p.v_head);
        k_row_bytes = uint32_t(p.k_token * 4);
        v_row_bytes = uint32_t(p.v_token * 4);
    }
    bool bad_page = false;
    struct Entries {
        uint32_t k, v[2];
    };
    auto load_entries = [&](uint32_t blk) {  // of this lane's K row and its two runs of V rows
        Entries e{};
        if constexpr (PAGED) {
            e.k = entries[min(blk * BN + perm32(col), last) >> p.shift];
#pragma unroll
            for (int c = 0; c < 2; ++c)
                e.v[c] = entries[min(blk * BN + 16 * c + 8 * hs, last) >> p.shift];
        }
        return e;
    };
    auto page_at = [&](const char* base, uint32_t entry) {
        if constexpr (!PAGED) return base;
        const bool in = entry < p.pages;
        bad_page |= !in;
        return base + uint64_t(in ? entry : 0u) * p.page_bytes;
    };
    f32x8 kreg[DC];
    float vreg[2][8][NT];
    auto load_keys = [&](uint32_t blk, const Entries& e) {
        const uint32_t key = min(blk * BN + perm32(col), last);
        const char* at = page_at(kbase, e.k) +
                         uint64_t(PAGED ? key & mask : key) * k_row_bytes + 32 * hs;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            f32x4 x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool in = FULL || uint32_t(16 * c + 8 * hs + 4 * i) < hd;
                x[i] = in ? *reinterpret_cast<const f32x4*>(at + 64 * c + 16 * i) : f32x4{};
            }
            kreg[c] = __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    auto load_values = [&](uint32_t blk, const Entries& e) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t run = blk * BN + 16 * c + 8 * hs;  // eight keys inside one page
            const char* base = page_at(vbase, e.v[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t key = min(run + i, last);
                const char* at = base + uint64_t(PAGED ? key & mask : key) * v_row_bytes;
                if constexpr (NT == 3) {  // element 32 t + col
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint32_t d = 32 * t + col;
                        vreg[c][i][t] =
                            *reinterpret_cast<const float*>(at + 4 * (FULL || d < hd ? d : 0u));
                    }
                } else {  // elements NT col .. + NT - 1
                    typedef typename VecOf<float, NT>::type VE;
                    const uint32_t d = NT * col;
                    const VE w = *reinterpret_cast<const VE*>(at + 4 * (FULL || d < hd ? d : 0u));
#pragma unroll
                    for (int t = 0; t < NT; ++t) vreg[c][i][t] = w[t];
                }
            }
        }
    };
    uint32_t blk = share;
    Entries e = load_entries(blk);
    if (blk < blocks) {
        load_keys(blk, e);
        load_values(blk, e);
    }

    Bf16x3 qf[DC];
    float widest = 0.0f;  // query element
    const float* qrow = q + (r.begin + token) * p.q_token + head * p.q_head + 8 * hs;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool in = row_valid && (FULL || uint32_t(16 * c + 8 * hs + 4 * i) < hd);
            const f32x4 w = in ? *reinterpret_cast<const f32x4*>(qrow + 16 * c + 4 * i) : f32x4{};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                widest = fmaxf(widest, fabsf(w[j]));
                x[4 * i + j] = w[j] * kPartScale;
            }
        }
        qf[c] = split_bf16(x);
    }
    const float scale_log2 = p.scale_log2 / kPartScale;  // of the scores, their queries scaled
    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (PAGED && blk + KS < blocks) e = load_entries(blk + KS);
    for (; blk < blocks; blk += KS) {
        const bool more = blk + KS < blocks;
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < DC; ++c) s = mfma_bf16x3(split_bf16(kreg[c]), qf[c], s);
        if (more) load_keys(blk + KS, e);
        // register i: key blk BN + 16 (i / 8) + 8 hs + i % 8
        if (blk * BN + BN > wave_least) {
            const int lim = limit - int(blk * BN) - int(8 * hs);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (16 * (i / 8) + i % 8 > lim) s[i] = -INFINITY;
        }
        float mx = -INFINITY, my = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            mx = max3(mx, s[i], s[i + 1]);
            my = max3(my, s[i + 2], s[i + 3]);
        }
        mx = max_halves(fmaxf(mx, my)) * scale_log2;
        if (__any(mx > m + kSlack)) {
            const float m_new = fmaxf(m, mx);
            const float alpha = m_new > m ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
        }
        const float neg_m = m == -INFINITY ? 0.0f : -m;
        Bf16x3 pb[2];
        float la = 0.0f, lb = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            f32x8 x;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * c + i], scale_log2, neg_m));
                x[i + 1] =
                    __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * c + i + 1], scale_log2, neg_m));
                la += x[i];
                lb += x[i + 1];
            }
            pb[c] = split_bf16(x * kPartScale);
        }
        l += la + lb;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            // the block's products apart, added to the output once
            f32x16 acc;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f32x8 x;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = vreg[c][i][t] * kPartScale;
                acc = mfma_bf16x3(split_bf16(x), pb[c], acc);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] += acc[i];
        }
        if (more) {
            load_values(blk + KS, e);
            if (PAGED && blk + 2 * KS < blocks) e = load_entries(blk + 2 * KS);
        }
    }
    if constexpr (KS > 1 || PAGED) __syncthreads();  // any_bad is set up
    if (PAGED && __any(bad_page) && lane == 0) any_bad = 1;

    if constexpr (KS > 1) {
        if (share > 0) {
            float* dst = merge + ((share - 1) * QW * 64 + qw * 64 + lane) * MERGE;
            dst[0] = m;
            dst[1] = l;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[2 + 16 * t + i] = o[t][i];
        }
        __syncthreads();
        if (share != 0) return;
#pragma unroll
        for (int x = 1; x < KS; ++x) {
            const float* src = merge + ((x - 1) * QW * 64 + qw * 64 + lane) * MERGE;
            const float m2 = src[0], top = fmaxf(m, m2);
            const float a1 = top > m ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            const float a2 = top > m2 ? __builtin_amdgcn_exp2f(m2 - top) : 1.0f;
            l = l * a1 + src[1] * a2;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] = o[t][i] * a1 + src[2 + 16 * t + i] * a2;
            m = top;
        }
    } else if (PAGED) {
        __syncthreads();
    }

    const float inv = kProductUnscale / (l + __shfl_xor(l, 32, 64));
    bool odd = (PAGED && any_bad != 0) || widest >= 0x1p60f;
    if (row_valid) {
        float* orow = out + (uint64_t(r.begin + token) * p.q_heads + head) * hd;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                // the tile's row, and its element
                const uint32_t at = 8 * (i / 4) + 4 * hs + i % 4;
                const uint32_t d = NT == 3 ? 32 * t + at : NT * at + t;
                if (!FULL && d >= hd) continue;
                const float x = limit < 0 ? 0.0f : o[t][i] * inv;
                odd |= !(fabsf(x) < INFINITY);
                orow[d] = r.bad ? NAN : x;
            }
    }
    if (r.bad) return;
    const uint64_t votes = __ballot(odd && row_valid);
    uint32_t redo = uint32_t(votes | votes >> 32);
    if (redo == 0) return;
    __builtin_amdgcn_s_waitcnt(0);
    for (; redo != 0; redo &= redo - 1) {
        const uint32_t again = wrow0 + __builtin_ctz(redo);
        row_by_wave<float, PAGED>(q, k, v, out, p, request, r, again / p.group,
                                  kvh * p.group + again % p.group);
    }
}

// ----------------------------------------------------------------- kernels

template <typename T, int DP, bool FULL>
__global__ __launch_bounds__(64 * kSplitWaves, 2) void k_ragged_split(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    T* __restrict__ out, RaggedParams p) {
    __shared__ __align__(16) SplitLds<DP> lds;
    split_rows<T, DP, FULL>(q, k, v, out, p, lds, blockIdx.x);
}

// A tile's LDS and body by type.
template <typename T, int NT, int QW, int KS, int BN>
struct Tile {
    typedef TileLds<NT, QW, KS, BN> Lds;
    static constexpr int kWaves = kTileWaves<NT, QW, KS, BN>;
    template <bool PAGED, bool FULL>
    __device__ static inline void run(const T* q, const T* k, const T* v, T* out,
                                      const RaggedParams& p, Lds& lds, uint32_t block,
                                      uint32_t blocks) {
        tile_rows<NT, QW, KS, BN, PAGED, FULL>(q, k, v, out, p, lds, block, blocks);
    }
};
template <int NT, int QW, int KS, int BN>
struct Tile<float, NT, QW, KS, BN> {
    typedef TileLdsF32<NT, QW, KS> Lds;
    static constexpr int kWaves = NT <= 2 ? 2 : 1;
    template <bool PAGED, bool FULL>
    __device__ static inline void run(const float* q, const float* k, const float* v, float* out,
                                      const RaggedParams& p, Lds& lds, uint32_t block,
                                      uint32_t blocks) {
        tile_rows_f32<NT, QW, KS, PAGED, FULL>(q, k, v, out, p, lds, block, blocks);
    }
};

template <typename T, int NT, int QW, int KS, int BN, bool FULL>
__global__ __launch_bounds__(64 * QW * KS, (Tile<T, NT, QW, KS, BN>::kWaves)) void k_packed_tiles(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    T* __restrict__ out, RaggedParams p) {
    typedef Tile<T, NT, QW, KS, BN> Body;
    __shared__ __align__(16) typename Body::Lds lds;
    Body::template run<false, FULL>(q, k, v, out, p, lds, blockIdx.x, gridDim.x);
}

// A paged batch of chunks and single tokens in one launch: the first
// split_blocks workgroups stream the keys of the requests of few rows, the
// others take tiles, so that the one's wait for memory runs beside the other's
// products (one MI355X: 65.5 us as two launches, 57 as one, 45.5 to 46.8 with the longest
// tiles first, for 4 chunks of 509 tokens and 20 single tokens over up to 4000 keys).
template <typename T, int NT, int QW, int KS, int BN, bool FULL>
__global__ __launch_bounds__(64 * QW * KS, (Tile<T, NT, QW, KS, BN>::kWaves)) void k_paged_mixed(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    T* __restrict__ out, RaggedParams p, uint32_t split_blocks) {
    static_assert(QW * KS == kSplitWaves, "both parts take four waves");
    typedef Tile<T, NT, QW, KS, BN> Body;
    constexpr int DP = NT <= 2 ? 64 : 128;
    union Lds {
        typename Body::Lds tile;
        SplitLds<DP> split;
    };
    __shared__ __align__(16) Lds lds;
    if (blockIdx.x < split_blocks)
        split_rows<T, DP, FULL && 32 * NT == DP>(q, k, v, out, p, lds.split, blockIdx.x);
    else
        Body::template run<true, FULL>(q, k, v, out, p, lds.tile, blockIdx.x - split_blocks,
                                       gridDim.x - split_blocks);
}

// -------------------------------------------------------------- workspace
//
// The split kernel's workgroups (two fit a CU: registers; three or four for the
// smaller ones of head size 64 gained nothing, 36.9 -> 38.1 / 38.9 us), their
// partials and tickets.
uint64_t split_slots(const rl_context* ctx, uint64_t kv_heads) {  // a KV head's
    return std::max<uint64_t>(2 * uint64_t(ctx->num_cus) / kv_heads, 1);
}

// What a call of these sizes needs; no less for more requests or KV heads.
rl_context::Workspace workspace_for(const rl_context* ctx, uint64_t sequences, uint64_t kv_heads) {
    const uint64_t groups = std::max<uint64_t>(2 * uint64_t(ctx->num_cus), kv_heads);
    return {sequences * kv_heads * kTicketStride * sizeof(uint32_t),
            2 * groups * kSplitRows * (128 + 2) * sizeof(float)};
}

// ------------------------------------------------------------- validation

constexpr uint64_t kMostRows = uint64_t(1) << 29;

// Checks shared by both attentions, the rows' part.
rl_status check_batch(uint64_t sequences, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads,
                      uint64_t head_dim, uint64_t max_queries, float scale) {
    if (sequences == 0 || tokens == 0 || q_heads == 0 || head_dim == 0 || max_queries == 0)
        return fail(RL_ERR_INVALID_SHAPE, "attention dimensions must be greater than zero");
    if (kv_heads == 0 || q_heads % kv_heads != 0)
        return fail(RL_ERR_MODEL_FORMAT, "Q heads %llu must be divisible by non-zero KV heads %llu",
                    (unsigned long long)q_heads, (unsigned long long)kv_heads);
    // a launch has fewer than 2^32 threads: of the tile kernels at most 8 a row and
    // 512 for each KV head of a request, beside 2^17 for the requests of few rows
    if (sequences > INT32_MAX || max_queries > UINT32_MAX || q_heads > kMostRows ||
        tokens > kMostRows / q_heads)
        return fail(RL_ERR_INVALID_SHAPE, "%llu rows of %llu heads exceed one launch",
                    (unsigned long long)tokens, (unsigned long long)q_heads);
    if (sequences * kv_heads >= (uint64_t(1) << 23) ||
        8 * tokens * q_heads + 512 * sequences * kv_heads + (1u << 17) > UINT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE,
                    "%llu requests of %llu KV heads exceed one launch beside %llu rows",
                    (unsigned long long)sequences, (unsigned long long)kv_heads,
                    (unsigned long long)(tokens * q_heads));
    if (head_dim > 512)
        return fail(RL_ERR_INVALID_SHAPE, "attention head size %llu exceeds 512",
                    (unsigned long long)head_dim);
    if (!(scale > 0.0f) || scale == INFINITY)
        return fail(RL_ERR_INVALID_SHAPE, "attention scale must be positive and finite, got %g",
                    double(scale));
    return RL_OK;
}

template <typename T, bool PAGED>
rl_status launch_rows(rl_context* ctx, const char* name, const T* q, const T* k, const T* v,
                      T* out, const RaggedParams& p) {
    if (uint64_t(p.tokens) * p.q_heads >= (uint64_t(1) << 26))
        return fail(RL_ERR_INVALID_SHAPE,
                    "%u rows of %u heads exceed one launch (head size, strides or alignment off "
                    "the matrix-core kernels')",
                    p.tokens, p.q_heads);
    const dim3 grid(p.tokens * p.q_heads), block(64);
    if (p.head_dim <= 64)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 1, PAGED>), grid, block, q, k, v, out, p);
    else if (p.head_dim <= 128)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 2, PAGED>), grid, block, q, k, v, out, p);
    else if (p.head_dim <= 256)
        RL_LAUNCH(ctx, (k_ragged_rows<T, 4, PAGED>), grid, block, q, k, v, out, p);
    else
        RL_LAUNCH(ctx, (k_ragged_rows<T, 8, PAGED>), grid, block, q, k, v, out, p);
    return after_launch(ctx, name);
}

// The tile kernels for a batch of at most `tokens` rows; paged ones with
// `split_blocks` workgroups for the requests of few rows.
template <typename T, int NT, int QW, int KS, int BN, bool PAGED>
void launch_tiles(rl_context* ctx, const T* q, const T* k, const T* v, T* out,
                  const RaggedParams& p, uint32_t split_blocks) {
    const uint64_t units =
        uint64_t(p.tokens) * p.group / kTileRows<QW> + p.sequences;
    const dim3 grid(uint32_t(units * p.kv_heads) + split_blocks), block(64 * QW * KS);
    const bool full = p.head_dim == 32 * NT;
    if constexpr (PAGED) {
        if (full)
            RL_LAUNCH(ctx, (k_paged_mixed<T, NT, QW, KS, BN, true>), grid, block, q, k, v, out, p,
                      split_blocks);
        else
            RL_LAUNCH(ctx, (k_paged_mixed<T, NT, QW, KS, BN, false>), grid, block, q, k, v, out,
                      p, split_blocks);
    } else {
        if (full)
            RL_LAUNCH(ctx, (k_packed_tiles<T, NT, QW, KS, BN, true>), grid, block, q, k, v, out,
                      p);
        else
            RL_LAUNCH(ctx, (k_packed_tiles<T, NT, QW, KS, BN, false>), grid, block, q, k, v, out,
                      p);
    }
}
// Which tiles, from the batch's 128-row tiles (`wide`) and how many of those run
// at once (`slots`).  Measured (one MI355X, us; 15/5 heads of 64 unless another
// head size is named, `wide` in brackets):
//   f16, packed: QW 8 (4 for head sizes other than 64) from `slots` on, 2 x 2 below:
//     22.6 / 16.7 [325], 50.7 / 45.6 [965], 75.7 / 75.2 [1675]; D 96 22.2 / 18.8 [261],
//     37.7 / 36.7 [537]; D 128 21.4 / 19.2 [352], 41.7 / 44.4 [712].  Packed, QW 8
//     against 4 at 64: 536 / 558 for 60 prompts; D 128 with blocks of 32 keys against
//     64 (three waves a SIMD against two): 357 / 368 for 8 prompts of up to 4096.
//     The mixed kernel does not leave the registers for either.
//   f16, paged, whose other part takes places too: QW 4 from half of `slots` on, 2 x 2
//     below: 55.4 / 49.2 [350], 65.2 / 76 [700]; D 128 67.5 / 71.4 [296].  Below half
//     a tile a CU, 1 x 4 at 64: 24.6 / 28.6 [35], 32.5 / 31.8 [80], 27.2 / 30.2
//     [115]; 40.1 / 32.6 [175].  Not at 128, where its LDS leaves one workgroup a CU:
//     36.5 / 45.0 [5], 44.1 / 47.4 [50], but 73.2 / 49.2 [75], and 18.9 / 16.2 [40] over
//     up to 500 keys.  At 96 and 32, where 2 x 2 is used, it would be the faster one:
//     39.5 / 43.6 [5], 42.2 / 45.9 [19] and 17.0 / 20.1 [5], 19.8 / 24.1 [56].
//   f32: 1 x 4 below a tile a CU, 2 x 2 from there on (4 x 1 for more than 64 elements):
//     24.5 / 30.7 [155], 61.7 / 49.7 [445]; D 128 50.7 / 53.9 [144], 116 / 76.4 [352].
// Longest tiles first (a search over the lengths in every workgroup, about 0.7 us)
// pays where the last tiles would decide:
//   f16, packed, `slots` to 8 `slots`: 11.1 without / 11.6 with [155], 92 / 75.8 [1675], 380 / 356
//     [6810]; D 96 135 / 119 [1611]; D 128 41.1 / 41.7 [712], 1326 / 1402 [11 thousand]
//   f16, paged, from 3/8 tile a CU on: 32.5 / 33.8 [80], 31.8 / 27.2 [115], 39.4 / 32.6
//     [175]; D 128 116 / 101 [600]
//   f32 below 4 tiles a CU: 28.9 / 27.5 [254], 50.6 / 40.9 [325], 61.4 / 62.6 [410],
//     though 23.6 / 24.5 at [155]; more than 64 elements from a tile a CU on:
//     48.2 / 50.7 [144], 135 / 126 [536]
template <typename T, bool PAGED>
void launch_tiles(rl_context* ctx, const T* q, const T* k, const T* v, T* out, RaggedParams p,
                  uint32_t sb) {
    const uint64_t cus = uint64_t(ctx->num_cus);
    const uint64_t wide = (uint64_t(p.tokens) * p.group / kTileRows<4>) * p.kv_heads;
    const uint32_t nt = (p.head_dim + 31) / 32;
    if constexpr (std::is_same<T, half_t>::value) {
        const uint64_t slots = (nt <= 2 ? 4 : 2) * cus;
        p.longest_first = p.sequences <= 64 && wide >= (PAGED ? 3 * cus / 8 : slots) &&
                          wide <= 8 * slots;
        if (wide >= (PAGED ? slots / 2 : slots)) {
            if (nt == 1) launch_tiles<T, 1, 4, 1, 64, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 2)
                launch_tiles<T, 2, PAGED ? 4 : 8, 1, 64, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 3) launch_tiles<T, 3, 4, 1, 64, PAGED>(ctx, q, k, v, out, p, sb);
            else launch_tiles<T, 4, 4, 1, PAGED ? 64 : 32, PAGED>(ctx, q, k, v, out, p, sb);
        } else if (PAGED && nt == 2 && wide < cus / 2) {
            launch_tiles<T, 2, 1, 4, 32, PAGED>(ctx, q, k, v, out, p, sb);
        } else {
            if (nt == 1) launch_tiles<T, 1, 2, 2, 64, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 2) launch_tiles<T, 2, 2, 2, 64, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 3) launch_tiles<T, 3, 2, 2, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else launch_tiles<T, 4, 2, 2, 32, PAGED>(ctx, q, k, v, out, p, sb);
        }
    } else {
        p.longest_first =
            p.sequences <= 64 && wide >= (nt >= 3 ? cus : 0) && wide < 4 * cus;
        if (wide >= cus) {
            if (nt == 1) launch_tiles<T, 1, 2, 2, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 2) launch_tiles<T, 2, 2, 2, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 3) launch_tiles<T, 3, 4, 1, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else launch_tiles<T, 4, 4, 1, 32, PAGED>(ctx, q, k, v, out, p, sb);
        } else {
            if (nt == 1) launch_tiles<T, 1, 1, 4, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 2) launch_tiles<T, 2, 1, 4, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else if (nt == 3) launch_tiles<T, 3, 1, 4, 32, PAGED>(ctx, q, k, v, out, p, sb);
            else launch_tiles<T, 4, 1, 4, 32, PAGED>(ctx, q, k, v, out, p, sb);
        }
    }
}

template <typename T>
void launch_split(rl_context* ctx, const T* q, const T* k, const T* v, T* out,
                  const RaggedParams& p) {
    const dim3 grid(p.slots * p.kv_heads), block(64 * kSplitWaves);
    if (p.head_dim == 64)
        RL_LAUNCH(ctx, (k_ragged_split<T, 64, true>), grid, block, q, k, v, out, p);
    else if (p.head_dim < 64)
        RL_LAUNCH(ctx, (k_ragged_split<T, 64, false>), grid, block, q, k, v, out, p);
    else if (p.head_dim == 128)
        RL_LAUNCH(ctx, (k_ragged_split<T, 128, true>), grid, block, q, k, v, out, p);
    else
        RL_LAUNCH(ctx, (k_ragged_split<T, 128, false>), grid, block, q, k, v, out, p);
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
    const T* qd = static_cast<const T*>(q->data);
    const T* kd = static_cast<const T*>(k->data);
    const T* vd = static_cast<const T*>(v->data);
    T* od = static_cast<T*>(out->data);
    // the matrix-core kernel: rows of whole 16-byte pieces on their grid, up to
    // 128 elements, row strides that fit its 32-bit byte steps
    bool matrix = D * es % 16 == 0 && D <= 128 && aligned_to(qd, 16) && aligned_to(kd, 16) &&
                  aligned_to(vd, 16) && aligned_to(od, 16);
    for (const uint64_t* strides : {q_strides, k_strides, v_strides})
        matrix = matrix && strides[0] * es % 16 == 0 && strides[1] * es % 16 == 0 &&
                 strides[0] <= UINT32_MAX / es;
    if (!matrix) return launch_rows<T, false>(ctx, name, qd, kd, vd, od, p);
    launch_tiles<T, false>(ctx, qd, kd, vd, od, p, 0);
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
    if (max_blocks > UINT32_MAX || max_context > INT32_MAX)
        return fail(RL_ERR_INVALID_SHAPE, "attention key range exceeds i32");
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
    const rl_context::Workspace need = workspace_for(ctx, sequences, kv_heads);
    const uint64_t slots = split_slots(ctx, kv_heads);
    const auto held = ctx->workspaces.find(workspace->data);
    if (held == ctx->workspaces.end())
        return fail(RL_ERR_INVALID_ARGUMENT,
                    "the workspace is not one of rl_paged_attention_workspace on this context");
    if (held->second.ticket_bytes < need.ticket_bytes ||
        held->second.partial_bytes < need.partial_bytes)
        return fail(RL_ERR_INVALID_SHAPE,
                    "the workspace holds %llu + %llu bytes, expected %llu + %llu",
                    (unsigned long long)held->second.ticket_bytes,
                    (unsigned long long)held->second.partial_bytes,
                    (unsigned long long)need.ticket_bytes,
                    (unsigned long long)need.partial_bytes);
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
    const T* qd = static_cast<const T*>(q->data);
    const T* kd = static_cast<const T*>(k_pages->data);
    const T* vd = static_cast<const T*>(v_pages->data);
    T* od = static_cast<T*>(out->data);
    // the matrix-core kernels: rows of whole 16-byte pieces up to 128 elements,
    // pages of at least the eight rows a lane's value loads take from one
    const uint64_t page_bytes = kv_heads * page_size * head_dim * es;
    const bool matrix = head_dim * es % 16 == 0 && head_dim <= 128 && page_size >= 8 &&
                        page_bytes <= UINT32_MAX && aligned_to(qd, 16) && aligned_to(kd, 16) &&
                        aligned_to(vd, 16) && aligned_to(od, 16);
    const uint64_t most_rows = std::min(max_queries, tokens) * p.group;
    uint32_t split_blocks = 0;
    p.page_bytes = uint32_t(page_bytes);
    p.head_bytes = uint32_t(page_size * head_dim * es);
    if (matrix && p.group <= kSplitRows) {
        char* ws = static_cast<char*>(workspace->data);
        p.small_rows = kSplitRows;
        p.slots = uint32_t(slots);
        p.tickets = reinterpret_cast<uint32_t*>(ws);
        p.part = reinterpret_cast<float*>(ws + held->second.ticket_bytes);
        p.part_ml = p.part + 2 * slots * kv_heads * kSplitRows * 128;
        if (most_rows <= kSplitRows) {
            launch_split<T>(ctx, qd, kd, vd, od, p);
            return after_launch(ctx, name);
        }
        // beside tiles: half of the workgroups that would fill the CUs (60 single tokens of
        // up to 8000 keys and a chunk of 30 tokens: 183 us, a quarter 295; 4 chunks and
        // 20 single tokens of up to 4000 keys: 57 / 56).  The host knows the bound alone, so
        // a batch of single tokens under a loose one has as few: 36.9 -> 41.8 us for 64 of
        // up to 4000 keys (15/5 heads of 64), 16.4 -> 18.2 for 16 of up to 1500 (32/8 of
        // 128), 155.8 -> 156.8 for 60 of up to 8000.
        p.slots = uint32_t(std::max<uint64_t>(slots / 2, 1));
        split_blocks = p.slots * p.kv_heads;
    }
    if (!matrix) return launch_rows<T, true>(ctx, name, qd, kd, vd, od, p);
    launch_tiles<T, true>(ctx, qd, kd, vd, od, p, split_blocks);
    return after_launch(ctx, name);
}

rl_status workspace_entry(rl_context* ctx, uint64_t sequences, uint64_t kv_heads,
                          rl_buffer* out) {
    if (out == nullptr) return fail(RL_ERR_INVALID_ARGUMENT, "output buffer pointer is null");
    *out = rl_buffer{nullptr, 0, 0};
    if (rl_status st = check_batch(sequences, 1, kv_heads, kv_heads, 1, 1, 1.0f)) return st;
    if (rl_status st = require_context(ctx)) return st;
    // this context's recording, or another's that reached its stream by an event
    hipStreamCaptureStatus recording = hipStreamCaptureStatusNone;
    const hipError_t known = hipStreamIsCapturing(ctx->stream, &recording);
    if (known != hipSuccess)
        return fail(RL_ERR_DEVICE, "workspace: %s", hipGetErrorString(known));
    if (ctx->capturing || recording != hipStreamCaptureStatusNone)
        return fail(RL_ERR_DEVICE, "a workspace cannot be made while recording a graph");
    const rl_context::Workspace size = workspace_for(ctx, sequences, kv_heads);
    const uint64_t bytes = size.ticket_bytes + size.partial_bytes;
    rl_buffer made{nullptr, 0, 0};
    if (rl_status st = rl_buffer_empty(ctx, bytes, 1, &made)) return st;
    const hipError_t err = hipMemsetAsync(made.data, 0, size.ticket_bytes, ctx->stream);
    if (err != hipSuccess) {
        rl_buffer_release(ctx, &made);
        return fail(RL_ERR_DEVICE, "workspace: %s", hipGetErrorString(err));
    }
    ctx->workspaces[made.data] = size;
    *out = made;
    return RL_OK;
}

}  // namespace
}  // namespace rl

using namespace rl;

extern "C" {

rl_status rl_paged_attention_workspace(rl_context* ctx, uint64_t sequences, uint64_t kv_heads,
                                       rl_buffer* out) {
    return guarded([&] { return workspace_entry(ctx, sequences, kv_heads, out); });
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
