// ragged.hpp -- shared by the paged cache (paged.hip) and the attentions over
// ragged batches (ragged_attention.hip): argument checks of their buffers.
#ifndef RUSTLLM_RAGGED_HPP
#define RUSTLLM_RAGGED_HPP

#include "common.hpp"

#include <exception>

namespace rl {

// A C entry's body: what it throws (an allocation that fails on the host)
// becomes a status.
template <typename F>
rl_status guarded(F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        return fail(RL_ERR_DEVICE, "%s", e.what());
    } catch (...) {
        return fail(RL_ERR_DEVICE, "unknown error");
    }
}

// A [tokens, heads, D] view of dims/strides with a unit innermost stride,
// all of it inside its buffer of `es`-byte elements.
rl_status check_token_view(const char* what, const rl_buffer* b, const uint64_t* dims,
                           const uint64_t* strides, uint64_t es);
// A buffer of exactly `len` u32 values.
rl_status check_u32(const char* what, const rl_buffer* b, uint64_t len);
// A power-of-two page size and slots that fit 32 bits.
rl_status check_pages(uint64_t pages, uint64_t page_size);
// A pool of [pages, kv_heads, page_size, head_dim] elements (after check_pages).
rl_status check_pool(const char* what, const rl_buffer* b, uint64_t pages, uint64_t kv_heads,
                     uint64_t page_size, uint64_t head_dim, uint64_t es);
uint32_t log2_of(uint64_t power);

}  // namespace rl

#endif
