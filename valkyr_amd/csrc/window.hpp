// What the windowed attention's kernel files share.
#pragma once

#include "ops.hpp"

namespace vkh {

// Query rows, keys and the first row's position of a sequence.
struct Span {
    int ql, kl, off;
};
VKH_DEV Span span_of(const WindowArgs &a, int b) {
    Span s;
    s.ql = a.q_len ? (int)min(a.q_len[b], (unsigned)a.n_q) : a.n_q;
    s.kl = a.kv_len ? (int)min(a.kv_len[b], (unsigned)a.n_kv) : a.n_kv;
    s.off = s.kl - s.ql;
    return s;
}

// The tile kernels on bf16 operands (k_attn_window16.hip): false, launching nothing, for a shape,
// stride or alignment that they do not take.
bool window16_forward(const WindowArgs &a, hipStream_t st);
bool window16_backward(const WindowArgs &a, hipStream_t st);
size_t window16_bwd_ws_bytes(const WindowArgs &a);

}  // namespace vkh
