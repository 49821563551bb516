// Attention with a sliding window and a few first keys that stay visible, forward (with the
// log-sum-exp) and backward.
//
// Query row r of a sequence with ql rows and kl keys is at position t = r + kl - ql and sees key
// j where j <= t and (j > t - window or j < n_sink).  With S = scale q k^T over the seen keys,
//   O = sum_j P_j v_j,  P = exp(S - LSE),  LSE = log sum_j exp(S_j)
//   D = sum_d O dO,  dS = P (dO v - D) scale,  dQ = dS K,  dK = dS^T Q,  dV = P^T dO
// and query heads h share KV head h / (n_heads / n_kv_heads), whose gradients are their sums.
// A row that sees no key (rows behind a sequence's last query; positions below 0) has O = 0,
// LSE = -inf and no gradient.  Pairs that are not seen take no part: what their keys, values or
// queries hold (an infinity, a NaN, memory never written) reaches no result.
//
// The kernels here take any head_dim up to 256, stride and alignment, one wave a row.
#include <algorithm>

#include "window.hpp"

namespace vkh {
namespace {

constexpr int WNT = 256, WPB = WNT / 64;
template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_fwd_any_k(WindowArgs a) {
    __shared__ float qs[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const long it = block_number() * WPB + w, row = it / a.n_heads;
    if (row >= (long)a.n_batch * a.n_q) return;
    window_fwd_row<T, TO>(a, (int)(row / a.n_q), (int)(row % a.n_q), (int)(it % a.n_heads), qs[w], lane);
}
template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_dq_any_k(WindowArgs a) {
    __shared__ float qs[WPB][256], gs[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const long it = block_number() * WPB + w, row = it / a.n_heads;
    if (row >= (long)a.n_batch * a.n_q) return;
    window_dq_row<T, TO>(a, (int)(row / a.n_q), (int)(row % a.n_q), (int)(it % a.n_heads), qs[w], gs[w], lane);
}
template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_dkv_any_k(WindowArgs a) {
    __shared__ float ks[WPB][256], vs[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
    const long it = block_number() * WPB + w, row = it / a.n_kv_heads;
    if (row >= (long)a.n_batch * a.n_kv) return;
    const int kh = (int)(it % a.n_kv_heads);
    window_dkv_row<T>(a, (int)(row / a.n_kv), (int)(row % a.n_kv), kh, ks[w], vs[w],
                      (TO *)a.dk + row * a.lddk + (long)kh * a.hd, (TO *)a.dv + row * a.lddv + (long)kh * a.hd, lane,
                      [](int, int) { return true; });
}

// f(operand type, result type)
template <class F>
void by_types(const WindowArgs &a, F f) {
    if (a.dt == DType::F32) f(float{}, float{});
    else if (a.odt == DType::F32) f(bf16{}, float{});
    else f(bf16{}, bf16{});
}
dim3 row_blocks(long rows) { return long_grid((rows + WPB - 1) / WPB); }

}  // namespace

size_t window_fwd_ws_bytes(const WindowArgs &a) { return window16_fwd_ws_bytes(a) + window32_fwd_ws_bytes(a); }
size_t window_bwd_ws_bytes(const WindowArgs &a) { return window16_bwd_ws_bytes(a) + window32_bwd_ws_bytes(a); }

hipError_t window_forward(const WindowArgs &a, hipStream_t st) {
    if (window16_forward(a, st) || window32_forward(a, st)) return hipGetLastError();
    by_types(a, [&](auto t, auto o) {
        hipLaunchKernelGGL((window_fwd_any_k<decltype(t), decltype(o)>),
                           row_blocks((long)a.n_batch * a.n_q * a.n_heads), dim3(WNT), 0, st, a);
    });
    return hipGetLastError();
}

hipError_t window_backward(const WindowArgs &a, hipStream_t st) {
    if (window16_backward(a, st) || window32_backward(a, st)) return hipGetLastError();
    by_types(a, [&](auto t, auto o) {
        hipLaunchKernelGGL((window_dq_any_k<decltype(t), decltype(o)>),
                           row_blocks((long)a.n_batch * a.n_q * a.n_heads), dim3(WNT), 0, st, a);
        if (hipPeekAtLastError() != hipSuccess) return;  // (D is not there)
        hipLaunchKernelGGL((window_dkv_any_k<decltype(t), decltype(o)>),
                           row_blocks((long)a.n_batch * a.n_kv * a.n_kv_heads), dim3(WNT), 0, st, a);
    });
    return hipGetLastError();
}

}  // namespace vkh
