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
// The per-row kernels here take any head_dim up to 256, stride and alignment: one wave per
// query row (dK/dV: per key row), 64 keys (queries) at a time with one dot product a lane, then
// the weighted sum with the head's values over the lanes.
#include <algorithm>

#include "window.hpp"

namespace vkh {
namespace {

constexpr int WNT = 256, WPB = WNT / 64;
constexpr int WE = 4;  // values of a head row per lane (head_dim <= 256)

// dot product of a row with `hd` values in LDS
template <class T>
VKH_DEV float row_dot(const T *r, const float *q, int hd) {
    float s = 0.f;
    for (int d = 0; d < hd; ++d) s = fmaf(to_f32(r[d]), q[d], s);
    return s;
}

template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_fwd_any_k(WindowArgs a) {
    __shared__ float qs[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64, hd = a.hd;
    const long it = (long)blockIdx.x * WPB + w;
    const bool live = it < (long)a.n_batch * a.n_q * a.n_heads;
    const int h = (int)(it % a.n_heads);
    const long row = it / a.n_heads;
    const int r = (int)(row % a.n_q), b = live ? (int)(row / a.n_q) : 0;
    if (live)
        for (int d = lane; d < hd; d += 64) qs[w][d] = to_f32(((const T *)a.q)[row * a.ldq + (long)h * hd + d]);
    __syncthreads();
    if (!live) return;
    const Span s = span_of(a, b);
    const int t = r + s.off;
    const int lo = max(0, t - a.window + 1), hi = r < s.ql ? t + 1 : 0;  // the window's keys
    const int ns = min(a.n_sink, lo), n = hi > 0 ? ns + max(0, hi - lo) : 0;
    const long kv0 = (long)b * a.n_kv, hk = (long)(h / (a.n_heads / a.n_kv_heads)) * hd;
    const T *K = (const T *)a.k + kv0 * a.ldk + hk, *V = (const T *)a.v + kv0 * a.ldv + hk;
    auto key = [&](int i) { return (long)(i < ns ? i : lo + i - ns); };
    float m = -INFINITY, l = 0.f, acc[WE] = {};
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        const float x = i < n ? a.scale * row_dot(K + key(i) * a.ldk, qs[w], hd) : -INFINITY;
        const float mn = fmaxf(m, wave_max(x)), ms = mn == -INFINITY ? 0.f : mn;
        const float p = i < n ? expf(x - ms) : 0.f, so = expf(m - ms);
        l = l * so + wave_sum(p);
        m = mn;
#pragma unroll
        for (int e = 0; e < WE; ++e) acc[e] *= so;
        for (int j = 0; j < min(64, n - i0); ++j) {
            const float pj = __shfl(p, j, 64);
            const T *vr = V + key(i0 + j) * a.ldv;
#pragma unroll
            for (int e = 0; e < WE; ++e)
                if (lane + 64 * e < hd) acc[e] = fmaf(pj, to_f32(vr[lane + 64 * e]), acc[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    TO *o = (TO *)a.o + row * a.ldo + (long)h * hd;
#pragma unroll
    for (int e = 0; e < WE; ++e)
        if (lane + 64 * e < hd) o[lane + 64 * e] = (TO)(l == 0.f ? 0.f : acc[e] * inv);
    if (a.lse && lane == 0) a.lse[row * a.n_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

// D and dQ of one query row.
template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_dq_any_k(WindowArgs a) {
    __shared__ float qs[WPB][256], os[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64, hd = a.hd;
    const long it = (long)blockIdx.x * WPB + w;
    const bool live = it < (long)a.n_batch * a.n_q * a.n_heads;
    const int h = (int)(it % a.n_heads);
    const long row = it / a.n_heads;
    const int r = (int)(row % a.n_q), b = live ? (int)(row / a.n_q) : 0;
    float dd = 0.f;
    if (live)
        for (int d = lane; d < hd; d += 64) {
            qs[w][d] = to_f32(((const T *)a.q)[row * a.ldq + (long)h * hd + d]);
            os[w][d] = to_f32(((const T *)a.dout)[row * a.lddo + (long)h * hd + d]);
            dd = fmaf(os[w][d], to_f32(((const TO *)a.o)[row * a.ldo + (long)h * hd + d]), dd);
        }
    __syncthreads();
    if (!live) return;
    const Span s = span_of(a, b);
    const int t = r + s.off;
    const float lse = a.lse[row * a.n_heads + h];
    const bool seen = r < s.ql && t >= 0 && lse != -INFINITY;
    const int lo = max(0, t - a.window + 1), ns = min(a.n_sink, lo), n = seen ? ns + t + 1 - lo : 0;
    dd = seen ? wave_sum(dd) : 0.f;
    if (lane == 0) a.d[row * a.n_heads + h] = dd;
    const long kv0 = (long)b * a.n_kv, hk = (long)(h / (a.n_heads / a.n_kv_heads)) * hd;
    const T *K = (const T *)a.k + kv0 * a.ldk + hk, *V = (const T *)a.v + kv0 * a.ldv + hk;
    auto key = [&](int i) { return (long)(i < ns ? i : lo + i - ns); };
    float acc[WE] = {};
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        float ds = 0.f;
        if (i < n) {
            const float p = expf(a.scale * row_dot(K + key(i) * a.ldk, qs[w], hd) - lse);
            ds = p * (row_dot(V + key(i) * a.ldv, os[w], hd) - dd);
        }
        for (int j = 0; j < min(64, n - i0); ++j) {
            const float dj = __shfl(ds, j, 64);
            const T *kr = K + key(i0 + j) * a.ldk;
#pragma unroll
            for (int e = 0; e < WE; ++e)
                if (lane + 64 * e < hd) acc[e] = fmaf(dj, to_f32(kr[lane + 64 * e]), acc[e]);
        }
    }
    TO *dq = (TO *)a.dq + row * a.lddq + (long)h * hd;
#pragma unroll
    for (int e = 0; e < WE; ++e)
        if (lane + 64 * e < hd) dq[lane + 64 * e] = (TO)(acc[e] * a.scale);
}

// dK and dV of one key row, over the query heads that share it and the rows that see it.
template <class T, class TO>
__global__ __launch_bounds__(WNT) void window_dkv_any_k(WindowArgs a) {
    __shared__ float ks[WPB][256], vs[WPB][256];
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64, hd = a.hd;
    const long it = (long)blockIdx.x * WPB + w;
    const bool live = it < (long)a.n_batch * a.n_kv * a.n_kv_heads;
    const int kh = (int)(it % a.n_kv_heads);
    const long row = it / a.n_kv_heads;
    const int j = (int)(row % a.n_kv), b = live ? (int)(row / a.n_kv) : 0;
    const Span s = span_of(a, b);
    if (live && j < s.kl)
        for (int d = lane; d < hd; d += 64) {
            ks[w][d] = to_f32(((const T *)a.k)[row * a.ldk + (long)kh * hd + d]);
            vs[w][d] = to_f32(((const T *)a.v)[row * a.ldv + (long)kh * hd + d]);
        }
    __syncthreads();
    if (!live) return;
    // rows at positions j .. j + window - 1, or from j on for a sink
    const int r0 = max(0, j - s.off), grp = a.n_heads / a.n_kv_heads;
    const long end = j < a.n_sink ? s.ql : min((long)s.ql, (long)j - s.off + a.window);
    const int n = j < s.kl ? (int)max(0L, end - r0) : 0;
    float dk[WE] = {}, dv[WE] = {};
    for (int h = kh * grp; h < (kh + 1) * grp; ++h) {
        const long q0 = (long)b * a.n_q + r0;
        const T *Q = (const T *)a.q + q0 * a.ldq + (long)h * hd, *G = (const T *)a.dout + q0 * a.lddo + (long)h * hd;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + lane;
            float p = 0.f, ds = 0.f;
            const float lse = i < n ? a.lse[(q0 + i) * a.n_heads + h] : -INFINITY;
            if (lse != -INFINITY) {
                p = expf(a.scale * row_dot(Q + i * a.ldq, ks[w], hd) - lse);
                ds = p * (row_dot(G + i * a.lddo, vs[w], hd) - a.d[(q0 + i) * a.n_heads + h]);
            }
            for (int x = 0; x < min(64, n - i0); ++x) {
                if (__shfl(lse, x, 64) == -INFINITY) continue;
                const float px = __shfl(p, x, 64), dx = __shfl(ds, x, 64);
                const T *qr = Q + (i0 + x) * a.ldq, *gr = G + (i0 + x) * a.lddo;
#pragma unroll
                for (int e = 0; e < WE; ++e)
                    if (lane + 64 * e < hd) {
                        dk[e] = fmaf(dx, to_f32(qr[lane + 64 * e]), dk[e]);
                        dv[e] = fmaf(px, to_f32(gr[lane + 64 * e]), dv[e]);
                    }
            }
        }
    }
    TO *ok = (TO *)a.dk + row * a.lddk + (long)kh * hd, *ov = (TO *)a.dv + row * a.lddv + (long)kh * hd;
#pragma unroll
    for (int e = 0; e < WE; ++e)
        if (lane + 64 * e < hd) {
            ok[lane + 64 * e] = (TO)(dk[e] * a.scale);
            ov[lane + 64 * e] = (TO)dv[e];
        }
}

// f(operand type, result type)
template <class F>
void by_types(const WindowArgs &a, F f) {
    if (a.dt == DType::F32) f(float{}, float{});
    else if (a.odt == DType::F32) f(bf16{}, float{});
    else f(bf16{}, bf16{});
}
unsigned row_blocks(long rows) { return (unsigned)((rows + WPB - 1) / WPB); }

}  // namespace

size_t window_fwd_ws_bytes(const WindowArgs &) { return 0; }
size_t window_bwd_ws_bytes(const WindowArgs &a) { return window16_bwd_ws_bytes(a); }

hipError_t window_forward(const WindowArgs &a, hipStream_t st) {
    if (window16_forward(a, st)) return hipGetLastError();
    by_types(a, [&](auto t, auto o) {
        hipLaunchKernelGGL((window_fwd_any_k<decltype(t), decltype(o)>),
                           dim3(row_blocks((long)a.n_batch * a.n_q * a.n_heads)), dim3(WNT), 0, st, a);
    });
    return hipGetLastError();
}

hipError_t window_backward(const WindowArgs &a, hipStream_t st) {
    if (window16_backward(a, st)) return hipGetLastError();
    by_types(a, [&](auto t, auto o) {
        hipLaunchKernelGGL((window_dq_any_k<decltype(t), decltype(o)>),
                           dim3(row_blocks((long)a.n_batch * a.n_q * a.n_heads)), dim3(WNT), 0, st, a);
        hipLaunchKernelGGL((window_dkv_any_k<decltype(t), decltype(o)>),
                           dim3(row_blocks((long)a.n_batch * a.n_kv * a.n_kv_heads)), dim3(WNT), 0, st, a);
    });
    return hipGetLastError();
}

}  // namespace vkh
