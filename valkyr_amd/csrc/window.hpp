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

// ── one row at a time ────────────────────────────────────────────────────
// A wave's work on one query row (dK/dV: key row), 64 keys (queries) at a time with one dot product
// a lane, then the weighted sum with the head's values over the lanes.  `q`, `g` (`k`, `v`) are
// head_dim floats of the wave's own LDS each.  Any head_dim up to 256, stride and alignment.
constexpr int WE = 4;  // values of a head row per lane

// dot product of a row with `hd` values in LDS
template <class T>
VKH_DEV float row_dot(const T *r, const float *q, int hd) {
    float s = 0.f;
    for (int d = 0; d < hd; ++d) s = fmaf(to_f32(r[d]), q[d], s);
    return s;
}
// LDS written by a wave for itself is read by its other lanes
VKH_DEV void wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// O and LSE of row r of head h of sequence b.
template <class T, class TO>
VKH_DEV void window_fwd_row(const WindowArgs &a, int b, int r, int h, float *q, int lane) {
    const int hd = a.hd;
    const long row = (long)b * a.n_q + r;
    wave_lds();
    for (int d = lane; d < hd; d += 64) q[d] = to_f32(((const T *)a.q)[row * a.ldq + (long)h * hd + d]);
    wave_lds();
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
        const float x = i < n ? a.scale * row_dot(K + key(i) * a.ldk, q, hd) : -INFINITY;
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

// D and dQ of row r of head h of sequence b.
template <class T, class TO>
VKH_DEV void window_dq_row(const WindowArgs &a, int b, int r, int h, float *q, float *g, int lane) {
    const int hd = a.hd;
    const long row = (long)b * a.n_q + r;
    float dd = 0.f;
    wave_lds();
    for (int d = lane; d < hd; d += 64) {
        q[d] = to_f32(((const T *)a.q)[row * a.ldq + (long)h * hd + d]);
        g[d] = to_f32(((const T *)a.dout)[row * a.lddo + (long)h * hd + d]);
        dd = fmaf(g[d], to_f32(((const TO *)a.o)[row * a.ldo + (long)h * hd + d]), dd);
    }
    wave_lds();
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
            const float p = expf(a.scale * row_dot(K + key(i) * a.ldk, q, hd) - lse);
            ds = p * (row_dot(V + key(i) * a.ldv, g, hd) - dd);
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

// dK and dV of key j of KV head kh of sequence b, over the query heads that share it and those of
// the rows that see it that mine(h, row) names: dk and dv point at head_dim results of type TR.
template <class T, class TR, class Mine>
VKH_DEV void window_dkv_row(const WindowArgs &a, int b, int j, int kh, float *k, float *v, TR *ok, TR *ov, int lane,
                            Mine mine) {
    const int hd = a.hd;
    const long row = (long)b * a.n_kv + j;
    const Span s = span_of(a, b);
    wave_lds();
    if (j < s.kl)
        for (int d = lane; d < hd; d += 64) {
            k[d] = to_f32(((const T *)a.k)[row * a.ldk + (long)kh * hd + d]);
            v[d] = to_f32(((const T *)a.v)[row * a.ldv + (long)kh * hd + d]);
        }
    wave_lds();
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
            const float lse = i < n && mine(h, r0 + i) ? a.lse[(q0 + i) * a.n_heads + h] : -INFINITY;
            if (lse != -INFINITY) {
                p = expf(a.scale * row_dot(Q + i * a.ldq, k, hd) - lse);
                ds = p * (row_dot(G + i * a.lddo, v, hd) - a.d[(q0 + i) * a.n_heads + h]);
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
#pragma unroll
    for (int e = 0; e < WE; ++e)
        if (lane + 64 * e < hd) {
            ok[lane + 64 * e] = (TR)(dk[e] * a.scale);
            ov[lane + 64 * e] = (TR)dv[e];
        }
}

// ── host ─────────────────────────────────────────────────────────────────
// The tile kernels on bf16 operands (k_attn_window16.hip): false, launching nothing, for a shape,
// stride or alignment that they do not take.
bool window16_forward(const WindowArgs &a, hipStream_t st);
bool window16_backward(const WindowArgs &a, hipStream_t st);
size_t window16_bwd_ws_bytes(const WindowArgs &a);

}  // namespace vkh
