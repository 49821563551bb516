// What the windowed attention's kernel files share.
#pragma once

#include <math.h>

#include <algorithm>

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

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int kAll = 0x7fffffff;  // the window of a sink

// The (sequence, KV head) of block x, and its turn y among that pair's blocks.  Blocks go round the
// 8 XCDs by their number; runs of up to `run` turns of one pair sit on one XCD and share its L2, and
// from run to run the pairs move on, so that pairs with little to do (short sequences of a padded
// batch) do not leave the XCD that would be theirs idle.
struct Pair {
    int bk, y;
};
VKH_DEV Pair pair_of(int x, int blocks, int pairs, int run) {
    const int y = x / pairs, r = max(1, min(run, blocks / pairs / pairs));
    return Pair{(x % pairs + y / r) % pairs, y};
}

// Whether position t sees key j (t = -1: a row that sees none).
VKH_DEV bool sees(const WindowArgs &a, int t, int j) {
    return (unsigned)(t - j) < (unsigned)(j < a.n_sink ? kAll : a.window);
}
// Whether all positions ta .. tb see all keys j0 .. j1, or none sees any.
VKH_DEV bool all_seen(const WindowArgs &a, int ta, int tb, int j0, int j1) {
    return j1 <= ta && (j0 > tb - a.window || j1 < a.n_sink);
}
VKH_DEV bool none_seen(const WindowArgs &a, int ta, int tb, int j0, int j1) {
    return tb < ta || j0 > tb || (j1 <= ta - a.window && j0 >= a.n_sink);
}

// hide(ks, r) for the keys k0 + 16 ks + 4 g + r, ks < KS, that position t does not see.
template <int KS, class F>
VKH_DEV void for_hidden(const WindowArgs &a, int t, int k0, int g, F hide) {
    int x = t - k0 - 4 * g;
    if (k0 < a.n_sink && k0 + 16 * KS > a.n_sink) {  // sinks and others: the others outside the window
        const int ns = a.n_sink - k0 - 4 * g;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * ks + r >= ns && x - 16 * ks - r >= a.window) hide(ks, r);
    }
    asm("" : "+v"(x));  // (the differences below are not kept from those above)
    const unsigned reach = k0 < a.n_sink ? kAll : a.window;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if ((unsigned)(x - 16 * ks - r) >= reach) hide(ks, r);
}

VKH_DEV void store4(float *p, float x, float y, float z, float w) {
    *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
}
VKH_DEV void store4(bf16 *p, float x, float y, float z, float w) {
    bf16x4 o;
    o[0] = (bf16)x; o[1] = (bf16)y; o[2] = (bf16)z; o[3] = (bf16)w;
    *reinterpret_cast<bf16x4 *>(p) = o;
}

// The key tiles (of BN keys) that a block of query rows r0 .. r1 - 1 walks: those of the sinks that
// lie before its window, then its window's.
struct KeyTiles {
    int ta, tb;     // live positions (tb < ta: none)
    int n_sink, w0, n;
    VKH_DEV int tile(int it) const { return it < n_sink ? it : w0 + it - n_sink; }
};
template <int BN>
VKH_DEV KeyTiles key_tiles(const WindowArgs &a, const Span &s, int r0, int r1) {
    KeyTiles k;
    k.ta = max(0, r0 + s.off);
    k.tb = min(r1, s.ql) - 1 + s.off;
    k.w0 = max(0, k.ta - a.window + 1) / BN;
    k.n_sink = min((a.n_sink + BN - 1) / BN, k.w0);
    k.n = k.tb >= k.ta ? k.n_sink + k.tb / BN - k.w0 + 1 : 0;
    return k;
}

// Which of those tiles some, and which all, of the positions ta .. tb among the block's see.  (Tiles of
// sinks that all see without being of sinks only are taken as not whole: they are masked.)
struct Reach {
    int n_sink, some0, some1, all0, n_all, n_sink_all;
    VKH_DEV bool none(int it) const { return it >= some1 || (it < some0 && it >= n_sink); }
    VKH_DEV bool whole(int it) const { return (unsigned)(it - all0) < (unsigned)n_all || it < n_sink_all; }
};
template <int BN>
VKH_DEV Reach reach(const WindowArgs &a, const KeyTiles &k, int ta, int tb) {
    const int to_it = k.n_sink - k.w0, last = (ta + 1) / BN;
    const bool dead = tb < ta;
    Reach r;
    r.n_sink = k.n_sink;
    r.some0 = a.n_sink > k.w0 * BN ? 0 : max(0, ta - a.window + 1) / BN + to_it;
    r.some1 = dead ? 0 : tb / BN + 1 + to_it;
    r.all0 = (int)((max(0, tb - a.window + 1) + (unsigned)BN - 1) / BN) + to_it;
    r.n_all = dead ? 0 : max(0, last + to_it - r.all0);
    r.n_sink_all = dead ? 0 : min(k.n_sink, a.n_sink / BN);
    return r;
}

// The same for the keys j0 .. j1 and tiles of BM query rows, by their first row q0.  (Tiles beside the
// reach of which no row sees a key may count as some.)
struct RowReach {
    int some0, n_some, all0, n_all;
    VKH_DEV bool some(int q0) const { return (unsigned)(q0 - some0) < (unsigned)n_some; }
    VKH_DEV bool whole(int q0) const { return (unsigned)(q0 - all0) < (unsigned)n_all; }
};
template <int BM>
VKH_DEV RowReach row_reach(const WindowArgs &a, const Span &s, int j0, int j1) {
    RowReach r;
    r.some0 = j0 - s.off - BM + 1;
    r.n_some = max(0, (j0 < a.n_sink ? s.ql : (int)min((long)s.ql, (long)j1 + a.window - s.off)) - r.some0);
    r.all0 = j1 - s.off;
    const int last = s.ql - BM + 1;
    r.n_all = max(0, (j1 < a.n_sink ? last : (int)min((long)last, (long)j0 + a.window - BM + 1 - s.off)) - r.all0);
    return r;
}

// A kernel's first argument, read anew from where the launch put it (the kernel arguments begin
// with it): its values need not stay in registers for the calls below.
VKH_DEV const WindowArgs &args_again() {
    unsigned long p = (unsigned long)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *reinterpret_cast<const WindowArgs *>(p);
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

// ── joined results ───────────────────────────────────────────────────────
struct DkvPlan {
    int key_blocks, sink_blocks;   // per KV head, of `keys` keys; the first sink_blocks hold sinks
    int sink_parts, parts;         // launched blocks per sink block, per other block
    int keys;
    // pairs of a sink and a row past its window: blocks of their own (0: the key blocks take them) per
    // slice of far_keys sinks, so that no key block has more steps than the others
    int far_parts, far_slices, far_keys;
    __host__ __device__ int blocks() const { return sink_blocks * sink_parts + (key_blocks - sink_blocks) * parts; }
    // slots of partial sums per KV head: those of the sink blocks, those of the others
    __host__ __device__ int sink_slots() const { return sink_parts > 1 || far_parts ? sink_blocks * sink_parts : 0; }
    __host__ __device__ int slots() const { return sink_slots() + (parts > 1 ? (key_blocks - sink_blocks) * parts : 0); }
    // key blocks whose sums window_dkv_sum_k writes
    __host__ __device__ int summed() const { return (sink_slots() ? sink_blocks : 0) + (parts > 1 ? key_blocks - sink_blocks : 0); }
};
// Key block kb, part z of `parts` and slot (-1: the block writes its results itself) of turn y.
VKH_DEV void dkv_block(const DkvPlan &p, int y, int &kb, int &z, int &parts, int &slot) {
    const int s = p.sink_blocks * p.sink_parts;
    if (y < s) {
        kb = y / p.sink_parts; z = y % p.sink_parts; parts = p.sink_parts;
        slot = p.sink_slots() ? y : -1;
    } else {
        kb = p.sink_blocks + (y - s) / p.parts; z = (y - s) % p.parts; parts = p.parts;
        slot = parts > 1 ? p.sink_slots() + y - s : -1;
    }
}

// The (query tile, head) steps of one part of a key block, as the dK/dV kernels walk them: tiles of
// 32 rows from the last one (`top`) down, heads inner; per: heads (alt: tiles) that one step takes.
struct Steps {
    int head0, qstart, top, nh;
    bool alt;
    int per, zpart, zparts;
    VKH_DEV bool mine(int h, int row) const {
        const int t = top - (row - qstart) / 32;
        return ((alt ? t / per : t) * nh + (alt ? h - head0 : (h - head0) / per)) % zparts == zpart;
    }
};
// dK and dV of the split key blocks: their parts and then those of the far pairs ([pair][slice][part] of
// [dK, dV][far_keys][HD] behind the key blocks' slots) added in order, four values a thread.
template <int HD, int BN, class TO>
__global__ __launch_bounds__(256) void window_dkv_sum_k(WindowArgs a, DkvPlan plan) {
    const int nbk = a.n_batch * a.n_kv_heads;
    const int bk = blockIdx.x % nbk, b = bk / a.n_kv_heads, kvh = bk % a.n_kv_heads;
    const int kb = blockIdx.x / nbk + (plan.sink_slots() ? 0 : plan.sink_blocks);
    const bool sink = kb < plan.sink_blocks;
    const int parts = sink ? plan.sink_parts : plan.parts;
    const int first = sink ? kb * parts : plan.sink_slots() + (kb - plan.sink_blocks) * parts;
    const float *ws = a.ws + ((long)bk * plan.slots() + first) * (2 * BN * HD);
    const int x = (blockIdx.y * 256 + threadIdx.x) * 4;  // of dK [BN][HD], then dV
    const bool v = x >= BN * HD;
    const int y = v ? x - BN * HD : x, key = kb * BN + y / HD;
    f32x4 t{0, 0, 0, 0};
#pragma unroll 8
    for (int p = 0; p < parts; ++p) t += *reinterpret_cast<const f32x4 *>(ws + (long)p * 2 * BN * HD + x);
    if (plan.far_parts && key / plan.far_keys < plan.far_slices) {
        const int fk = plan.far_keys;
        const float *far = a.ws + (long)nbk * plan.slots() * (2 * BN * HD) +
                           ((long)bk * plan.far_slices + key / fk) * plan.far_parts * (2 * fk * HD) + (v ? fk * HD : 0) + key % fk * HD + y % HD;
#pragma unroll 8
        for (int p = 0; p < plan.far_parts; ++p) t += *reinterpret_cast<const f32x4 *>(far + (long)p * 2 * fk * HD);
    }
    if (key >= a.n_kv) return;
    const long row = (long)b * a.n_kv + key;
    TO *out = v ? (TO *)a.dv + row * a.lddv : (TO *)a.dk + row * a.lddk;
    store4(out + kvh * HD + y % HD, t[0], t[1], t[2], t[3]);
}

// The splits' results of one (row, head) per 16 lanes, joined in order: lane i holds the factors of
// splits i, i + 16, ...  Latency: all loads are on their way at once (3 to 5 us).
template <int HD, class TO>
__global__ __launch_bounds__(256) void window_join_k(WindowArgs a, int splits) {
    constexpr int E = HD / 16;
    const int lane = threadIdx.x % 64, i16 = lane % 16;
    const long rows = (long)a.n_batch * a.n_q * a.n_heads, at0 = (long)blockIdx.x * 16 + threadIdx.x / 16;
    const long at = min(at0, rows - 1);
    const float *st = a.ws + splits * rows * HD;
    float m[4], f[4], mx = -INFINITY, sum = 0.f, o[E] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool on = 16 * k + i16 < splits;
        const float2 x = on ? *reinterpret_cast<const float2 *>(st + ((16 * k + i16) * rows + at) * 2) : make_float2(-INFINITY, 0.f);
        m[k] = x.x;
        f[k] = x.y;
        mx = fmaxf(mx, x.x);
    }
    mx = row16_max(mx);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float w = f[k] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[k] - (mx == -INFINITY ? 0.f : mx));
        sum = f[k] == 0.f ? sum : fmaf(f[k], w, sum);
        f[k] = f[k] == 0.f ? -1.f : w;  // (a split without keys has no result)
    }
    sum = row16_sum(sum);
    const float *src = a.ws + at * HD + i16 * E;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (16 * k >= splits) break;
        f32x4 v[16][E / 4];  // all on their way at once (the last split's again past the end)
#pragma unroll
        for (int x = 0; x < 16; ++x)
#pragma unroll
            for (int e = 0; e < E / 4; ++e)
                v[x][e] = *reinterpret_cast<const f32x4 *>(src + min(16 * k + x, splits - 1) * rows * HD + 4 * e);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const float w = __shfl(f[k], (lane & 48) + x, 64);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = w < 0.f ? o[e] : fmaf(v[x][e / 4][e % 4], w, o[e]);
        }
    }
    if (at0 >= rows) return;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const long row = at / a.n_heads;
    const int h = (int)(at % a.n_heads);
    TO *out = (TO *)a.o + row * a.ldo + h * HD + i16 * E;
#pragma unroll
    for (int e = 0; e < E; e += 4) store4(out + e, o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
    if (a.lse && i16 == 0) a.lse[row * a.n_heads + h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * LN2;
}

// ── host ─────────────────────────────────────────────────────────────────
inline size_t dkv_ws_bytes(const WindowArgs &a, const DkvPlan &p) {
    const size_t nbk = (size_t)a.n_batch * a.n_kv_heads;
    return nbk * ((size_t)p.slots() * p.keys + (size_t)p.far_slices * p.far_parts * p.far_keys) * 2 * a.hd * sizeof(float);
}
// keys: per key block; cu_blocks: that fill the chip; least: steps that a part keeps; far: whether the
// far pairs of up to 128 sinks may have blocks of their own.  At most 256 MiB of partial sums.
inline DkvPlan dkv_plan(const WindowArgs &a, bool ws, int keys, long cu_blocks, long most_parts, long least, bool far) {
    DkvPlan p;
    p.keys = keys;
    p.key_blocks = (a.n_kv + keys - 1) / keys;
    p.sink_blocks = a.window < a.n_kv ? std::min(p.key_blocks, (a.n_sink + keys - 1) / keys) : 0;
    p.sink_parts = p.parts = 1;
    p.far_parts = p.far_slices = p.far_keys = 0;
    if (!ws) return p;
    const long nbk = (long)a.n_batch * a.n_kv_heads, blocks = nbk * p.key_blocks, hpk = a.n_heads / a.n_kv_heads;
    const long most = hpk * ((a.n_q + 31) / 32), usual = std::min(most, hpk * ((std::min<long>(a.n_kv, a.window) + keys + 31) / 32));
    const long slot = 2l * keys * a.hd * 4;
    p.parts = (int)std::max(1l, std::min({most_parts, cu_blocks / blocks, usual / least}));
    while (p.parts > 1 && blocks * slot * p.parts > (64l << 20)) --p.parts;
    // A sink block's steps over the usual block's; the sink blocks start first, so a part may take as
    // long as the rounds of the others.  Fewer parts where they would not all start at once.
    const int parts = p.parts;
    for (;; --p.parts) {
        const double rounds = std::max(1.0, (double)blocks * p.parts / cu_blocks);
        p.sink_parts = p.sink_blocks ? (int)std::max(1.0, std::min(64.0, ceil((double)most / usual * p.parts / rounds))) : 1;
        if (p.parts == 1 || nbk * p.blocks() <= cu_blocks) break;
    }
    // Far pairs apart (two launches, 15 to 20 us) where the sink blocks' parts do not all start at once or take
    // many steps from the others.  Backward in us, with the sink blocks / apart: 3 x 21 tokens, window 13: 16 / 27;
    // 2 x 1001, window 256, 16 / 4 heads of 128: 59 / 67; 2048, window 16, 16 / 8 heads: 44 / 58; 4 x 1001, window
    // 256, 16 / 8 heads: 103 / 95; 4 x 2048, window 16: 130 / 119; 4000, window 1024, 100 sinks: 213 / 180.
    // They make every sink block's sums go through a slot: not where the slots of a large batch pass the bound
    // (forward and backward in ms, with the sink blocks / apart: 512 x 256 tokens, window 64, 16 / 8 heads of 128,
    // 576 MiB of slots: 2.31 / 2.62; 256 x 1024, window 256, 288 MiB: 6.61 / 6.69).
    if (far && p.sink_blocks && a.n_sink <= 128 &&
        (nbk * p.blocks() > cu_blocks || usual * (1.0 / p.parts - 1.0 / parts) > 24)) {
        DkvPlan f = p;
        f.sink_parts = f.parts = parts;
        f.far_keys = a.n_sink > 16 ? 32 : 16;
        f.far_slices = (a.n_sink + f.far_keys - 1) / f.far_keys;
        // four waves a CU in all, while each keeps three steps
        f.far_parts = (int)std::max(1l, std::min(256 / (nbk * f.far_slices), most / 12));
        if (dkv_ws_bytes(a, f) <= (256u << 20)) return f;
    }
    while (p.sink_parts > 1 && p.sink_blocks * nbk * slot * p.sink_parts > (192l << 20)) --p.sink_parts;
    return p;
}
template <int HD, int BN, class TO>
void launch_dkv_sum(const WindowArgs &a, const DkvPlan &p, hipStream_t st) {
    if (p.summed())
        hipLaunchKernelGGL((window_dkv_sum_k<HD, BN, TO>), dim3((unsigned)((long)a.n_batch * a.n_kv_heads * p.summed()), BN * HD / 512),
                           dim3(256), 0, st, a, p);
}

// The kernels of few rows: 16 rows of a KV head's query heads a block, whose keys several blocks share.
// Calls of at most kFewRows query rows take them; of longer calls those whose 16-row tiles are few
// (`max_tiles`) and see many keys (`min_span`), for which the tile kernels leave CUs without a block
// and each block a long chain of steps.
constexpr int kFewRows = 16;
inline long row_tiles(const WindowArgs &a) {
    return (long)a.n_batch * a.n_kv_heads * (((long)a.n_q * (a.n_heads / a.n_kv_heads) + 15) / 16);
}
inline bool few_rows_of(const WindowArgs &a, long max_tiles, int min_span) {
    return a.n_q <= kFewRows || (row_tiles(a) <= max_tiles && std::min<long>(a.n_kv, (long)a.window + 64) >= min_span);
}
// Blocks that share a KV head's keys: towards `fill` blocks, while each of a block's four waves keeps a
// tile of `keys` keys.
inline int step_splits(const WindowArgs &a, int keys, long fill) {
    const long base = row_tiles(a);
    const long tiles = (std::min<long>(a.n_kv, (long)a.window + a.n_q) + a.n_sink + 2 * keys - 1) / keys;
    return (int)std::max(1l, std::min({64l, fill / base, (tiles + 3) / 4}));
}
inline size_t step_ws_bytes(const WindowArgs &a, int splits) {
    return splits > 1 ? (size_t)splits * a.n_batch * a.n_q * a.n_heads * (a.hd + 2) * sizeof(float) : 0;
}
template <int HD, class TO>
void launch_join(const WindowArgs &a, int splits, hipStream_t st) {
    const long rows = (long)a.n_batch * a.n_q * a.n_heads;
    hipLaunchKernelGGL((window_join_k<HD, TO>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a, splits);
}
// A launch takes fewer than 2^32 threads along x.  Calls of more tiles go row by row (k_attn_window.hip).
inline bool launchable(long blocks, int threads) { return blocks < (1l << 32) / threads; }
// the launches of a backward pass: dQ's blocks, dK/dV's with its sums and far pairs
inline bool launchable(const WindowArgs &a, const DkvPlan &p, long dq_blocks, int threads) {
    const long nbk = (long)a.n_batch * a.n_kv_heads;
    return launchable(dq_blocks, threads) && launchable(nbk * p.blocks(), 512) && launchable(nbk * p.summed(), 256) &&
           launchable(nbk * p.far_slices * p.far_parts, 256);
}
inline bool aligned_rows(const void *x, long ld, int align, int es) { return (uintptr_t)x % align == 0 && ld * es % align == 0; }

// The tile kernels on bf16 (k_attn_window16.hip) and fp32 operands (k_attn_window32.hip): false,
// launching nothing, for a shape, stride or alignment that they do not take.
bool window16_forward(const WindowArgs &a, hipStream_t st);
bool window16_backward(const WindowArgs &a, hipStream_t st);
size_t window16_fwd_ws_bytes(const WindowArgs &a);
size_t window16_bwd_ws_bytes(const WindowArgs &a);
bool window32_forward(const WindowArgs &a, hipStream_t st);
bool window32_backward(const WindowArgs &a, hipStream_t st);
size_t window32_fwd_ws_bytes(const WindowArgs &a);
size_t window32_bwd_ws_bytes(const WindowArgs &a);

}  // namespace vkh
