// Rotary positions and the per-head Q/K RMSNorm with the rotation in the same pass.
//
// A head row x of head_dim values at position t: its first `rot` values are turned pair by
// pair, (x_i, x_{i + rot/2}) (half layout) or (x_2i, x_{2i+1}) (interleaved), by the angle
// t f_i, and multiplied by the plan's scale a; the rest passes through.
//
//   rotary       y  = a R(t f) x                      backward  dx = a R(-t f) dy
//   norm+rotary  y  = a R(t f) (x rstd w),  rstd = 1 / sqrt(mean(x^2) + eps)
//   its backward g  = a R(-t f) dy,  xh = x rstd
//                dx = rstd (w g - xh mean(xh w g)),  dw = sum over rows and heads of g xh
//
// The angle is formed in turns, in 64 bits (t up to 2^32 times a frequency loses whole
// radians in 32), reduced to [-1/2, 1/2] and only then rounded to 32 bits.  A wave computes
// the cosines and sines of its row once for all heads; head rows are held by 2 V values a
// lane (both members of V pairs), so neither layout exchanges values between lanes, and a
// lane's loads and stores are 8 or 16 bytes.  Every pass reads and writes each value once: bound
// by HBM for long batches and by the launch for a few tokens.
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int RNT = 256;

VKH_DEV unsigned position(const RotaryArgs &a, long row) {
    return a.pos ? a.pos[row] : a.pos0 + (unsigned)row % a.seq;
}
VKH_DEV float2 cos_sin(const RotaryArgs &a, unsigned t, int j) {
    double turn = (double)t * a.turns[j];
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    return make_float2(a.scale * c, a.sign * a.scale * s);
}

template <int V>
VKH_DEV void load_v(const float *p, float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p + i);
        o[i] = f.x; o[i + 1] = f.y; o[i + 2] = f.z; o[i + 3] = f.w;
    }
}
template <int V>
VKH_DEV void load_v(const bf16 *p, float (&o)[V]) {
    typedef bf16 vec __attribute__((ext_vector_type(V)));
    const vec f = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)f[i];
}
template <int V>
VKH_DEV void store_v(float *p, const float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4 *>(p + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
}
// Past the caches: what is written is read by another kernel, and each store covers whole lines over its
// lanes (16384 rows, 32 / 8 heads of 128: norm and rotation 69 us through the caches, 62 past them, their backward
// 112 and 102; fp32 stores of 8 values a lane, in two halves, go through them).
template <int V>
VKH_DEV void store_v(bf16 *p, const float (&o)[V]) {
    typedef bf16 vec __attribute__((ext_vector_type(V)));
    vec f;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (bf16)o[i];
    __builtin_nontemporal_store(f, reinterpret_cast<vec *>(p));
}

// gains (any alignment)
template <int V>
VKH_DEV void load_gain(const float *p, float (&o)[V], float quirk) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = p[i] + quirk;
}

// The V pairs that a lane holds as two chunks, turned.  Half layout: pair i is (a[i], b[i]);
// interleaved: neighbours within a, then within b.  SELECT: lanes that are not `turned` (their cs is (1, 0))
// may call it too; what their sines multiply is taken as 0, since 0 times an infinity or a NaN is NaN.  (For the
// norm's backward: with a branch around the call it has four waves a SIMD in place of five, 140 us for 100.)
template <bool SELECT, int V>
VKH_DEV void turn_pairs(float (&a)[V], float (&b)[V], const float2 (&cs)[V], bool interleaved, bool turned = true) {
    auto part = [&](float x) { return !SELECT || turned ? x : 0.f; };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 u = cs[i], w = cs[V / 2 + i];
            const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
            a[2 * i] = a0 * u.x - part(a1) * u.y;
            a[2 * i + 1] = a1 * u.x + part(a0) * u.y;
            b[2 * i] = b0 * w.x - part(b1) * w.y;
            b[2 * i + 1] = b1 * w.x + part(b0) * w.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 u = cs[i];
            const float a0 = a[i], b0 = b[i];
            a[i] = a0 * u.x - part(b0) * u.y;
            b[i] = b0 * u.x + part(a0) * u.y;
        }
    }
}

// sum over the LP lanes (a power of two, at most 32) of a head row
VKH_DEV float row_sum(float v, int LP) {
    if (LP > 1) v += dpp_f<0xB1>(v);   // quad_perm [1,0,3,2]
    if (LP > 2) v += dpp_f<0x4E>(v);   // quad_perm [2,3,0,1]
    if (LP > 4) v += dpp_f<0x141>(v);  // row_half_mirror
    if (LP > 8) v += dpp_f<0x140>(v);  // row_mirror
    if (LP > 16) v += __shfl_xor(v, 16, 64);
    return v;
}

// Lane t of a head row: its two chunks start at values e0 and e1, of the turned part's halves or of the
// rest's (all of the row where nothing is turned): what a load or store of one chunk touches is contiguous
// over the lanes of either part.
VKH_DEV void chunks(const RotaryArgs &a, int t, int V, int &e0, int &e1) {
    const bool turned = 2 * t * V < a.rot;
    const int lo = turned ? 0 : a.rot, n = turned ? a.rot : a.hd - a.rot;
    e0 = lo + t * V - lo / 2;
    e1 = e0 + n / 2;
}

// The cosines and sines of a row for the V pairs of each lane: a wave computes one pair a lane and
// hands them round through its own LDS (128 pairs).  True where the lane's values are turned.
template <int V>
VKH_DEV bool row_angles(const RotaryArgs &a, unsigned pos, float2 *sh, int lane, int t, float2 (&cs)[V]) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last row's are read
    for (int j = lane; j < a.rot / 2; j += 64) sh[j] = cos_sin(a, pos, j);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const bool turned = 2 * t * V < a.rot;
    if (turned) {
        // half layout: pairs t V ..; neighbours: half of them in either chunk
        const int p0 = a.interleaved ? t * V / 2 : t * V, p1 = a.interleaved ? a.rot / 4 + p0 : p0 + V / 2;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) cs[i] = sh[p0 + i], cs[V / 2 + i] = sh[p1 + i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) cs[i] = make_float2(1.f, 0.f);
    }
    return turned;
}

// Forward of both operators, and the rotary backward (a.sign = -1, dy in, dx out).  HS waves share
// a row (4 where rows are few: one token's latency; 1 where they fill the chip), 64 / LP heads at a
// time; the next heads' values are on their way while the present ones are turned.
// 16384 rows, 32 / 8 heads of 128, bf16 (0.34 GB): 68 us a rotation of 64 neighbouring pairs' values (4.9
// TB/s; 71 with both chunks of a lane side by side), 62 with the norm (5.4 TB/s); a block per 4 rows over a
// flat list of heads took 73 and 105.
template <class TX, class TY, int V, bool NORM>
__global__ __launch_bounds__(RNT) void rotary_fwd_k(RotaryArgs a, int HS, int LP) {
    __shared__ float2 sh[RNT / 64][128];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int t = lane % LP, grp = lane / LP, NG = 64 / LP, hd = a.hd;
    const long row = block_number() * (RNT / 64 / HS) + wave / HS;
    if (row >= a.n_rows) return;
    const bool act = 2 * t * V < hd;
    const int step = NG * HS, first = wave % HS * NG;
    int e0, e1;
    chunks(a, t, V, e0, e1);
    const float inv_hd = 1.0f / (float)hd;
    float2 cs[V];
    bool angles = false, turned = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const RotarySide &s = a.s[k];
        const int H = a.nh[k];
        if (first >= H) continue;
        const TX *x = (const TX *)s.x + row * s.ldx;
        TY *y = (TY *)s.y + row * s.ldy;
        auto fetch = [&](int h, float (&u)[V], float (&v)[V]) {
            if (h < H && act) {
                load_v<V>(x + h * hd + e0, u);
                load_v<V>(x + h * hd + e1, v);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) u[i] = v[i] = 0.f;
            }
        };
        float u[V], v[V], w0[V], w1[V];
        fetch(first + grp, u, v);
        if constexpr (NORM) {
            if (act) {
                load_gain<V>(s.w + e0, w0, a.quirk);
                load_gain<V>(s.w + e1, w1, a.quirk);
            }
        }
        if (!angles) turned = row_angles<V>(a, position(a, row), sh[wave], lane, t, cs);
        angles = true;
        for (int h0 = first; h0 < H; h0 += step) {
            float nu[V], nv[V];
            if (h0 + step < H) fetch(h0 + step + grp, nu, nv);
            if constexpr (NORM) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
                const float r = rsqrtf(fmaf(row_sum(ss, LP), inv_hd, a.eps));
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u[i] = u[i] * r * w0[i];
                    v[i] = v[i] * r * w1[i];
                }
            }
            if (turned) turn_pairs<false>(u, v, cs, a.interleaved);
            if (h0 + grp < H && act) {
                store_v<V>(y + (h0 + grp) * hd + e0, u);
                store_v<V>(y + (h0 + grp) * hd + e1, v);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = nu[i], v[i] = nv[i];
        }
    }
}

// Backward of norm + rotary.  The first parts.q blocks take the query heads, the others the key
// heads: a lane then has one set of sums for its gain's gradient (it holds the same values of every
// head row), and registers for more waves.  A wave walks rows, 64 / LP heads at a time; the next
// heads' values, also the next row's, are on their way while the present ones are worked on.  A
// block's sums go to its row of `partial` ([blocks][hd]), which rotary_dw_k adds in block order.
// 16384 rows, 32 / 8 heads of 128, bf16 (0.5 GB): 102 us, 4.9 TB/s; rotary_dw_k 6.
// REST: some values of a head are not turned (five waves a SIMD asked for: without, 99 registers leave four).
template <class TX, class TG, class TD, int V, bool REST>
__global__ __launch_bounds__(RNT, REST ? 5 : 1) void rotary_norm_bwd_k(RotaryArgs a, int LP, RotaryParts parts, float *partial) {
    __shared__ float2 sh[RNT / 64][128];
    extern __shared__ float sums[];  // 256 / LP head rows of hd gain sums
    const bool isk = (int)blockIdx.x >= parts.q;
    const RotarySide s = isk ? a.s[1] : a.s[0];
    const int H = isk ? a.nh[1] : a.nh[0], blk = blockIdx.x - (isk ? parts.q : 0);
    const long stride = (long)(isk ? parts.k : parts.q) * (RNT / 64);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int t = lane % LP, grp = lane / LP, NG = 64 / LP, hd = a.hd;
    const bool act = 2 * t * V < hd;
    const float inv_hd = 1.0f / (float)hd;
    int e0, e1;
    chunks(a, t, V, e0, e1);
    float dw[2 * V] = {}, w0[V] = {}, w1[V] = {};
    if (act) {
        load_gain<V>(s.w + e0, w0, a.quirk);
        load_gain<V>(s.w + e1, w1, a.quirk);
    }
    float2 cs[V];
    float x0[V], x1[V], g0[V], g1[V];
    auto fetch = [&](long row, int h, float (&x0)[V], float (&x1)[V], float (&g0)[V], float (&g1)[V]) {
        if (row < a.n_rows && h < H && act) {
            const TX *x = (const TX *)s.x + row * s.ldx + h * hd;
            const TG *dy = (const TG *)s.dy + row * s.lddy + h * hd;
            load_v<V>(x + e0, x0);
            load_v<V>(x + e1, x1);
            load_v<V>(dy + e0, g0);
            load_v<V>(dy + e1, g1);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x0[i] = x1[i] = g0[i] = g1[i] = 0.f;
        }
    };
    long row = (long)blk * (RNT / 64) + wave;
    unsigned pos = row < a.n_rows ? position(a, row) : 0;
    fetch(row, grp, x0, x1, g0, g1);
    while (row < a.n_rows) {
        const long next = row + stride;
        const unsigned npos = next < a.n_rows ? position(a, next) : 0;
        const bool turned = row_angles<V>(a, pos, sh[wave], lane, t, cs);
        for (int h0 = 0; h0 < H; h0 += NG) {
            float nx0[V], nx1[V], ng0[V], ng1[V];
            const bool same = h0 + NG < H;
            fetch(same ? row : next, (same ? h0 + NG : 0) + grp, nx0, nx1, ng0, ng1);
            float ss = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
            turn_pairs<REST>(g0, g1, cs, a.interleaved, turned);
            // lanes without a head add nothing to the gains' sums (0 times the root of eps = 0 would be NaN)
            const float root = rsqrtf(fmaf(row_sum(ss, LP), inv_hd, a.eps)), r = h0 + grp < H ? root : 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x0[i] *= r;
                x1[i] *= r;
                dw[i] = fmaf(g0[i], x0[i], dw[i]);
                dw[V + i] = fmaf(g1[i], x1[i], dw[V + i]);
                g0[i] *= w0[i];
                g1[i] *= w1[i];
                dot = fmaf(x0[i], g0[i], fmaf(x1[i], g1[i], dot));
            }
            const float m = row_sum(dot, LP) * inv_hd;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                g0[i] = (g0[i] - x0[i] * m) * r;
                g1[i] = (g1[i] - x1[i] * m) * r;
            }
            if (h0 + grp < H && act) {
                TD *dx = (TD *)s.dx + row * s.lddx + (h0 + grp) * hd;
                store_v<V>(dx + e0, g0);
                store_v<V>(dx + e1, g1);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) x0[i] = nx0[i], x1[i] = nx1[i], g0[i] = ng0[i], g1[i] = ng1[i];
        }
        row = next;
        pos = npos;
    }
    if (!partial) return;
    if (act) {
        float *mine = sums + (wave * NG + grp) * hd;
#pragma unroll
        for (int i = 0; i < V; ++i) mine[e0 + i] = dw[i], mine[e1 + i] = dw[V + i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < hd; c += RNT) {
        float x = 0.f;
        for (int g = 0; g < RNT / LP; ++g) x += sums[g * hd + c];
        partial[(long)blockIdx.x * hd + c] = x;
    }
}

// Any head_dim up to 256, rotary span, stride and alignment: one wave per head row, lane l
// holds the items l, l + 64, ... of the row's rot / 2 pairs and hd - rot single values.
constexpr int GI = 4;
struct RotItem {
    int e0, e1;  // values (e1 < 0: a single one; e0 < 0: none)
};
VKH_DEV RotItem rot_item(const RotaryArgs &a, int i) {
    const int half = a.rot / 2;
    if (i < half) return a.interleaved ? RotItem{2 * i, 2 * i + 1} : RotItem{i, half + i};
    const int e = a.rot + i - half;
    return RotItem{e < a.hd ? e : -1, -1};
}
template <class TX, class TY, bool NORM>
__global__ __launch_bounds__(RNT) void rotary_fwd_any_k(RotaryArgs a) {
    const int lane = threadIdx.x % 64, H = a.nh[0] + a.nh[1];
    const long it = block_number() * (RNT / 64) + threadIdx.x / 64;
    if (it >= a.n_rows * H) return;
    const long row = it / H;
    const int hh = (int)(it % H);
    const bool isk = hh >= a.nh[0];
    const RotarySide &s = isk ? a.s[1] : a.s[0];
    const long h = (long)(isk ? hh - a.nh[0] : hh) * a.hd;
    const TX *x = (const TX *)s.x + row * s.ldx + h;
    TY *y = (TY *)s.y + row * s.ldy + h;
    float u[GI], v[GI], ss = 0.f;
#pragma unroll
    for (int i = 0; i < GI; ++i) {
        const RotItem e = rot_item(a, lane + 64 * i);
        u[i] = e.e0 >= 0 ? to_f32(x[e.e0]) : 0.f;
        v[i] = e.e1 >= 0 ? to_f32(x[e.e1]) : 0.f;
        ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
    }
    const float r = NORM ? 1.0f / sqrtf(wave_sum(ss) / (float)a.hd + a.eps) : 1.f;
#pragma unroll
    for (int i = 0; i < GI; ++i) {
        const RotItem e = rot_item(a, lane + 64 * i);
        if (e.e0 < 0) continue;
        if (NORM) {
            u[i] = u[i] * r * (s.w[e.e0] + a.quirk);
            if (e.e1 >= 0) v[i] = v[i] * r * (s.w[e.e1] + a.quirk);
        }
        if (e.e1 >= 0) {
            const float2 c = cos_sin(a, position(a, row), lane + 64 * i);
            const float p = u[i] * c.x - v[i] * c.y;
            v[i] = v[i] * c.x + u[i] * c.y;
            u[i] = p;
            y[e.e1] = (TY)v[i];
        }
        y[e.e0] = (TY)u[i];
    }
}
template <class TX, class TG, class TD>
__global__ __launch_bounds__(RNT) void rotary_norm_bwd_any_k(RotaryArgs a, RotaryParts parts, float *partial) {
    __shared__ float sh[RNT / 64][256];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    {
        const bool isk = (int)blockIdx.x >= parts.q;
        const RotarySide s = isk ? a.s[1] : a.s[0];
        const int H = isk ? a.nh[1] : a.nh[0], blk = blockIdx.x - (isk ? parts.q : 0);
        float du[GI] = {}, dv[GI] = {};
        for (long it = (long)blk * (RNT / 64) + wave; it < a.n_rows * H; it += (long)(isk ? parts.k : parts.q) * (RNT / 64)) {
            const long row = it / H, h = it % H * a.hd;
            const TX *x = (const TX *)s.x + row * s.ldx + h;
            const TG *dy = (const TG *)s.dy + row * s.lddy + h;
            TD *dx = (TD *)s.dx + row * s.lddx + h;
            float u[GI], v[GI], p[GI], q[GI], ss = 0.f;
#pragma unroll
            for (int i = 0; i < GI; ++i) {
                const RotItem e = rot_item(a, lane + 64 * i);
                u[i] = e.e0 >= 0 ? to_f32(x[e.e0]) : 0.f;
                v[i] = e.e1 >= 0 ? to_f32(x[e.e1]) : 0.f;
                p[i] = e.e0 >= 0 ? to_f32(dy[e.e0]) : 0.f;
                q[i] = e.e1 >= 0 ? to_f32(dy[e.e1]) : 0.f;
                ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
                if (e.e1 >= 0) {
                    const float2 c = cos_sin(a, position(a, row), lane + 64 * i);
                    const float g = p[i] * c.x - q[i] * c.y;
                    q[i] = q[i] * c.x + p[i] * c.y;
                    p[i] = g;
                }
            }
            const float r = 1.0f / sqrtf(wave_sum(ss) / (float)a.hd + a.eps);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < GI; ++i) {
                const RotItem e = rot_item(a, lane + 64 * i);
                u[i] *= r;
                v[i] *= r;
                du[i] = fmaf(p[i], u[i], du[i]);
                dv[i] = fmaf(q[i], v[i], dv[i]);
                p[i] *= e.e0 >= 0 ? s.w[e.e0] + a.quirk : 0.f;
                q[i] *= e.e1 >= 0 ? s.w[e.e1] + a.quirk : 0.f;
                dot = fmaf(u[i], p[i], fmaf(v[i], q[i], dot));
            }
            const float m = wave_sum(dot) / (float)a.hd;
#pragma unroll
            for (int i = 0; i < GI; ++i) {
                const RotItem e = rot_item(a, lane + 64 * i);
                if (e.e0 >= 0) dx[e.e0] = (TD)((p[i] - u[i] * m) * r);
                if (e.e1 >= 0) dx[e.e1] = (TD)((q[i] - v[i] * m) * r);
            }
        }
        if (!partial) return;
#pragma unroll
        for (int i = 0; i < GI; ++i) {
            const RotItem e = rot_item(a, lane + 64 * i);
            if (e.e0 >= 0) sh[wave][e.e0] = du[i];
            if (e.e1 >= 0) sh[wave][e.e1] = dv[i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.hd; c += RNT) {
            float t = 0.f;
            for (int w = 0; w < RNT / 64; ++w) t += sh[w][c];
            partial[(long)blockIdx.x * a.hd + c] = t;
        }
    }
}

// The gain gradients: four columns of one side's partial sums a block; thread r adds every 256th
// block's row, then the threads' sums are added by halves.
__global__ __launch_bounds__(RNT) void rotary_dw_k(const float *partial, RotaryParts parts, int hd, float *dwq, float *dwk) {
    __shared__ f32x4 sh[RNT];
    const int r = threadIdx.x, col = blockIdx.x * 4;
    const bool isk = blockIdx.y;
    float *out = isk ? dwk : dwq;
    if (!out) return;
    partial += isk ? (long)parts.q * hd : 0;
    f32x4 s{0, 0, 0, 0};
    for (int b = r; b < (isk ? parts.k : parts.q); b += RNT)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < hd) s[i] += partial[(long)b * hd + col + i];
    sh[r] = s;
    for (int o = RNT / 2; o; o /= 2) {
        __syncthreads();
        if (r < o) sh[r] += sh[r + o];
    }
    if (r) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < hd) out[col + i] = sh[0][i];
}

// Chunk width: 8 values where both dtypes' rows allow 16-byte (fp32: two 16-byte) accesses,
// 4 where they allow 16 bytes of fp32 and 8 of bf16, 0 for the per-value kernels.
int chunk_width(const RotaryArgs &a, std::initializer_list<std::pair<DType, int>> which) {
    for (int V : {8, 4}) {
        bool ok = a.hd % (2 * V) == 0 && a.rot % (2 * V) == 0;
        for (int k = 0; k < 2; ++k) {
            if (!a.nh[k]) continue;
            for (auto &w : which) {
                const RotarySide &s = a.s[k];
                const void *p = w.second == 0 ? s.x : w.second == 1 ? s.y : w.second == 2 ? s.dy : s.dx;
                const long ld = w.second == 0 ? s.ldx : w.second == 1 ? s.ldy : w.second == 2 ? s.lddy : s.lddx;
                const int es = w.first == DType::F32 ? 4 : 2, al = std::min(16, V * es);
                ok = ok && (uintptr_t)p % al == 0 && ld * es % al == 0;
            }
        }
        if (ok) return V;
    }
    return 0;
}
int lanes(int hd, int V) {
    int l = 1;
    while (l * 2 * V < hd) l *= 2;
    return l;
}

}  // namespace

// Blocks of each side: five a CU in all (as many as fit at 4-value chunks), shared by the sides'
// heads, at most one a wave's row.  16384 rows, 32 / 8 heads of 128, bf16, as first measured: 114 us; 8-value
// chunks fill the registers with three a CU and take 123; 2048 rows, 16 / 8 heads, fp32 to bf16: 14 against 18.
RotaryParts rotary_parts(const RotaryArgs &a) {
    const long H = a.nh[0] + a.nh[1], rows = (a.n_rows + RNT / 64 - 1) / (RNT / 64);
    auto of = [&](int nh) { return nh ? (int)std::max(1l, std::min(rows, 1280 * nh / H)) : 0; };
    return RotaryParts{of(a.nh[0]), of(a.nh[1])};
}

hipError_t rotary_forward(const RotaryArgs &a, bool norm, DType xt, DType yt, hipStream_t st) {
    const int H = a.nh[0] + a.nh[1];
    if (a.n_rows <= 0 || !H) return hipSuccess;
    const int V = chunk_width(a, {{xt, 0}, {yt, 1}});
    if (!V) {
        const dim3 grid = long_grid((a.n_rows * H + RNT / 64 - 1) / (RNT / 64));
        by_type(xt, [&](auto x) {
            by_type(yt, [&](auto y) {
                auto k = norm ? rotary_fwd_any_k<decltype(x), decltype(y), true> : rotary_fwd_any_k<decltype(x), decltype(y), false>;
                hipLaunchKernelGGL(k, grid, dim3(RNT), 0, st, a);
            });
        });
        return hipGetLastError();
    }
    const int LP = lanes(a.hd, V), HS = a.n_rows >= 2048 ? 1 : a.n_rows >= 1024 ? 2 : 4, per = RNT / 64 / HS;
    const dim3 grid = long_grid((a.n_rows + per - 1) / per);
    by_type(xt, [&](auto x) {
        by_type(yt, [&](auto y) {
            using X = decltype(x);
            using Y = decltype(y);
            auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(RNT), 0, st, a, HS, LP); };
            if (V == 8) norm ? go(rotary_fwd_k<X, Y, 8, true>) : go(rotary_fwd_k<X, Y, 8, false>);
            else norm ? go(rotary_fwd_k<X, Y, 4, true>) : go(rotary_fwd_k<X, Y, 4, false>);
        });
    });
    return hipGetLastError();
}

hipError_t rotary_norm_backward(const RotaryArgs &a, DType xt, DType gt, DType dt, float *partial,
                                float *dwq, float *dwk, hipStream_t st) {
    if (a.n_rows <= 0 || !(a.nh[0] + a.nh[1])) return hipSuccess;
    const bool chunked = chunk_width(a, {{xt, 0}, {gt, 2}, {dt, 3}}) != 0;
    const RotaryParts parts = rotary_parts(a);
    const dim3 grid(parts.q + parts.k);
    by_type(xt, [&](auto x) {
        by_type(gt, [&](auto g) {
            by_type(dt, [&](auto d) {
                using X = decltype(x);
                using G = decltype(g);
                using D = decltype(d);
                if (!chunked) {
                    hipLaunchKernelGGL((rotary_norm_bwd_any_k<X, G, D>), grid, dim3(RNT), 0, st, a, parts, partial);
                    return;
                }
                const int LP = lanes(a.hd, 4);
                auto k = a.rot < a.hd ? rotary_norm_bwd_k<X, G, D, 4, true> : rotary_norm_bwd_k<X, G, D, 4, false>;
                hipLaunchKernelGGL(k, grid, dim3(RNT), RNT / LP * a.hd * sizeof(float), st, a, LP, parts, partial);
            });
        });
    });
    if (partial)
        hipLaunchKernelGGL(rotary_dw_k, dim3((a.hd + 3) / 4, 2), dim3(RNT), 0, st, partial, parts, a.hd, dwq, dwk);
    return hipGetLastError();
}

}  // namespace vkh
