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
// radians in 32), reduced to [-1/2, 1/2] and only then rounded to 32 bits.  A block computes
// the cosines and sines of its rows once, in LDS, for all heads; head rows are held by
// 2 V values a lane (both members of V pairs), so neither layout exchanges values between
// lanes, and a lane's loads and stores are 8 or 16 bytes.  Every pass reads and writes each
// value once: bound by HBM for long batches and by the launch for a few tokens.
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int RNT = 256;

VKH_DEV float2 cos_sin(const RotaryArgs &a, long row, int j) {
    const unsigned t = a.pos ? a.pos[row] : a.pos0 + (unsigned)row % a.seq;
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
template <int V>
VKH_DEV void store_v(bf16 *p, const float (&o)[V]) {
    typedef bf16 vec __attribute__((ext_vector_type(V)));
    vec f;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (bf16)o[i];
    *reinterpret_cast<vec *>(p) = f;
}

// The V pairs that a lane holds as two chunks, turned.  Half layout: pair i is (a[i], b[i]);
// interleaved: neighbours within a, then within b.
template <int V>
VKH_DEV void turn_pairs(float (&a)[V], float (&b)[V], const float2 *cs, bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 u = cs[i], w = cs[V / 2 + i];
            const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
            a[2 * i] = a0 * u.x - a1 * u.y;
            a[2 * i + 1] = a1 * u.x + a0 * u.y;
            b[2 * i] = b0 * w.x - b1 * w.y;
            b[2 * i + 1] = b1 * w.x + b0 * w.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 u = cs[i];
            const float a0 = a[i], b0 = b[i];
            a[i] = a0 * u.x - b0 * u.y;
            b[i] = b0 * u.x + a0 * u.y;
        }
    }
}

// sum over the LP lanes (a power of two) of a head row
VKH_DEV float row_sum(float v, int LP) {
    for (int o = LP / 2; o; o /= 2) v += __shfl_xor(v, o, 64);
    return v;
}

// Lane t of a head row: its two chunks start at values e0 and e1.
VKH_DEV void chunks(const RotaryArgs &a, int t, int V, int &e0, int &e1) {
    const bool turned = 2 * t * V < a.rot;
    e0 = 2 * t * V;
    e1 = e0 + V;
    if (!a.interleaved && turned) e0 = t * V, e1 = a.rot / 2 + t * V;
}

// Forward of both operators, and the rotary backward (a.sign = -1, dy in, dx out).  A block
// takes RB rows; grid.y > 1 (RB = 1) shares a row's heads between blocks.  The next head
// row's values are loaded before the present one is stored.
template <class TX, class TY, int V, bool NORM>
__global__ __launch_bounds__(RNT) void rotary_fwd_k(RotaryArgs a, int RB, int LP) {
    extern __shared__ float2 cs[];
    const int tid = threadIdx.x, t = tid % LP, grp = tid / LP, NG = RNT / LP;
    const int half = a.rot / 2, hd = a.hd, H = a.nh[0] + a.nh[1];
    const long row0 = (long)blockIdx.x * RB;
    const int nr = (int)min((long)RB, a.n_rows - row0), items = nr * H;
    const bool act = 2 * t * V < hd, turned = 2 * t * V < a.rot;
    int e0, e1;
    chunks(a, t, V, e0, e1);
    auto src = [&](int it) {
        const long row = row0 + it / H;
        const int h = it % H;
        return h < a.nh[0] ? (const TX *)a.s[0].x + row * a.s[0].ldx + (long)h * hd
                           : (const TX *)a.s[1].x + row * a.s[1].ldx + (long)(h - a.nh[0]) * hd;
    };
    auto fetch = [&](int it, float (&u)[V], float (&v)[V]) {
        if (it >= items || !act) {
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = v[i] = 0.f;
            return;
        }
        const TX *p = src(it);
        load_v<V>(p + e0, u);
        load_v<V>(p + e1, v);
    };
    const int step = NG * gridDim.y;
    const int first = blockIdx.y * NG + grp, wave0 = blockIdx.y * NG + (tid - tid % 64) / LP;
    float u[V], v[V], wg[2][2 * V];
    fetch(first, u, v);
    if constexpr (NORM) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool on = act && a.nh[k];
                wg[k][i] = on ? a.s[k].w[e0 + i] + a.quirk : 0.f;
                wg[k][V + i] = on ? a.s[k].w[e1 + i] + a.quirk : 0.f;
            }
    }
    for (int i = tid; i < nr * half; i += RNT) cs[i] = cos_sin(a, row0 + i / half, i % half);
    __syncthreads();
    const float inv_hd = 1.0f / (float)hd;
    for (int w0 = wave0, it = first; w0 < items; w0 += step, it += step) {
        float nu[V], nv[V];
        fetch(it + step, nu, nv);
        const int h = it % H;
        const bool isk = h >= a.nh[0];
        if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
            const float r = 1.0f / sqrtf(row_sum(ss, LP) * inv_hd + a.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                u[i] = u[i] * r * (isk ? wg[1][i] : wg[0][i]);
                v[i] = v[i] * r * (isk ? wg[1][V + i] : wg[0][V + i]);
            }
        }
        if (it < items && act) {
            const long row = row0 + it / H;
            if (turned) turn_pairs<V>(u, v, cs + (it / H) * half + t * V, a.interleaved);
            TY *p = isk ? (TY *)a.s[1].y + row * a.s[1].ldy + (long)(h - a.nh[0]) * hd
                        : (TY *)a.s[0].y + row * a.s[0].ldy + (long)h * hd;
            store_v<V>(p + e0, u);
            store_v<V>(p + e1, v);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = nu[i], v[i] = nv[i];
    }
}

// Backward of norm + rotary.  Blocks walk tiles of RB rows, the query heads of a tile first
// and then its key heads, so each gain's gradient has one set of sums per lane (a lane holds
// the same values of every head row); a block's sums go to its row of `partial`
// ([blocks][2 hd]), which rotary_dw_k adds in block order.
template <class TX, class TG, class TD, int V>
__global__ __launch_bounds__(RNT) void rotary_norm_bwd_k(RotaryArgs a, int RB, int LP, float *partial) {
    extern __shared__ float2 cs[];  // RB rot / 2 cosines and sines; afterwards NG hd gain sums
    const int tid = threadIdx.x, t = tid % LP, grp = tid / LP, NG = RNT / LP;
    const int half = a.rot / 2, hd = a.hd;
    const bool act = 2 * t * V < hd, turned = 2 * t * V < a.rot;
    const float inv_hd = 1.0f / (float)hd;
    int e0, e1;
    chunks(a, t, V, e0, e1);
    float dw[2][2 * V] = {};
    for (long row0 = (long)blockIdx.x * RB; row0 < a.n_rows; row0 += (long)gridDim.x * RB) {
        const int nr = (int)min((long)RB, a.n_rows - row0);
        __syncthreads();  // everyone is done with the last tile's angles
        for (int i = tid; i < nr * half; i += RNT) cs[i] = cos_sin(a, row0 + i / half, i % half);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const RotarySide &s = a.s[k];
            const int H = a.nh[k], items = nr * H;
            if (!H) continue;
            float w[2 * V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                w[i] = act ? s.w[e0 + i] + a.quirk : 0.f;
                w[V + i] = act ? s.w[e1 + i] + a.quirk : 0.f;
            }
            for (int w0 = (tid - tid % 64) / LP, it = grp; w0 < items; w0 += NG, it += NG) {
                const bool on = it < items && act;
                const long row = row0 + it / H;
                const long h = (long)(it % H) * hd;
                float x0[V] = {}, x1[V] = {}, g0[V] = {}, g1[V] = {};
                if (on) {
                    const TX *xp = (const TX *)s.x + row * s.ldx + h;
                    const TG *gp = (const TG *)s.dy + row * s.lddy + h;
                    load_v<V>(xp + e0, x0);
                    load_v<V>(xp + e1, x1);
                    load_v<V>(gp + e0, g0);
                    load_v<V>(gp + e1, g1);
                }
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
                if (on && turned) turn_pairs<V>(g0, g1, cs + (it / H) * half + t * V, a.interleaved);
                const float r = 1.0f / sqrtf(row_sum(ss, LP) * inv_hd + a.eps);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x0[i] *= r;
                    x1[i] *= r;
                    dw[k][i] = fmaf(g0[i], x0[i], dw[k][i]);
                    dw[k][V + i] = fmaf(g1[i], x1[i], dw[k][V + i]);
                    g0[i] *= w[i];
                    g1[i] *= w[V + i];
                    dot = fmaf(x0[i], g0[i], fmaf(x1[i], g1[i], dot));
                }
                const float m = row_sum(dot, LP) * inv_hd;
                if (on) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        g0[i] = (g0[i] - x0[i] * m) * r;
                        g1[i] = (g1[i] - x1[i] * m) * r;
                    }
                    TD *dp = (TD *)s.dx + row * s.lddx + h;
                    store_v<V>(dp + e0, g0);
                    store_v<V>(dp + e1, g1);
                }
            }
        }
    }
    if (!partial) return;
    float *sh = reinterpret_cast<float *>(cs);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
        if (act) {
#pragma unroll
            for (int i = 0; i < V; ++i) sh[grp * hd + e0 + i] = dw[k][i], sh[grp * hd + e1 + i] = dw[k][V + i];
        }
        __syncthreads();
        for (int c = tid; c < hd; c += RNT) {
            float s = 0.f;
            for (int g = 0; g < NG; ++g) s += sh[g * hd + c];
            partial[(long)blockIdx.x * 2 * hd + k * hd + c] = s;
        }
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
    const long it = (long)blockIdx.x * (RNT / 64) + threadIdx.x / 64;
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
            const float2 c = cos_sin(a, row, lane + 64 * i);
            const float p = u[i] * c.x - v[i] * c.y;
            v[i] = v[i] * c.x + u[i] * c.y;
            u[i] = p;
            y[e.e1] = (TY)v[i];
        }
        y[e.e0] = (TY)u[i];
    }
}
template <class TX, class TG, class TD>
__global__ __launch_bounds__(RNT) void rotary_norm_bwd_any_k(RotaryArgs a, float *partial) {
    __shared__ float sh[RNT / 64][256];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        const RotarySide &s = a.s[k];
        float du[GI] = {}, dv[GI] = {};
        for (long it = (long)blockIdx.x * (RNT / 64) + wave; it < a.n_rows * a.nh[k]; it += (long)gridDim.x * (RNT / 64)) {
            const long row = it / a.nh[k], h = it % a.nh[k] * a.hd;
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
                    const float2 c = cos_sin(a, row, lane + 64 * i);
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
        if (!partial) continue;
        __syncthreads();
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
            partial[(long)blockIdx.x * 2 * a.hd + k * a.hd + c] = t;
        }
    }
}

// dw of both gains: column c of the 2 hd partial sums, 16 columns a block, each added by 16
// threads over every 16th block's row and then in thread order.
__global__ __launch_bounds__(RNT) void rotary_dw_k(const float *partial, int parts, int hd, float *dwq, float *dwk) {
    __shared__ float sh[16][17];
    const int c = threadIdx.x % 16, r = threadIdx.x / 16, col = blockIdx.x * 16 + c;
    float s = 0.f;
    if (col < 2 * hd)
        for (int b = r; b < parts; b += 16) s += partial[(long)b * 2 * hd + col];
    sh[r][c] = s;
    __syncthreads();
    if (r || col >= 2 * hd) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += sh[i][c];
    float *out = col < hd ? dwq : dwk;
    if (out) out[col % hd] = t;
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

template <class F>
void by_type(DType d, F f) {
    if (d == DType::F32) f(float{});
    else f(bf16{});
}

}  // namespace

// Partial rows of the gain sums: at most kRotaryParts blocks.
constexpr int kRotaryParts = 512;
static int bwd_rows(const RotaryArgs &a) { return a.n_rows >= 4 * kRotaryParts ? 4 : a.n_rows >= 2 * kRotaryParts ? 2 : 1; }
int rotary_parts(const RotaryArgs &a) {
    const int RB = bwd_rows(a);
    return (int)std::min<long>(kRotaryParts, (a.n_rows + RB - 1) / RB);
}

hipError_t rotary_forward(const RotaryArgs &a, bool norm, DType xt, DType yt, hipStream_t st) {
    const int H = a.nh[0] + a.nh[1];
    if (a.n_rows <= 0 || !H) return hipSuccess;
    const int V = chunk_width(a, {{xt, 0}, {yt, 1}});
    if (!V) {
        const long blocks = (a.n_rows * H + RNT / 64 - 1) / (RNT / 64);
        if (blocks >= (1L << 31)) return hipErrorInvalidValue;
        by_type(xt, [&](auto x) {
            by_type(yt, [&](auto y) {
                auto k = norm ? rotary_fwd_any_k<decltype(x), decltype(y), true> : rotary_fwd_any_k<decltype(x), decltype(y), false>;
                hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(RNT), 0, st, a);
            });
        });
        return hipGetLastError();
    }
    const int LP = lanes(a.hd, V), NG = RNT / LP;
    const int RB = a.n_rows >= 4096 ? 4 : a.n_rows >= 2048 ? 2 : 1;
    const unsigned gy = RB == 1 && a.n_rows < 256 ? (unsigned)((H + NG - 1) / NG) : 1u;
    const dim3 grid((unsigned)((a.n_rows + RB - 1) / RB), gy);
    const unsigned lds = std::max(1, RB * a.rot / 2) * sizeof(float2);
    by_type(xt, [&](auto x) {
        by_type(yt, [&](auto y) {
            using X = decltype(x);
            using Y = decltype(y);
            auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(RNT), lds, st, a, RB, LP); };
            if (V == 8) norm ? go(rotary_fwd_k<X, Y, 8, true>) : go(rotary_fwd_k<X, Y, 8, false>);
            else norm ? go(rotary_fwd_k<X, Y, 4, true>) : go(rotary_fwd_k<X, Y, 4, false>);
        });
    });
    return hipGetLastError();
}

hipError_t rotary_norm_backward(const RotaryArgs &a, DType xt, DType gt, DType dt, float *partial,
                                float *dwq, float *dwk, hipStream_t st) {
    if (a.n_rows <= 0 || !(a.nh[0] + a.nh[1])) return hipSuccess;
    const int V = chunk_width(a, {{xt, 0}, {gt, 2}, {dt, 3}});
    const int parts = rotary_parts(a), RB = bwd_rows(a);
    by_type(xt, [&](auto x) {
        by_type(gt, [&](auto g) {
            by_type(dt, [&](auto d) {
                using X = decltype(x);
                using G = decltype(g);
                using D = decltype(d);
                if (!V) {
                    hipLaunchKernelGGL((rotary_norm_bwd_any_k<X, G, D>), dim3(parts), dim3(RNT), 0, st, a, partial);
                    return;
                }
                const int LP = lanes(a.hd, V);
                const unsigned lds = std::max<unsigned>(RB * a.rot / 2 * sizeof(float2), RNT / LP * a.hd * sizeof(float));
                auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3(parts), dim3(RNT), lds, st, a, RB, LP, partial); };
                if (V == 8) go(rotary_norm_bwd_k<X, G, D, 8>);
                else go(rotary_norm_bwd_k<X, G, D, 4>);
            });
        });
    });
    if (partial)
        hipLaunchKernelGGL(rotary_dw_k, dim3((2 * a.hd + 15) / 16), dim3(RNT), 0, st, partial, parts, a.hd, dwq, dwk);
    return hipGetLastError();
}

}  // namespace vkh
