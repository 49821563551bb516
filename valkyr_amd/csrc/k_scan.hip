// A gated linear recurrence over time, every channel on its own:
//
//   h_t = a_t h_{t-1} + u_t,  a = sigmoid(g) or g,  u = x or (1 - a) x
//
// and its gradients, with R_t = a_t G_t (what G hands on to the row before):
//
//   G_t = dh_t + R_{t+1},  du = G_t,  da = G_t h_{t-1}  (coupled: dx = (1 - a) G, da = G (h_{t-1} - x))
//   dg = da, or da a (1 - a),  dh0 = R_0
//
// A stretch of rows maps the state before it to the one behind it as h -> A h + B (A the product of its a, B what
// the stretch makes of h = 0), and the same A carries R the other way: R -> A R + Q.  A block takes 64 V
// channels and walks tiles of kScanTile rows: each of its waves holds kRows rows of all these channels in
// registers, forms A and B of them, and adds up the others' before it through LDS; then it runs its rows again from
// the state that they start from.  Each value is read and written once: bound by HBM.  The forward keeps the state
// before every tile, from which the backward forms h again.
#include <type_traits>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int kRows = 16;
constexpr int kWaves = kScanTile / kRows;

template <class F>
void by_type(DType d, F f) {
    if (d == DType::F32) f(float{});
    else f(bf16{});
}

template <class T, int V>
VKH_DEV void load_v(const T *p, float (&o)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) {
        o[0] = to_f32(p[0]);
    } else {
        const vec f = *reinterpret_cast<const vec *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (float)f[i];
    }
}
template <class T, int V>
VKH_DEV void store_v(T *p, const float (&o)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) {
        p[0] = (T)o[0];
    } else {
        vec f;
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (T)o[i];
        *reinterpret_cast<vec *>(p) = f;
    }
}

// a and 1 - a of a gate, each to its own last digits: e = exp(-|g|) from a product in two parts (one alone is
// off by |g| steps), 1 / (1 + e) and e / (1 + e).
template <bool SIG>
VKH_DEV void gate(float g, float &a, float &rest) {
    if constexpr (SIG) {
        float m = fabsf(g);
        m = m > 200.f ? 200.f : m;  // (a NaN stays)
        const float p = m * -1.44269504f, lo = fmaf(m, -1.44269504f, -p) + m * -1.92596299e-8f;
        float e = __builtin_amdgcn_exp2f(p);
        e = fmaf(e, lo * 0.693147181f, e);
        const float s = 1.0f / (1.0f + e), t = e * s;
        a = g >= 0.f ? s : t;
        rest = g >= 0.f ? t : s;
        if (g != g) a = rest = g;
    } else {
        a = g;
        rest = 1.0f - g;
    }
}

VKH_DEV int rows_of(const ScanArgs &a, int b) {
    if (!a.len) return a.n_pos;
    const unsigned n = a.len[b];
    return n < (unsigned)a.n_pos ? (int)n : a.n_pos;
}

// What a wave holds of its rows: gates, inputs (x and 1 - a).  Rows from `len` on leave the state alone.
template <class T, int V, bool SIG, bool COUP>
struct Rows {
    float a[kRows][V], rest[kRows][V], x[kRows][V];
    VKH_DEV float u(int i, int v) const { return COUP ? rest[i][v] * x[i][v] : x[i][v]; }
    VKH_DEV void load(const ScanArgs &s, long row0, int t0, int len, int c, bool act) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (act && t0 + i < len) {
                load_v<T, V>((const T *)s.x + (row0 + i) * s.ldx + c, x[i]);
                load_v<T, V>((const T *)s.g + (row0 + i) * s.ldg + c, a[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (act && t0 + i < len) gate<SIG>(a[i][v], a[i][v], rest[i][v]);
                else a[i][v] = 1.f, rest[i][v] = x[i][v] = 0.f;
            }
    }
};

template <class TI, class TO, int V, bool SIG, bool COUP>
__global__ __launch_bounds__(kWaves * 64) void scan_fwd_k(ScanArgs s) {
    __shared__ float shA[2][kWaves][64 * V], shB[2][kWaves][64 * V];
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), b = blockIdx.y;
    const int c = (blockIdx.x * 64 + lane) * V, tiles = (s.n_pos + kScanTile - 1) / kScanTile;
    const bool act = c < s.dim;
    const int len = rows_of(s, b);
    float H[V] = {};
    if (act && s.h0) load_v<float, V>(s.h0 + (long)b * s.dim + c, H);
    for (int k = 0; k < tiles; ++k) {
        const int t0 = k * kScanTile + w * kRows;
        const long row0 = (long)b * s.n_pos + t0;
        Rows<TI, V, SIG, COUP> r;
        r.load(s, row0, t0, len, c, act);
        float (&A)[kWaves][64 * V] = shA[k & 1], (&B)[kWaves][64 * V] = shB[k & 1];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float p = 1.f, q = 0.f;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                p *= r.a[i][v];
                q = fmaf(r.a[i][v], q, r.u(i, v));
            }
            A[w][lane * V + v] = p;
            B[w][lane * V + v] = q;
        }
        if (s.states && w == 0 && act) store_v<float, V>(s.states + ((long)b * tiles + k) * s.dim + c, H);
        __syncthreads();
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = H[v];
        for (int j = 0; j < kWaves; ++j) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                H[v] = fmaf(A[j][lane * V + v], H[v], B[j][lane * V + v]);
                if (j < w) h[v] = H[v];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (!act || t0 + i >= s.n_pos) break;
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = fmaf(r.a[i][v], h[v], r.u(i, v));
                o[v] = t0 + i < len ? h[v] : 0.f;
            }
            store_v<TO, V>((TO *)s.h + (row0 + i) * s.ldh + c, o);
        }
    }
    if (s.h_last && w == 0 && act) store_v<float, V>(s.h_last + (long)b * s.dim + c, H);
}

template <class TI, class TO, int V, bool SIG, bool COUP>
__global__ __launch_bounds__(kWaves * 64) void scan_bwd_k(ScanArgs s) {
    __shared__ float shA[2][kWaves][64 * V], shB[2][kWaves][64 * V], shQ[2][kWaves][64 * V];
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), b = blockIdx.y;
    const int c = (blockIdx.x * 64 + lane) * V, tiles = (s.n_pos + kScanTile - 1) / kScanTile;
    const bool act = c < s.dim;
    const int len = rows_of(s, b);
    float R[V] = {};
    if (act && s.dh_last) load_v<float, V>(s.dh_last + (long)b * s.dim + c, R);
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * kScanTile + w * kRows;
        const long row0 = (long)b * s.n_pos + t0;
        Rows<TI, V, SIG, COUP> r;
        float d[kRows][V], hp[kRows][V], h[V] = {};
        r.load(s, row0, t0, len, c, act);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (act && t0 + i < len) {
                load_v<TI, V>((const TI *)s.dh + (row0 + i) * s.lddh + c, d[i]);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) d[i][v] = 0.f;
            }
        }
        // (a tile behind the sequence's end has no state, and needs none)
        if (act && k * kScanTile < len) load_v<float, V>(s.states + ((long)b * tiles + k) * s.dim + c, h);
        float (&A)[kWaves][64 * V] = shA[k & 1], (&B)[kWaves][64 * V] = shB[k & 1], (&Q)[kWaves][64 * V] = shQ[k & 1];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float p = 1.f, q = 0.f, z = 0.f;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                p *= r.a[i][v];
                q = fmaf(r.a[i][v], q, r.u(i, v));
            }
#pragma unroll
            for (int i = kRows - 1; i >= 0; --i) z = r.a[i][v] * (d[i][v] + z);
            A[w][lane * V + v] = p;
            B[w][lane * V + v] = q;
            Q[w][lane * V + v] = z;
        }
        __syncthreads();
        for (int j = 0; j < w; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = fmaf(A[j][lane * V + v], h[v], B[j][lane * V + v]);
        float e[V];
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = R[v];
        for (int j = kWaves - 1; j >= 0; --j) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                R[v] = fmaf(A[j][lane * V + v], R[v], Q[j][lane * V + v]);
                if (j > w) e[v] = R[v];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                hp[i][v] = h[v];
                h[v] = fmaf(r.a[i][v], h[v], r.u(i, v));
            }
#pragma unroll
        for (int i = kRows - 1; i >= 0; --i) {
            float dx[V], dg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float G = d[i][v] + e[v];
                e[v] = r.a[i][v] * G;
                dx[v] = COUP ? r.rest[i][v] * G : G;
                dg[v] = COUP ? G * (hp[i][v] - r.x[i][v]) : G * hp[i][v];
                if (SIG) dg[v] *= r.a[i][v] * r.rest[i][v];
                if (t0 + i >= len) dx[v] = dg[v] = 0.f;
            }
            if (act && t0 + i < s.n_pos) {
                store_v<TO, V>((TO *)s.dx + (row0 + i) * s.lddx + c, dx);
                store_v<TO, V>((TO *)s.dg + (row0 + i) * s.lddg + c, dg);
            }
        }
    }
    if (s.dh0 && w == 0 && act) store_v<float, V>(s.dh0 + (long)b * s.dim + c, R);
}

// Two channels a lane where every row of them can be read as pairs, else one.
bool pairs(const ScanArgs &s, bool back) {
    bool ok = s.dim % 2 == 0;
    auto may = [&](const void *p, long ld, DType t) {
        ok = ok && (uintptr_t)p % (t == DType::F32 ? 8 : 4) == 0 && ld % 2 == 0;
    };
    may(s.x, s.ldx, s.dt);
    may(s.g, s.ldg, s.dt);
    may(s.states, 0, DType::F32);
    if (back) {
        may(s.dh, s.lddh, s.dt);
        may(s.dx, s.lddx, s.odt);
        may(s.dg, s.lddg, s.odt);
        may(s.dh0, 0, DType::F32);
        may(s.dh_last, 0, DType::F32);
    } else {
        may(s.h, s.ldh, s.odt);
        may(s.h0, 0, DType::F32);
        may(s.h_last, 0, DType::F32);
    }
    return ok;
}

template <class F>
void by_form(const ScanArgs &s, bool pair, F f) {
    by_type(s.dt, [&](auto ti) {
        by_type(s.odt, [&](auto to) {
            auto gates = [&](auto v) {
                auto coup = [&](auto sig) {
                    if (s.coupled) f(ti, to, v, sig, std::true_type{});
                    else f(ti, to, v, sig, std::false_type{});
                };
                if (s.sigmoid) coup(std::true_type{});
                else coup(std::false_type{});
            };
            if (pair) gates(std::integral_constant<int, 2>{});
            else gates(std::integral_constant<int, 1>{});
        });
    });
}

dim3 grid_of(const ScanArgs &s, int V) { return dim3(ceil_div(s.dim, 64 * V), s.n_batch); }

}  // namespace

size_t scan_states_floats(const ScanArgs &s) {
    return (size_t)s.n_batch * ((s.n_pos + kScanTile - 1) / kScanTile) * s.dim;
}
size_t scan_ws_bytes(const ScanArgs &) { return 0; }

hipError_t scan_forward(const ScanArgs &s, hipStream_t st) {
    by_form(s, pairs(s, false), [&](auto ti, auto to, auto v, auto sig, auto coup) {
        constexpr int V = decltype(v)::value;
        hipLaunchKernelGGL((scan_fwd_k<decltype(ti), decltype(to), V, decltype(sig)::value, decltype(coup)::value>),
                           grid_of(s, V), dim3(kWaves * 64), 0, st, s);
    });
    return hipGetLastError();
}

hipError_t scan_backward(const ScanArgs &s, hipStream_t st) {
    by_form(s, pairs(s, true), [&](auto ti, auto to, auto v, auto sig, auto coup) {
        constexpr int V = decltype(v)::value;
        hipLaunchKernelGGL((scan_bwd_k<decltype(ti), decltype(to), V, decltype(sig)::value, decltype(coup)::value>),
                           grid_of(s, V), dim3(kWaves * 64), 0, st, s);
    });
    return hipGetLastError();
}

}  // namespace vkh
