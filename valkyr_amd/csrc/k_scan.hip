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
// channels and tiles of a few rows for each of its waves: a wave holds its rows of all these channels in
// registers, forms A and B of them, and joins the others' before it through LDS; then it runs its rows again from
// the state that they start from.  Each value is read and written once: bound by HBM.  The forward keeps the state
// before every kScanTile rows, from which the backward forms h again.
//
// Where channels are few, the tiles of a sequence go to blocks of their own.  A tile's block publishes its A and B
// as soon as it has them, looks for the nearest tile before it whose state behind it is known, applies the A and B
// of the tiles between in their order, and publishes its own state.  That is the same arithmetic whichever tile it
// starts from, so results do not depend on timing, nor on whether a sequence is split.  Blocks take their tiles
// by a ticket, in order of time: a tile waits only for tiles that running blocks hold already, and the first of
// those waits for none.  Published words are single atomic stores past the XCDs' own caches, valid once they differ
// from kUnset, so nothing has to be ordered.
#include <algorithm>
#include <type_traits>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int kFwdWaves = 8, kBwdWaves = 16;
constexpr int kFwdRows = 16, kBwdRows = 8;  // a wave's
constexpr int kFwdTile = kFwdWaves * kFwdRows, kBwdTile = kBwdWaves * kBwdRows;
static_assert(kScanTile % kFwdRows == 0 && kFwdTile % kScanTile == 0 && kBwdTile == kScanTile, "states");
constexpr int kFew = 16;  // rows of a short sequence
constexpr int kPerSimd = 4;  // waves: registers for 16 a CU
constexpr int kLook = 4;  // tiles looked back over at a time
constexpr uint32_t kUnset = 0xffffffffu;

template <class F>
void by_type(DType d, F f) {
    if (d == DType::F32) f(float{});
    else f(bf16{});
}

// V values from any address of T
template <class T, int V> struct Vec;
template <int V> struct Vec<float, V> { typedef float type __attribute__((ext_vector_type(V), aligned(4))); };
template <int V> struct Vec<bf16, V> { typedef bf16 type __attribute__((ext_vector_type(V), aligned(2))); };
template <class T, int V>
using Raw = std::conditional_t<V == 1, T, typename Vec<T, V>::type>;

template <class T, int V>
VKH_DEV Raw<T, V> load_raw(const T *p) { return *reinterpret_cast<const Raw<T, V> *>(p); }
// A matrix's rows from `row` on: a pointer that is the same for all lanes, which add their channel's bytes to it in 32
// bits.  (Both are kept from being joined into vector registers, two for each row of each matrix.)
typedef __attribute__((address_space(1))) char *Row;
template <class T>
struct Walk {
    uintptr_t p, step;
    VKH_DEV Walk(const void *m, long row, long ld) : p((uintptr_t)m + row * ld * (long)sizeof(T)), step(ld * sizeof(T)) {
        asm volatile("" : "+s"(p));
    }
    VKH_DEV Row at(unsigned bytes) const {
        asm volatile("" : "+v"(bytes));
        return (Row)p + bytes;
    }
    template <int V>
    VKH_DEV Raw<T, V> load(unsigned bytes) const { return *(__attribute__((address_space(1))) Raw<T, V> *)at(bytes); }
    template <int V>
    VKH_DEV void store(unsigned bytes, const float (&o)[V]) const;
    VKH_DEV void next(bool more = true) { p += more ? step : 0; }
    VKH_DEV void back() { p -= step; }
};
template <class T, int V>
VKH_DEV float part(const Raw<T, V> &r, int v) {
    if constexpr (V == 1) return (float)r;
    else return (float)r[v];
}
template <class T, int V>
VKH_DEV void load_v(const T *p, float (&o)[V]) {
    const Raw<T, V> r = load_raw<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = part<T, V>(r, i);
}
template <class T, int V>
VKH_DEV Raw<T, V> raw_of(const float (&o)[V]) {
    Raw<T, V> r;
    if constexpr (V == 1) {
        r = (T)o[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = (T)o[i];
    }
    return r;
}
template <class T, int V>
VKH_DEV void store_v(T *p, const float (&o)[V]) { *reinterpret_cast<Raw<T, V> *>(p) = raw_of<T, V>(o); }
template <class T>
template <int V>
VKH_DEV void Walk<T>::store(unsigned bytes, const float (&o)[V]) const {
    *(__attribute__((address_space(1))) Raw<T, V> *)at(bytes) = raw_of<T, V>(o);
}

// a and 1 - a of a gate, each to its own last digits: e = exp(-|g|) from a product in two parts (one alone is
// off by |g| steps), 1 / (1 + e) and e / (1 + e).
template <bool SIG>
VKH_DEV void gate(float g, float &a, float &rest) {
    if constexpr (SIG) {
        float m = fabsf(g);
        m = m > 200.f ? 200.f : m;  // (a NaN stays)
        const float p = m * -1.44269504f, lo = fmaf(m, -1.92596299e-8f, fmaf(m, -1.44269504f, -p));
        float e = __builtin_amdgcn_exp2f(p);
        e = fmaf(e, lo * 0.693147181f, e);
        const float s = __builtin_amdgcn_rcpf(1.0f + e), t = e * s;
        a = g >= 0.f ? s : t;
        rest = g >= 0.f ? t : s;
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

// The workspace of a split call: a ticket, then each tile's A and B (a 64-bit word a channel) and the state behind it.
struct Words {
    unsigned *ticket;
    uint64_t *ab;
    uint32_t *h;
};
__host__ __device__ inline Words words_of(void *ws, size_t channels) {
    Words w;
    w.ticket = (unsigned *)ws;
    w.ab = (uint64_t *)((char *)ws + 64);
    w.h = (uint32_t *)(w.ab + channels);
    return w;
}
__global__ __launch_bounds__(256) void scan_clear_k(uint4 *ws, size_t n) {
    const size_t step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step)
        ws[i] = i ? make_uint4(kUnset, kUnset, kUnset, kUnset) : make_uint4(0, 0, 0, 0);
}

VKH_DEV uint32_t bits_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return u == kUnset ? 0x7fc00000u : u;  // (one NaN for another)
}
VKH_DEV uint64_t word_of(float a, float b) { return (uint64_t)bits_of(b) << 32 | bits_of(a); }
VKH_DEV float low_of(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)w); }
VKH_DEV float high_of(uint64_t w) { return __builtin_bit_cast(float, (uint32_t)(w >> 32)); }
// A word of the workspace: `at` the same for all lanes, `bytes` the lane's.
template <class T>
VKH_DEV T peek(const void *at, unsigned bytes) {
    const Walk<T> w(at, 0, 0);
    return __hip_atomic_load((__attribute__((address_space(1))) T *)w.at(bytes), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
VKH_DEV void publish(void *at, unsigned bytes, T v) {
    const Walk<T> w(at, 0, 0);
    __hip_atomic_store((__attribute__((address_space(1))) T *)w.at(bytes), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int V>
using States = std::conditional_t<V == 1, uint32_t, uint64_t>;

// By one wave, for the 64 V channels at `base` of the words (tile s of the sequence at s 64 V after it): publishes
// this tile's A and B, sets H (given for the first tile) to the state before tile s, and publishes the one behind it.
// A tile's states of a lane are one word.
template <int V>
VKH_DEV void look_back(const Words &W, size_t base, int s, unsigned lane, const float (&A)[V], const float (&B)[V], float (&H)[V]) {
    const unsigned lab = lane * V * 8, lh = lane * V * 4;
    auto ab = [&](int k) { return W.ab + base + (size_t)k * 64 * V; };
    auto hs = [&](int k) { return W.h + base + (size_t)k * 64 * V; };
    if (s) {
#pragma unroll
        for (int v = 0; v < V; ++v) publish(ab(s), lab + v * 8, word_of(A[v], B[v]));
    }
    for (bool found = s == 0; !found;) {
        uint64_t w[kLook][V];
        States<V> h[kLook];
#pragma unroll
        for (int d = 0; d < kLook; ++d) {  // tile s - 1 - d
            const int k = max(s - 1 - d, 0);
            h[d] = peek<States<V>>(hs(k), lh);
#pragma unroll
            for (int v = 0; v < V; ++v) w[d][v] = peek<uint64_t>(ab(k), lab + v * 8);
        }
        int n = 0;  // tiles between the nearest known state and this tile
        bool going = true;
#pragma unroll
        for (int d = 0; d < kLook; ++d) {
            const bool known = (uint32_t)h[d] != kUnset && (V == 1 || (uint32_t)((uint64_t)h[d] >> 32) != kUnset);
            if (going && __ballot(!known) == 0) {
                going = false;
                found = true;
                n = d;
#pragma unroll
                for (int v = 0; v < V; ++v) H[v] = __builtin_bit_cast(float, (uint32_t)((uint64_t)h[d] >> 32 * v));
            }
            bool there = s - 1 - d > 0;  // (the first tile publishes its state alone)
#pragma unroll
            for (int v = 0; v < V; ++v) there = there && (uint32_t)(w[d][v] >> 32) != kUnset;
            going = going && __ballot(!there) == 0;
        }
        if (found) {
#pragma unroll
            for (int d = kLook - 2; d >= 0; --d)
                if (d < n)
#pragma unroll
                    for (int v = 0; v < V; ++v) H[v] = fmaf(low_of(w[d][v]), H[v], high_of(w[d][v]));
        } else {
            __builtin_amdgcn_s_sleep(1);
        }
    }
    uint64_t out = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) out |= (uint64_t)bits_of(fmaf(A[v], H[v], B[v])) << 32 * v;
    publish(hs(s), lh, (States<V>)out);
}

// The tiles of a block: of a split call those that its tickets name, in order of time from the side that the scan
// starts from (s: the how manieth), each ticket fetched while the tile before it is worked on; else all tiles of a
// sequence and channel group.
template <bool SPLIT>
struct Tiles {
    int b, grp, s = -1, groups, n_batch, tiles;
    unsigned *sh, next;
    VKH_DEV Tiles(const Words &W, int groups_, int n_batch_, int tiles_, unsigned *sh_)
        : b(blockIdx.y), grp(blockIdx.x), groups(groups_), n_batch(n_batch_), tiles(tiles_), sh(sh_) {
        if (SPLIT && threadIdx.x == 0) next = atomicAdd(W.ticket, 1u);
    }
    VKH_DEV bool take(const Words &W) {
        if (!SPLIT) return ++s < tiles;
        if (threadIdx.x == 0) *sh = next;
        __syncthreads();  // (also behind the last tile's reads of LDS)
        const unsigned t = __builtin_amdgcn_readfirstlane(*sh), per = groups * n_batch, at = t % per;
        s = t / per, b = at / groups, grp = at % groups;
        if (s >= tiles) return false;
        if (threadIdx.x == 0) next = atomicAdd(W.ticket, 1u);
        return true;
    }
};

template <class TI, class TO, int V, bool SIG, bool COUP, bool SPLIT>
__global__ __launch_bounds__(kFwdWaves * 64, kPerSimd) void scan_fwd_k(ScanArgs s, int groups) {
    constexpr int R = kFwdRows;
    __shared__ float shA[2][kFwdWaves][64 * V], shB[2][kFwdWaves][64 * V], shH[64 * V];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles = (s.n_pos + kFwdTile - 1) / kFwdTile, marks = (s.n_pos + kScanTile - 1) / kScanTile;
    const Words W = words_of(s.ws, (size_t)s.n_batch * groups * tiles * 64 * V);
    Tiles<SPLIT> at(W, groups, s.n_batch, tiles, &ticket);
    float H[V];
    while (at.take(W)) {
        const int k = at.s, b = at.b, c = (at.grp * 64 + lane) * V, len = rows_of(s, b);
        const bool act = c < s.dim;
        const unsigned in_bytes = (act ? c : s.dim - V) * sizeof(TI), out_bytes = c * sizeof(TO);  // (lanes past the channels read the last ones)
        if (SPLIT || k == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) H[v] = 0.f;
            if (k == 0 && act && s.h0) load_v<float, V>(s.h0 + (long)b * s.dim + c, H);
        }
        const int t0 = k * kFwdTile + w * R;
        const long row0 = (long)b * s.n_pos + t0;
        Raw<TI, V> xr[R], gr[R];
        if (t0 < len) {  // (rows behind the end: the last one again)
            Walk<TI> g(s.g, row0, s.ldg), x(s.x, row0, s.ldx);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                gr[i] = g.template load<V>(in_bytes);
                xr[i] = x.template load<V>(in_bytes);
                g.next(t0 + i + 1 < len);
                x.next(t0 + i + 1 < len);
            }
        }
        float a[R][V], u[R][V], p[V], q[V];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float rest;
                gate<SIG>(part<TI, V>(gr[i], v), a[i][v], rest);
                u[i][v] = part<TI, V>(xr[i], v);
                if (COUP) u[i][v] *= rest;
            }
        if (t0 + R > len) {  // rows behind the end leave the state alone
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (t0 + i >= len) a[i][v] = 1.f, u[i][v] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            p[v] = 1.f, q[v] = 0.f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                p[v] *= a[i][v];
                q[v] = fmaf(a[i][v], q[v], u[i][v]);
            }
        }
        float (&A)[kFwdWaves][64 * V] = shA[k & 1], (&B)[kFwdWaves][64 * V] = shB[k & 1];
#pragma unroll
        for (int v = 0; v < V; ++v) A[w][lane * V + v] = p[v], B[w][lane * V + v] = q[v];
        __syncthreads();
        // of the waves before this one, and of the tile
        float pa[V], pb[V], ta[V], tb[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            ta[v] = 1.f, tb[v] = 0.f;
#pragma unroll
            for (int j = 0; j < kFwdWaves; ++j) {
                if (j == w) pa[v] = ta[v], pb[v] = tb[v];
                ta[v] *= A[j][lane * V + v];
                tb[v] = fmaf(A[j][lane * V + v], tb[v], B[j][lane * V + v]);
            }
        }
        if (SPLIT) {
            if (w == 0) {
                look_back<V>(W, ((size_t)b * groups + at.grp) * tiles * 64 * V, k, lane, ta, tb, H);
#pragma unroll
                for (int v = 0; v < V; ++v) shH[lane * V + v] = H[v];
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v) H[v] = shH[lane * V + v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = fmaf(pa[v], H[v], pb[v]);
            H[v] = fmaf(ta[v], H[v], tb[v]);
        }
        if (s.states && w * R % kScanTile == 0 && t0 < s.n_pos && act)
            store_v<float, V>(s.states + ((long)b * marks + t0 / kScanTile) * s.dim + c, h);
        if (act) {
            Walk<TO> out(s.h, row0, s.ldh);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                float o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = fmaf(a[i][v], h[v], u[i][v]);
                    o[v] = t0 + i < len ? h[v] : 0.f;
                }
                if (t0 + i < s.n_pos) out.store(out_bytes, o);
                out.next();
            }
        }
        if (k + 1 == tiles && s.h_last && w == 0 && act) store_v<float, V>(s.h_last + (long)b * s.dim + c, H);
    }
}

template <class TI, class TO, int V, bool SIG, bool COUP, bool SPLIT>
__global__ __launch_bounds__(kBwdWaves * 64, kPerSimd) void scan_bwd_k(ScanArgs s, int groups) {
    constexpr int N = kBwdRows;
    __shared__ float shA[2][kBwdWaves][64 * V], shB[2][kBwdWaves][64 * V], shQ[2][kBwdWaves][64 * V], shR[64 * V];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles = (s.n_pos + kBwdTile - 1) / kBwdTile;
    const Words W = words_of(s.ws, (size_t)s.n_batch * groups * tiles * 64 * V);
    Tiles<SPLIT> at(W, groups, s.n_batch, tiles, &ticket);
    float R[V];
    while (at.take(W)) {
        const int k = tiles - 1 - at.s, b = at.b, c = (at.grp * 64 + lane) * V, len = rows_of(s, b);
        const bool act = c < s.dim;
        const unsigned in_bytes = (act ? c : s.dim - V) * sizeof(TI), out_bytes = c * sizeof(TO);  // (lanes past the channels read the last ones)
        if (SPLIT || at.s == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) R[v] = 0.f;
            if (at.s == 0 && act && s.dh_last) load_v<float, V>(s.dh_last + (long)b * s.dim + c, R);
        }
        const int t0 = k * kBwdTile + w * N;
        const long row0 = (long)b * s.n_pos + t0;
        Raw<TI, V> xr[N], gr[N], dr[N];
        float h[V] = {};
        if (t0 < len) {  // (rows behind the end: the last one again)
            Walk<TI> g(s.g, row0, s.ldg), d(s.dh, row0, s.lddh), x(s.x, row0, s.ldx);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                gr[i] = g.template load<V>(in_bytes);
                dr[i] = d.template load<V>(in_bytes);
                xr[i] = x.template load<V>(in_bytes);
                g.next(t0 + i + 1 < len);
                d.next(t0 + i + 1 < len);
                x.next(t0 + i + 1 < len);
            }
        }
        // (a tile behind the sequence's end has no state, and needs none)
        if (act && k * kBwdTile < len) load_v<float, V>(s.states + ((long)b * tiles + k) * s.dim + c, h);
        float a[N][V], rest[N][V], x[N][V], d[N][V];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gate<SIG>(part<TI, V>(gr[i], v), a[i][v], rest[i][v]);
                x[i][v] = part<TI, V>(xr[i], v);
                d[i][v] = part<TI, V>(dr[i], v);
            }
        if (t0 + N > len) {  // rows behind the end leave state and gradient alone
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (t0 + i >= len) a[i][v] = 1.f, rest[i][v] = x[i][v] = d[i][v] = 0.f;
        }
        auto u = [&](int i, int v) { return COUP ? rest[i][v] * x[i][v] : x[i][v]; };
        float (&A)[kBwdWaves][64 * V] = shA[k & 1], (&B)[kBwdWaves][64 * V] = shB[k & 1], (&Q)[kBwdWaves][64 * V] = shQ[k & 1];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float p = 1.f, q = 0.f, z = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p *= a[i][v];
                q = fmaf(a[i][v], q, u(i, v));
            }
#pragma unroll
            for (int i = N - 1; i >= 0; --i) z = a[i][v] * (d[i][v] + z);
            A[w][lane * V + v] = p;
            B[w][lane * V + v] = q;
            Q[w][lane * V + v] = z;
        }
        __syncthreads();
        // of the waves behind this one, and of the tile; and the state before this wave's rows
        float pa[V], pb[V], ta[V], tb[V], e[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            ta[v] = 1.f, tb[v] = 0.f;
#pragma unroll
            for (int j = kBwdWaves - 1; j >= 0; --j) {
                if (j == w) pa[v] = ta[v], pb[v] = tb[v];
                ta[v] *= A[j][lane * V + v];
                tb[v] = fmaf(A[j][lane * V + v], tb[v], Q[j][lane * V + v]);
            }
#pragma unroll
            for (int j = 0; j < w; ++j) h[v] = fmaf(A[j][lane * V + v], h[v], B[j][lane * V + v]);
        }
        if (SPLIT) {
            if (w == 0) {
                look_back<V>(W, ((size_t)b * groups + at.grp) * tiles * 64 * V, at.s, lane, ta, tb, R);
#pragma unroll
                for (int v = 0; v < V; ++v) shR[lane * V + v] = R[v];
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v) R[v] = shR[lane * V + v];
        }
        float hp[N][V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            e[v] = fmaf(pa[v], R[v], pb[v]);
            R[v] = fmaf(ta[v], R[v], tb[v]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                hp[i][v] = h[v];
                h[v] = fmaf(a[i][v], h[v], u(i, v));
            }
        }
        Walk<TO> ox(s.dx, row0 + N - 1, s.lddx), og(s.dg, row0 + N - 1, s.lddg);
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            float dx[V], dg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float G = d[i][v] + e[v];
                e[v] = a[i][v] * G;
                dx[v] = COUP ? rest[i][v] * G : G;
                dg[v] = COUP ? G * (hp[i][v] - x[i][v]) : G * hp[i][v];
                if (SIG) dg[v] *= a[i][v] * rest[i][v];
                if (t0 + i >= len) dx[v] = dg[v] = 0.f;
            }
            if (act && t0 + i < s.n_pos) {
                ox.store(out_bytes, dx);
                og.store(out_bytes, dg);
            }
            ox.back();
            og.back();
        }
        if (k == 0 && s.dh0 && w == 0 && act) store_v<float, V>(s.dh0 + (long)b * s.dim + c, R);
    }
}

// Sequences of up to kFew rows (the next token of each, above all): a thread takes V channels through all rows.
template <class TI, class TO, int V, bool SIG, bool COUP>
__global__ __launch_bounds__(256) void scan_few_fwd_k(ScanArgs s) {
    const int b = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * V, len = rows_of(s, b);
    if (c >= s.dim) return;
    const long row0 = (long)b * s.n_pos, state = (long)b * s.dim + c;
    float h[V] = {};
    if (s.h0) load_v<float, V>(s.h0 + state, h);
    if (s.states && s.n_pos) store_v<float, V>(s.states + state, h);
#pragma unroll 4
    for (int t = 0; t < s.n_pos; ++t) {
        float g[V], x[V], o[V] = {};
        if (t < len) {
            load_v<TI, V>((const TI *)s.g + (row0 + t) * s.ldg + c, g);
            load_v<TI, V>((const TI *)s.x + (row0 + t) * s.ldx + c, x);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                gate<SIG>(g[v], a, rest);
                o[v] = h[v] = fmaf(a, h[v], COUP ? rest * x[v] : x[v]);
            }
        }
        store_v<TO, V>((TO *)s.h + (row0 + t) * s.ldh + c, o);
    }
    if (s.h_last) store_v<float, V>(s.h_last + state, h);
}

template <class TI, class TO, bool SIG, bool COUP>
__global__ __launch_bounds__(256) void scan_few_bwd_k(ScanArgs s) {
    const int b = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x, len = rows_of(s, b);
    if (c >= s.dim) return;
    const long row0 = (long)b * s.n_pos, state = (long)b * s.dim + c;
    float hp[kFew], a[kFew], rest[kFew], x[kFew], h = len ? s.states[state] : 0.f, R = s.dh_last ? s.dh_last[state] : 0.f;
#pragma unroll
    for (int t = 0; t < kFew; ++t) {
        if (t >= len) continue;
        gate<SIG>(to_f32(((const TI *)s.g)[(row0 + t) * s.ldg + c]), a[t], rest[t]);
        x[t] = to_f32(((const TI *)s.x)[(row0 + t) * s.ldx + c]);
        hp[t] = h;
        h = fmaf(a[t], h, COUP ? rest[t] * x[t] : x[t]);
    }
#pragma unroll
    for (int t = kFew - 1; t >= 0; --t) {
        if (t >= s.n_pos) continue;
        float dx = 0.f, dg = 0.f;
        if (t < len) {
            const float G = to_f32(((const TI *)s.dh)[(row0 + t) * s.lddh + c]) + R;
            R = a[t] * G;
            dx = COUP ? rest[t] * G : G;
            dg = COUP ? G * (hp[t] - x[t]) : G * hp[t];
            if (SIG) dg *= a[t] * rest[t];
        }
        ((TO *)s.dx)[(row0 + t) * s.lddx + c] = (TO)dx;
        ((TO *)s.dg)[(row0 + t) * s.lddg + c] = (TO)dg;
    }
    if (s.dh0) s.dh0[state] = R;
}

// How a call is laid out: channels a lane, channel groups, and whether its tiles go to blocks of their own.
struct Plan {
    int groups;
    bool split;
    size_t blocks, channels;  // of a split call; its words' channels
};
Plan plan_of(const ScanArgs &s, int tile) {
    Plan p;
    p.groups = (int)ceil_div(s.dim, 64);
    const size_t rows = (size_t)p.groups * s.n_batch, tiles = (s.n_pos + tile - 1) / tile;
    p.blocks = rows * tiles;
    p.channels = p.blocks * 64;
    p.split = s.n_pos > kFew && tiles > 1 && rows < 1024 && p.blocks < (1u << 20);
    return p;
}
size_t words_bytes(const Plan &p) { return p.split ? (64 + p.channels * 12 + 15) / 16 * 16 : 0; }

template <class F>
void by_form(const ScanArgs &s, F f) {
    by_type(s.dt, [&](auto ti) {
        by_type(s.odt, [&](auto to) {
            auto coup = [&](auto sig) {
                if (s.coupled) f(ti, to, sig, std::true_type{});
                else f(ti, to, sig, std::false_type{});
            };
            if (s.sigmoid) coup(std::true_type{});
            else coup(std::false_type{});
        });
    });
}

// The plan of a call, its workspace ready
Plan ready(const ScanArgs &s, int tile, hipStream_t st) {
    Plan p = plan_of(s, tile);
    if (!s.ws) p.split = false;
    const size_t n = words_bytes(p) / 16;
    if (p.split) hipLaunchKernelGGL(scan_clear_k, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1024)), dim3(256), 0, st, (uint4 *)s.ws, n);
    return p;
}
dim3 grid_of(const ScanArgs &s, const Plan &p, int waves) {
    return p.split ? dim3((unsigned)std::min<size_t>(p.blocks, (size_t)cu_count() * kPerSimd * 4 / waves)) : dim3(p.groups, s.n_batch);
}

}  // namespace

size_t scan_states_floats(const ScanArgs &s) {
    return (size_t)s.n_batch * ((s.n_pos + kScanTile - 1) / kScanTile) * s.dim;
}
size_t scan_ws_bytes(const ScanArgs &s) {
    return std::max(words_bytes(plan_of(s, kFwdTile)), words_bytes(plan_of(s, kBwdTile)));
}

hipError_t scan_forward(const ScanArgs &s, hipStream_t st) {
    by_form(s, [&](auto ti, auto to, auto sig, auto coup) {
        using TI = decltype(ti);
        using TO = decltype(to);
        constexpr bool SIG = decltype(sig)::value, COUP = decltype(coup)::value;
        if (s.n_pos <= kFew) {
            const int V = s.dim % 4 ? 1 : 4;
            auto k = V == 4 ? scan_few_fwd_k<TI, TO, 4, SIG, COUP> : scan_few_fwd_k<TI, TO, 1, SIG, COUP>;
            hipLaunchKernelGGL(k, dim3(ceil_div(s.dim, 256 * V), s.n_batch), dim3(256), 0, st, s);
            return;
        }
        const Plan p = ready(s, kFwdTile, st);
        auto k = p.split ? scan_fwd_k<TI, TO, 1, SIG, COUP, true> : scan_fwd_k<TI, TO, 1, SIG, COUP, false>;
        hipLaunchKernelGGL(k, grid_of(s, p, kFwdWaves), dim3(kFwdWaves * 64), 0, st, s, p.groups);
    });
    return hipGetLastError();
}

hipError_t scan_backward(const ScanArgs &s, hipStream_t st) {
    by_form(s, [&](auto ti, auto to, auto sig, auto coup) {
        using TI = decltype(ti);
        using TO = decltype(to);
        constexpr bool SIG = decltype(sig)::value, COUP = decltype(coup)::value;
        if (s.n_pos <= kFew) {
            hipLaunchKernelGGL((scan_few_bwd_k<TI, TO, SIG, COUP>), dim3(ceil_div(s.dim, 256), s.n_batch), dim3(256), 0, st, s);
            return;
        }
        const Plan p = ready(s, kBwdTile, st);
        auto k = p.split ? scan_bwd_k<TI, TO, 1, SIG, COUP, true> : scan_bwd_k<TI, TO, 1, SIG, COUP, false>;
        hipLaunchKernelGGL(k, grid_of(s, p, kBwdWaves), dim3(kBwdWaves * 64), 0, st, s, p.groups);
    });
    return hipGetLastError();
}

}  // namespace vkh
