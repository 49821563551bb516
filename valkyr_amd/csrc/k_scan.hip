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
// the stretch makes of h = 0), and the same A carries R the other way: R -> A R + Q.  A block takes 64
// channels and tiles of a few rows for each of its waves: a wave holds its rows of all these channels in
// registers, forms A and B of them, and joins the others' before it through LDS; then it runs its rows again from
// the state that they start from.  Each value is read and written once: bound by HBM.  The forward keeps the state
// before every kScanTile rows, from which the backward forms h again.
//
// Where channels are few, the tiles of a sequence go to blocks of their own.  A tile's block publishes its A and B
// as soon as it has them, looks for the nearest tile before it whose state behind it is known, applies the A and B
// of the tiles between in their order, and publishes its own state.  That is the same arithmetic whichever tile it
// starts from, so results do not depend on timing, nor on whether a sequence is split.  Blocks take a sequence's
// tiles by tickets, in order of time: a tile waits only for tiles that running blocks hold already, and the first of
// those waits for none.  Published words are single atomic stores past the XCDs' own caches, valid once they differ
// from kUnset, so nothing has to be ordered.
#include <algorithm>
#include <type_traits>

#include "ops.hpp"

namespace vkh {
namespace {

// 16 rows a wave in the forward, whose values, gates and inputs fit 128 registers so; 8 in the backward, which holds five
// numbers of each, and twice the waves, so that a tile has as many rows: fewer tiles have fewer words to publish and to
// look back over (16384 x 4096 bf16, a forward of 64 rows a tile 120 us beside 113, a backward of 8 waves and 64 rows 196
// beside 185).  Registers for three blocks a CU spill and are slower (128 and 210).
constexpr int kFwdWaves = 8, kBwdWaves = 16;
constexpr int kFwdRows = 16, kBwdRows = 8;
constexpr int kFwdTile = kFwdWaves * kFwdRows, kBwdTile = kBwdWaves * kBwdRows;
static_assert(kFwdTile == kScanTile && kBwdTile == kScanTile, "states");
constexpr int kPerSimd = 4;  // waves: 128 registers
constexpr int kFold = 4;     // waves whose A and B are read at a time
constexpr int kLook = 4;     // tiles looked back over at a time (one: a forward of 131 us beside 118; eight: 114 beside 113)
constexpr size_t kMostChannels = 80l << 20;  // of a split call's words (12 bytes each)
constexpr uint32_t kUnset = 0xffffffffu;
// Rows of a sequence that a thread takes alone.  64 sequences of 16 rows of 4096 bf16, forward and backward, their inputs
// in the last cache: 14 and 17 us (22 and 25 where they are not), 30 and 66 in tiles; 8 of them, 10 and 9, in tiles 8 and 10.
constexpr int kFew = 16;

// V values from any address of T
template <class T, int V>
using Raw = std::conditional_t<V == 1, T, typename Vec<T, V>::type>;

template <class T, int V>
VKH_DEV Raw<T, V> load_raw(const T *p) { return *reinterpret_cast<const Raw<T, V> *>(p); }
// A matrix's rows from `row` on: a pointer that is the same for all lanes, which add their channel's bytes to it in 32
// bits.  (Both are kept from being joined into vector registers, two for each row of each matrix: the pointer here,
// the bytes by here() at each row, after which they are a new value.)
VKH_DEV unsigned here(unsigned bytes) {
    asm volatile("" : "+v"(bytes));
    return bytes;
}
typedef __attribute__((address_space(1))) char *Row;
template <class T>
struct Walk {
    uintptr_t p, step;
    VKH_DEV Walk(const void *m, long row, long ld) : p((uintptr_t)m + row * ld * (long)sizeof(T)), step(ld * sizeof(T)) {
        p = (uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)p);
        asm volatile("" : "+s"(p));
    }
    VKH_DEV Row at(unsigned bytes) const { return (Row)p + bytes; }
    VKH_DEV T load(unsigned bytes) const { return *(__attribute__((address_space(1))) T *)at(bytes); }
    // past the caches: what is written is read by another kernel
    VKH_DEV void store(unsigned bytes, float v) const { __builtin_nontemporal_store((T)v, (__attribute__((address_space(1))) T *)at(bytes)); }
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
// a and 1 - a of a gate, each to its own last digits (the smaller one may be 0 past |g| = 87, where it would be less than
// fp32's normal numbers): e = exp(-|g|), 1 / (1 + e) and e / (1 + e).  The exponential takes
// its product with 1 / ln 2 in two parts (one alone is off by |g| steps): exact with the first 16 bits of it for a
// bf16, the rounded one and what its rounding left for an fp32.
template <bool SIG, class T>
VKH_DEV void gate(T logit, float &a, float &rest) {
    const float g = (float)logit;
    if constexpr (SIG) {
        float m = fabsf(g), p, less;  // e = 2^p (1 - less)
        m = m > 200.f ? 200.f : m;    // (a NaN stays)
        if constexpr (sizeof(T) == 2) {
            p = m * -0x1.7154p+0f;
            less = m * 4.88849537e-06f;
        } else {
            p = m * -1.44269502f;
            less = fmaf(fmaf(m, 1.44269502f, p), 0.693147182f, m * 1.33497577e-08f);
        }
        float e = __builtin_amdgcn_exp2f(p);
        e = fmaf(-e, less, e);
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

// The workspace of a split call: a counter for each sequence and channel group, in lines of their own, then each
// tile's A and B (a 64-bit word a channel) and the state behind it.
constexpr int kTicketBytes = 128;
struct Words {
    char *tickets;
    uint64_t *ab;
    uint32_t *h;
};
__host__ __device__ inline Words words_of(void *ws, size_t lines, size_t channels) {
    Words w;
    w.tickets = (char *)ws;
    w.ab = (uint64_t *)((char *)ws + lines * kTicketBytes);
    w.h = (uint32_t *)(w.ab + channels);
    return w;
}
__global__ __launch_bounds__(256) void scan_clear_k(uint4 *ws, size_t zeros, size_t n) {
    const size_t step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step)
        ws[i] = i < zeros ? make_uint4(0, 0, 0, 0) : make_uint4(kUnset, kUnset, kUnset, kUnset);
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
    return __hip_atomic_load((__attribute__((address_space(1))) T *)w.at(here(bytes)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
VKH_DEV void publish(void *at, unsigned bytes, T v) {
    const Walk<T> w(at, 0, 0);
    __hip_atomic_store((__attribute__((address_space(1))) T *)w.at(here(bytes)), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// By one wave, for the 64 channels at `base` of the words (tile s of the sequence at 64 s after it): publishes this
// tile's A and B, sets H (given for the first tile) to the state before tile s, and publishes the one behind it.
VKH_DEV void look_back(const Words &W, size_t base, int s, unsigned lane, float A, float B, float &H) {
    auto ab = [&](int k) { return W.ab + base + (size_t)k * 64; };
    auto hs = [&](int k) { return W.h + base + (size_t)k * 64; };
    if (s) publish(ab(s), lane * 8, word_of(A, B));
    for (bool found = s == 0; !found;) {
        uint64_t w[kLook];
        uint32_t h[kLook];
#pragma unroll
        for (int d = 0; d < kLook; ++d) {  // tile s - 1 - d
            const int k = max(s - 1 - d, 0);
            h[d] = peek<uint32_t>(hs(k), lane * 4);
            w[d] = peek<uint64_t>(ab(k), lane * 8);
        }
        int n = 0;  // tiles between the nearest known state and this tile
        bool going = true;
#pragma unroll
        for (int d = 0; d < kLook; ++d) {
            if (going && __ballot(h[d] == kUnset) == 0) {
                going = false;
                found = true;
                n = d;
                H = __builtin_bit_cast(float, h[d]);
            }
            // (the first tile publishes its state alone)
            going = going && s - 1 - d > 0 && __ballot((uint32_t)(w[d] >> 32) == kUnset) == 0;
        }
        if (found) {
#pragma unroll
            for (int d = kLook - 2; d >= 0; --d)
                if (d < n) H = fmaf(low_of(w[d]), H, high_of(w[d]));
        } else {
            __builtin_amdgcn_s_sleep(1);
        }
    }
    publish(hs(s), lane * 4, bits_of(fmaf(A, H, B)));
}

// The tiles of a block, all of one sequence and channel group.  In a split call several blocks share them, each
// taking the tiles that its tickets name: a ticket is handed round at a barrier of the tile before, and the next one
// fetched from there on, while that tile is worked on.  (One counter for all of them took 15 ns a tile: atomics on one
// address wait for each other.)
template <bool SPLIT>
struct Tiles {
    unsigned *ticket, *sh, next = 0;  // sh: two, in turn, as a wave may still read one when the next is handed round
    int turn = 0;
    VKH_DEV void fetch() {
        if (SPLIT && threadIdx.x == 0) next = atomicAdd(ticket, 1u);
    }
    VKH_DEV void hand_round() {  // ahead of a barrier
        if (SPLIT && threadIdx.x == 0) sh[turn] = next;
    }
    VKH_DEV int take(int now) {  // behind it
        if (!SPLIT) return now + 1;
        const int t = __builtin_amdgcn_readfirstlane(sh[turn]);
        turn ^= 1;
        fetch();
        return t;
    }
    VKH_DEV int first() {
        if (!SPLIT) return 0;
        fetch();
        hand_round();
        __syncthreads();
        return take(0);
    }
};

// Both kernels: a tile's values are asked for as soon as the one before is in use, by the wave that looks back once it
// has (a wave's loads return in order), so they arrive while that tile is joined and stored.  (Backward of 16384 x 4096
// bf16: 208 us without, 185 with; the forward 113 and 111.)
//
// 16384 x 4096 bf16 (0.40 and 0.67 GB): forward 105 us, 3.8 TB/s, backward 179, 3.75, and 5 or 6 each for the launch that
// makes the words ready; fp32, 8192 rows (the same bytes): 84 and 128, 4.8 and 5.2, and the same launch (with it, back to
// back: 110 and 185, 90 and 137).  bf16 has twice the values of its bytes and reaches neither HBM's rate nor that of the
// vector instructions (26 and 46 for each value, 40 % of the cycles): all waves of a block wait while one looks back, a
// third of a tile's time, and a CU has one other block to go on with in the forward and none in the backward.  16 sequences of
// 1024 rows, a block each: 90 and 162.
template <class TI, class TO, bool SIG, bool COUP, bool SPLIT>
__global__ __launch_bounds__(kFwdWaves * 64, kPerSimd) void scan_fwd_k(ScanArgs s, int groups) {
    constexpr int R = kFwdRows;
    __shared__ float shA[2][kFwdWaves][64], shB[2][kFwdWaves][64], shH[64];
    __shared__ unsigned ticket[2];
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles = (s.n_pos + kFwdTile - 1) / kFwdTile;
    const long blk = SPLIT ? blockIdx.x % (groups * s.n_batch) : block_number<kFwdWaves * 64>();
    if (blk >= groups * s.n_batch) return;
    const int line = __builtin_amdgcn_readfirstlane((int)blk), b = __builtin_amdgcn_readfirstlane(line / groups);
    const int c = (line - b * groups) * 64 + lane, len = __builtin_amdgcn_readfirstlane(rows_of(s, b));
    const bool act = c < s.dim;
    const unsigned in_bytes = min(c, s.dim - 1) * sizeof(TI);  // (lanes past the channels: the last one)
    const Words W = words_of(s.ws, (size_t)s.n_batch * groups, (size_t)s.n_batch * groups * tiles * 64);
    Tiles<SPLIT> order{(unsigned *)(W.tickets + (size_t)line * kTicketBytes), ticket};
    TI xr[R], gr[R];
    // FULL: all rows of the wave are in the sequence; else rows behind its end are the last one again
    auto load = [&](int t0, auto full) {
        constexpr bool FULL = decltype(full)::value;
        const long row0 = (long)b * s.n_pos + t0;
        Walk<TI> g(s.g, row0, s.ldg), x(s.x, row0, s.ldx);
        unsigned at = in_bytes;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            at = here(at);
            gr[i] = g.load(at);
            xr[i] = x.load(at);
            g.next(FULL || t0 + i + 1 < len);
            x.next(FULL || t0 + i + 1 < len);
        }
    };
    auto store = [&](int t0, float h, const float (&a)[R], const float (&u)[R], auto full) {
        constexpr bool FULL = decltype(full)::value;
        Walk<TO> out(s.h, (long)b * s.n_pos + t0, s.ldh);
        unsigned at = c * sizeof(TO);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            h = fmaf(a[i], h, u[i]);
            at = here(at);
            if (FULL || t0 + i < s.n_pos) out.store(at, FULL || t0 + i < len ? h : 0.f);
            out.next();
        }
    };
    float H = 0.f;
    int at = order.first();
    if (at >= tiles) return;
    auto ask = [&](int tile) {
        const int t0 = tile * kFwdTile + w * R;
        if (t0 + R <= len) load(t0, std::true_type{});
        else if (t0 < len) load(t0, std::false_type{});
    };
    ask(at);
    for (int turn = 0;; turn ^= 1) {
        const int k = at, t0 = k * kFwdTile + w * R;
        const bool full = t0 + R <= len;
        if (k == 0) {
            H = act && s.h0 ? s.h0[(long)b * s.dim + c] : 0.f;
            asm volatile("" : "+v"(H));  // (it has been read when the block meets at its barrier: h_last may be h0)
        }
        float a[R], u[R], p = 1.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float rest;
            gate<SIG>(gr[i], a[i], rest);
            u[i] = COUP ? rest * (float)xr[i] : (float)xr[i];
        }
        if (!full) {  // rows behind the end leave the state alone
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (t0 + i >= len) a[i] = 1.f, u[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            p *= a[i];
            q = fmaf(a[i], q, u[i]);
        }
        float (&A)[kFwdWaves][64] = shA[turn], (&B)[kFwdWaves][64] = shB[turn];
        A[w][lane] = p;
        B[w][lane] = q;
        order.hand_round();
        __syncthreads();
        const int then = order.take(at);
        const bool more = then < tiles;
        if (more && (!SPLIT || w)) ask(then);
        // of the waves before this one, and of the tile
        float pa = 1.f, pb = 0.f, ta = 1.f, tb = 0.f;
#pragma unroll kFold
        for (int j = 0; j < kFwdWaves; ++j) {
            if (j == w) pa = ta, pb = tb;
            ta *= A[j][lane];
            tb = fmaf(A[j][lane], tb, B[j][lane]);
        }
        if (SPLIT) {
            if (w == 0) {
                __builtin_amdgcn_s_setprio(3);  // (others wait for it: 1 % of a long scan)
                look_back(W, (size_t)line * tiles * 64, at, lane, ta, tb, H);
                __builtin_amdgcn_s_setprio(0);
                shH[lane] = H;
            }
            __syncthreads();
            H = shH[lane];
            if (more && !w) ask(then);
        }
        float h = fmaf(pa, H, pb);
        H = fmaf(ta, H, tb);
        if (act) {
            if (s.states && w == 0) s.states[((long)b * tiles + k) * s.dim + c] = h;
            if (full) store(t0, h, a, u, std::true_type{});
            else store(t0, h, a, u, std::false_type{});
            if (k + 1 == tiles && s.h_last && w == 0) s.h_last[(long)b * s.dim + c] = H;
        }
        if (!more) return;
        at = then;
    }
}

template <class TI, class TO, bool SIG, bool COUP, bool SPLIT>
__global__ __launch_bounds__(kBwdWaves * 64, kPerSimd) void scan_bwd_k(ScanArgs s, int groups) {
    constexpr int N = kBwdRows;
    __shared__ float shA[2][kBwdWaves][64], shB[2][kBwdWaves][64], shQ[2][kBwdWaves][64], shR[64];
    __shared__ unsigned ticket[2];
    const int lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int tiles = (s.n_pos + kBwdTile - 1) / kBwdTile;
    const long blk = SPLIT ? blockIdx.x % (groups * s.n_batch) : block_number<kBwdWaves * 64>();
    if (blk >= groups * s.n_batch) return;
    const int line = __builtin_amdgcn_readfirstlane((int)blk), b = __builtin_amdgcn_readfirstlane(line / groups);
    const int c = (line - b * groups) * 64 + lane, len = __builtin_amdgcn_readfirstlane(rows_of(s, b));
    const bool act = c < s.dim;
    const unsigned in_bytes = min(c, s.dim - 1) * sizeof(TI);  // (lanes past the channels: the last one)
    const Words W = words_of(s.ws, (size_t)s.n_batch * groups, (size_t)s.n_batch * groups * tiles * 64);
    Tiles<SPLIT> order{(unsigned *)(W.tickets + (size_t)line * kTicketBytes), ticket};
    TI xr[N], gr[N], dr[N];
    // (FULL: as in the forward)
    auto load = [&](int t0, auto full) {
        constexpr bool FULL = decltype(full)::value;
        const long row0 = (long)b * s.n_pos + t0;
        Walk<TI> g(s.g, row0, s.ldg), d(s.dh, row0, s.lddh), x(s.x, row0, s.ldx);
        unsigned at = in_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            at = here(at);
            gr[i] = g.load(at);
            dr[i] = d.load(at);
            xr[i] = x.load(at);
            g.next(FULL || t0 + i + 1 < len);
            d.next(FULL || t0 + i + 1 < len);
            x.next(FULL || t0 + i + 1 < len);
        }
    };
    float R = 0.f;
    int at = order.first();
    if (at >= tiles) return;
    auto ask = [&](int tile) {
        const int t0 = (tiles - 1 - tile) * kBwdTile + w * N;
        if (t0 + N <= len) load(t0, std::true_type{});
        else if (t0 < len) load(t0, std::false_type{});
    };
    ask(at);
    for (int turn = 0;; turn ^= 1) {
        const int k = tiles - 1 - at, t0 = k * kBwdTile + w * N;
        const bool full = t0 + N <= len;
        // the state before the tile (one behind the sequence's end has none, and needs none)
        float h = act && k * kBwdTile < len ? s.states[((long)b * tiles + k) * s.dim + c] : 0.f;
        if (at == 0) {
            R = act && s.dh_last ? s.dh_last[(long)b * s.dim + c] : 0.f;
            asm volatile("" : "+v"(R));  // (as in the forward: dh0 may be dh_last)
        }
        float a[N], rest[N], x[N], d[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            gate<SIG>(gr[i], a[i], rest[i]);
            x[i] = (float)xr[i];
            d[i] = (float)dr[i];
        }
        if (!full) {  // rows behind the end leave state and gradient alone
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (t0 + i >= len) a[i] = 1.f, rest[i] = x[i] = d[i] = 0.f;
        }
        auto u = [&](int i) { return COUP ? rest[i] * x[i] : x[i]; };
        float p = 1.f, q = 0.f, z = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p *= a[i];
            q = fmaf(a[i], q, u(i));
        }
#pragma unroll
        for (int i = N - 1; i >= 0; --i) z = a[i] * (d[i] + z);
        float (&A)[kBwdWaves][64] = shA[turn], (&B)[kBwdWaves][64] = shB[turn], (&Q)[kBwdWaves][64] = shQ[turn];
        A[w][lane] = p;
        B[w][lane] = q;
        Q[w][lane] = z;
        order.hand_round();
        __syncthreads();
        const int then = order.take(at);
        const bool more = then < tiles;
        if (more && (!SPLIT || w)) ask(then);
        // of the waves behind this one, and of the tile; and the state before this wave's rows
        float pa = 1.f, pb = 0.f, ta = 1.f, tb = 0.f;
#pragma unroll kFold
        for (int j = kBwdWaves - 1; j >= 0; --j) {
            if (j == w) pa = ta, pb = tb;
            ta *= A[j][lane];
            tb = fmaf(A[j][lane], tb, Q[j][lane]);
        }
#pragma unroll kFold
        for (int j = 0; j < kBwdWaves; ++j)
            if (j < w) h = fmaf(A[j][lane], h, B[j][lane]);
        if (SPLIT) {
            if (w == 0) {
                __builtin_amdgcn_s_setprio(3);
                look_back(W, (size_t)line * tiles * 64, at, lane, ta, tb, R);
                __builtin_amdgcn_s_setprio(0);
                shR[lane] = R;
            }
            __syncthreads();
            R = shR[lane];
            if (more && !w) ask(then);
        }
        float hp[N], e = fmaf(pa, R, pb);
        R = fmaf(ta, R, tb);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            hp[i] = h;
            h = fmaf(a[i], h, u(i));
        }
        if (act) {
            auto store = [&](auto full) {
                constexpr bool FULL = decltype(full)::value;
                const long row = (long)b * s.n_pos + t0 + N - 1;
                Walk<TO> ox(s.dx, row, s.lddx), og(s.dg, row, s.lddg);
                unsigned at = c * sizeof(TO);
#pragma unroll
                for (int i = N - 1; i >= 0; --i) {
                    const float G = d[i] + e;
                    e = a[i] * G;
                    float dx = COUP ? rest[i] * G : G, dg = COUP ? G * (hp[i] - x[i]) : G * hp[i];
                    if (SIG) dg *= a[i] * rest[i];
                    at = here(at);
                    if (FULL || t0 + i < s.n_pos) {
                        ox.store(at, FULL || t0 + i < len ? dx : 0.f);
                        og.store(at, FULL || t0 + i < len ? dg : 0.f);
                    }
                    ox.back();
                    og.back();
                }
            };
            if (full) store(std::true_type{});
            else store(std::false_type{});
            if (k == 0 && s.dh0 && w == 0) s.dh0[(long)b * s.dim + c] = R;
        }
        if (!more) return;
        at = then;
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
        float x[V], o[V] = {};
        if (t < len) {
            const Raw<TI, V> g = load_raw<TI, V>((const TI *)s.g + (row0 + t) * s.ldg + c);
            load_v<TI, V>((const TI *)s.x + (row0 + t) * s.ldx + c, x);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                if constexpr (V == 1) gate<SIG>(g, a, rest);
                else gate<SIG>((TI)g[v], a, rest);
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
        gate<SIG>(((const TI *)s.g)[(row0 + t) * s.ldg + c], a[t], rest[t]);
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

// How a call is laid out: channel groups, and the blocks that share the tiles of each sequence and group (0: one has
// them all).
struct Plan {
    int groups, sharing;
    size_t lines, channels;  // sequences times groups; a split call's words' channels
};
Plan plan_of(const ScanArgs &s, bool back) {
    Plan p;
    p.groups = (int)ceil_div(s.dim, 64);
    p.lines = (size_t)p.groups * s.n_batch;
    const int tile = back ? kBwdTile : kFwdTile;
    const size_t tiles = (s.n_pos + tile - 1) / tile, resident = (size_t)cu_count() * (kPerSimd * 4 / (back ? kBwdWaves : kFwdWaves));
    p.channels = p.lines * tiles * 64;
    // The same number of blocks for every line: what is left of the resident ones has no work, and lines past half of them
    // are a block's each.  4 x 4096 x 2560 bf16, of 160 lines, 72 and 160 us (3.5 and 2.6 TB/s), 5 x 4096 x 4096, of 320 lines and
    // more than one round of blocks, 160 and 291 (3.1 and 2.9); of 256 lines, 4 x 4096 x 4096, 102 and 162 (4.0 and 4.1).
    p.sharing = (int)std::min(tiles, resident / p.lines);
    // Two tiles (forward: three) one after the other cost less than the launch that makes the words ready: 200 x 1024
    // bf16, forward and backward, 8.3 and 8.8 us in one block a line, 10.6 and 10.4 shared; 512 x 1024 mixed, of four tiles,
    // 11.6 and 17.8, shared 10.2 and 11.7.
    if (s.n_pos <= kFew || p.sharing < 2 || tiles < (back ? 3 : 4) || p.channels > kMostChannels) p.sharing = 0;
    return p;
}
size_t words_bytes(const Plan &p) { return p.sharing ? p.lines * kTicketBytes + (p.channels * 12 + 15) / 16 * 16 : 0; }

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
Plan ready(const ScanArgs &s, bool back, hipStream_t st) {
    Plan p = plan_of(s, back);
    if (!s.ws) p.sharing = 0;
    const size_t n = words_bytes(p) / 16;
    if (n)
        hipLaunchKernelGGL(scan_clear_k, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1024)), dim3(256), 0, st, (uint4 *)s.ws,
                           p.lines * kTicketBytes / 16, n);
    return p;
}
dim3 grid_of(const Plan &p, int threads) { return p.sharing ? dim3((unsigned)p.lines * p.sharing) : long_grid((long)p.lines, threads); }

}  // namespace

size_t scan_states_floats(const ScanArgs &s) {
    return (size_t)s.n_batch * ((s.n_pos + kScanTile - 1) / kScanTile) * s.dim;
}
size_t scan_ws_bytes(const ScanArgs &s) {
    return std::max(words_bytes(plan_of(s, false)), words_bytes(plan_of(s, true)));
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
        const Plan p = ready(s, false, st);
        auto k = p.sharing ? scan_fwd_k<TI, TO, SIG, COUP, true> : scan_fwd_k<TI, TO, SIG, COUP, false>;
        hipLaunchKernelGGL(k, grid_of(p, kFwdWaves * 64), dim3(kFwdWaves * 64), 0, st, s, p.groups);
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
        const Plan p = ready(s, true, st);
        auto k = p.sharing ? scan_bwd_k<TI, TO, SIG, COUP, true> : scan_bwd_k<TI, TO, SIG, COUP, false>;
        hipLaunchKernelGGL(k, grid_of(p, kBwdWaves * 64), dim3(kBwdWaves * 64), 0, st, s, p.groups);
    });
    return hipGetLastError();
}

}  // namespace vkh
