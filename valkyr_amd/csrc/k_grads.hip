// The norm of a list of gradients, and the gradients scaled down to a largest norm.
//
//   norm = sqrt(sum of g^2),  c = max_norm / norm where norm > max_norm and norm is finite, else 1,  out = c g
//
// Squares are formed and summed in 64 bits: gradients near either end of fp32 neither overflow nor vanish, and
// long sums lose nothing.  Two passes: the squares, one partial sum a block; then every block adds the partial
// sums (in their order) and scales its part.  Which values a block takes follows from the sizes of the list's tensors
// alone, wherever they and their outputs lie, so results do not change from run to run.
#include <algorithm>
#include <type_traits>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int GNT = 256;
constexpr int kChunk = 8192;    // values: a block's unit of work, of one tensor
constexpr int kParts = 2048;    // partial sums of all sections, but for one more a section
// Tensors whose chunks are shared by blocks of their own: a launch takes two or three whole sections, as its table holds
// by where the tensors lie, and the partial sums are the same in either case.
constexpr int kSection = 90;

// The tensors of one launch, an argument of the kernel.  Tensor i takes chunks first[i] .. first[i + 1], the last of them
// of (tail & 0x7fff) + 1 values; section s has the blocks from block[s] on.  NEAR: addresses are 32-bit numbers of 2-byte
// units past the lowest one, so that a launch holds more tensors (224 adapters in one launch a pass in place of two: 16
// us, not 24); for gradients, and outputs, within 8 GiB of each other.
template <bool NEAR>
struct Table {
    static constexpr bool near = NEAR;
    static constexpr int sections = NEAR ? 3 : 2, most = sections * kSection;
    typedef std::conditional_t<NEAR, unsigned, uintptr_t> At;
    int n;
    unsigned block[sections];
    uintptr_t g0, out0;
    At g[most], out[most];
    unsigned first[most + 1];
    uint16_t tail[most];  // bit 15: bf16
    VKH_DEV const void *grad(int i) const { return (const void *)(g0 + (NEAR ? 2ull : 1ull) * g[i]); }
    VKH_DEV void *dest(int i) const { return (void *)(out0 + (NEAR ? 2ull : 1ull) * out[i]); }
};
static_assert(sizeof(Table<true>) + 64 <= 4096 && sizeof(Table<false>) + 64 <= 4096, "kernel arguments");

// The chunks of this block: an equal share of its section's, one after the other.
struct Share {
    unsigned c, end;
    int t;
};
template <bool NEAR>
VKH_DEV Share share(const Table<NEAR> &T) {
    int s0 = 0;
    unsigned b0 = 0, b1 = gridDim.x;
#pragma unroll
    for (int i = 1; i < Table<NEAR>::sections; ++i) {  // (a section that the launch does not have: block[i] = gridDim.x)
        if (blockIdx.x >= T.block[i]) s0 = i, b0 = T.block[i];
        else b1 = min(b1, T.block[i]);
    }
    const int t0 = s0 * kSection, t1 = min(t0 + kSection, T.n);
    const unsigned c0 = T.first[t0], chunks = T.first[t1] - c0, blocks = b1 - b0;
    const unsigned per = chunks / blocks, more = chunks % blocks, b = blockIdx.x - b0;
    Share s;
    s.c = c0 + b * per + (b < more ? b : more);
    s.end = s.c + per + (b < more ? 1 : 0);
    int lo = t0, hi = t1 - 1;  // the last tensor that starts at or before c
    while (lo < hi) {
        const int m = (lo + hi + 1) / 2;
        if (T.first[m] <= s.c) lo = m;
        else hi = m - 1;
    }
    s.t = lo;
    return s;
}

VKH_DEV double block_sum64(double v, double *sh) {
    v = wave_sum(v);
    if (threadIdx.x % 64 == 0) sh[threadIdx.x / 64] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < GNT / 64; ++i) t += sh[i];
    return t;
}

// 16 bytes of a tensor, which may start at any of its values: two neighbouring lines at most take a lane's load, and
// the lanes of a wave whole lines but for the first and last.
template <class T>
using Bytes16 = typename Vec<T, 16 / (int)sizeof(T)>::type;

// f(vector of U at i) over the chunk's n values, 16 bytes a lane and 32 KiB under way, and f1(value) behind the last
// whole vector.
template <bool PAST, class T, class F, class F1>
VKH_DEV void over_chunk(const T *g, int n, F f, F1 f1) {
    typedef Bytes16<T> V;
    constexpr int W = 16 / sizeof(T), U = kChunk / W / GNT;
    if (n == kChunk) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const V *p = reinterpret_cast<const V *>(g + (u * GNT + threadIdx.x) * W);
            v[u] = PAST ? __builtin_nontemporal_load(p) : *p;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) f((u * GNT + threadIdx.x) * W, v[u]);
        return;
    }
    for (int i = threadIdx.x * W; i + W <= n; i += GNT * W) f(i, *reinterpret_cast<const V *>(g + i));
    const int i = n / W * W + threadIdx.x;
    if (i < n) f1(i, g[i]);
}

// The chunk c of tensor t: its values from `at` on, and how many.
template <bool NEAR>
VKH_DEV size_t chunk_at(const Table<NEAR> &T, int t, unsigned c, int &n) {
    n = c + 1 == T.first[t + 1] ? (T.tail[t] & 0x7fff) + 1 : kChunk;
    return (size_t)(c - T.first[t]) * kChunk;
}

template <bool PAST, class T>
VKH_DEV void squares_of(const T *g, int n, double (&s)[4]) {
    constexpr int W = 16 / sizeof(T);
    over_chunk<PAST>(
        g, n,
        [&](int, Bytes16<T> v) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const double d = (float)v[i];
                s[i % 4] = fma(d, d, s[i % 4]);
            }
        },
        [&](int, T v) {
            const double d = (float)v;
            s[0] = fma(d, d, s[0]);
        });
}

template <bool NEAR, bool PAST>
__global__ __launch_bounds__(GNT) void grad_squares_k(Table<NEAR> T, double *part) {
    __shared__ double sh[GNT / 64];
    double s[4] = {};
    Share w = share(T);
    for (; w.c < w.end; ++w.c) {
        while (w.c >= T.first[w.t + 1]) ++w.t;
        int n;
        const size_t at = chunk_at(T, w.t, w.c, n);
        if (T.tail[w.t] >> 15) squares_of<PAST>((const bf16 *)T.grad(w.t) + at, n, s);
        else squares_of<PAST>((const float *)T.grad(w.t) + at, n, s);
    }
    const double sum = block_sum64((s[0] + s[1]) + (s[2] + s[3]), sh);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

VKH_DEV double norm_of(const double *part, int n_part, double *sh) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_part; i += GNT) s += part[i];
    return sqrt(block_sum64(s, sh));
}

__global__ __launch_bounds__(GNT) void grad_norm_k(const double *part, int n_part, float *norm) {
    __shared__ double sh[GNT / 64];
    const double n = norm_of(part, n_part, sh);
    if (threadIdx.x == 0) norm[0] = (float)n;
}

// (scaled = false: the bits as they are)
template <bool PAST, class T>
VKH_DEV void scale_of(const T *g, T *out, int n, bool scaled, double c) {
    typedef Bytes16<T> V;
    auto one = [&](T v) { return scaled ? (T)(float)((double)(float)v * c) : v; };
    over_chunk<PAST>(
        g, n,
        [&](int i, V v) {
#pragma unroll
            for (int k = 0; k < (int)(16 / sizeof(T)); ++k) v[k] = one(v[k]);
            __builtin_nontemporal_store(v, reinterpret_cast<V *>(out + i));
        },
        [&](int i, T v) { out[i] = one(v); });
}

template <bool NEAR, bool PAST>
__global__ __launch_bounds__(GNT) void grad_scale_k(Table<NEAR> T, const double *part, int n_part, float max_norm, float *norm) {
    __shared__ double sh[GNT / 64];
    const double n = norm_of(part, n_part, sh);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
    const bool scaled = n > (double)max_norm && n <= 1.7976931348623157e308;
    const double c = scaled ? (double)max_norm / n : 1.0;
    Share w = share(T);
    for (; w.c < w.end; ++w.c) {
        while (w.c >= T.first[w.t + 1]) ++w.t;
        if (!scaled && T.grad(w.t) == T.dest(w.t)) continue;
        int n;
        const size_t at = chunk_at(T, w.t, w.c, n);
        if (T.tail[w.t] >> 15) scale_of<PAST>((const bf16 *)T.grad(w.t) + at, (bf16 *)T.dest(w.t) + at, n, scaled, c);
        else scale_of<PAST>((const float *)T.grad(w.t) + at, (float *)T.dest(w.t) + at, n, scaled, c);
    }
}

unsigned chunks_of(const GradTensor &t) { return (unsigned)((t.n + kChunk - 1) / kChunk); }

}  // namespace

size_t grad_ws_bytes(size_t n) { return (kParts + n / kSection + 1) * sizeof(double); }

hipError_t grad_clip(const GradTensor *t, size_t n, bool clip, float max_norm, float *norm, void *ws, hipStream_t st) {
    double *part = (double *)ws;
    size_t total = 0, bytes = 0;
    for (size_t i = 0; i < n; ++i) total += chunks_of(t[i]), bytes += t[i].n * (t[i].dt == DType::F32 ? 4 : 2);
    // More than the chip's last cache holds of it from one pass to the next goes past the caches (2.4 GB: 1422 us through
    // them, 1366 past them; 128 MB: 68 and 77).  Results always do (2.4 GB: 1448 through them; 128 MB: 86).
    const bool past = bytes > (256ull << 20);
    if (!total) return norm ? fill_f32(norm, 1, 0.f, st) : hipSuccess;
    // f(table, blocks) for each launch of whole sections, each with its share of kParts blocks, at most one a chunk
    auto each = [&](auto f) {
        for (size_t i = 0; i < n;) {
            // how many of the next tensors are near each other, in whole sections
            uintptr_t g0 = (uintptr_t)t[i].g, g1 = g0, o0 = (uintptr_t)t[i].out, o1 = o0;
            size_t near = i;
            for (; near < n && near - i < (size_t)Table<true>::most; ++near) {
                const uintptr_t g = (uintptr_t)t[near].g, o = (uintptr_t)t[near].out;
                const uintptr_t a0 = std::min(g0, g), a1 = std::max(g1, g), b0 = std::min(o0, o), b1 = std::max(o1, o);
                if ((a1 - a0) >> 33 || (b1 - b0) >> 33) break;
                g0 = a0, g1 = a1, o0 = b0, o1 = b1;
            }
            auto go = [&](auto T, size_t end, uintptr_t gb, uintptr_t ob, unsigned unit) {
                T.n = (int)(end - i);
                T.g0 = gb;
                T.out0 = ob;
                unsigned c = 0, blocks = 0;
                for (int s = 0; s < decltype(T)::sections; ++s) {
                    T.block[s] = blocks;
                    const unsigned c0 = c;
                    for (int k = s * kSection; k < (s + 1) * kSection && i < end; ++i, ++k) {
                        T.first[k] = c;
                        T.tail[k] = (uint16_t)((t[i].n - 1) % kChunk | (t[i].dt == DType::BF16 ? 0x8000 : 0));
                        T.g[k] = (typename decltype(T)::At)(((uintptr_t)t[i].g - gb) / unit);
                        T.out[k] = (typename decltype(T)::At)(((uintptr_t)t[i].out - ob) / unit);
                        c += chunks_of(t[i]);
                    }
                    if (c > c0) blocks += (unsigned)std::min<size_t>(c - c0, (size_t)kParts * (c - c0) / total + 1);
                }
                T.first[T.n] = c;
                f(T, (int)blocks);
            };
            const size_t far = std::min(n, i + Table<false>::most);
            if (near < n) near -= (near - i) % kSection;
            if (near >= far) go(Table<true>(), near, g0, o0, 2);
            else go(Table<false>(), far, 0, 0, 1);
        }
    };
    int parts = 0;
    each([&](const auto &T, int blocks) {
        constexpr bool NEAR = std::decay_t<decltype(T)>::near;
        auto k = past ? grad_squares_k<NEAR, true> : grad_squares_k<NEAR, false>;
        hipLaunchKernelGGL(k, dim3(blocks), dim3(GNT), 0, st, T, part + parts);
        parts += blocks;
    });
    if (!clip) {
        hipLaunchKernelGGL(grad_norm_k, dim3(1), dim3(GNT), 0, st, part, parts, norm);
        return hipGetLastError();
    }
    bool first = true;
    each([&](const auto &T, int blocks) {
        constexpr bool NEAR = std::decay_t<decltype(T)>::near;
        auto k = past ? grad_scale_k<NEAR, true> : grad_scale_k<NEAR, false>;
        hipLaunchKernelGGL(k, dim3(blocks), dim3(GNT), 0, st, T, part, parts, max_norm, first ? norm : nullptr);
        first = false;
    });
    return hipGetLastError();
}

}  // namespace vkh
