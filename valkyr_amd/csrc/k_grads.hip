// The norm of a list of gradients, and the gradients scaled down to a largest norm.
//
//   norm = sqrt(sum of g^2),  c = max_norm / norm where norm > max_norm and norm is finite, else 1,  out = c g
//
// Squares are formed and summed in 64 bits: gradients near either end of fp32 neither overflow nor vanish, and
// long sums lose nothing.  Two passes: the squares, one partial sum a block; then every block adds the partial
// sums (in their order) and scales its part.  Which values a block takes follows from the sizes alone, so results
// do not change from run to run.
#include <algorithm>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int GNT = 256;
constexpr int kChunk = 4096;    // values: a block's unit of work, of one tensor
constexpr int kTensors = 112;   // of one launch: its table is an argument of the kernel
constexpr int kParts = 2048;    // partial sums of all launches, but for one more a launch

// Tensor i takes chunks first[i] .. first[i + 1].
struct Table {
    int n;
    unsigned chunks;
    unsigned first[kTensors + 1];
    uint8_t bf16s[kTensors];
    const void *g[kTensors];
    void *out[kTensors];
    size_t len[kTensors];
};
static_assert(sizeof(Table) + 64 < 4096, "kernel arguments");

// The chunks of this block: an equal share, one after the other.
struct Share {
    unsigned c, end;
    int t;
};
VKH_DEV Share share(const Table &T) {
    const unsigned per = T.chunks / gridDim.x, more = T.chunks % gridDim.x, b = blockIdx.x;
    Share s;
    s.c = b * per + (b < more ? b : more);
    s.end = s.c + per + (b < more ? 1 : 0);
    int lo = 0, hi = T.n - 1;  // the last tensor that starts at or before c
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

__global__ __launch_bounds__(GNT) void grad_squares_k(Table T, double *part) {
    __shared__ double sh[GNT / 64];
    double s = 0.0;
    Share w = share(T);
    for (; w.c < w.end; ++w.c) {
        while (w.c >= T.first[w.t + 1]) ++w.t;
        const size_t at = (size_t)(w.c - T.first[w.t]) * kChunk;
        const size_t n = T.len[w.t] - at < kChunk ? T.len[w.t] - at : kChunk;
        for (size_t i = threadIdx.x; i < n; i += GNT) {
            const double v = T.bf16s[w.t] ? (float)((const bf16 *)T.g[w.t])[at + i] : ((const float *)T.g[w.t])[at + i];
            s = fma(v, v, s);
        }
    }
    s = block_sum64(s, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
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

__global__ __launch_bounds__(GNT) void grad_scale_k(Table T, const double *part, int n_part, float max_norm, float *norm) {
    __shared__ double sh[GNT / 64];
    const double n = norm_of(part, n_part, sh);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n;
    const bool scaled = n > (double)max_norm && n <= 1.7976931348623157e308;
    const double c = scaled ? (double)max_norm / n : 1.0;
    Share w = share(T);
    for (; w.c < w.end; ++w.c) {
        while (w.c >= T.first[w.t + 1]) ++w.t;
        if (!scaled && T.g[w.t] == T.out[w.t]) continue;
        const size_t at = (size_t)(w.c - T.first[w.t]) * kChunk;
        const size_t n = T.len[w.t] - at < kChunk ? T.len[w.t] - at : kChunk;
        for (size_t i = threadIdx.x; i < n; i += GNT) {
            if (T.bf16s[w.t]) {
                const bf16 v = ((const bf16 *)T.g[w.t])[at + i];
                ((bf16 *)T.out[w.t])[at + i] = scaled ? (bf16)(float)((double)(float)v * c) : v;
            } else {
                const float v = ((const float *)T.g[w.t])[at + i];
                ((float *)T.out[w.t])[at + i] = scaled ? (float)((double)v * c) : v;
            }
        }
    }
}

unsigned chunks_of(const GradTensor &t) { return (unsigned)((t.n + kChunk - 1) / kChunk); }

}  // namespace

size_t grad_ws_bytes(size_t n) { return (kParts + (n + kTensors - 1) / kTensors) * sizeof(double); }

hipError_t grad_clip(const GradTensor *t, size_t n, bool clip, float max_norm, float *norm, void *ws, hipStream_t st) {
    double *part = (double *)ws;
    size_t total = 0;
    for (size_t i = 0; i < n; ++i) total += chunks_of(t[i]);
    if (!total) return norm ? fill_f32(norm, 1, 0.f, st) : hipSuccess;
    // each launch's blocks: its share of kParts, at most one a chunk
    auto each = [&](auto f) {
        for (size_t i = 0; i < n;) {
            Table T;
            T.n = 0;
            T.chunks = 0;
            for (; i < n && T.n < kTensors; ++i) {
                if (!t[i].n) continue;
                T.first[T.n] = T.chunks;
                T.bf16s[T.n] = t[i].dt == DType::BF16;
                T.g[T.n] = t[i].g;
                T.out[T.n] = t[i].out;
                T.len[T.n++] = t[i].n;
                T.chunks += chunks_of(t[i]);
            }
            if (!T.n) break;
            T.first[T.n] = T.chunks;
            f(T, (int)std::min<size_t>(T.chunks, (size_t)kParts * T.chunks / total + 1));
        }
    };
    int parts = 0;
    each([&](const Table &T, int blocks) {
        hipLaunchKernelGGL(grad_squares_k, dim3(blocks), dim3(GNT), 0, st, T, part + parts);
        parts += blocks;
    });
    if (!clip) {
        hipLaunchKernelGGL(grad_norm_k, dim3(1), dim3(GNT), 0, st, part, parts, norm);
        return hipGetLastError();
    }
    bool first = true;
    each([&](const Table &T, int blocks) {
        hipLaunchKernelGGL(grad_scale_k, dim3(blocks), dim3(GNT), 0, st, T, part, parts, max_norm, first ? norm : nullptr);
        first = false;
    });
    return hipGetLastError();
}

}  // namespace vkh
