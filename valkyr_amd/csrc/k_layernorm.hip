// Layer norm of rows, forward and backward.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), xh = (x - mu) r
//   forward   y = xh w + b
//   backward  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)) (+ residual)
//             dw = sum over rows of dy xh,  db = sum over rows of dy
//
// The variance is that of the centred values (a row far from 0 keeps its digits), statistics and sums
// are fp32, and the backward forms the statistics again from x, which it reads anyway.
#include "ops.hpp"

namespace vkh {
namespace {

constexpr int LNT = 256;
constexpr int kBlocks = 512;  // of the backward: rows of partial gain gradients

template <class F>
void by_type(DType d, F f) {
    if (d == DType::F32) f(float{});
    else f(bf16{});
}

// A block per row, which reads it once for the mean, once for the variance and once more.
template <class T>
VKH_DEV void row_stats(const T *x, int dim, float eps, float *sh, float &mu, float &r) {
    float s = 0.f;
    for (int i = threadIdx.x; i < dim; i += LNT) s += to_f32(x[i]);
    mu = block_sum<LNT>(s, sh) / (float)dim;
    float q = 0.f;
    for (int i = threadIdx.x; i < dim; i += LNT) {
        const float c = to_f32(x[i]) - mu;
        q = fmaf(c, c, q);
    }
    r = 1.0f / sqrtf(block_sum<LNT>(q, sh) / (float)dim + eps);
}

template <class TX, class TY>
__global__ __launch_bounds__(LNT) void layernorm_fwd_k(LayernormArgs a) {
    __shared__ float sh[LNT / 64];
    const long row = block_number();
    if (row >= a.n_rows) return;
    const TX *x = (const TX *)a.x + row * a.ldx;
    TY *y = (TY *)a.y + row * a.ldy;
    float mu, r;
    row_stats(x, a.dim, a.eps, sh, mu, r);
    for (int i = threadIdx.x; i < a.dim; i += LNT)
        y[i] = (TY)((to_f32(x[i]) - mu) * r * (a.w ? a.w[i] : 1.f) + (a.b ? a.b[i] : 0.f));
}

// Block b takes rows b, b + gridDim.x, ..; its sums for dw and db are its row of `partial` ([blocks][2][dim]).
template <class TX, class TG, class TD>
__global__ __launch_bounds__(LNT) void layernorm_bwd_k(LayernormArgs a) {
    __shared__ float sh[LNT / 64];
    const int dim = a.dim;
    float *pw = a.partial ? a.partial + (long)blockIdx.x * 2 * dim : nullptr, *pb = pw ? pw + dim : nullptr;
    if (pw)
        for (int i = threadIdx.x; i < 2 * dim; i += LNT) pw[i] = 0.f;
    for (long row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
        const TX *x = (const TX *)a.x + row * a.ldx;
        const TG *dy = (const TG *)a.dy + row * a.lddy;
        TD *dx = (TD *)a.dx + row * a.lddx;
        const TD *res = a.res ? (const TD *)a.res + row * a.lddx : nullptr;
        float mu, r, s = 0.f, q = 0.f;
        row_stats(x, dim, a.eps, sh, mu, r);
        for (int i = threadIdx.x; i < dim; i += LNT) {
            const float d = to_f32(dy[i]), xh = (to_f32(x[i]) - mu) * r, g = d * (a.w ? a.w[i] : 1.f);
            s += g;
            q = fmaf(g, xh, q);
            if (pw) {
                pw[i] = fmaf(d, xh, pw[i]);
                pb[i] += d;
            }
        }
        s = block_sum<LNT>(s, sh) / (float)dim;
        q = block_sum<LNT>(q, sh) / (float)dim;
        for (int i = threadIdx.x; i < dim; i += LNT) {
            const float xh = (to_f32(x[i]) - mu) * r, g = to_f32(dy[i]) * (a.w ? a.w[i] : 1.f);
            dx[i] = (TD)((g - s - xh * q) * r + (res ? to_f32(res[i]) : 0.f));
        }
    }
}

// dw and db: a column a thread, the blocks' rows added in their order.
__global__ __launch_bounds__(LNT) void layernorm_dw_k(const float *partial, int n, int dim, float *dw, float *db) {
    const int c = blockIdx.x * LNT + threadIdx.x;
    if (c >= 2 * dim) return;
    float *out = c < dim ? dw : db;
    if (!out) return;
    float s = 0.f;
    for (int b = 0; b < n; ++b) s += partial[(long)b * 2 * dim + c];
    out[c < dim ? c : c - dim] = s;
}

int bwd_blocks(const LayernormArgs &a) { return (int)(a.n_rows < kBlocks ? a.n_rows : kBlocks); }

}  // namespace

size_t layernorm_partial_floats(const LayernormArgs &a) { return (size_t)bwd_blocks(a) * 2 * a.dim; }

hipError_t layernorm_forward(const LayernormArgs &a, DType xt, DType yt, hipStream_t st) {
    if (a.n_rows <= 0) return hipSuccess;
    by_type(xt, [&](auto x) {
        by_type(yt, [&](auto y) {
            hipLaunchKernelGGL((layernorm_fwd_k<decltype(x), decltype(y)>), long_grid(a.n_rows), dim3(LNT), 0, st, a);
        });
    });
    return hipGetLastError();
}

hipError_t layernorm_backward(const LayernormArgs &a, DType xt, DType gt, DType dt, hipStream_t st) {
    if (a.n_rows <= 0) return hipSuccess;
    by_type(xt, [&](auto x) {
        by_type(gt, [&](auto g) {
            by_type(dt, [&](auto d) {
                hipLaunchKernelGGL((layernorm_bwd_k<decltype(x), decltype(g), decltype(d)>), dim3(bwd_blocks(a)), dim3(LNT), 0, st, a);
            });
        });
    });
    if (a.partial)
        hipLaunchKernelGGL(layernorm_dw_k, dim3(ceil_div(2 * (size_t)a.dim, LNT)), dim3(LNT), 0, st, a.partial, bwd_blocks(a), a.dim, a.dw, a.db);
    return hipGetLastError();
}

}  // namespace vkh
