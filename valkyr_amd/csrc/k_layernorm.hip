// Layer norm of rows, forward and backward.
//
//   mu = mean(x), v = mean((x - mu)^2), r = 1 / sqrt(v + eps), xh = (x - mu) r
//   forward   y = xh w + b
//   backward  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)) (+ residual)
//             dw = sum over rows of dy xh,  db = sum over rows of dy
//
// The variance is that of the centred values (a row far from 0 keeps its digits), statistics and sums
// are fp32, and the backward forms the statistics again from x, which it reads anyway.  Each row is read once
// and held in registers, 16 values a lane in the forward and 8 in the backward, which has the sums of two
// gradients beside them: by a wave where that holds it, by up to sixteen waves beyond that, by a block that reads it
// several times where even those do not hold it.  Rows may start at any value; their last values, less than a vector, are
// taken one by one (16384 rows of 777 bf16: 17 and 47 us, 2.9 and 2.2 TB/s; of 4096 58 and 106, 4.6 and 5.0).  Bound by
// HBM for long batches and by the launch for a few tokens.
#include <algorithm>
#include <type_traits>

#include "ops.hpp"

namespace vkh {
namespace {

constexpr int kFwdHeld = 16, kBwdHeld = 8;  // values of a row in a lane (the backward's longest rows: kFwdHeld)
constexpr int kWide = 16384;  // the longest row that is held
constexpr int LNT = 256;           // threads on a longer one

// The sum over a wave, in its lanes' order by halves of 16 and then row by row.
VKH_DEV float lanes_sum(float v) {
    v = row16_sum(v);
    auto at = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (at(0) + at(16)) + (at(32) + at(48));
}

// A row's values from `e` on, what is past its end as 0: chunk k of thread t of the NT on a row starts at (k NT + t) W.
// TAIL: the row's last chunk is not whole (dim % W), else a chunk is in the row or behind it.
template <int W, bool TAIL, class T>
VKH_DEV typename Vec<T, W>::type raw_chunk(const T *p, int e, int dim) {
    typename Vec<T, W>::type v = {};
    if (e + W <= dim) {
        v = *reinterpret_cast<const typename Vec<T, W>::type *>(p + e);
    } else if constexpr (TAIL) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (e + i < dim) v[i] = p[e + i];
    }
    return v;
}
template <class T, int W>
VKH_DEV void widen(T v, float (&o)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = (float)v[i];
}
template <bool TAIL, class T, int W>
VKH_DEV void load_chunk(const T *p, int e, int dim, float (&o)[W]) { widen(raw_chunk<W, TAIL>(p, e, dim), o); }
// Results go past the caches: they are read by another kernel, each store covers whole lines over its lanes, and the
// inputs stay in the last cache for the backward (16384 rows of 4096 bf16, inputs that are in no cache: both directions
// 160 us, through the caches 169; 8192 rows of fp32 148 and 168.  One direction alone 57 and 106 us, through them 58 and 109).
template <bool TAIL, bool PAST = true, class T, int W>
VKH_DEV void store_chunk(T *p, int e, int dim, const float (&o)[W]) {
    if (e + W <= dim) {
        typename Vec<T, W>::type v;
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (T)o[i];
        if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<typename Vec<T, W>::type *>(p + e));
        else *reinterpret_cast<typename Vec<T, W>::type *>(p + e) = v;
    } else if (TAIL) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (e + i < dim) p[e + i] = (T)o[i];
    }
}

// The NT threads on a row (BT in the block).  Lane j of each 16 takes wave j's part of an exchange: sums over the waves are
// sums over a row of lanes.
template <int NT, int BT, int W, int HELD>
struct Group {
    static constexpr int waves = NT / 64;
    float2 (*sh)[BT / 64];    // two, in turn: one barrier an exchange
    int first, turn = 0;      // the group's first wave
    float mine, of_j, inv_j;  // 1 / values of a row in this wave, values in wave j, 1 / them (0 for none)

    VKH_DEV Group(float2 (*s)[BT / 64], int grp, int dim) : sh(s), first(grp * waves) {
        if constexpr (waves > 1) {
            auto held = [&](int w) {
                int n = 0;
#pragma unroll
                for (int k = 0; k < HELD / W; ++k) n += min(max(dim - (k * NT + w * 64) * W, 0), 64 * W);
                return n;
            };
            const int j = threadIdx.x % 16, n = j < waves ? held(j) : 0, m = held(threadIdx.x % NT / 64);
            of_j = (float)n;
            inv_j = n ? 1.0f / (float)n : 0.f;
            mine = m ? 1.0f / (float)m : 0.f;
        }
    }
    // (a, b) of wave j
    VKH_DEV float2 exchange(float a, float b) {
        if (threadIdx.x % 64 == 0) sh[turn][threadIdx.x / 64] = make_float2(a, b);
        __syncthreads();
        const int j = threadIdx.x % 16;
        const float2 v = sh[turn][first + j % waves];
        turn ^= 1;
        return j < waves ? v : make_float2(0.f, 0.f);
    }
};

// 1 / deviation of the row in x; leaves x centred and scaled (0 past its end).  Each wave centres its values about its
// own mean; the waves' sums of squares are joined with n (mean_w - mean)^2 each.
template <bool TAIL, int NT, int BT, int W, int HELD>
VKH_DEV float normalise(float (&x)[HELD / W][W], int t, int dim, float inv_dim, float eps, Group<NT, BT, W, HELD> &g) {
    auto centred = [&](int k, int i, float m) { return (k * NT + t) * W + (TAIL ? i : 0) < dim ? x[k][i] - m : 0.f; };
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < HELD / W; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) s += x[k][i];
    s = lanes_sum(s);
    float mu = s * (NT == 64 ? inv_dim : g.mine);
#pragma unroll
    for (int k = 0; k < HELD / W; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float c = centred(k, i, mu);
            q = fmaf(c, c, q);
        }
    q = lanes_sum(q);
    if constexpr (NT > 64) {
        const float2 v = g.exchange(s, q);
        mu = row16_sum(v.x) * inv_dim;
        const float d = v.x * g.inv_j - mu;
        q = row16_sum(g.of_j > 0.f ? fmaf(d * d, g.of_j, v.y) : 0.f);
    }
    const float r = 1.0f / sqrtf(fmaf(q, inv_dim, eps));
#pragma unroll
    for (int k = 0; k < HELD / W; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) x[k][i] = centred(k, i, mu) * r;
    return r;
}

template <class TX, class TY, int NT, bool TAIL>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void layernorm_fwd_held_k(LayernormArgs a) {
    constexpr int BT = NT < 256 ? 256 : NT, W = 16 / (int)sizeof(TX), NI = kFwdHeld / W;
    __shared__ float2 sh[2][BT / 64];
    const int t = threadIdx.x % NT, dim = a.dim;
    const long row = block_number<BT>() * (BT / NT) + __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
    const bool live = row < a.n_rows;
    Group<NT, BT, W, kFwdHeld> g(sh, threadIdx.x / NT, dim);
    typename Vec<TX, W>::type xr[NI];  // (all asked for before the first is used)
    float x[NI][W];
#pragma unroll
    for (int k = 0; k < NI; ++k) xr[k] = raw_chunk<W, TAIL>((const TX *)a.x + (live ? row : 0) * a.ldx, (k * NT + t) * W, dim);
#pragma unroll
    for (int k = 0; k < NI; ++k) widen(xr[k], x[k]);
    normalise<TAIL>(x, t, dim, 1.0f / (float)dim, a.eps, g);
    if (!live) return;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        const int e = (k * NT + t) * W;
        float v[W];
        if (a.w) {
            load_chunk<TAIL>(a.w, e, dim, v);
#pragma unroll
            for (int i = 0; i < W; ++i) x[k][i] *= v[i];
        }
        if (a.b) {
            load_chunk<TAIL>(a.b, e, dim, v);
#pragma unroll
            for (int i = 0; i < W; ++i) x[k][i] += v[i];
        }
        store_chunk<TAIL>((TY *)a.y + row * a.ldy, e, dim, x[k]);
    }
}

// Values a vector: 16 bytes of the widest type.
template <class TX, class TG, class TD>
constexpr int bwd_vector() {
    return sizeof(TX) + sizeof(TG) + sizeof(TD) == 6 ? 8 : 4;
}

// Rows are dealt to the blocks' groups of NT threads in turn.  A lane sums its columns' gradients of w and b over its
// rows; the groups of a block add theirs through LDS, one after the other, and the block writes them to its row of
// `partial` ([blocks][2][dim]), which layernorm_dw_k adds in block order.
template <class TX, class TG, class TD, int NT, int BT, int HELD, bool TAIL>
__global__ __launch_bounds__(BT) void layernorm_bwd_held_k(LayernormArgs a) {
    constexpr int W = bwd_vector<TX, TG, TD>(), NI = HELD / W, GR = BT / NT;
    __shared__ float2 sh[2][BT / 64];
    extern __shared__ float sums[];  // [2][dim] with more than one group
    const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), t = threadIdx.x % NT, dim = a.dim;
    const long stride = (long)gridDim.x * GR;
    Group<NT, BT, W, HELD> g(sh, grp, dim);
    const float inv_dim = 1.0f / (float)dim;
    float dw[NI][W] = {}, db[NI][W] = {}, w[NI][W];
#pragma unroll
    for (int k = 0; k < NI; ++k) {
        if (a.w) {
            load_chunk<TAIL>(a.w, (k * NT + t) * W, dim, w[k]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) w[k][i] = 1.f;
        }
    }
    for (long row0 = (long)blockIdx.x * GR; row0 < a.n_rows; row0 += stride) {  // (all groups of a block take every barrier)
        const bool live = row0 + grp < a.n_rows;
        const long row = live ? row0 + grp : row0;
        typename Vec<TX, W>::type xr[NI];  // (all asked for before the first is used)
        typename Vec<TG, W>::type dr[NI];
        typename Vec<TD, W>::type rr[NI] = {};
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            xr[k] = raw_chunk<W, TAIL>((const TX *)a.x + row * a.ldx, (k * NT + t) * W, dim);
            dr[k] = raw_chunk<W, TAIL>((const TG *)a.dy + row * a.lddy, (k * NT + t) * W, dim);
        }
        if (a.res) {
#pragma unroll
            for (int k = 0; k < NI; ++k) rr[k] = raw_chunk<W, TAIL>((const TD *)a.res + row * a.lddx, (k * NT + t) * W, dim);
        }
        float x[NI][W], d[NI][W];
#pragma unroll
        for (int k = 0; k < NI; ++k) widen(xr[k], x[k]), widen(dr[k], d[k]);
        const float r = normalise<TAIL>(x, t, dim, inv_dim, a.eps, g);
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (live) {
                    dw[k][i] = fmaf(d[k][i], x[k][i], dw[k][i]);
                    db[k][i] += d[k][i];
                }
                d[k][i] *= w[k][i];
                s += d[k][i];
                q = fmaf(d[k][i], x[k][i], q);
            }
        s = lanes_sum(s);
        q = lanes_sum(q);
        if constexpr (NT > 64) {
            const float2 v = g.exchange(s, q);
            s = row16_sum(v.x);
            q = row16_sum(v.y);
        }
        s *= inv_dim;
        q *= inv_dim;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            float o[W];
            widen(rr[k], o);
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] = fmaf(d[k][i] - s - x[k][i] * q, r, o[i]);
            store_chunk<TAIL>((TD *)a.dx + row * a.lddx, (k * NT + t) * W, dim, o);
        }
    }
    if (!a.partial) return;
    float *out = a.partial + (long)blockIdx.x * 2 * dim;
#pragma unroll 1
    for (int j = 0; j < GR; ++j) {
        if (GR > 1) __syncthreads();
        if (grp != j) continue;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
            const int e = (k * NT + t) * W;
            if (j) {
                float u[W], v[W];
                load_chunk<TAIL>(sums, e, dim, u);
                load_chunk<TAIL>(sums + dim, e, dim, v);
#pragma unroll
                for (int i = 0; i < W; ++i) dw[k][i] += u[i], db[k][i] += v[i];
            }
            store_chunk<TAIL, false>(j + 1 < GR ? sums : out, e, dim, dw[k]);
            store_chunk<TAIL, false>((j + 1 < GR ? sums : out) + dim, e, dim, db[k]);
        }
    }
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

// dw and db: 64 columns a block, each thread every 16th of the blocks' rows, and then the 16 sums of a column in order.
__global__ __launch_bounds__(1024) void layernorm_dw_k(const float *partial, int n, int dim, float *dw, float *db) {
    __shared__ float sh[16][64];
    const int l = threadIdx.x % 64, part = threadIdx.x / 64;
    const long c = (long)blockIdx.x * 64 + l;
    float s = 0.f;
    if (c < 2l * dim) {
#pragma unroll 8
        for (int b = part; b < n; b += 16) s += partial[(long)b * 2 * dim + c];
    }
    sh[part][l] = s;
    __syncthreads();
    float *out = c < dim ? dw : db;
    if (part || c >= 2l * dim || !out) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sh[i][l];
    out[c < dim ? c : c - dim] = s;
}

// Threads on a row: as many as hold it.
int threads_of(int dim, int held) {
    int n = 64;
    while (n * held < dim) n *= 2;
    return n;
}
template <class F>
void by_threads(int n, F f) {
    switch (n) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    case 512: return f(std::integral_constant<int, 512>{});
    default: return f(std::integral_constant<int, 1024>{});
    }
}

// The backward's threads a block and blocks: 512 threads where there are rows for more than 512 blocks of 256, and as
// many blocks as give every CU sixteen waves.  Two blocks of 512 threads a CU work while the other waits (16384
// rows of 4096 bf16: 106 us; one block of 1024 threads 118, three of 512 119, with the partial sums of half as many more
// blocks; 16 values a lane 135 to 181).
struct Bwd {
    int threads, blocks;
};
Bwd bwd_of(const LayernormArgs &a) {
    // Rows of more than kWide values: partial sums of up to 64 MiB, or of one block (more than 2^22 values), which then adds
    // all rows one after the other.
    if (a.dim > kWide) {
        const long most = std::min(512l, std::max(1l, (8l << 20) / a.dim));
        return {LNT, (int)std::min(a.n_rows, most)};
    }
    const int nt = std::min(1024, threads_of(a.dim, kBwdHeld)), bt = std::max(nt, a.n_rows * nt / 256 > 512 ? 512 : 256);
    return {bt, (int)std::min((a.n_rows * nt + bt - 1) / bt, 256l * 1024 / bt)};
}

}  // namespace

size_t layernorm_partial_floats(const LayernormArgs &a) { return (size_t)bwd_of(a).blocks * 2 * a.dim; }

hipError_t layernorm_forward(const LayernormArgs &a, DType xt, DType yt, hipStream_t st) {
    if (a.n_rows <= 0) return hipSuccess;
    by_type(xt, [&](auto x) {
        by_type(yt, [&](auto y) {
            using X = decltype(x);
            using Y = decltype(y);
            if (a.dim > kWide) {
                hipLaunchKernelGGL((layernorm_fwd_k<X, Y>), long_grid(a.n_rows), dim3(LNT), 0, st, a);
                return;
            }
            by_threads(threads_of(a.dim, kFwdHeld), [&](auto nt) {
                constexpr int NT = decltype(nt)::value, BT = std::max(NT, 256), per = BT / NT;
                auto k = a.dim % (16 / sizeof(X)) ? layernorm_fwd_held_k<X, Y, NT, true> : layernorm_fwd_held_k<X, Y, NT, false>;
                hipLaunchKernelGGL(k, long_grid((a.n_rows + per - 1) / per, BT), dim3(BT), 0, st, a);
            });
        });
    });
    return hipGetLastError();
}

hipError_t layernorm_backward(const LayernormArgs &a, DType xt, DType gt, DType dt, hipStream_t st) {
    if (a.n_rows <= 0) return hipSuccess;
    const Bwd n = bwd_of(a);
    by_type(xt, [&](auto x) {
        by_type(gt, [&](auto g) {
            by_type(dt, [&](auto d) {
                using X = decltype(x);
                using G = decltype(g);
                using D = decltype(d);
                if (a.dim > kWide) {
                    hipLaunchKernelGGL((layernorm_bwd_k<X, G, D>), dim3(n.blocks), dim3(LNT), 0, st, a);
                    return;
                }
                by_threads(std::min(1024, threads_of(a.dim, kBwdHeld)), [&](auto nt) {
                    constexpr int NT = decltype(nt)::value;
                    auto go = [&](auto bt) {
                        constexpr int BT = std::max(NT, decltype(bt)::value);
                        const size_t lds = BT > NT && a.partial ? 2 * a.dim * sizeof(float) : 0;
                        auto pick = [&](auto held) {
                            constexpr int H = decltype(held)::value;
                            auto k = a.dim % bwd_vector<X, G, D>() ? layernorm_bwd_held_k<X, G, D, NT, BT, H, true>
                                                                   : layernorm_bwd_held_k<X, G, D, NT, BT, H, false>;
                            hipLaunchKernelGGL(k, dim3(n.blocks), dim3(BT), lds, st, a);
                        };
                        if constexpr (NT == 1024) {
                            if (a.dim > 1024 * kBwdHeld) return pick(std::integral_constant<int, kFwdHeld>{});
                        }
                        pick(std::integral_constant<int, kBwdHeld>{});
                    };
                    if (n.threads == 256) go(std::integral_constant<int, 256>{});
                    else go(std::integral_constant<int, 512>{});
                });
            });
        });
    });
    if (a.partial)
        hipLaunchKernelGGL(layernorm_dw_k, dim3(ceil_div(2 * (size_t)a.dim, 64)), dim3(1024), 0, st, a.partial, n.blocks, a.dim, a.dw, a.db);
    return hipGetLastError();
}

}  // namespace vkh
