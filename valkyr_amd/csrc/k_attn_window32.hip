// Windowed attention on fp32 operands: the tile kernels (64- and 128-wide heads, aligned rows) of the
// operator that k_attn_window.hip describes, on v_mfma_f32_16x16x4_f32.
//
// Tiles of 32 keys (dK/dV: 32 queries) come by DMA into swizzled LDS rows, the next one while one computes; each
// of a block's 4 waves holds 16 query (key) rows in registers.  Lane (g, c) = (lane / 16, lane % 16) gives A[c][g]
// and B[g][c] and holds C[4 g + r][c]: over the head, step (u, e) stands for value 16 u + 4 g + e (one 16-byte
// read covers four), and an accumulator is the next product's B operand as it stands:
//   forward  S^T = K Q^T, O^T += V^T P^T          dQ  S^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   dK/dV    S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// A score is the sum of HD / 16 side-by-side chains (one chain of 128 terms rounds three times as
// coarsely, and each product would wait for the one before).  Bound by the fp32 matrix cores, and on
// short sequences by the few steps that each block has: 4 x 2048 tokens, window 2048, 16 / 8 heads of 128,
// forward / backward 563 / 2091 us, 122 / 82 TFLOP/s; 2 x 1001 tokens, window 256, 16 / 4 heads of 64, half of them
// padding: 23.5 + 33 (dQ) + 44 us (dK/dV), about 40 TFLOP/s each.
//
// As in the bf16 kernels, a block that meets an infinity or a NaN in a tile that its rows do not see
// in full forms its rows anew one at a time.
#include "attn16.hpp"
#include "window.hpp"

#pragma clang fp contract(off)

namespace vkh {
namespace {

constexpr int FNT = 256, FT = 32;

VKH_DEV float4 f4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
VKH_DEV f32x4 mfma4(const float4 &a, const float4 &b, f32x4 c) {
    c = mfma16x16x4(a.x, b.x, c);
    c = mfma16x16x4(a.y, b.y, c);
    c = mfma16x16x4(a.z, b.z, c);
    return mfma16x16x4(a.w, b.w, c);
}
// LDS tiles of FT head rows as the DMA writes them: 16-byte chunk n of row r at chunk n ^ (r & 15), so
// that the 16 rows of a fragment read lie in 16 different chunk columns of LDS's 256 bytes a cycle.
template <int HD>
struct Rows32 {
    static constexpr int TILE = FT * HD, RPI = 256 / HD, IPT = FT / RPI;  // floats; rows a DMA of 1 KB; DMAs
    int row[4], col[4];  // a lane's offsets: of values 16 u + 4 g .. of row c (u % 4), of values 4 c .. of row 4 g + e
    VKH_DEV Rows32(int g, int c) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            row[x] = c * HD + 4 * ((4 * x + g) ^ c);
            col[x] = (4 * g + x) * HD + 4 * (c ^ (4 * g + x));
        }
    }
    // a lane's byte offset in a tile's DMA number q
    static VKH_DEV unsigned dma(int q, int lane, int ld) {
        const int r = q * RPI + lane / (HD / 4), n = (lane % (HD / 4)) ^ (r & 15);
        return (unsigned)((r * ld + 4 * n) * 4);
    }
    static VKH_DEV unsigned bytes(int rows, int ld) { return rows > 0 ? (unsigned)(((min(rows, FT) - 1) * ld + HD) * 4) : 0u; }
};
// Whether a group of 256 threads' tile holds an infinity or a NaN (exponent bits of all ones, to which
// one more carries into the sign's place): each thread's share.
template <int HD>
VKH_DEV bool scan32(const float *tile, int tid) {
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < FT * HD / 1024; ++i) {
        const uint4 v = *reinterpret_cast<const uint4 *>(tile + (i * 256 + tid) * 4);
        carry |= ((v.x & 0x7f800000u) + 0x00800000u) | ((v.y & 0x7f800000u) + 0x00800000u);
        carry |= ((v.z & 0x7f800000u) + 0x00800000u) | ((v.w & 0x7f800000u) + 0x00800000u);
    }
    return carry & 0x80000000u;
}
template <int NU>
VKH_DEV f32x4 chains(f32x4 (&a)[NU]) {
#pragma unroll
    for (int w = NU / 2; w; w /= 2)
#pragma unroll
        for (int u = 0; u < w; ++u) a[u] += a[u + w];
    return a[0];
}
// the lane's element of 16 tile rows' products with its column of f
template <int HD>
VKH_DEV f32x4 head_dot(const float *tile, const Rows32<HD> &t, const float4 (&f)[HD / 16]) {
    constexpr int NU = HD / 16;
    f32x4 a[NU] = {};
#pragma unroll
    for (int u = 0; u < NU; ++u) a[u] = mfma4(f4(tile + t.row[u % 4] + 64 * (u / 4)), f[u], a[u]);
    return chains(a);
}
// acc += T^T w over 16 rows of an LDS tile: element e of w is row 4 g + e.  Matrix row i of acc[4 J + j]
// is column 64 J + 4 i + j of the tile, so that one 16-byte read feeds four products (a 4-byte read for
// each left them waiting on LDS: see acc_cols for the way back).  `at(e)` is values 4 c .. of row 4 g + e.
template <int NU, class At>
VKH_DEV void add_rows_at(f32x4 (&acc)[NU], At at, const f32x4 &w) {
#pragma unroll
    for (int J = 0; J < NU / 4; ++J) {
        float4 t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = f4(at(e) + 64 * J);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[4 * J] = mfma16x16x4(t[e].x, w[e], acc[4 * J]);
            acc[4 * J + 1] = mfma16x16x4(t[e].y, w[e], acc[4 * J + 1]);
            acc[4 * J + 2] = mfma16x16x4(t[e].z, w[e], acc[4 * J + 2]);
            acc[4 * J + 3] = mfma16x16x4(t[e].w, w[e], acc[4 * J + 3]);
        }
    }
}
template <int HD>
VKH_DEV void add_rows(f32x4 (&acc)[HD / 16], const float *tile, const Rows32<HD> &t, const f32x4 &w) {
    add_rows_at(acc, [&](int e) { return tile + t.col[e]; }, w);
}
// e^x with one rounding more than the instruction's: that of x log2(e), relative to x
VKH_DEV float exp_(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// Four columns of the lane's item: f(first column, their values) for columns 64 J + 16 g + 4 r.
template <int NU, class F>
VKH_DEV void acc_cols(const f32x4 (&acc)[NU], int g, F f) {
#pragma unroll
    for (int J = 0; J < NU / 4; ++J)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            f(64 * J + 16 * g + 4 * r, f32x4{acc[4 * J][r], acc[4 * J + 1][r], acc[4 * J + 2][r], acc[4 * J + 3][r]});
}

// R rows of HD floats moved by NT threads, global -> registers -> LDS (pitch HD + 4).
template <int HD, int R, int NT>
struct Tile32 {
    static constexpr int P = HD + 4, N4 = R * HD / 4 / NT;
    static_assert(N4 * NT * 4 == R * HD, "tile / thread count");
    float4 v[N4];
    VKH_DEV void load(const float *base, long ld, int tid, int rows) {  // rows from `rows` on are zero
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            const int x = tid + NT * i, r = x / (HD / 4), c = x % (HD / 4);
            v[i] = r < rows ? f4(base + (long)r * ld + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    VKH_DEV void store(float *lds, int tid) const {
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            const int x = tid + NT * i, r = x / (HD / 4), c = x % (HD / 4);
            *reinterpret_cast<float4 *>(lds + r * P + 4 * c) = v[i];
        }
    }
    VKH_DEV bool odd() const {  // holds an infinity or a NaN (0 times which is NaN)
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < N4; ++i) {
            z = fmaf(v[i].x, 0.f, z); z = fmaf(v[i].y, 0.f, z);
            z = fmaf(v[i].z, 0.f, z); z = fmaf(v[i].w, 0.f, z);
        }
        return !(z == 0.f);
    }
};

__device__ __attribute__((noinline)) void fwd_rows32(const WindowArgs &a, int b, int r, int end, int h, float *q, int lane) {
    for (; r < end; r += 4) window_fwd_row<float, float>(a, b, r, h, q, lane);
}
__device__ __attribute__((noinline)) void dq_rows32(const WindowArgs &a, int b, int r, int end, int h, float *q, float *g, int lane) {
    for (; r < end; r += 4) window_dq_row<float, float>(a, b, r, h, q, g, lane);
}
__device__ __attribute__((noinline)) void dkv_rows32(const WindowArgs &a, const Steps &st, int b, int kvh, int k0, int wave,
                                                     float *ws, float *k, float *v, int lane) {
    auto mine = [&](int h, int row) { return st.mine(h, row); };
    for (int x = wave; x < 64; x += 4) {
        if (k0 + x >= a.n_kv) {  // (their slots are read)
            for (int d = lane; ws && d < a.hd; d += 64) ws[x * a.hd + d] = ws[(64 + x) * a.hd + d] = 0.f;
            continue;
        }
        const long row = (long)b * a.n_kv + k0 + x;
        window_dkv_row<float>(a, b, k0 + x, kvh, k, v, ws ? ws + x * a.hd : (float *)a.dk + row * a.lddk + kvh * a.hd,
                              ws ? ws + (64 + x) * a.hd : (float *)a.dv + row * a.lddv + kvh * a.hd, lane, mine);
    }
}

// ── forward: block = 64 query rows of one head ───────────────────────────
// KG groups of four waves take every KG-th key tile each (from LDS of their own) and join their results
// at the end: short sequences leave a CU one block, whose steps then wait for themselves.
template <int HD, int KG>
__global__ __launch_bounds__(256 * KG, KG == 1 ? 2 : 1) void window_fwd32_k(WindowArgs a) {
    using T = Rows32<HD>;
    constexpr int NU = HD / 16, TILE = T::TILE, C = T::IPT / 2;  // DMAs per wave and step
    __shared__ __attribute__((aligned(16))) float tiles[KG][2][2][TILE];  // [group][buffer][K, V]
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, nqt = (a.n_q + 63) / 64;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4 * grp);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, h = kvh * grp + pr.y % grp, qt = nqt - 1 - pr.y / grp;
    const int tid = threadIdx.x % 256, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % 4, kg = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    const Span s = span_of(a, b);
    const int r0 = qt * 64, qw = r0 + 16 * wave, r = qw + c;
    const KeyTiles kt = key_tiles<FT>(a, s, r0, r0 + 64);
    const int wta = max(0, qw + s.off), wtb = min(qw + 16, s.ql) - 1 + s.off;
    const int pos = r < s.ql ? max(-1, r + s.off) : -1;
    const long row = (long)b * a.n_q + r;
    Reach mine = reach<FT>(a, kt, wta, wtb);
    if (qw + 16 > s.ql || qw + s.off < 0) mine.n_all = mine.n_sink_all = 0;  // rows that are not there
    const Reach block = reach<FT>(a, kt, kt.ta, kt.tb);
    const int steps = (kt.n + KG - 1) / KG, n = (kt.n - kg + KG - 1) / KG;  // the block's; the group's
    float4 qf[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u)
        qf[u] = pos >= 0 ? f4((const float *)a.q + row * a.ldq + h * HD + 4 * g + 16 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
    // waves 0 and 1 move K, 2 and 3 V
    const int ld = (int)(wave < 2 ? a.ldk : a.ldv);
    const float *src = (const float *)(wave < 2 ? a.k : a.v) + (long)b * a.n_kv * ld + kvh * HD;
    const unsigned dst = lds_addr(tiles[kg][0][wave / 2]) + wave % 2 * C * 1024;
    unsigned off[C];
#pragma unroll
    for (int i = 0; i < C; ++i) off[i] = T::dma(wave % 2 * C + i, lane, ld);
    wait_vm0();  // Q is in registers before any DMA is queued
    auto dma = [&](int it, int buf) {
        const int k0 = kt.tile(KG * it + kg) * FT;
        const sgpr4 rs = rsrc4(src + (long)k0 * ld, T::bytes(s.kl - k0, ld));
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rs, dst + buf * 2 * TILE * 4 + i * 1024, off[i]);
    };
    const T t(g, c);
    const float c2 = a.scale * LOG2E;
    f32x4 ot[NU];  // O^T, columns as acc_cols has them
#pragma unroll
    for (int j = 0; j < NU; ++j) ot[j] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;  // running maximum of q k; this lane's share of the sum
    bool odd = false;              // in V of a tile that is not seen in full
    if (n > 0) dma(0, 0);
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        wait_vm0();
        lds_barrier();  // tile it landed; everyone is done with tile it - 1
        if (it + 1 < n) dma(it + 1, buf ^ 1);
        if (KG > 1 && it >= n) return;
        const float *Kl = tiles[kg][buf][0], *Vl = tiles[kg][buf][1];
        const int tile = KG * it + kg;
        if (!block.whole(tile) && scan32<HD>(Vl, tid)) odd = true;
        if (mine.none(tile)) return;
        const int k0 = kt.tile(tile) * FT;
        f32x4 st[2];
        bool live[2] = {true, true};
        if (mine.whole(tile)) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) st[ks] = head_dot<HD>(Kl + 16 * ks * HD, t, qf);
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                live[ks] = !none_seen(a, wta, wtb, k0 + 16 * ks, k0 + 16 * ks + 15);  // wave-uniform
                st[ks] = f32x4{0, 0, 0, 0};
                if (live[ks]) st[ks] = head_dot<HD>(Kl + 16 * ks * HD, t, qf);
            }
            for_hidden<2>(a, pos, k0, g, [&](int ks, int r) { st[ks][r] = -INFINITY; });
        }
        // The maximum moves only when a row's scores pass it by more than 8 (in log2 units): P stays
        // under 2^8, which fp32 holds as exactly.
        float mt = -INFINITY;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) mt = fmaxf(mt, st[ks][e]);
        if (__any(m == -INFINITY ? mt > m : (mt - m) * c2 > 8.f)) {
            const float mn = xrow_max(mt), mo = m;
            if (mo == -INFINITY || (mn - mo) * c2 > 8.f) m = mn;
            const float alpha = m == mo ? 1.f : __builtin_amdgcn_exp2f((mo - m) * c2);
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NU; ++j) ot[j] *= alpha;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                st[ks][e] = __builtin_amdgcn_exp2f((st[ks][e] - ms) * c2);
                l += st[ks][e];
            }
        // O^T += V^T P^T
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
            if (live[ks]) add_rows<HD>(ot, Vl + 16 * ks * HD, t, st[ks]);
    };
    for (int it0 = 0; it0 < steps; it0 += 2) {
        step(it0, std::integral_constant<int, 0>{});
        if (it0 + 1 < steps) step(it0 + 1, std::integral_constant<int, 1>{});
    }
    if (__syncthreads_or(odd)) {
        if (kg == 0) fwd_rows32(args_again(), b, r0 + wave, min(r0 + 64, a.n_q), h, tiles[0][0][0] + wave * HD, lane);
        return;
    }
    l = xrow_sum(l);
    if constexpr (KG > 1) {  // the groups' results, joined in order through LDS
        constexpr int W = (NU + 1) * 4 * 64;  // floats of a wave's result: columns of 64 lanes
        static_assert(4 * W <= 4 * TILE, "a group's results fit its tiles");
        auto column = [&](int k, int j) { return reinterpret_cast<f32x4 *>(tiles[k][0][0] + wave * W + j * 256) + lane; };
        if (kg) {
#pragma unroll
            for (int j = 0; j < NU; ++j) *column(kg, j) = ot[j];
            *column(kg, NU) = f32x4{m, l, 0, 0};
        }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int k = 1; k < KG; ++k) {
            const f32x4 st = *column(k, NU);
            const float mn = fmaxf(m, st[0]), ms = mn == -INFINITY ? 0.f : mn;
            const float f0 = __builtin_amdgcn_exp2f((m - ms) * c2), f1 = __builtin_amdgcn_exp2f((st[0] - ms) * c2);
            m = mn;
            l = l * f0 + st[1] * f1;
#pragma unroll
            for (int j = 0; j < NU; ++j) ot[j] = ot[j] * f0 + *column(k, j) * f1;
        }
    }
    if (r >= a.n_q) return;
    const bool dead = l == 0.f;
    const float inv = 1.0f / l;
    float *o = (float *)a.o + row * a.ldo + h * HD;
    acc_cols<NU>(ot, g, [&](int d, f32x4 x) {
        x = dead ? f32x4{0, 0, 0, 0} : x * inv;
        store4(o + d, x[0], x[1], x[2], x[3]);
    });
    if (a.lse && g == 0) a.lse[row * a.n_heads + h] = dead ? -INFINITY : fmaf(m, a.scale, logf(l));
}

// ── forward of a few rows ────────────────────────────────────────────────
// As in bf16 (window_step16_k), with 16-key tiles that a wave moves through its registers into LDS rows of
// HD + 4 floats.  One row, window 4096, 16 / 8 heads of 128: 20 us with the join.
template <int HD>
__global__ __launch_bounds__(FNT, 2) void window_step32_k(WindowArgs a, int splits) {
    constexpr int BN = 16, NU = HD / 16;
    using T = Tile32<HD, BN, 64>;
    constexpr int P = T::P;
    __shared__ __attribute__((aligned(16))) float tiles[4][2][BN * P];
    __shared__ float ml[4][2][16];
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, M = a.n_q * grp, RT = (M + 15) / 16;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, rt = pr.y % RT, split = pr.y / RT;
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const Span s = span_of(a, b);
    const KeyTiles kt = key_tiles<BN>(a, s, rt * 16 / grp, (min(M, rt * 16 + 16) - 1) / grp + 1);
    const int per = (kt.n + splits - 1) / splits, last = min(kt.n, (split + 1) * per);
    const float c2 = a.scale * LOG2E;
    const int mi = rt * 16 + c, row = mi / grp, h = kvh * grp + mi % grp;
    const int pos = mi < M && row < s.ql ? max(-1, row + s.off) : -1;
    float4 qf[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u)
        qf[u] = pos >= 0 ? f4((const float *)a.q + ((long)b * a.n_q + row) * a.ldq + h * HD + 4 * g + 16 * u)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
    const float *kb = (const float *)a.k + (long)b * a.n_kv * a.ldk + kvh * HD;
    const float *vb = (const float *)a.v + (long)b * a.n_kv * a.ldv + kvh * HD;
    float *Kl = tiles[wave][0], *Vl = tiles[wave][1];
    T tk, tv;
    auto load = [&](int it) {
        const int k0 = kt.tile(it) * BN;
        tk.load(kb + (long)k0 * a.ldk, a.ldk, lane, s.kl - k0);
        tv.load(vb + (long)k0 * a.ldv, a.ldv, lane, s.kl - k0);
    };
    f32x4 acc[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) acc[j] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;  // maximum in log2 units
    int it = split * per + wave;
    if (it < last) load(it);
    for (; it < last; it += 4) {
        const int k0 = kt.tile(it) * BN;
        const bool odd = !all_seen(a, kt.ta, kt.tb, k0, k0 + BN - 1) && __any(tv.odd());
        wave_lds();  // the last tile's reads are done
        tk.store(Kl, lane);
        tv.store(Vl, lane);
        if (it + 4 < last) load(it + 4);
        wave_lds();
        f32x4 a0[NU] = {};
#pragma unroll
        for (int u = 0; u < NU; ++u) a0[u] = mfma4(f4(Kl + c * P + 4 * g + 16 * u), qf[u], a0[u]);
        f32x4 st = chains(a0) * c2;
        float mt = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!sees(a, pos, k0 + 4 * g + e)) st[e] = -INFINITY;
            mt = fmaxf(mt, st[e]);
        }
        const float mn = fmaxf(m, xrow_max(mt)), ms = mn == -INFINITY ? 0.f : mn;
        const float so = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        l *= so;
#pragma unroll
        for (int j = 0; j < NU; ++j) acc[j] *= so;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            st[e] = __builtin_amdgcn_exp2f(st[e] - ms);
            l += st[e];
        }
        if (odd) {  // pair by pair, seen pairs only
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll 1
                for (int g2 = 0; g2 < 4; ++g2) {
                    const float w = __shfl(st[e], 16 * g2 + c, 64);
                    if (!sees(a, pos, k0 + 4 * g2 + e)) continue;
#pragma unroll
                    for (int j = 0; j < NU; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            acc[j][x] = fmaf(Vl[(4 * g2 + e) * P + 64 * (j / 4) + 16 * g + 4 * x + j % 4], w, acc[j][x]);
                }
            continue;
        }
        add_rows_at(acc, [&](int e) { return Vl + (4 * g + e) * P + 4 * c; }, st);
    }
    wave_lds();
    float *res = tiles[wave][0];  // rows of P floats
    const float lt = xrow_sum(l);
    acc_cols<NU>(acc, g, [&](int d, f32x4 x) { *reinterpret_cast<f32x4 *>(res + c * P + d) = x; });
    if (g == 0) ml[wave][0][c] = m, ml[wave][1][c] = lt;
    __syncthreads();
    constexpr int E = HD / 16;
    const int r = tid / 16, d0 = tid % 16 * E;
    float mx = -INFINITY, sum = 0.f, o[E] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[w][0][r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float lw = ml[w][1][r];
        if (lw == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(ml[w][0][r] - (mx == -INFINITY ? 0.f : mx));
        sum = fmaf(lw, f, sum);
        const float *src = tiles[w][0] + r * P + d0;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(src[e], f, o[e]);
    }
    const int mr = rt * 16 + r;
    if (mr >= M) return;
    const long orow = (long)b * a.n_q + mr / grp;
    const int oh = kvh * grp + mr % grp;
    if (splits > 1) {  // as in bf16
        const long rows = (long)a.n_batch * a.n_q * a.n_heads, at = (split * rows) + orow * a.n_heads + oh;
        float *dst = a.ws + at * HD + d0;
#pragma unroll
        for (int e = 0; e < E; e += 4) store4(dst + e, o[e], o[e + 1], o[e + 2], o[e + 3]);
        if (d0 == 0) {
            float *st = a.ws + splits * rows * HD + at * 2;
            st[0] = mx;
            st[1] = sum;
        }
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    float *out = (float *)a.o + orow * a.ldo + oh * HD + d0;
#pragma unroll
    for (int e = 0; e < E; e += 4) store4(out + e, o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
    if (a.lse && d0 == 0) a.lse[orow * a.n_heads + oh] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * LN2;
}

// ── backward: D and dQ, block = 64 query rows of one head ────────────────
// Key groups as in the forward.
template <int HD, int KG>
__global__ __launch_bounds__(256 * KG, KG == 1 ? 2 : 1) void window_dq32_k(WindowArgs a) {
    using T = Rows32<HD>;
    constexpr int NU = HD / 16, TILE = T::TILE, C = T::IPT / 2;
    __shared__ __attribute__((aligned(16))) float tiles[KG][2][2][TILE];  // [group][buffer][K, V]
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, nqt = (a.n_q + 63) / 64;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4 * grp);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, h = kvh * grp + pr.y % grp, qt = nqt - 1 - pr.y / grp;
    const int tid = threadIdx.x % 256, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % 4, kg = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    const Span s = span_of(a, b);
    const int r0 = qt * 64, qw = r0 + 16 * wave, r = qw + c;
    const KeyTiles kt = key_tiles<FT>(a, s, r0, r0 + 64);
    const int wta = max(0, qw + s.off), wtb = min(qw + 16, s.ql) - 1 + s.off;
    const long row = (long)b * a.n_q + r;
    const float lse = r < s.ql && r + s.off >= 0 ? a.lse[row * a.n_heads + h] : -INFINITY;
    const int pos = lse == -INFINITY ? -1 : r + s.off;
    float4 qf[NU], of[NU];
    double acc = 0;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const long col = h * HD + 4 * g + 16 * u;
        qf[u] = of[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (pos >= 0) {
            qf[u] = f4((const float *)a.q + row * a.ldq + col);
            of[u] = f4((const float *)a.dout + row * a.lddo + col);
            const float4 o = f4((const float *)a.o + row * a.ldo + col);
            acc += (double)o.x * of[u].x + (double)o.y * of[u].y + (double)o.z * of[u].z + (double)o.w * of[u].w;
        }
    }
    acc += __shfl_xor(acc, 16, 64);
    acc += __shfl_xor(acc, 32, 64);
    const float dd = (float)acc;
    if (kg == 0 && r < a.n_q && g == 0) a.d[row * a.n_heads + h] = dd;
    Reach mine = reach<FT>(a, kt, wta, wtb);
    if (!__all(pos >= 0)) mine.n_all = mine.n_sink_all = 0;  // rows of no gradient
    const Reach block = reach<FT>(a, kt, kt.ta, kt.tb);
    const int steps = (kt.n + KG - 1) / KG, n = (kt.n - kg + KG - 1) / KG;
    const int ld = (int)(wave < 2 ? a.ldk : a.ldv);
    const float *src = (const float *)(wave < 2 ? a.k : a.v) + (long)b * a.n_kv * ld + kvh * HD;
    const unsigned dst = lds_addr(tiles[kg][0][wave / 2]) + wave % 2 * C * 1024;
    unsigned off[C];
#pragma unroll
    for (int i = 0; i < C; ++i) off[i] = T::dma(wave % 2 * C + i, lane, ld);
    wait_vm0();
    auto dma = [&](int it, int buf) {
        const int k0 = kt.tile(KG * it + kg) * FT;
        const sgpr4 rs = rsrc4(src + (long)k0 * ld, T::bytes(s.kl - k0, ld));
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rs, dst + buf * 2 * TILE * 4 + i * 1024, off[i]);
    };
    const T t(g, c);
    f32x4 dqt[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) dqt[j] = f32x4{0, 0, 0, 0};
    bool odd = false;  // in K of a tile that is not seen in full
    if (n > 0) dma(0, 0);
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        wait_vm0();
        lds_barrier();
        if (it + 1 < n) dma(it + 1, buf ^ 1);
        if (KG > 1 && it >= n) return;
        const float *Kl = tiles[kg][buf][0], *Vl = tiles[kg][buf][1];
        const int tile = KG * it + kg;
        if (!block.whole(tile) && scan32<HD>(Kl, tid)) odd = true;
        if (mine.none(tile)) return;
        const int k0 = kt.tile(tile) * FT;
        const bool whole = mine.whole(tile);
        f32x4 da[2];
        bool live[2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            live[ks] = whole || !none_seen(a, wta, wtb, k0 + 16 * ks, k0 + 16 * ks + 15);  // wave-uniform
            da[ks] = f32x4{0, 0, 0, 0};
            if (!live[ks]) continue;
            const f32x4 sa = head_dot<HD>(Kl + 16 * ks * HD, t, qf);
            da[ks] = head_dot<HD>(Vl + 16 * ks * HD, t, of);
#pragma unroll
            for (int e = 0; e < 4; ++e) da[ks][e] = exp_(fmaf(sa[e], a.scale, -lse)) * (da[ks][e] - dd);
        }
        if (!whole) for_hidden<2>(a, pos, k0, g, [&](int ks, int r) { da[ks][r] = 0.f; });
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
            if (live[ks]) add_rows<HD>(dqt, Kl + 16 * ks * HD, t, da[ks]);
    };
    for (int it0 = 0; it0 < steps; it0 += 2) {
        step(it0, std::integral_constant<int, 0>{});
        if (it0 + 1 < steps) step(it0 + 1, std::integral_constant<int, 1>{});
    }
    if (__syncthreads_or(odd)) {
        float *sh = tiles[0][0][0] + wave * 2 * HD;
        if (kg == 0) dq_rows32(args_again(), b, r0 + wave, min(r0 + 64, a.n_q), h, sh, sh + HD, lane);
        return;
    }
    if constexpr (KG > 1) {
        auto column = [&](int k, int j) { return reinterpret_cast<f32x4 *>(tiles[k][0][0] + (wave * NU + j) * 256) + lane; };
        if (kg)
#pragma unroll
            for (int j = 0; j < NU; ++j) *column(kg, j) = dqt[j];
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
            for (int j = 0; j < NU; ++j) dqt[j] += *column(k, j);
    }
    if (r >= a.n_q) return;
    float *dq = (float *)a.dq + row * a.lddq + h * HD;
    acc_cols<NU>(dqt, g, [&](int d, f32x4 x) {
        x = pos >= 0 ? x * a.scale : f32x4{0, 0, 0, 0};
        store4(dq + d, x[0], x[1], x[2], x[3]);
    });
}

// ── backward: dK and dV, block = 64 keys of one KV head ──────────────────
// Steps and parts as in bf16 (window_dkv16_k), one head a step; KG groups of waves take every KG-th of
// the block's steps each and add their sums at the end.
template <int HD, int KG>
__global__ __launch_bounds__(256 * KG, KG == 1 ? 2 : 1) void window_dkv32_k(WindowArgs a, DkvPlan plan) {
    using T = Rows32<HD>;
    constexpr int NU = HD / 16, BN = 64, TILE = T::TILE, C = T::IPT / 2;
    __shared__ __attribute__((aligned(16))) float tiles[KG][2][2][TILE];  // [group][buffer][Q, dO]
    __shared__ __attribute__((aligned(16))) float stat[KG][2][2][64];     // [group][buffer][LSE, D]
    const int nbk = a.n_batch * a.n_kv_heads;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4);
    const int bk = pr.bk, b = bk / a.n_kv_heads, kvh = bk % a.n_kv_heads;
    int kb, zpart, zparts, slot;
    dkv_block(plan, pr.y, kb, zpart, zparts, slot);
    const int nh = a.n_heads / a.n_kv_heads;
    const int tid = threadIdx.x % 256, lane = tid % 64, g = lane / 16, c = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) % 4, kg = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    const Span s = span_of(a, b);
    const int k0 = kb * BN, kw = k0 + 16 * wave, key = kw + c;
    const long krow = (long)b * a.n_kv + key, row0 = (long)b * a.n_q;
    float4 kf[NU], vf[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const long col = kvh * HD + 4 * g + 16 * u;
        kf[u] = vf[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (key < s.kl) {
            kf[u] = f4((const float *)a.k + krow * a.ldk + col);
            vf[u] = f4((const float *)a.v + krow * a.ldv + col);
        }
    }
    const int k1 = min(k0 + BN, s.kl) - 1;  // the block's last key
    const int qstart = max(0, k0 - s.off);
    const int qend = k0 < a.n_sink ? s.ql : (int)min((long)s.ql, (long)k1 + a.window - s.off);
    const int nqt = k1 >= k0 && qend > qstart ? (qend - qstart + FT - 1) / FT : 0;
    const int niter = max(0, (nh * nqt - zpart + zparts - 1) / zparts), top = nqt - 1;
    // The group's steps kg, kg + KG, ... of the block's zpart, zpart + zparts, ... of (query tile, head),
    // heads inner: head and tile of one, moved on by steps of `stride`.
    const int stride = KG * zparts, dh = stride % nh, dt = stride / nh;
    struct Cursor {
        int head, tile;
    };
    auto advance = [&](Cursor &x) {
        x.head += dh;
        x.tile += dt;
        if (x.head >= nh) x.head -= nh, ++x.tile;
    };
    const int x0 = kg * zparts + zpart;
    Cursor ahead{x0 % nh, x0 / nh}, now = ahead;
    const int steps = (niter + KG - 1) / KG, n = (niter - kg + KG - 1) / KG;  // the block's; the group's
    // waves 0 and 1 move Q, 2 and 3 dO; 0 the rows' LSE too, 2 their D
    const int ld = (int)(wave < 2 ? a.ldq : a.lddo);
    const float *src = (const float *)(wave < 2 ? a.q : a.dout) + row0 * ld + kvh * nh * HD;
    const float *stat_src = (wave < 2 ? a.lse : a.d) + row0 * a.n_heads + kvh * nh;
    const unsigned dst = lds_addr(tiles[kg][0][wave / 2]) + wave % 2 * C * 1024;
    const unsigned off_stat = lane < FT ? (unsigned)(lane * a.n_heads * 4) : kOOB;
    unsigned off[C];
#pragma unroll
    for (int i = 0; i < C; ++i) off[i] = T::dma(wave % 2 * C + i, lane, ld);
    wait_vm0();  // K and V are in registers before any DMA is queued
    auto dma = [&](int buf) {
        const int h = ahead.head, q0 = qstart + (top - ahead.tile) * FT, rows = s.ql - q0;
        advance(ahead);
        const sgpr4 rs = rsrc4(src + (long)q0 * ld + h * HD, T::bytes(rows, ld));
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rs, dst + buf * 2 * TILE * 4 + i * 1024, off[i]);
        if (wave % 2 == 0) {
            const sgpr4 r1 = rsrc4(stat_src + (long)q0 * a.n_heads + h, (unsigned)(((min(rows, FT) - 1) * a.n_heads + 1) * 4));
            dma4_at(r1, lds_addr(stat[kg][buf][wave / 2]), off_stat);
        }
    };
    const T t(g, c);
    bool odd = false;  // in Q or dO of a tile whose rows do not all see all keys, or have no gradient
    f32x4 dvt[NU], dkt[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) dvt[j] = dkt[j] = f32x4{0, 0, 0, 0};
    if (n > 0) dma(0);
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        wait_vm0();
        lds_barrier();
        if (it + 1 < n) dma(buf ^ 1);
        if (KG > 1 && it >= n) return;
        const int q0 = qstart + (top - now.tile) * FT, ta = q0 + s.off, tb = min(q0 + FT, s.ql) - 1 + s.off;
        advance(now);
        const float *Ql = tiles[kg][buf][0], *Ol = tiles[kg][buf][1], *Ll = stat[kg][buf][0] + 4 * g, *Dl = stat[kg][buf][1] + 4 * g;
        const bool all = all_seen(a, ta, tb, k0, k0 + BN - 1);
        if (!all && (scan32<HD>(Ql, tid) || scan32<HD>(Ol, tid))) odd = true;
        if (none_seen(a, ta, tb, kw, kw + 15)) return;
        const bool whole = q0 + FT <= s.ql && all_seen(a, ta, tb, kw, kw + 15);
        f32x4 sa[2], da[2];  // S / dP[q0 + 16 qs + 4 g + e][key]
        bool live[2], dead = false;
#pragma unroll
        for (int qs = 0; qs < 2; ++qs) {
            sa[qs] = da[qs] = f32x4{0, 0, 0, 0};
            live[qs] = whole || !none_seen(a, ta + 16 * qs, min(ta + 16 * qs + 15, s.kl - 1), kw, kw + 15);  // wave-uniform
            if (!live[qs]) continue;
            sa[qs] = head_dot<HD>(Ql + 16 * qs * HD, t, kf);
            da[qs] = head_dot<HD>(Ol + 16 * qs * HD, t, vf);
            const f32x4 l = *reinterpret_cast<const f32x4 *>(Ll + 16 * qs), d = *reinterpret_cast<const f32x4 *>(Dl + 16 * qs);
            // (a row of no gradient has an LSE of -inf: P = 0 for it and, behind the last row, below)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sa[qs][e] = l[e] == -INFINITY ? 0.f : exp_(fmaf(sa[qs][e], a.scale, -l[e]));
                da[qs][e] = l[e] == -INFINITY ? 0.f : sa[qs][e] * (da[qs][e] - d[e]);
                dead = dead || l[e] == -INFINITY;
            }
        }
        if (all && __any(dead) && (scan32<HD>(Ql, tid) || scan32<HD>(Ol, tid))) odd = true;  // (every wave's rows here)
        if (!whole) {
#pragma unroll
            for (int qs = 0; qs < 2; ++qs)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = q0 + 16 * qs + 4 * g + e;
                    if (x >= s.ql || !sees(a, x + s.off, key)) sa[qs][e] = da[qs][e] = 0.f;
                }
        }
        // dV^T += dO^T P, dK^T += Q^T dS
#pragma unroll
        for (int qs = 0; qs < 2; ++qs) {
            if (!live[qs]) continue;
            add_rows<HD>(dvt, Ol + 16 * qs * HD, t, sa[qs]);
            add_rows<HD>(dkt, Ql + 16 * qs * HD, t, da[qs]);
        }
    };
    for (int it0 = 0; it0 < steps; it0 += 2) {
        step(it0, std::integral_constant<int, 0>{});
        if (it0 + 1 < steps) step(it0 + 1, std::integral_constant<int, 1>{});
    }
    float *ws = slot >= 0 ? a.ws + ((long)bk * plan.slots() + slot) * (2 * BN * HD) : nullptr;
    if (__syncthreads_or(odd)) {
        float *sh = tiles[0][0][0] + wave * 2 * HD;
        const Steps st{kvh * nh, qstart, top, nh, false, 1, zpart, zparts};
        if (kg == 0) dkv_rows32(args_again(), st, b, kvh, k0, wave, ws, sh, sh + HD, lane);
        return;
    }
    if constexpr (KG > 1) {
        static_assert(2 * NU * 4 * 256 <= 4 * TILE, "a group's sums fit its tiles");
        auto column = [&](int k, int j) { return reinterpret_cast<f32x4 *>(tiles[k][0][0] + (wave * 2 * NU + j) * 256) + lane; };
        if (kg)
#pragma unroll
            for (int j = 0; j < NU; ++j) *column(kg, j) = dkt[j], *column(kg, NU + j) = dvt[j];
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int k = 1; k < KG; ++k)
#pragma unroll
            for (int j = 0; j < NU; ++j) dkt[j] += *column(k, j), dvt[j] += *column(k, NU + j);
    }
    if (!ws && key >= a.n_kv) return;
    float *dk = ws ? ws + (16 * wave + c) * HD : (float *)a.dk + krow * a.lddk + kvh * HD;
    float *dv = ws ? ws + (BN + 16 * wave + c) * HD : (float *)a.dv + krow * a.lddv + kvh * HD;
    const bool live = key < s.kl;
    acc_cols<NU>(dkt, g, [&](int d, f32x4 x) {
        x = live ? x * a.scale : f32x4{0, 0, 0, 0};
        store4(dk + d, x[0], x[1], x[2], x[3]);
    });
    acc_cols<NU>(dvt, g, [&](int d, f32x4 x) {
        x = live ? x : f32x4{0, 0, 0, 0};
        store4(dv + d, x[0], x[1], x[2], x[3]);
    });
}

bool shape_ok(const WindowArgs &a) { return a.dt == DType::F32 && (a.hd == 64 || a.hd == 128) && a.scale > 0.f && a.scale < INFINITY && a.n_heads < (1 << 16); }
bool ok(const void *p, long ld) { return aligned_rows(p, ld, 16, 4) && ld < (1l << 23); }
bool fwd_ok(const WindowArgs &a) { return shape_ok(a) && ok(a.q, a.ldq) && ok(a.k, a.ldk) && ok(a.v, a.ldv) && ok(a.o, a.ldo); }
// Against the tile kernel, us: 64 rows, window 4096, 16 / 8 heads of 128: 45 against 294; 500 tokens, 4 / 1
// heads (125 tiles) 23 against 43; 300 tokens, 8 / 4 heads of 64: 12 against 17; 8 x 32 rows, window 2048,
// 32 / 4 heads (512 tiles) 80 against 83; 1000 tokens, window 64 (252 tiles) 13.5 against 11.8.
bool few_rows(const WindowArgs &a) { return few_rows_of(a, 512, 192); }
int splits32(const WindowArgs &a) { return step_splits(a, 16, 1024); }
// Two groups of waves a block where the chip has at most two blocks a CU.  One or two groups, forward /
// backward in us: 2 x 1024 tokens, 16 / 16 heads of 128, window 1024 (512 blocks): 111 / 387 and 94 / 315; heads
// of 64: 60 / 211 and 57 / 179; 4 x 1024 tokens, 16 / 8 heads of 64, window 256 (1024 blocks): 51 / 212 and 55 / 215.
bool grouped(const WindowArgs &a) { return (long)a.n_heads * a.n_batch * ((a.n_q + 63) / 64) <= 512; }
bool grouped_dkv(const WindowArgs &a) { return (long)a.n_kv_heads * a.n_batch * ((a.n_kv + 63) / 64) <= 512; }
// Parts of two steps (backward in us, parts of four / of two: 50 tokens, 4 / 2 heads of 128: 41 / 33; 2 x 92, 16 / 8
// heads: 55 / 42), as many as the CUs take at once: two blocks each, one of two groups of 128-wide heads (2 x 473
// tokens, window 18, 16 / 8 heads, one sink: 70 us, with parts for two a CU 90).
DkvPlan plan32(const WindowArgs &a, bool ws) { return dkv_plan(a, ws, 64, grouped_dkv(a) && a.hd == 128 ? 256 : 512, 16, 2, false); }

}  // namespace

size_t window32_fwd_ws_bytes(const WindowArgs &a) { return shape_ok(a) && few_rows(a) ? step_ws_bytes(a, splits32(a)) : 0; }
size_t window32_bwd_ws_bytes(const WindowArgs &a) { return shape_ok(a) ? dkv_ws_bytes(a, plan32(a, true)) : 0; }

bool window32_forward(const WindowArgs &a, hipStream_t st) {
    if (!fwd_ok(a)) return false;
    if (few_rows(a) && (a.n_q <= kFewRows || a.ws)) {
        const int grp = a.n_heads / a.n_kv_heads, splits = a.ws ? splits32(a) : 1;
        const long blocks = (long)a.n_batch * a.n_kv_heads * ((a.n_q * grp + 15) / 16) * splits;
        if (!launchable(blocks, FNT)) return false;
        const dim3 grid((unsigned)blocks);
        if (a.hd == 128) hipLaunchKernelGGL(window_step32_k<128>, grid, dim3(FNT), 0, st, a, splits);
        else hipLaunchKernelGGL(window_step32_k<64>, grid, dim3(FNT), 0, st, a, splits);
        if (splits > 1) a.hd == 128 ? launch_join<128, float>(a, splits, st) : launch_join<64, float>(a, splits, st);
        return true;
    }
    const long blocks = (long)a.n_heads * a.n_batch * ((a.n_q + 63) / 64);
    if (!launchable(blocks, 256)) return false;
    const dim3 grid((unsigned)blocks);
    auto by = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (grouped(a)) hipLaunchKernelGGL((window_fwd32_k<HD, 2>), grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((window_fwd32_k<HD, 1>), grid, dim3(256), 0, st, a);
    };
    if (a.hd == 128) by(std::integral_constant<int, 128>{});
    else by(std::integral_constant<int, 64>{});
    return true;
}

bool window32_backward(const WindowArgs &a, hipStream_t st) {
    if (!fwd_ok(a) || !ok(a.dout, a.lddo) || !ok(a.dq, a.lddq) || !ok(a.dk, a.lddk) || !ok(a.dv, a.lddv)) return false;
    const DkvPlan plan = plan32(a, a.ws != nullptr);
    const long blocks = (long)a.n_heads * a.n_batch * ((a.n_q + 63) / 64);
    if (!launchable(a, plan, blocks, 256)) return false;
    const dim3 gq((unsigned)blocks);
    const dim3 gk((unsigned)((long)a.n_batch * a.n_kv_heads * plan.blocks()));
    auto by = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (grouped(a)) hipLaunchKernelGGL((window_dq32_k<HD, 2>), gq, dim3(512), 0, st, a);
        else hipLaunchKernelGGL((window_dq32_k<HD, 1>), gq, dim3(256), 0, st, a);
        if (hipPeekAtLastError() != hipSuccess) return;  // (D is not there)
        if (grouped_dkv(a)) hipLaunchKernelGGL((window_dkv32_k<HD, 2>), gk, dim3(512), 0, st, a, plan);
        else hipLaunchKernelGGL((window_dkv32_k<HD, 1>), gk, dim3(256), 0, st, a, plan);
        launch_dkv_sum<HD, 64, float>(a, plan, st);
    };
    if (a.hd == 128) by(std::integral_constant<int, 128>{});
    else by(std::integral_constant<int, 64>{});
    return true;
}

}  // namespace vkh
