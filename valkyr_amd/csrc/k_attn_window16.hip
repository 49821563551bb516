// Windowed attention on bf16 operands: the tile kernels (64- and 128-wide heads, aligned rows) of
// the operator that k_attn_window.hip describes.
//
// v_mfma_f32_16x16x32_bf16 with fp32 accumulation; scores are formed transposed where that lets P
// and dS go from the accumulators straight into the next product as its B operand:
//   forward  S^T = K Q^T, O^T += V^T P^T          dQ  S^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   dK/dV    S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// P and dS are rounded to bf16 for those products, as their other operands are (the sum of P that
// divides O is of the unrounded values; the kernel of few rows, which waits for memory, holds P as two bf16
// terms); everything else is fp32.
//
// A block walks only the tiles of its window and, before them, those of the sinks.  Tiles come
// by DMA into swizzled LDS rows, through a buffer resource that is set on the tile's first row:
// its offsets stay small however long the cache is, a lane's offset is the same for every tile,
// and rows past a sequence's end read as zero by the range check.  Masks cost nothing in tiles
// that every row sees in full.  In the others a masked pair has P = dS = 0, selected, and since
// 0 times an infinity or a NaN is NaN, the tile that multiplies them is scanned for such values: a
// block that meets one (none does, in a healthy run) forms its rows anew one at a time, from seen
// pairs only.
#include <algorithm>

#include "attn16.hpp"
#include "window.hpp"

namespace vkh {
namespace {

// Whether any of the thread's share of BYTES of LDS holds an infinity or a NaN: exponent bits of all
// ones, to which one more carries into the sign's place (of either half of a word).
template <int BYTES, int NT>
VKH_DEV bool scan(const char *lds, int tid) {
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < (BYTES + 16 * NT - 1) / (16 * NT); ++i)
        if ((i + 1) * 16 * NT <= BYTES || (i * NT + tid) * 16 < BYTES) {
            const uint4 v = *reinterpret_cast<const uint4 *>(lds + (i * NT + tid) * 16);
#pragma unroll
            for (unsigned w : {v.x, v.y, v.z, v.w}) carry |= (w & 0x7f807f80u) + 0x00800080u;
        }
    return carry & 0x80008000u;
}

// The resource of rows row0 .. row0 + rows - 1 of one head (rows <= 0: of none).
template <int HD>
VKH_DEV sgpr4 head_rows(const void *p, long row0, long ld, int col, int rows) {
    return rsrc4((const bf16 *)p + row0 * ld + col, rows > 0 ? (unsigned)(((rows - 1) * (int)ld + HD) * 2) : 0u);
}
// A lane's byte offset in a DMA of 1 KB: row r0 + lane / (HD / 8) of the tile, its chunk swizzled.
template <int HD>
VKH_DEV unsigned dma_off(int r0, int lane, int ld) {
    const int r = r0 + lane / (HD / 8), c = (lane % (HD / 8)) ^ TileRows<HD>::swz(r);
    return (unsigned)((r * ld + 8 * c) * 2);
}

// A block's rows one at a time, for blocks that met an infinity or a NaN in a tile which some of
// their rows do not see in full (0 times either is NaN).  Out of line: their registers are not the
// tile loops'.
template <class TO>
__device__ __attribute__((noinline)) void fwd_rows(const WindowArgs &a, int b, int r, int end, int step, int h, float *q,
                                                   int lane) {
    for (; r < end; r += step) window_fwd_row<bf16, TO>(a, b, r, h, q, lane);
}
template <class TO>
__device__ __attribute__((noinline)) void dq_rows(const WindowArgs &a, int b, int r, int end, int step, int h, float *q,
                                                  float *g, int lane) {
    for (; r < end; r += step) window_dq_row<bf16, TO>(a, b, r, h, q, g, lane);
}
template <int HD, class TO>
__device__ __attribute__((noinline)) void dkv_rows(const WindowArgs &a, const Steps &st, int b, int kvh, int k0, int wave,
                                                   float *ws, float *k, float *v, int lane) {
    auto mine = [&](int h, int row) { return st.mine(h, row); };
    for (int x = wave; x < 128; x += 8) {
        if (k0 + x >= a.n_kv) {  // (their slots are read)
            for (int d = lane; ws && d < HD; d += 64) ws[x * HD + d] = ws[(128 + x) * HD + d] = 0.f;
            continue;
        }
        const long row = (long)b * a.n_kv + k0 + x;
        if (ws) window_dkv_row<bf16>(a, b, k0 + x, kvh, k, v, ws + x * HD, ws + (128 + x) * HD, lane, mine);
        else window_dkv_row<bf16>(a, b, k0 + x, kvh, k, v, (TO *)a.dk + row * a.lddk + kvh * HD,
                                  (TO *)a.dv + row * a.lddv + kvh * HD, lane, mine);
    }
}

// ── forward ──────────────────────────────────────────────────────────────
// Block = 64 QS query rows of one head, 4 waves of 16 QS; 32-key tiles, three buffers (two tiles on
// their way).  The heaviest (last) rows start first.  Matrix cores, vector ALU and LDS each have about
// as much to do and take turns within a wave, so it is waves that overlap them: 32-key tiles leave
// registers for three a SIMD.  16384 tokens, window 2048, 32 / 8 heads of 128: 513 to 536 us, 1.0 PFLOP/s;
// as first measured 534, 64-key tiles on two waves a SIMD 566, the next tile's scores formed beside this
// one's exponentials (two waves) 710.
// On short grids (64-row blocks) a wave's own chain of steps is the time: heads of 64, whose registers
// allow it, take 64-key tiles there (2048 tokens, window 2048, 8 / 8 heads: 26 against 32 us).
template <int HD, int QS, int KG, class TO>
__global__ __launch_bounds__(256 * KG, KG == 2 ? 2 : HD == 64 && QS == 2 ? 4 : 3) void window_fwd16_k(WindowArgs a) {
    using R = TileRows<HD>;
    constexpr int DS = HD / 32, DSUB = HD / 16, BM = 64 * QS, BN = HD == 64 && QS == 1 ? 64 : 32, KS = BN / 16, TILE = BN * HD * 2, NBUF = 3;
    constexpr int RPI = 512 / HD, IPT = BN / RPI, C = 2 * IPT / 4;  // rows per DMA, DMAs per tile and tensor, per wave
    __shared__ __attribute__((aligned(16))) char Kts[KG][NBUF][TILE], Vts[KG][NBUF][TILE];
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, nqt = (a.n_q + BM - 1) / BM;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4 * grp);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, h = kvh * grp + pr.y % grp, qt = nqt - 1 - pr.y / grp;
    const int tid = threadIdx.x % 256, lane = tid % 64, g = lane / 16, c16 = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), kg = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    char(*Kt)[TILE] = Kts[kg], (*Vt)[TILE] = Vts[kg];
    const Span s = span_of(a, b);
    const int r0 = qt * BM, qw0 = r0 + wave * 16 * QS;
    const KeyTiles kt = key_tiles<BN>(a, s, r0, r0 + BM);
    const int steps = (kt.n + KG - 1) / KG, n = (kt.n - kg + KG - 1) / KG;  // the block's; the group's
    const int wta = max(0, qw0 + s.off), wtb = min(qw0 + 16 * QS, s.ql) - 1 + s.off;
    Reach mine = reach<BN>(a, kt, wta, wtb);
    if (qw0 + 16 * QS > s.ql || qw0 + s.off < 0) mine.n_all = mine.n_sink_all = 0;  // rows that are not there
    const Reach block = reach<BN>(a, kt, kt.ta, kt.tb);
    const float c2 = a.scale * LOG2E;
    const long row0 = (long)b * a.n_q, key0 = (long)b * a.n_kv;

    bf16x8 qf[QS][DS];
    int pos[QS];
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        const int r = qw0 + 16 * qs + c16;
        pos[qs] = r < s.ql ? max(-1, r + s.off) : -1;
        const bf16 *qr = (const bf16 *)a.q + (row0 + r) * a.ldq + h * HD + 8 * g;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) qf[qs][ds] = pos[qs] >= 0 ? ld_frag(qr + 32 * ds) : bf16x8{};
    }
    // the wave's DMAs: number q = C wave + i of the 2 IPT of a tile, K's first
    const bool isk = C * wave < IPT;  // (a wave's DMAs are all K's or all V's)
    const int ld = (int)(isk ? a.ldk : a.ldv), row = C * wave - (isk ? 0 : IPT);
    const bf16 *src = (const bf16 *)(isk ? a.k : a.v) + key0 * ld + kvh * HD;
    const unsigned dst = lds_addr(isk ? Kt[0] : Vt[0]) + row * 1024;
    unsigned off[C];
#pragma unroll
    for (int i = 0; i < C; ++i) off[i] = dma_off<HD>((row + i) * RPI, lane, ld);
    wait_vm0();  // Q fragments are in registers before any DMA is queued
    auto dma = [&](int it, int buf) {
        const int k0 = kt.tile(KG * it + kg) * BN;
        const sgpr4 rs = rsrc4(src + (long)k0 * ld, (unsigned)(((min(BN, s.kl - k0) - 1) * ld + HD) * 2));
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rs, dst + buf * TILE + i * 1024, off[i]);
    };
    static_assert(IPT % C == 0, "a wave's DMAs are of one tensor");
    f32x4 oacc[QS][DSUB], st[KS][QS];
    float m[QS], l[QS];  // running maximum in log2 units; this lane's share of the sum
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        m[qs] = -INFINITY;
        l[qs] = 0.f;
#pragma unroll
        for (int i = 0; i < DSUB; ++i) oacc[qs][i] = f32x4{0, 0, 0, 0};
    }
    auto scores = [&](const char *Kb, f32x4 (&x)[KS][QS]) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) x[ks][qs] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 kf = R::frag_row(Kb, 16 * ks + c16, 32 * ds + 8 * g);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) x[ks][qs] = mfma16x16x32(kf, qf[qs][ds], x[ks][qs]);
            }
    };
    bool odd = false;  // an infinity or a NaN in V of a tile that is not seen in full
    if (n > 0) dma(0, 0);
    if (n > 1) dma(1, 1);
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        const int k0 = kt.tile(KG * it + kg) * BN;
        if (it + 1 < n) wait_vm<C>();
        else wait_vm0();
        lds_barrier();  // tile it landed; everyone is done with tile it - 1
        if (it + 2 < n) dma(it + 2, (buf + 2) % NBUF);
        if (KG > 1 && it >= n) return;
        const char *Kb = Kt[buf], *Vb = Vt[buf];
        if (!block.whole(KG * it + kg) && scan<TILE, 256>(Vb, tid)) odd = true;
        if (mine.none(KG * it + kg)) return;
        scores(Kb, st);
        if (!mine.whole(KG * it + kg)) {
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) for_hidden<KS>(a, pos[qs], k0, g, [&](int ks, int r) { st[ks][qs][r] = -INFINITY; });
        }
        // The maximum that P is taken against moves only when a row's scores pass it by more than 8 (in
        // log2 units): P stays under 2^8, where bf16 and fp32 hold it as exactly, and the accumulators
        // are rescaled in few tiles after the first.  A row's decision is its own.
        float mt[QS];
        bool moved = false;
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            mt[qs] = -INFINITY;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt[qs] = fmaxf(mt[qs], st[ks][qs][r]);
            moved = moved || mt[qs] * c2 > m[qs] + 8.f;
        }
        if (__any(moved)) {
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
                const float mn = xrow_max(mt[qs]) * c2, mo = m[qs];
                if (mn > mo + 8.f) m[qs] = mn;
                const float so = m[qs] == mo ? 1.f : __builtin_amdgcn_exp2f(mo - m[qs]);
                l[qs] *= so;
#pragma unroll
                for (int i = 0; i < DSUB; ++i) oacc[qs][i] *= so;
            }
        }
        bf16x8 pf[KS / 2][QS];
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            const float ms = m[qs] == -INFINITY ? 0.f : m[qs];  // no score above -inf yet: P = 0
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[ks][qs][r], c2, -ms));
                    st[ks][qs][r] = p;
                    l[qs] += p;
                }
#pragma unroll
            for (int ks = 0; ks < KS; ks += 2) pf[ks / 2][qs] = frag_acc(st[ks][qs], st[ks + 1][qs]);
        }
#pragma unroll
        for (int i = 0; i < DSUB; ++i)
#pragma unroll
            for (int k2 = 0; k2 < KS / 2; ++k2) {
                const bf16x8 vf = R::frag_t(Vb, 16 * i, 32 * k2, g, c16);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) oacc[qs][i] = mfma16x16x32(vf, pf[k2][qs], oacc[qs][i]);
            }
    };
    for (int it0 = 0; it0 < steps; it0 += NBUF) {
        step(it0, std::integral_constant<int, 0>{});
        if (it0 + 1 < steps) step(it0 + 1, std::integral_constant<int, 1>{});
        if (it0 + 2 < steps) step(it0 + 2, std::integral_constant<int, 2>{});
    }
    if (__syncthreads_or(odd)) {
        if (kg == 0) fwd_rows<TO>(args_again(), b, r0 + wave, min(r0 + BM, a.n_q), 4, h, (float *)Kts + wave * HD, lane);
        return;
    }
    if constexpr (KG > 1) {  // the groups' results, joined in order through LDS
        constexpr int W = (DSUB + 1) * 64 * 16;  // bytes of a wave's result: columns of 64 lanes
        static_assert(KG == 2 && QS == 1 && 4 * W <= (int)sizeof(Kts), "the results fit the tiles");
        auto column = [&](int j) { return reinterpret_cast<f32x4 *>((char *)Kts + wave * W + j * 1024) + lane; };
        if (kg) {
#pragma unroll
            for (int i = 0; i < DSUB; ++i) *column(i) = oacc[0][i];
            *column(DSUB) = f32x4{m[0], l[0], 0, 0};
        }
        __syncthreads();
        if (kg) return;
        const f32x4 ml = *column(DSUB);
        const float mn = fmaxf(m[0], ml[0]), ms = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m[0] - ms), f1 = __builtin_amdgcn_exp2f(ml[0] - ms);
        m[0] = mn;
        l[0] = l[0] * f0 + ml[1] * f1;
#pragma unroll
        for (int i = 0; i < DSUB; ++i) oacc[0][i] = oacc[0][i] * f0 + *column(i) * f1;
    }
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        const int r = qw0 + 16 * qs + c16;
        const float lt = xrow_sum(l[qs]);
        if (r >= a.n_q) continue;
        const bool dead = lt == 0.f;
        const float inv = 1.0f / lt;
        TO *o = (TO *)a.o + (row0 + r) * a.ldo + h * HD + 4 * g;
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            const f32x4 x = dead ? f32x4{0, 0, 0, 0} : oacc[qs][i] * inv;
            store4(o + 16 * i, x[0], x[1], x[2], x[3]);
        }
        if (a.lse && g == 0)
            a.lse[(row0 + r) * a.n_heads + h] = dead ? -INFINITY : (m[qs] + log2f(lt)) * LN2;
    }
}

// ── forward of a few rows ────────────────────────────────────────────────
// One new token against a cache, or a few: bound by reading K and V.  The rows of all query heads
// of a KV head (row m = query row m / group, head m % group) share each key that is read, 16 at a
// time; each of the 4 waves streams 32-key tiles of its own (two in LDS, no barrier between the
// waves), every fourth of the block's, and their results are joined at the end.  `splits` blocks
// share a KV head's tiles; their results (maximum, sum, O in fp32) go to a.ws and
// window_join_k joins them in order.  32 sequences of up to 32768 tokens, window 4096, 32 / 8 heads of
// 128 (0.52 GB of K and V): 92 to 98 us, 5.3 to 5.6 TB/s, and 4 to join; one sequence, window 1024: 6 and 3,
// two launches' latency.
// acc[i][r] += sum over the tile's rows x that `see` names of T[x][16 i + 4 g + r] w[x], where w is
// held as a B operand: element 4 u + e is row 16 u + 4 g + e.  It goes through `wl`, 1 KB of the
// wave's own LDS.
template <int HD, class See>
VKH_DEV void add_pairs(f32x4 (&acc)[HD / 16], const char *T, const bf16x8 &w, bf16x8 *wl, int lane, See see) {
    const int g = lane / 16, c16 = lane % 16;
    wl[lane] = w;
    wave_lds();
#pragma unroll 1
    for (int x = 0; x < 32; ++x) {
        const float wx = (float)reinterpret_cast<const bf16 *>(wl + x % 16 / 4 * 16 + c16)[x / 16 * 4 + x % 4];
        if (!see(x)) continue;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            const bf16x4 t = *reinterpret_cast<const bf16x4 *>(T + TileRows<HD>::toff(x, 16 * i + 4 * g));
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][r] = fmaf((float)t[r], wx, acc[i][r]);
        }
    }
}
template <int HD, class TO>
__global__ __launch_bounds__(256, 1) void window_step16_k(WindowArgs a, int splits) {
    using R = TileRows<HD>;
    constexpr int DS = HD / 32, DSUB = HD / 16, BN = 32, TILE = BN * HD * 2, RPI = 512 / HD, IPT = BN / RPI;
    constexpr int RL = HD + 4;  // floats of a result row in LDS
    __shared__ __attribute__((aligned(16))) char tiles[4][2][2][TILE];
    __shared__ bf16x8 wl[4][64];
    __shared__ float ml[4][2][16];
    static_assert(16 * RL * 4 <= 4 * TILE, "a wave's result fits its tiles");
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, M = a.n_q * grp, RT = (M + 15) / 16;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, rt = pr.y % RT, split = pr.y / RT;
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c16 = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const Span s = span_of(a, b);
    const KeyTiles kt = key_tiles<BN>(a, s, rt * 16 / grp, (min(M, rt * 16 + 16) - 1) / grp + 1);
    const int per = (kt.n + splits - 1) / splits, last = min(kt.n, (split + 1) * per);
    const float c2 = a.scale * LOG2E;
    const long key0 = (long)b * a.n_kv;
    char *Kt = tiles[wave][0][0], *Vt = tiles[wave][1][0];

    const int m16 = rt * 16 + c16, row = m16 / grp, h = kvh * grp + m16 % grp;
    const int pos = m16 < M && row < s.ql ? max(-1, row + s.off) : -1;
    bf16x8 qf[DS];
    {
        const bf16 *qr = (const bf16 *)a.q + ((long)b * a.n_q + row) * a.ldq + h * HD + 8 * g;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) qf[ds] = pos >= 0 ? ld_frag(qr + 32 * ds) : bf16x8{};
    }
    unsigned ko[IPT], vo[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
        ko[i] = dma_off<HD>(RPI * i, lane, (int)a.ldk);
        vo[i] = dma_off<HD>(RPI * i, lane, (int)a.ldv);
    }
    const bool live = __all(pos >= 0);
    wait_vm0();
    auto dma = [&](int it, int buf) {
        const int k0 = kt.tile(it) * BN, rows = min(BN, s.kl - k0);
        const sgpr4 rk = head_rows<HD>(a.k, key0 + k0, a.ldk, kvh * HD, rows);
        const sgpr4 rv = head_rows<HD>(a.v, key0 + k0, a.ldv, kvh * HD, rows);
#pragma unroll
        for (int i = 0; i < IPT; ++i) dma16_at(rk, lds_addr(Kt + buf * TILE + i * 1024), ko[i]);
#pragma unroll
        for (int i = 0; i < IPT; ++i) dma16_at(rv, lds_addr(Vt + buf * TILE + i * 1024), vo[i]);
    };
    f32x4 acc[DSUB];
#pragma unroll
    for (int i = 0; i < DSUB; ++i) acc[i] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;
    const int it0 = split * per + wave;
    if (it0 < last) dma(it0, 0);
    if (it0 + 4 < last) dma(it0 + 4, 1);
    for (int it = it0, buf = 0; it < last; it += 4, buf ^= 1) {
        const int k0 = kt.tile(it) * BN;
        const char *Kb = Kt + buf * TILE, *Vb = Vt + buf * TILE;
        // its K and V are here (the next tile's may still be on their way)
        if (it + 4 < last) wait_vm<2 * IPT>();
        else wait_vm0();
        asm volatile("" ::: "memory");
        const bool whole = live && all_seen(a, kt.ta, kt.tb, k0, k0 + BN - 1);
        f32x4 st[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
                st[ks] = mfma16x16x32(R::frag_row(Kb, 16 * ks + c16, 32 * ds + 8 * g), qf[ds], st[ks]);
        if (!whole) for_hidden<2>(a, pos, k0, g, [&](int ks, int r) { st[ks][r] = -INFINITY; });
        float mt = -INFINITY;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int r = 0; r < 4; ++r) mt = fmaxf(mt, st[ks][r]);
        if (__any(mt * c2 > m + 8.f)) {  // (as in the forward above)
            const float mn = xrow_max(mt) * c2, mo = m;
            if (mn > mo + 8.f) m = mn;
            const float so = m == mo ? 1.f : __builtin_amdgcn_exp2f(mo - m);
            l *= so;
#pragma unroll
            for (int i = 0; i < DSUB; ++i) acc[i] *= so;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(st[ks][r], c2, -ms));
                st[ks][r] = p;
                l += p;
            }
        // P as two bf16 terms: rounded once it is off by as much as O's own rounding (O in bf16 off by 0.0020 to
        // 0.0023 of its norm in place of 0.0017), and the second product hides behind the reading of K and V
        // (99.5 against 99.2 us on the 32 sequences above; calls of more rows 1 to 2.5 %)
        const bf16x8 pf = frag_acc(st[0], st[1]);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int r = 0; r < 4; ++r) st[ks][r] -= (float)pf[4 * ks + r];
        const bf16x8 pl = frag_acc(st[0], st[1]);
        if (!whole && __any(scan<TILE, 64>(Vb, lane))) {
            auto see = [&](int x) { return sees(a, pos, k0 + x); };
            add_pairs<HD>(acc, Vb, pf, wl[wave], lane, see);
            wave_lds();
            add_pairs<HD>(acc, Vb, pl, wl[wave], lane, see);
        } else {
#pragma unroll
            for (int i = 0; i < DSUB; ++i) {
                const bf16x8 vf = R::frag_t(Vb, 16 * i, 0, g, c16);
                acc[i] = mfma16x16x32(vf, pf, acc[i]);
                acc[i] = mfma16x16x32(vf, pl, acc[i]);
            }
        }
        if (it + 8 < last) {
            wave_lds();  // this buffer's reads are done
            dma(it + 8, buf);
        }
    }
    // the four waves' results: rows of HD floats over their own tiles, maximum and sum beside them
    wave_lds();
    float *res = reinterpret_cast<float *>(tiles[wave]);
    const float lt = xrow_sum(l);
#pragma unroll
    for (int i = 0; i < DSUB; ++i) *reinterpret_cast<f32x4 *>(res + c16 * RL + 16 * i + 4 * g) = acc[i];
    if (g == 0) ml[wave][0][c16] = m, ml[wave][1][c16] = lt;
    __syncthreads();
    constexpr int E = HD / 16;  // values per thread
    const int r = tid / 16, d0 = tid % 16 * E;
    float mx = -INFINITY, sum = 0.f, o[E] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[w][0][r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float lw = ml[w][1][r], f = lw == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[w][0][r] - (mx == -INFINITY ? 0.f : mx));
        if (lw == 0.f) continue;
        sum = fmaf(lw, f, sum);
        const float *src = reinterpret_cast<const float *>(tiles[w]) + r * RL + d0;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(src[e], f, o[e]);
    }
    const int mr = rt * 16 + r;
    if (mr >= M) return;
    const long orow = (long)b * a.n_q + mr / grp;
    const int oh = kvh * grp + mr % grp;
    if (splits > 1) {  // [split][row][head]: HD values; behind them all, maximum and sum
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
    TO *out = (TO *)a.o + orow * a.ldo + oh * HD + d0;
#pragma unroll
    for (int e = 0; e < E; e += 4) store4(out + e, o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
    if (a.lse && d0 == 0) a.lse[orow * a.n_heads + oh] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * LN2;
}

// ── backward: D and dQ ───────────────────────────────────────────────────
// Block = BQ query rows of one head on 4 waves of 16 QSUB rows, whose Q and dO fragments stay in
// registers; 32-key tiles of K and V through three buffers (two in flight, the wait counted).
// D = rowsum(O dO) of the block's rows is formed first (fp64 sums of the bf16 products) and
// stored for the dK/dV kernel, which runs after this one.  As the forward, it is bound by what a wave
// does between its products (softmax, rounding, LDS reads) and by masked tiles: 16384 tokens, window
// 2048, 32 / 8 heads of 128: 760 to 773 us, 1.0 PFLOP/s; 4 x 2048, window 512, 16 / 8 heads: 77 us, 0.59 PFLOP/s.  KG = 2 (short
// grids: one block a CU): two groups of waves take every other tile; 2048 tokens, window 2048, 8 / 8
// heads of 64, forward / backward: 24.8 / 73 us without, 19.3 / 63 with.
template <int HD, int BQ, int KG, class TO>
__global__ __launch_bounds__(256 * KG, 2) void window_dq16_k(WindowArgs a) {
    using R = TileRows<HD>;
    constexpr int NWV = 4;
    constexpr int QSUB = BQ / 16 / NWV, BN = 32, KS = 2, NBUF = 3, TILE = BN * HD * 2;
    constexpr int DS = HD / 32, DSUB = HD / 16, NF = 2 * DS;
    constexpr int RPI = 512 / HD, IPT = BN / RPI, C = 2 * IPT / NWV;  // DMAs per tile and tensor, per wave
    static_assert(C >= 1 && C * NWV == 2 * IPT, "DMA share");
    __shared__ __attribute__((aligned(16))) char Kts[KG][NBUF][TILE], Vts[KG][NBUF][TILE];
    const int nbk = a.n_batch * a.n_kv_heads, grp = a.n_heads / a.n_kv_heads, nqb = (a.n_q + BQ - 1) / BQ;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4 * grp);
    const int b = pr.bk / a.n_kv_heads, kvh = pr.bk % a.n_kv_heads, h = kvh * grp + pr.y % grp, qb = nqb - 1 - pr.y / grp;
    const int tid = threadIdx.x % 256, lane = tid % 64, g = lane / 16, c16 = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64), kg = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
    char(*Kt)[TILE] = Kts[kg], (*Vt)[TILE] = Vts[kg];
    const Span s = span_of(a, b);
    const int r0 = qb * BQ, qw0 = r0 + wave * 16 * QSUB;
    const KeyTiles kt = key_tiles<BN>(a, s, r0, r0 + BQ);
    const int steps = (kt.n + KG - 1) / KG, nt = (kt.n - kg + KG - 1) / KG;  // the block's; the group's
    const int wta = max(0, qw0 + s.off), wtb = min(qw0 + 16 * QSUB, s.ql) - 1 + s.off;
    Reach mine = reach<BN>(a, kt, wta, wtb);
    const Reach block = reach<BN>(a, kt, kt.ta, kt.tb);
    const float c2 = a.scale * LOG2E;
    const long row0 = (long)b * a.n_q, key0 = (long)b * a.n_kv;

    bf16x8 qr[QSUB][DS], orr[QSUB][DS];
    float lq[QSUB], dd[QSUB];
    int pos[QSUB];
#pragma unroll
    for (int j = 0; j < QSUB; ++j) {
        const int r = qw0 + 16 * j + c16;
        const long t = row0 + r;
        const float l = r < s.ql && r + s.off >= 0 ? a.lse[t * a.n_heads + h] : -INFINITY;
        const bool live = l != -INFINITY;  // no gradient for a row whose scores are all -inf either
        pos[j] = live ? r + s.off : -1;
        lq[j] = l * LOG2E;
        const bf16 *qp = (const bf16 *)a.q + t * a.ldq + h * HD + 8 * g;
        const bf16 *gp = (const bf16 *)a.dout + t * a.lddo + h * HD + 8 * g;
        const TO *op = (const TO *)a.o + t * a.ldo + h * HD + 8 * g;
        double acc = 0;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            qr[j][ds] = live ? ld_frag(qp + 32 * ds) : bf16x8{};
            orr[j][ds] = live ? ld_frag(gp + 32 * ds) : bf16x8{};
            if (live) {
                typedef TO vec __attribute__((ext_vector_type(8)));
                const vec o = *reinterpret_cast<const vec *>(op + 32 * ds);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc += (double)(float)o[e] * (double)(float)orr[j][ds][e];
            }
        }
        acc += __shfl_xor(acc, 16, 64);
        acc += __shfl_xor(acc, 32, 64);
        dd[j] = (float)acc;
        if (r < a.n_q && g == 0 && kg == 0) a.d[t * a.n_heads + h] = dd[j];
    }
    bool live = true;
#pragma unroll
    for (int j = 0; j < QSUB; ++j) live = live && pos[j] >= 0;
    if (!__all(live)) mine.n_all = mine.n_sink_all = 0;  // rows of no gradient
    // the wave's DMAs: number q = C wave + i of the 2 IPT of a tile, K's first
    const bool isk = C * wave < IPT;  // (a wave's DMAs are all K's or all V's)
    const int ld = (int)(isk ? a.ldk : a.ldv), row = C * wave - (isk ? 0 : IPT);
    const bf16 *src = (const bf16 *)(isk ? a.k : a.v) + key0 * ld + kvh * HD;
    const unsigned dst = lds_addr(isk ? Kt[0] : Vt[0]) + row * 1024;
    unsigned off[C];
#pragma unroll
    for (int i = 0; i < C; ++i) off[i] = dma_off<HD>((row + i) * RPI, lane, ld);
    wait_vm0();
    auto dma = [&](int it, int buf) {
        const int k0 = kt.tile(KG * it + kg) * BN;
        const sgpr4 rs = rsrc4(src + (long)k0 * ld, (unsigned)(((min(BN, s.kl - k0) - 1) * ld + HD) * 2));
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rs, dst + buf * TILE + i * 1024, off[i]);
    };
    static_assert(IPT % C == 0, "a wave's DMAs are of one tensor");
    f32x4 acc[QSUB][DSUB];
#pragma unroll
    for (int j = 0; j < QSUB; ++j)
#pragma unroll
        for (int i = 0; i < DSUB; ++i) acc[j][i] = f32x4{0, 0, 0, 0};
    if (nt > 0) dma(0, 0);
    if (nt > 1) dma(1, 1);
    // unrolled over the three buffers: every LDS address is a lane's base plus a constant
    bool odd = false;  // an infinity or a NaN in K of a tile that is not seen in full
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        if (it + 1 < nt) wait_vm<C>();
        else wait_vm0();
        lds_barrier();
        if (it + 2 < nt) dma(it + 2, (buf + 2) % NBUF);
        if (KG > 1 && it >= nt) return;
        const int k0 = kt.tile(KG * it + kg) * BN;
        const char *Kb = Kt[buf], *Vb = Vt[buf];
        if (!block.whole(KG * it + kg) && scan<TILE, NWV * 64>(Kb, tid)) odd = true;
        if (mine.none(KG * it + kg)) return;
        // the dP^T accumulators start at -D (one query per lane), so they end as dP^T - D
        f32x4 st[KS][QSUB], dpt[KS][QSUB];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < QSUB; ++j) {
                st[ks][j] = f32x4{0, 0, 0, 0};
                dpt[ks][j] = f32x4{-dd[j], -dd[j], -dd[j], -dd[j]};
            }
        // The three phases walk their operand fragments in one sequence (K rows for S^T, V rows
        // for dP^T, transposed K for dQ^T), each slot's LDS read issued PD slots ahead of its MFMAs.
        constexpr int PD = 2, RING = PD + 1;
        auto ldslot = [&](int n) -> bf16x8 {
            if (n < NF) return R::frag_row(Kb, 16 * (n % 2) + c16, 32 * (n / 2) + 8 * g);
            if (n < 2 * NF) return R::frag_row(Vb, 16 * ((n - NF) % 2) + c16, 32 * ((n - NF) / 2) + 8 * g);
            return R::frag_t(Kb, 16 * (n - 2 * NF), 0, g, c16);
        };
        bf16x8 fr[RING];
#pragma unroll
        for (int n = 0; n < PD; ++n) fr[n] = ldslot(n);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            fr[(f + PD) % RING] = ldslot(f + PD);
#pragma unroll
            for (int j = 0; j < QSUB; ++j) st[f % 2][j] = mfma16x16x32(fr[f % RING], qr[j][f / 2], st[f % 2][j]);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int n = NF + f;
            fr[(n + PD) % RING] = ldslot(n + PD);
#pragma unroll
            for (int j = 0; j < QSUB; ++j) dpt[f % 2][j] = mfma16x16x32(fr[n % RING], orr[j][f / 2], dpt[f % 2][j]);
            // P^T = exp2(S^T c - lse) of one (ks, j) tile rides along
            constexpr int EVERY = NF / (KS * QSUB);
            static_assert(EVERY >= 1 && EVERY * KS * QSUB == NF, "exp schedule");
            if (f % EVERY == 0) {
                const int t2 = f / EVERY, ks2 = t2 / QSUB, j2 = t2 % QSUB;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    st[ks2][j2][r] = __builtin_amdgcn_exp2f(fmaf(st[ks2][j2][r], c2, -lq[j2]));
            }
        }
        const bool whole = mine.whole(KG * it + kg);
        bf16x8 sb[QSUB];
#pragma unroll
        for (int j = 0; j < QSUB; ++j) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int r = 0; r < 4; ++r) dpt[ks][j][r] = st[ks][j][r] * dpt[ks][j][r];
            if (!whole) for_hidden<KS>(a, pos[j], k0, g, [&](int ks, int r) { dpt[ks][j][r] = 0.f; });
            sb[j] = frag_acc(dpt[0][j], dpt[1][j]);
        }
        // dQ^T += K^T dS^T
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            const int n = 2 * NF + i;
            if (n + PD < 2 * NF + DSUB) fr[(n + PD) % RING] = ldslot(n + PD);
#pragma unroll
            for (int j = 0; j < QSUB; ++j) acc[j][i] = mfma16x16x32(fr[n % RING], sb[j], acc[j][i]);
        }
    };
    for (int t0 = 0; t0 < steps; t0 += NBUF) {
        step(t0, std::integral_constant<int, 0>{});
        if (t0 + 1 < steps) step(t0 + 1, std::integral_constant<int, 1>{});
        if (t0 + 2 < steps) step(t0 + 2, std::integral_constant<int, 2>{});
    }
    if (__syncthreads_or(odd)) {
        if (kg) return;
        float *sh = (float *)Kts + wave * 2 * HD;
        dq_rows<TO>(args_again(), b, r0 + wave, min(r0 + BQ, a.n_q), NWV, h, sh, sh + HD, lane);
        return;
    }
    if constexpr (KG > 1) {  // the groups' sums, added through LDS
        static_assert(KG == 2 && QSUB == 1 && 4 * DSUB * 1024 <= (int)sizeof(Kts), "the sums fit the tiles");
        auto column = [&](int j) { return reinterpret_cast<f32x4 *>((char *)Kts + (wave * DSUB + j) * 1024) + lane; };
        if (kg) {
#pragma unroll
            for (int i = 0; i < DSUB; ++i) *column(i) = acc[0][i];
        }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int i = 0; i < DSUB; ++i) acc[0][i] += *column(i);
    }
#pragma unroll
    for (int j = 0; j < QSUB; ++j) {
        const int r = qw0 + 16 * j + c16;
        if (r >= a.n_q) continue;
        TO *dq = (TO *)a.dq + (row0 + r) * a.lddq + h * HD + 4 * g;
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            const f32x4 x = pos[j] >= 0 ? acc[j][i] * a.scale : f32x4{0, 0, 0, 0};
            store4(dq + 16 * i, x[0], x[1], x[2], x[3]);
        }
    }
}

// ── backward: dK and dV ──────────────────────────────────────────────────
// Block = 128 keys of one KV head; 8 waves = 4 slices of 32 keys x 2 groups.  A wave holds K of its
// slice in registers (V of the block sits in LDS) and takes 32-query tiles of the query heads that
// share the KV head: group 0 every other head, group 1 the rest, or for an odd number of heads
// alternate query tiles of every head.  Each group streams its Q and dO tiles through three
// buffers.  Query tiles run from the first row that sees the block's first key to the last in
// its window, or to the last row of all where the block holds sinks (unless window_far16_k takes
// the rows past their window); such a block has a share of work as many times the others' as the
// sequence is longer than the window, and is split between `sink_parts` blocks, as the others are between
// `parts` where they are too few for the chip.  Parts write fp32 sums
// to their slots of a.ws, which window_dkv_sum_k adds in order.  Bound by the one block a CU that
// the dK and dV accumulators (2 x 32 x HD a wave) and their registers leave: eight waves, half of whose
// time goes to waiting for each other and for LDS.  16384 tokens, window 2048, 32 / 8 heads of 128: 1140
// us, 0.91 PFLOP/s; 4 x 2048, window 512, 16 / 8 heads: 112 us, 0.54 PFLOP/s.
template <int HD, class TO>
__global__ __launch_bounds__(512, 1) void window_dkv16_k(WindowArgs a, DkvPlan plan) {
    using R = TileRows<HD>;
    constexpr int NS = 4, BM = 32, BN = 128, KW = 32, KS = 2, QS = 2, NBUF = 3, TILE = BM * HD * 2;
    constexpr int STREAM = NBUF * 2 * TILE, DS = HD / 32, DSUB = HD / 16, NF = 2 * DS;
    constexpr int XSLOT = DSUB * KS * 64 * 16;  // one wave's dK^T or dV^T
    constexpr int LDS = 8 * XSLOT > 2 * STREAM + BN * HD * 2 ? 8 * XSLOT : 2 * STREAM + BN * HD * 2;
    constexpr int RPI = 512 / HD, C = 16 / RPI;  // rows per DMA; a wave's DMAs per tile (16 rows)
    __shared__ __attribute__((aligned(16))) char smem[LDS];
    __shared__ __attribute__((aligned(16))) float Ls[2][NBUF][64], Dd[2][NBUF][64];

    const int nbk = a.n_batch * a.n_kv_heads;
    const Pair pr = pair_of(blockIdx.x, gridDim.x, nbk, 4);
    const int bk = pr.bk, b = bk / a.n_kv_heads, kvh = bk % a.n_kv_heads;
    int kb, zpart, zparts, slot;
    dkv_block(plan, pr.y, kb, zpart, zparts, slot);
    const int hpk = a.n_heads / a.n_kv_heads;
    const bool alt = hpk & 1;
    const int nh = alt ? hpk : hpk / 2;  // heads per group
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c16 = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int sl = wave % NS, hg = wave / NS;
    const bool tdo = sl >= NS / 2;  // this wave moves dO and D (else Q and LSE), rows 16 part ..
    const int part = sl % (NS / 2);
    const Span s = span_of(a, b);
    const int k0 = kb * BN, kw0 = k0 + sl * KW;
    const float c2 = a.scale * LOG2E;
    const long row0 = (long)b * a.n_q, key0 = (long)b * a.n_kv;

    // K of the slice as B operands (keys past the end read the last row: not stored)
    bf16x8 kr[KS][DS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const bf16 *kp = (const bf16 *)a.k + (key0 + min(kw0 + 16 * ks + c16, a.n_kv - 1)) * a.ldk + kvh * HD + 8 * g;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) kr[ks][ds] = ld_frag(kp + 32 * ds);
    }
    char *vsl = smem + 2 * STREAM + sl * KW * HD * 2;
    if (hg == 0) {
        const sgpr4 rv = head_rows<HD>(a.v, key0 + kw0, a.ldv, kvh * HD, min(KW, s.kl - kw0));
#pragma unroll
        for (int i = 0; i < KW / RPI; ++i) dma16_at(rv, lds_addr(vsl + i * 1024), dma_off<HD>(RPI * i, lane, (int)a.ldv));
    }
    wait_vm0();
    __syncthreads();
    f32x4 dvt[KS][DSUB], dkt[KS][DSUB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < DSUB; ++i) dvt[ks][i] = dkt[ks][i] = f32x4{0, 0, 0, 0};

    const int k1 = min(k0 + BN, s.kl) - 1;  // the block's last key
    const int qstart = max(0, k0 - s.off);
    const int qend = k0 < a.n_sink ? s.ql : (int)min((long)s.ql, (long)k1 + a.window - s.off);
    const int nqt = k1 >= k0 && qend > qstart ? (qend - qstart + BM - 1) / BM : 0;
    const int nsteps = nh * (alt ? (nqt + 1) / 2 : nqt);
    const int niter = max(0, (nsteps - zpart + zparts - 1) / zparts);
    char *strm = smem + hg * STREAM;
    // A cursor runs over the block's steps zpart, zpart + zparts, ... of (query tile, head), heads
    // inner: the group's first row and head (of the KV head's) of a step.
    struct Cursor {
        int h, q0;
    };
    const int span = alt ? 2 * BM : BM, dh = zparts % nh * (alt ? 1 : 2), dq = zparts / nh * span;
    auto advance = [&](Cursor &c) {
        c.h += dh;
        c.q0 -= dq;
        if (c.h >= hpk) c.h -= hpk, c.q0 -= span;
    };
    const int top = alt ? (nqt + 1) / 2 * 2 - 1 : nqt - 1;  // the last tile (alt: of a pair)
    Cursor ahead{zpart % nh * (alt ? 1 : 2) + (alt ? 0 : hg), qstart + (top - (alt ? hg : 0)) * BM - zpart / nh * span};
    Cursor now = ahead;
    // C DMAs per wave and tile, and one more for the waves that move LSE or D.  (The lane id is
    // laundered so that the offsets are formed here rather than held in registers across the loop:
    // spilled, their reloads would wait for the DMA in flight.)
    const int ldt = (int)(tdo ? a.lddo : a.ldq);
    const bf16 *tp = (const bf16 *)(tdo ? a.dout : a.q) + (row0 + 16 * part) * ldt + kvh * hpk * HD;
    const float *sp = (tdo ? a.d : a.lse) + row0 * a.n_heads + kvh * hpk;
    const unsigned dst = lds_addr(strm) + (tdo ? TILE : 0) + part * 16 * HD * 2;
    const unsigned dst_stat = lds_addr(tdo ? Dd[hg][0] : Ls[hg][0]);
    auto dma = [&](int buf) {
        const int rows = s.ql - ahead.q0 - 16 * part;
        const sgpr4 rt = rsrc4(tp + (long)ahead.q0 * ldt + ahead.h * HD, rows > 0 ? (unsigned)(((min(rows, 16) - 1) * ldt + HD) * 2) : 0u);
        int ln = lane;
        asm volatile("" : "+v"(ln));
        // row r = RPI i + ln / (HD / 8) of the 16, chunk ln % (HD / 8) ^ swz(r): the part of i is 4 i
        const unsigned x = (unsigned)(ln % (HD / 8) ^ ln / 16) * 16, ro = __umul24(ln / (HD / 8), 2 * ldt);
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rt, dst + buf * 2 * TILE + i * 1024, (x ^ 64 * i) + (ro + i * RPI * 2 * ldt));
        if (part == 0) {
            const sgpr4 rs = rsrc4(sp + (long)ahead.q0 * a.n_heads + ahead.h, rows > 0 ? (unsigned)(((min(rows, BM) - 1) * a.n_heads + 1) * 4) : 0u);
            dma4_at(rs, dst_stat + buf * 256, ln < BM ? (unsigned)__umul24(ln, a.n_heads * 4) : kOOB);
        }
        advance(ahead);
    };
    const RowReach block = row_reach<BM>(a, s, k0, k0 + BN - 1), mine = row_reach<BM>(a, s, kw0, kw0 + KW - 1);
    if (niter > 0) dma(0);
    if (niter > 1) dma(1);
    bool odd = false;  // an infinity or a NaN in Q or dO of a tile whose rows do not all see all keys, or have no gradient
    auto step = [&](const int it, auto bufc) {
        constexpr int buf = decltype(bufc)::value;
        if (it + 1 < niter) {
            if (part == 0) wait_vm<C + 1>();
            else wait_vm<C>();
        } else {
            wait_vm0();
        }
        lds_barrier();
        if (it + 2 < niter) dma((buf + 2) % NBUF);
        const int q0 = now.q0;
        advance(now);
        const char *Qb = strm + buf * 2 * TILE, *Ob = Qb + TILE;
        if (!block.whole(q0)) odd |= scan<2 * TILE, 256>(Qb, tid % 256);
        if (!mine.some(q0)) return;
        auto dval = [&](int qs, int r) { return Dd[hg][buf][16 * qs + 4 * g + r]; };
        auto prob = [&](float x, int qs, int r) {
            return __builtin_amdgcn_exp2f(fmaf(x, c2, -(Ls[hg][buf][16 * qs + 4 * g + r] * LOG2E)));
        };
        // the dP accumulators start at -D, so they end as dP - D
        f32x4 sc[QS][KS], dp[QS][KS];
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            const f32x4 nd{-dval(qs, 0), -dval(qs, 1), -dval(qs, 2), -dval(qs, 3)};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                sc[qs][ks] = f32x4{0, 0, 0, 0};
                dp[qs][ks] = nd;
            }
        }
        // each phase's next fragment is read ahead of this one's MFMAs; the arithmetic of one score
        // tile rides along with each step of the phase after it
        bf16x8 fr[2];
        fr[0] = R::frag_row(Qb, c16, 8 * g);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int ds = f / 2, qs = f % 2, n = f + 1;
            fr[n & 1] = n < NF ? R::frag_row(Qb, 16 * (n % 2) + c16, 32 * (n / 2) + 8 * g) : R::frag_row(Ob, c16, 8 * g);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) sc[qs][ks] = mfma16x16x32(fr[f & 1], kr[ks][ds], sc[qs][ks]);
        }
        bf16x8 vf[KS];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int ds = f / 2, qs = f % 2, n = f + 1;
            if (qs == 0)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) vf[ks] = R::frag_row(vsl, 16 * ks + c16, 32 * ds + 8 * g);
            fr[n & 1] = n < NF ? R::frag_row(Ob, 16 * (n % 2) + c16, 32 * (n / 2) + 8 * g) : R::frag_t(Ob, 0, 0, g, c16);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dp[qs][ks] = mfma16x16x32(fr[f & 1], vf[ks], dp[qs][ks]);
            constexpr int EVERY = NF / (QS * KS);
            static_assert(EVERY >= 1 && EVERY * QS * KS == NF, "exp schedule");
            if (f % EVERY == 0) {
                const int t2 = f / EVERY, qs2 = t2 / KS, ks2 = t2 % KS;
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[qs2][ks2][r] = prob(sc[qs2][ks2][r], qs2, r);
            }
        }
        const bool dead = __any(lane < BM && Ls[hg][buf][lane % BM] == -INFINITY);  // a row of no gradient
        if (dead || !mine.whole(q0)) {
            if (block.whole(q0)) odd |= scan<2 * TILE, 256>(Qb, tid % 256);  // (every wave of the group is here)
#pragma unroll
            for (int qs = 0; qs < QS; ++qs)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = q0 + 16 * qs + 4 * g + r;
                    const bool live = row < s.ql && Ls[hg][buf][16 * qs + 4 * g + r] != -INFINITY;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
                        if (!sees(a, live ? row + s.off : -1, kw0 + 16 * ks + c16)) sc[qs][ks][r] = dp[qs][ks][r] = 0.f;
                }
        }
        bf16x8 pb[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) pb[ks] = frag_acc(sc[0][ks], sc[1][ks]);
        // dV^T += dO^T P, with dS = P (dP - D)
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            const int n = i + 1;
            fr[n & 1] = n < DSUB ? R::frag_t(Ob, 16 * n, 0, g, c16) : R::frag_t(Qb, 0, 0, g, c16);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dvt[ks][i] = mfma16x16x32(fr[i & 1], pb[ks], dvt[ks][i]);
            constexpr int EVERY = DSUB / (QS * KS);
            static_assert(EVERY >= 1 && EVERY * QS * KS == DSUB, "dS schedule");
            if (i % EVERY == 0) {
                const int t2 = i / EVERY, qs2 = t2 / KS, ks2 = t2 % KS;
#pragma unroll
                for (int r = 0; r < 4; ++r) dp[qs2][ks2][r] = sc[qs2][ks2][r] * dp[qs2][ks2][r];
            }
        }
        // dK^T += Q^T dS
        bf16x8 sb[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) sb[ks] = frag_acc(dp[0][ks], dp[1][ks]);
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            if (i + 1 < DSUB) fr[(i + 1) & 1] = R::frag_t(Qb, 16 * (i + 1), 0, g, c16);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dkt[ks][i] = mfma16x16x32(fr[i & 1], sb[ks], dkt[ks][i]);
        }
    };
    for (int it0 = 0; it0 < niter; it0 += NBUF) {
        step(it0, std::integral_constant<int, 0>{});
        if (it0 + 1 < niter) step(it0 + 1, std::integral_constant<int, 1>{});
        if (it0 + 2 < niter) step(it0 + 2, std::integral_constant<int, 2>{});
    }
    float *ws = slot >= 0 ? a.ws + ((long)bk * plan.slots() + slot) * (2 * BN * HD) : nullptr;
    if (__syncthreads_or(odd)) {
        float *sh = (float *)smem + wave * 2 * HD;
        const Steps st{kvh * hpk, qstart, top, nh, alt, 2, zpart, zparts};
        dkv_rows<HD, TO>(args_again(), st, b, kvh, k0, wave, ws, sh, sh + HD, lane);
        return;
    }
    // the two groups' sums through the (now idle) tile arena: group 0 hands over dK^T and keeps dV^T
    wait_vm0();
    __syncthreads();
    f32x4 *xs = reinterpret_cast<f32x4 *>(smem + (sl * 2 + hg) * XSLOT);
    const f32x4 *xp = reinterpret_cast<const f32x4 *>(smem + (sl * 2 + (1 - hg)) * XSLOT);
    auto give = [&](const f32x4 (&x)[KS][DSUB]) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < DSUB; ++i) xs[(i * KS + ks) * 64 + lane] = x[ks][i];
    };
    if (hg == 0) give(dkt);
    else give(dvt);
    __syncthreads();
    auto keep = [&](const f32x4 (&x)[KS][DSUB], auto *base, long ld, bool raw, float mul) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int key = sl * KW + 16 * ks + c16;  // of the block
            if (!raw && k0 + key >= a.n_kv) continue;
            const bool live = k0 + key < s.kl;
            auto *out = base + key * ld + 4 * g;
#pragma unroll
            for (int i = 0; i < DSUB; ++i) {
                const f32x4 v = live ? (x[ks][i] + xp[(i * KS + ks) * 64 + lane]) * mul : f32x4{0, 0, 0, 0};
                store4(out + 16 * i, v[0], v[1], v[2], v[3]);
            }
        }
    };
    if (ws) {
        if (hg == 0) keep(dvt, ws + BN * HD, HD, true, 1.f);
        else keep(dkt, ws, HD, true, a.scale);
        return;
    }
    if (hg == 0) keep(dvt, (TO *)a.dv + (key0 + k0) * a.lddv + kvh * HD, a.lddv, false, 1.f);
    else keep(dkt, (TO *)a.dk + (key0 + k0) * a.lddk + kvh * HD, a.lddk, false, a.scale);
}

// ── backward: dK and dV of the sinks from rows past their window ─────────
// A wave holds 16 or 32 sinks' K and V in registers and streams 32-query tiles of its own (Q and dO, two
// tiles in LDS, no barrier between the waves) from the first row past a sink's window to the last,
// over the query heads of the KV head; the block's four waves and then the blocks' parts are added in
// order.  The key blocks leave these pairs out: with them, the sink blocks' steps past the window, for
// which three waves of four had nothing to do, took 1442 us of dK/dV to 1177 without (16384 tokens,
// window 2048, 4 sinks, 32 / 8 heads of 128).  Bound by reading Q and dO
// once more (51 to 56 us there, 5 TB/s); on shorter sequences by the chain of loads, steps and join (4 x 2048
// tokens, window 512, 16 / 8 heads: 18 us; with 32 sinks a wave, 4 of them there, 20).
template <int HD, int KS>
__global__ __launch_bounds__(256, 1) void window_far16_k(WindowArgs a, DkvPlan plan) {
    using R = TileRows<HD>;
    constexpr int NK = 16 * KS, QS = 2, BM = 32, TILE = BM * HD * 2, DS = HD / 32, DSUB = HD / 16, RPI = 512 / HD, C = BM / RPI;
    __shared__ __attribute__((aligned(16))) char tiles[4][2][2 * TILE];
    __shared__ __attribute__((aligned(16))) float stat[4][2][2][64];  // LSE and D of a tile's rows
    __shared__ bf16x8 wl[4][64];
    const int nbk = a.n_batch * a.n_kv_heads, hpk = a.n_heads / a.n_kv_heads;
    const int bk = blockIdx.x % nbk, b = bk / a.n_kv_heads, kvh = bk % a.n_kv_heads;
    const int slice = blockIdx.x / nbk % plan.far_slices, part = blockIdx.x / nbk / plan.far_slices;
    const int tid = threadIdx.x, lane = tid % 64, g = lane / 16, c16 = lane % 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const Span s = span_of(a, b);
    const int k0 = NK * slice, nk = min(min(a.n_sink, s.kl) - k0, NK);  // this slice's sinks
    const float c2 = a.scale * LOG2E;
    const long row0 = (long)b * a.n_q, key0 = (long)b * a.n_kv;
    unsigned qo[C], go[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        qo[i] = dma_off<HD>(RPI * i, lane, (int)a.ldq);
        go[i] = dma_off<HD>(RPI * i, lane, (int)a.lddo);
    }
    const unsigned so = lane < BM ? (unsigned)(lane * a.n_heads * 4) : kOOB;
    f32x4 dvt[KS][DSUB], dkt[KS][DSUB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < DSUB; ++i) dvt[ks][i] = dkt[ks][i] = f32x4{0, 0, 0, 0};
    const int qstart = max(0, k0 + a.window - s.off);  // the first row past the first sink's window
    const int nqt = nk > 0 && s.ql > qstart ? (s.ql - qstart + BM - 1) / BM : 0, n = nqt * hpk;
    const int step = 4 * plan.far_parts;
    wait_vm0();
    auto dma = [&](int it, int buf) {
        const int h = kvh * hpk + it % hpk, q0 = qstart + it / hpk * BM, rows = min(BM, s.ql - q0);
        const sgpr4 rq = head_rows<HD>(a.q, row0 + q0, a.ldq, h * HD, rows);
        const sgpr4 rg = head_rows<HD>(a.dout, row0 + q0, a.lddo, h * HD, rows);
        const long at = (row0 + q0) * a.n_heads + h;
        const unsigned bytes = (unsigned)(((rows - 1) * a.n_heads + 1) * 4);
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rq, lds_addr(tiles[wave][buf] + i * 1024), qo[i]);
#pragma unroll
        for (int i = 0; i < C; ++i) dma16_at(rg, lds_addr(tiles[wave][buf] + TILE + i * 1024), go[i]);
        dma4_at(rsrc4(a.lse + at, bytes), lds_addr(stat[wave][buf][0]), so);
        dma4_at(rsrc4(a.d + at, bytes), lds_addr(stat[wave][buf][1]), so);
    };
    const int it0 = 4 * part + wave;
    if (it0 < n) dma(it0, 0);
    if (it0 + step < n) dma(it0 + step, 1);
    bf16x8 kr[KS][DS], vr[KS][DS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const long row = key0 + min(k0 + 16 * ks + c16, a.n_kv - 1);
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            kr[ks][ds] = ld_frag((const bf16 *)a.k + row * a.ldk + kvh * HD + 8 * g + 32 * ds);
            vr[ks][ds] = ld_frag((const bf16 *)a.v + row * a.ldv + kvh * HD + 8 * g + 32 * ds);
        }
    }
    for (int it = it0, buf = 0; it < n; it += step, buf ^= 1) {
        const int q0 = qstart + it / hpk * BM;
        const char *Qb = tiles[wave][buf], *Ob = Qb + TILE;
        const float *L = stat[wave][buf][0], *D = stat[wave][buf][1];
        if (it + step < n) wait_vm<2 * C + 2>();
        else wait_vm0();
        asm volatile("" ::: "memory");
        // whether row q0 + x is past the window of key (ks, c16); all rows' past all keys'
        auto far = [&](int x, int ks) { return q0 + x < s.ql && q0 + x + s.off - k0 - 16 * ks - c16 >= a.window; };
        const bool whole = q0 + BM <= s.ql && q0 + s.off - k0 - NK + 1 >= a.window;
        f32x4 sc[QS][KS], dp[QS][KS];
        bool dead = false;
#pragma unroll
        for (int qs = 0; qs < QS; ++qs)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) sc[qs][ks] = dp[qs][ks] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
                const bf16x8 fq = R::frag_row(Qb, 16 * qs + c16, 32 * ds + 8 * g), fo = R::frag_row(Ob, 16 * qs + c16, 32 * ds + 8 * g);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    sc[qs][ks] = mfma16x16x32(fq, kr[ks][ds], sc[qs][ks]);
                    dp[qs][ks] = mfma16x16x32(fo, vr[ks][ds], dp[qs][ks]);
                }
            }
#pragma unroll
        for (int qs = 0; qs < QS; ++qs)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int x = 16 * qs + 4 * g + r;
                const float l2 = L[x] * LOG2E, d = D[x];
                dead = dead || L[x] == -INFINITY;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bool on = L[x] != -INFINITY && (whole || far(x, ks));  // (-inf: no gradient)
                    const float p = __builtin_amdgcn_exp2f(fmaf(sc[qs][ks][r], c2, -l2));
                    sc[qs][ks][r] = on ? p : 0.f;
                    dp[qs][ks][r] = on ? p * (dp[qs][ks][r] - d) : 0.f;
                }
            }
        // the first tiles hold rows that are past some sinks' windows only; any tile may hold rows of no gradient
        const bool odd = (!whole || __any(dead)) && __any(scan<2 * TILE, 64>(Qb, lane));
        bf16x8 pb[KS], sb[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            pb[ks] = frag_acc(sc[0][ks], sc[1][ks]);
            sb[ks] = frag_acc(dp[0][ks], dp[1][ks]);
        }
        if (odd) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                add_pairs<HD>(dvt[ks], Ob, pb[ks], wl[wave], lane, [&](int x) { return L[x] != -INFINITY && far(x, ks); });
                wave_lds();
                add_pairs<HD>(dkt[ks], Qb, sb[ks], wl[wave], lane, [&](int x) { return L[x] != -INFINITY && far(x, ks); });
                wave_lds();
            }
        } else {
#pragma unroll
            for (int i = 0; i < DSUB; ++i) {
                const bf16x8 fo = R::frag_t(Ob, 16 * i, 0, g, c16), fq = R::frag_t(Qb, 16 * i, 0, g, c16);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    dvt[ks][i] = mfma16x16x32(fo, pb[ks], dvt[ks][i]);
                    dkt[ks][i] = mfma16x16x32(fq, sb[ks], dkt[ks][i]);
                }
            }
        }
        if (it + 2 * step < n) {
            wave_lds();  // this buffer's reads are done
            dma(it + 2 * step, buf);
        }
    }
    // the four waves' sums, each [dK, dV][NK][HD] floats over its own tiles
    wave_lds();
    static_assert(2 * NK * HD * 4 <= (int)sizeof(tiles[0]), "a wave's sums fit its tiles");
    float *mine = reinterpret_cast<float *>(tiles[wave]);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < DSUB; ++i) {
            *reinterpret_cast<f32x4 *>(mine + (16 * ks + c16) * HD + 16 * i + 4 * g) = dkt[ks][i] * a.scale;
            *reinterpret_cast<f32x4 *>(mine + (NK + 16 * ks + c16) * HD + 16 * i + 4 * g) = dvt[ks][i];
        }
    __syncthreads();
    float *ws = a.ws + (long)nbk * plan.slots() * (2 * 128 * HD) + (((long)bk * plan.far_slices + slice) * plan.far_parts + part) * (2 * NK * HD);
#pragma unroll
    for (int i = 0; i < 2 * NK * HD / 1024; ++i) {
        const int x = (i * 256 + tid) * 4;
        f32x4 t{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) t += *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(tiles[w]) + x);
        if (x / HD % NK >= nk) t = f32x4{0, 0, 0, 0};
        *reinterpret_cast<f32x4 *>(ws + x) = t;
    }
}

// Heads of 64 or 128 values in rows of aligned 16-byte chunks, a tile's rows within 31 bits of
// offset, and a scale that keeps the order of the scores.
bool shape_ok(const WindowArgs &a) {
    return a.dt == DType::BF16 && (a.hd == 64 || a.hd == 128) && a.scale > 0.f && a.scale < INFINITY &&
           std::max({a.ldq, a.ldk, a.ldv, a.lddo}) < (1l << 23) && a.n_heads < (1 << 16);
}
bool fwd_ok(const WindowArgs &a) {
    const int es = a.odt == DType::F32 ? 4 : 2;
    return shape_ok(a) && aligned_rows(a.q, a.ldq, 16, 2) && aligned_rows(a.k, a.ldk, 16, 2) && aligned_rows(a.v, a.ldv, 16, 2) && aligned_rows(a.o, a.ldo, 4 * es, es);
}
bool bwd_ok(const WindowArgs &a) {
    const int es = a.odt == DType::F32 ? 4 : 2;
    return fwd_ok(a) && aligned_rows(a.dout, a.lddo, 16, 2) && aligned_rows(a.o, a.ldo, 16, es) && aligned_rows(a.dq, a.lddq, 4 * es, es) &&
           aligned_rows(a.dk, a.lddk, 4 * es, es) && aligned_rows(a.dv, a.lddv, 4 * es, es);
}

// Against the tile kernel, us: 64 / 24 rows, window 4096, 16 / 8 heads of 128: 22 against 48, 17.5
// against 52; 200 rows, 2000 keys, 8 / 8 heads of 64 (104 tiles) 12.5 against 19; 500 tokens, 4 / 1 heads
// (125 tiles) 14.3 against 11.1; 8 x 16 rows, window 2048, 32 / 4 heads of 64 (256 tiles) 28.5 against 25.5.
bool few_rows(const WindowArgs &a) { return few_rows_of(a, 192, 1536); }
// two rounds of one block per CU
int splits16(const WindowArgs &a) { return step_splits(a, 32, 512); }
// dK/dV: one block per CU, at least two steps of both groups each (of four / of two, backward in us: 2 x 2989
// tokens, window 9, 3 / 1 heads: 64 / 55; 300 tokens, 8 / 4 heads of 64: 25 / 23; 4 x 430, 4 / 4 heads: 37 / 38)
DkvPlan plan16(const WindowArgs &a, bool ws) { return dkv_plan(a, ws, 128, 256, 8, 4, true); }

// Two groups of waves a block where the chip has at most one block a CU (up to two: 1 x 4096 tokens, window
// 512, 8 / 8 heads of 128, 512 blocks: forward 30 us with two groups, 24 with one).
bool grouped(const WindowArgs &a) { return (long)a.n_heads * a.n_batch * ((a.n_q + 63) / 64) <= cu_count(); }

}  // namespace

size_t window16_fwd_ws_bytes(const WindowArgs &a) { return shape_ok(a) && few_rows(a) ? step_ws_bytes(a, splits16(a)) : 0; }
size_t window16_bwd_ws_bytes(const WindowArgs &a) {
    if (!shape_ok(a)) return 0;
    return dkv_ws_bytes(a, plan16(a, true));
}

bool window16_forward(const WindowArgs &a, hipStream_t st) {
    if (!fwd_ok(a)) return false;
    if (few_rows(a) && (a.n_q <= kFewRows || a.ws)) {
        const int grp = a.n_heads / a.n_kv_heads, rt = (a.n_q * grp + 15) / 16, splits = a.ws ? splits16(a) : 1;
        const long blocks = (long)a.n_batch * a.n_kv_heads * rt * splits;
        if (!launchable(blocks, 256)) return false;
        auto by = [&](auto hd, auto to) {
            constexpr int HD = decltype(hd)::value;
            using TO = decltype(to);
            hipLaunchKernelGGL((window_step16_k<HD, TO>), dim3((unsigned)blocks), dim3(256), 0, st, a, splits);
            if (splits > 1) launch_join<HD, TO>(a, splits, st);
        };
        auto by_head = [&](auto to) {
            if (a.hd == 128) by(std::integral_constant<int, 128>{}, to);
            else by(std::integral_constant<int, 64>{}, to);
        };
        a.odt == DType::F32 ? by_head(float{}) : by_head(bf16{});
        return true;
    }
    const long per = (long)a.n_heads * a.n_batch;
    // 64-row blocks where 128-row ones would be two a CU or fewer, with small windows (more of whose tiles are
    // masked in part) four of 128-wide heads.  With 128 / 64 rows, us: 5000 tokens, window 256, 8 / 8 heads of 64 (320
    // blocks of 128): 16 / 12; 3377, window 2000, 16 / 8 heads of 128 (432): 67 / 60; 4 x 2048 (1024), windows 64, 256,
    // 512, 2048: 35.5 / 32.5, 47 / 43, 61 / 59, 94 / 100, heads of 64, window 512: 33 / 37; 16384, window 256: 173 / 196.
    const long blocks = per * ((a.n_q + 127) / 128);
    const bool small = blocks <= 2l * cu_count() || (a.hd == 128 && a.window <= 512 && blocks <= 4l * cu_count()), pairs = grouped(a);
    if (!launchable(small ? per * ((a.n_q + 63) / 64) : blocks, 256)) return false;
    auto go = [&](auto kernel, int bm, int kg) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(per * ((a.n_q + bm - 1) / bm))), dim3(256 * kg), 0, st, a);
    };
    auto by = [&](auto hd, auto to) {
        constexpr int HD = decltype(hd)::value;
        using TO = decltype(to);
        if (pairs) go(window_fwd16_k<HD, 1, 2, TO>, 64, 2);
        else if (small) go(window_fwd16_k<HD, 1, 1, TO>, 64, 1);
        else go(window_fwd16_k<HD, 2, 1, TO>, 128, 1);
    };
    auto by_head = [&](auto to) {
        if (a.hd == 128) by(std::integral_constant<int, 128>{}, to);
        else by(std::integral_constant<int, 64>{}, to);
    };
    a.odt == DType::F32 ? by_head(float{}) : by_head(bf16{});
    return true;
}

bool window16_backward(const WindowArgs &a, hipStream_t st) {
    if (!bwd_ok(a)) return false;
    const long per = (long)a.n_heads * a.n_batch, nbk = (long)a.n_batch * a.n_kv_heads;
    // 128-row dQ blocks on 4 waves, two a CU (256 rows on 8 waves, one a CU, wait for each other over
    // twice the span of masked tiles: 16384 tokens, window 2048, 996 against 881 us; 4 x 2048, window
    // 512, 112 against 90); 64 rows where those would be less than two a CU (backward of 3377 tokens, window
    // 2000, 16 / 8 heads: 227 us with 128, 219 with 64; of 2 x 4096, window 800, 8 / 4 heads, 512 blocks of
    // 128: 140 and 146), and on windows whose tiles are masked in large part (16384 tokens, window 256, 621
    // and 596; 4 x 2048, window 512, 224 and 222; window 1024, 294 and 298)
    const int bq = per * ((a.n_q + 127) / 128) >= 2l * cu_count() && a.window > 512 ? 128 : 64;
    const DkvPlan plan = plan16(a, a.ws != nullptr);
    if (!launchable(a, plan, per * ((a.n_q + bq - 1) / bq), 256)) return false;
    auto by = [&](auto hd, auto to) {
        constexpr int HD = decltype(hd)::value;
        using TO = decltype(to);
        auto dq = [&](auto kernel, int kg) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)(per * ((a.n_q + bq - 1) / bq))), dim3(256 * kg), 0, st, a);
        };
        if (bq == 128) dq(window_dq16_k<HD, 128, 1, TO>, 1);
        else if (grouped(a)) dq(window_dq16_k<HD, 64, 2, TO>, 2);
        else dq(window_dq16_k<HD, 64, 1, TO>, 1);
        if (hipPeekAtLastError() != hipSuccess) return;  // (D is not there)
        WindowArgs near = a;
        if (plan.far_parts) {
            near.n_sink = 0;
            const dim3 grid((unsigned)(nbk * plan.far_slices * plan.far_parts));
            if (plan.far_keys == 16) hipLaunchKernelGGL((window_far16_k<HD, 1>), grid, dim3(256), 0, st, a, plan);
            else hipLaunchKernelGGL((window_far16_k<HD, 2>), grid, dim3(256), 0, st, a, plan);
        }
        hipLaunchKernelGGL((window_dkv16_k<HD, TO>), dim3((unsigned)(nbk * plan.blocks())), dim3(512), 0, st, near, plan);
        launch_dkv_sum<HD, 128, TO>(a, plan, st);
    };
    auto by_head = [&](auto to) {
        if (a.hd == 128) by(std::integral_constant<int, 128>{}, to);
        else by(std::integral_constant<int, 64>{}, to);
    };
    a.odt == DType::F32 ? by_head(float{}) : by_head(bf16{});
    return true;
}

}  // namespace vkh
