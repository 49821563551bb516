"""Attention with a sliding window and sinks through the C ABI against its formula in 64 bits.

Bars (relative 2-norm of each output): fp32 1e-5, the repository's bar for fp32 sums.  bf16
operands round P (and dS) once, half a step of 2^-8, which O, dQ, dK and dV feel as sums of
independent roundings, and gradients feel O's rounding through D: 2^-8 for fp32 outputs' O, 2 * 2^-8
for their gradients, and 2^-8 more where the outputs are bf16 themselves.  The log-sum-exp is fp32
from exact products of its operands: |S| of hd terms is within (hd / 16 + 8) 2^-24 sum |q k| scale
(16 partial sums side by side, then their own), and the sum's logarithm adds 8 * 2^-24.  dP - D
cancels where a row sees few keys (one key: dS = 0): both are fp32 sums of hd terms, so whatever they
are rounded to, dQ and dK may be off by the products of (hd / 16 + 8) 2^-24 P (sum |dO v| + sum |dO O|)
with |K| and |Q| as well ("edq", "edk").  And P = exp(S - LSE) holds the roundings of S and LSE to fp32,
one step of |LSE| for both: 2 * 2^-24 |LSE| more on everything ("large").
"""
import math

import numpy as np
import pytest

from helpers import bf16_dev, dev, host, note, rel_l2

U, U16 = 2.0 ** -24, 2.0 ** -8


def refused(call, *args, **kw):
    import valkyr_amd as v

    with pytest.raises(v.VkhError) as e:
        call(*args, **kw)
    return e.value.name


# ── refusals (no GPU) ────────────────────────────────────────────────────

def test_call_refusals():
    """Arguments are checked before any device work (the addresses here are not memory)."""
    from valkyr_amd import kernels as K

    def both(*a, **kw):
        p = K.window_params(*a, **kw)
        names = {refused(K.fa_window_forward, p, 256, 256, 256, 256, 256),
                 refused(K.fa_window_backward, p, *([256] * 10))}
        assert K.fa_window_forward_workspace_bytes(p) == K.fa_window_backward_workspace_bytes(p) == 0
        assert len(names) == 1
        return names.pop()

    assert both(0, 4, 2, 1, 64) == "InvalidArgument"
    assert both(4, 0, 2, 1, 64) == "InvalidArgument"
    assert both(4, 4, 3, 2, 64) == "InvalidArgument"
    assert both(5, 4, 2, 1, 64) == "InvalidArgument"  # more queries than keys
    assert both(4, 4, 2, 1, 64, dtype=2) == "InvalidArgument"
    assert both(4, 4, 2, 1, 64, dtype=K.F32, out_dtype=K.BF16) == "InvalidArgument"
    assert both(4, 4, 2, 1, 64, ld_q=127) == "InvalidArgument"
    assert both(4, 4, 2, 1, 64, ld_dv=63) == "InvalidArgument"
    assert both(4, 4, 2, 1, 257) == "Unsupported"
    assert both(4, 1 << 30, 2, 1, 64) == "Unsupported"
    assert both(1 << 16, 1 << 16, 2, 1, 64, n_batch=1 << 15) == "Unsupported"
    p = K.window_params(4, 4, 2, 1, 64, 2, 1)
    args = [256] * 10
    for i in range(4):
        for bad in (None, 258):
            a = args[:4]
            a[i] = bad
            assert refused(K.fa_window_forward, p, *a) == "InvalidArgument"
    assert refused(K.fa_window_forward, p, *args[:4], 258) == "InvalidArgument"  # lse
    for i in range(10):
        for bad in (None, 258):
            a = args[:]
            a[i] = bad
            assert refused(K.fa_window_backward, p, *a) == "InvalidArgument"
    one = K.window_params(1, 65536, 8, 1, 128, dtype=K.BF16)
    assert refused(K.fa_window_forward, one, 256, 256, 256, 257) == "InvalidArgument"
    if K.fa_window_forward_workspace_bytes(one):
        assert refused(K.fa_window_forward, one, *([256] * 5), workspace=264) == "InvalidArgument"


# ── the formula ──────────────────────────────────────────────────────────

def visible(nq, nk, ql, kl, window, sinks):
    """[n_q, n_kv] truth: which keys a query row sees."""
    t = np.arange(nq)[:, None] + kl - ql
    j = np.arange(nk)[None, :]
    see = (j <= t) & (j < kl) & (np.arange(nq)[:, None] < ql)
    return see & ((j > t - window) | (j < sinks)) if window else see


def attention64(q, k, v, do, see, scale):
    """One sequence: q, do [nq, H, hd], k, v [nk, Hkv, hd].  Rows of k, v, q and do that no visible pair
    names are not looked at."""
    nq, H, hd = q.shape
    g = H // k.shape[1]
    k, v = (np.where(see.any(0)[:, None, None], x, 0) for x in (k, v))
    q, do = (np.where(see.any(1)[:, None, None], x, 0) for x in (q, do))
    o, lse = np.zeros_like(q), np.full((nq, H), -np.inf)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    size, edq, edk = np.zeros((nq, H)), np.zeros_like(q), np.zeros_like(k)
    for h in range(H):
        s = np.where(see, q[:, h] @ k[:, h // g].T * scale, -np.inf)
        m = s.max(1, keepdims=True)
        m = np.where(np.isfinite(m), m, 0)
        e = np.exp(s - m)
        total = e.sum(1, keepdims=True)
        p = np.divide(e, total, out=np.zeros_like(e), where=total > 0)
        with np.errstate(divide="ignore"):
            lse[:, h] = (m + np.log(total))[:, 0]
        o[:, h] = p @ v[:, h // g]
        dp = do[:, h] @ v[:, h // g].T
        ds = p * (dp - (do[:, h] * o[:, h]).sum(1, keepdims=True)) * scale
        dq[:, h] = ds @ k[:, h // g]
        dk[:, h // g] += ds.T @ q[:, h]
        dv[:, h // g] += p.T @ do[:, h]
        size[:, h] = np.where(see, np.abs(q[:, h]) @ np.abs(k[:, h // g]).T * scale, 0).max(1)
        e = p * (np.abs(do[:, h]) @ np.abs(v[:, h // g]).T + (np.abs(do[:, h] * o[:, h])).sum(1, keepdims=True)) * scale
        e *= (hd / 16 + 8) * U
        edq[:, h] = e @ np.abs(k[:, h // g])
        edk[:, h // g] += e.T @ np.abs(q[:, h])
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv, size=size, edq=edq, edk=edk)


class Call:
    """One attention call's buffers and its values in 64 bits."""

    def __init__(self, b, nq, nk, H, Hkv, hd, window, sinks, form, lens=None, pad=0, seed=0, spoil=None, fused=False):
        from valkyr_amd import kernels as K

        self.K, self.shape, self.form = K, (b, nq, nk, H, Hkv, hd, window, sinks), form
        rng = np.random.default_rng(seed)
        self.bf, self.obf = form != "fp32", form == "bf16"
        ql, kl = lens if lens else ([nq] * b, [nk] * b)
        self.ql, self.kl = np.minimum(ql, nq), np.minimum(kl, nk)
        self.scale = 1 / math.sqrt(hd)
        vals = dict(q=rng.standard_normal((b, nq, H, hd)) * 1.5, k=rng.standard_normal((b, nk, Hkv, hd)) * 1.5,
                    v=rng.standard_normal((b, nk, Hkv, hd)), do=rng.standard_normal((b, nq, H, hd)))
        if spoil:
            spoil(vals)
        self.pad = {n: pad for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv")}
        up = {}
        for n, x in vals.items():
            width = x.shape[2] * hd
            m = np.full((x.shape[0] * x.shape[1], width + pad), np.nan if pad else 0, np.float32)
            m[:, :width] = x.reshape(-1, width)
            up[n], w = bf16_dev(m) if self.bf else (dev(m), m)
            vals[n] = np.asarray(w, np.float64)[:, :width].reshape(x.shape)
        self.vals, self.up = vals, up
        self.lens = dict(q_len=dev(np.array(ql, np.uint32)), kv_len=dev(np.array(kl, np.uint32))) if lens else {}
        ld = {f"ld_{n}": (H if n in ("q", "o", "do", "dq") else Hkv) * hd + pad for n in self.pad} if pad else {}
        self.p = K.window_params(nq, nk, H, Hkv, hd, window, sinks, n_batch=b, dtype=int(self.bf),
                                 out_dtype=int(self.obf), **ld)
        self.out = {n: self.empty(n) for n in ("o", "dq", "dk", "dv")}
        self.lse, self.d = (dev(np.full(b * nq * H, 7.0, np.float32)) for _ in range(2))

    def empty(self, n):
        b, nq, nk, H, Hkv, hd = self.shape[:6]
        rows, width = (b * nq, H * hd) if n in ("o", "dq") else (b * nk, Hkv * hd)
        x = np.full((rows, width + self.pad[n]), 7.0, np.float32)
        return bf16_dev(x)[0] if self.obf else dev(x)

    def forward(self, **kw):
        u = self.up
        self.K.fa_window_forward(self.p, u["q"], u["k"], u["v"], self.out["o"], self.lse, **self.lens, **kw)

    def backward(self, **kw):
        u, o = self.up, self.out
        self.K.fa_window_backward(self.p, u["q"], u["k"], u["v"], o["o"], u["do"], self.lse, self.d, o["dq"], o["dk"],
                                  o["dv"], **self.lens, **kw)

    def read(self):
        from valkyr_amd.device import bf16_bits_to_f32

        b, nq, nk, H, Hkv, hd = self.shape[:6]
        got = {}
        for n, buf in self.out.items():
            x = bf16_bits_to_f32(host(buf, dtype=np.uint16)) if self.obf else host(buf)
            rows, heads = (nq, H) if n in ("o", "dq") else (nk, Hkv)
            x = x.reshape(b * rows, heads * hd + self.pad[n])
            assert np.all(x[:, heads * hd:] == 7.0), n  # between the rows
            got[n] = x[:, :heads * hd].reshape(b, rows, heads, hd).astype(np.float64)
        got["lse"] = host(self.lse).reshape(b, nq, H).astype(np.float64)
        return got

    def want(self):
        b, nq, nk, H, Hkv, hd, window, sinks = self.shape
        each = [attention64(*(self.vals[n][i] for n in ("q", "k", "v", "do")),
                            visible(nq, nk, self.ql[i], self.kl[i], window, sinks), self.scale) for i in range(b)]
        return {n: np.stack([e[n] for e in each]) for n in each[0]}

    def bar(self, n):
        if self.form == "fp32":
            return 1e-5
        return (1 if n == "o" else 2) * U16 + (U16 if self.obf else 0)

    def check(self, got, want, names=("o", "lse", "dq", "dk", "dv")):
        hd = self.shape[5]
        dead = np.isneginf(want["lse"])
        large = 2 * U * np.abs(want["lse"][~dead]).max(initial=0)
        for n in names:
            if n == "lse":
                assert np.array_equal(dead, np.isneginf(got["lse"]))
                off = np.abs(np.where(dead, 0, got["lse"]) - np.where(dead, 0, want["lse"]))[~dead]
                assert np.all(off <= ((hd / 16 + 8) * U * want["size"] + 8 * U * (1 + np.abs(want["lse"])))[~dead])
                continue
            zero = ~want[n].any(-1) & ~want.get("e" + n, want[n]).any(-1)  # rows of nothing are exact zeros
            assert not got[n][zero].any(), n
            slack = np.linalg.norm(want["e" + n]) if "e" + n in want else 0.0
            off, size = np.linalg.norm(got[n] - want[n]), np.linalg.norm(want[n])
            assert off <= (self.bar(n) + large) * size + slack, (n, off, size, slack)


FORMS = ["fp32", "bf16", "bf16-fp32"]
# batch, n_q, n_kv, heads, kv heads, head_dim, window, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 128, 1, 0),
    (2, 1, 300, 4, 2, 128, 64, 4),
    (1, 1, 700, 8, 1, 64, 0, 0),
    (2, 4, 513, 6, 2, 128, 200, 70),
    (1, 3, 70, 4, 4, 64, 7, 1),
    (1, 65, 65, 2, 1, 128, 64, 0),
    (2, 129, 129, 4, 2, 128, 33, 5),
    (1, 200, 200, 3, 1, 64, 1, 1),
    (1, 100, 357, 6, 3, 64, 65, 130),
    (2, 257, 257, 4, 1, 128, 128, 1),
    (1, 300, 300, 2, 2, 64, 0, 0),
    (1, 321, 400, 4, 2, 128, 500, 3),
    (1, 330, 330, 4, 2, 64, 90, 600),
    (1, 13, 1200, 8, 1, 64, 500, 2),
    (2, 16, 300, 6, 2, 128, 40, 35),
    (1, 17, 300, 6, 2, 128, 40, 35),
    # other head widths
    (1, 37, 50, 4, 2, 32, 20, 2),
    (2, 33, 33, 2, 1, 80, 9, 1),
    (1, 20, 90, 2, 1, 256, 40, 3),
    (1, 18, 18, 3, 3, 7, 5, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s))
def test_matches_the_formula(shape, form):
    note(f"window attention {shape} {form}")
    c = Call(*shape, form)
    c.forward()
    c.backward()
    c.check(c.read(), c.want())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("hd,pad", [(64, 0), (128, 64), (128, 1), (40, 3)])
@pytest.mark.parametrize("nq,nk,window,sinks,ql,kl", [
    (130, 130, 50, 3, [130, 0, 1, 65, 64], [130, 0, 1, 65, 64]),   # a padded training batch
    (2, 333, 100, 4, [2, 2, 2, 1, 2], [333, 1, 0, 77, 200]),       # caches of any length, some shorter than the rows
    (150, 400, 0, 0, [150, 9, 150, 400, 20], [400, 260, 149, 150, 4000]),  # values beyond the room are the room's
])
def test_lengths_and_strides(nq, nk, window, sinks, ql, kl, hd, pad, form):
    note(f"window attention lens {ql} {kl} hd={hd} pad={pad} {form}")

    def spoil(v):  # memory behind each sequence's end holds anything
        for i, (a, b) in enumerate(zip(ql, kl)):
            v["k"][i, b:] = v["v"][i, b:] = np.nan
            v["q"][i, a:] = v["do"][i, a:] = np.inf

    c = Call(5, nq, nk, 4, 2, hd, window, sinks, form, lens=(ql, kl), pad=pad, spoil=spoil)
    c.forward()
    c.backward()
    c.check(c.read(), c.want())


# grids of more blocks than the chip has CUs (by 64 and by 128 rows), more than one group's steps, and
# longer calls whose few rows' tiles see many keys
LARGER = [
    (1, 700, 700, 32, 8, 64, 130, 3),
    (1, 1100, 1100, 32, 8, 128, 600, 70),
    (1, 1100, 1100, 64, 8, 128, 600, 70),
    (1, 1100, 1100, 64, 16, 64, 700, 3),
    (1, 1100, 1100, 32, 32, 64, 90, 1),
    (2, 520, 520, 32, 32, 64, 40, 40),
    (1, 1030, 1030, 32, 32, 128, 200, 100),
    (1, 90, 2000, 4, 2, 128, 1900, 70),
    (2, 200, 1700, 3, 1, 64, 0, 0),
    (1, 40, 700, 8, 4, 64, 300, 5),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", LARGER, ids=lambda s: "-".join(str(x) for x in s))
def test_larger_calls(shape, form, ragged):
    note(f"larger window attention {shape} {form} {ragged}")
    b, nq, nk = shape[:3]
    ql, kl = [nq - 45 * i - 7 for i in range(b)], [nk - 77 * i - 30 for i in range(b)]

    def spoil(v):
        for i in range(b if ragged else 0):
            v["k"][i, kl[i]:] = v["v"][i, kl[i]:] = np.nan
            v["q"][i, ql[i]:] = v["do"][i, ql[i]:] = np.inf

    c = Call(*shape, form, lens=(ql, kl) if ragged else None, spoil=spoil)
    c.forward()
    c.backward()
    c.check(c.read(), c.want())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, -np.inf])
@pytest.mark.parametrize("form", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1100, 1100, 32, 8, 64, 600, 3), (1, 1100, 1100, 64, 8, 128, 600, 3), (1, 700, 700, 32, 32, 128, 48, 2), (1, 1100, 1100, 32, 32, 64, 90, 40),
                                   (1, 90, 2000, 4, 2, 128, 1600, 3),
                                   (1, 40, 700, 4, 2, 64, 250, 1)], ids=lambda s: "-".join(str(x) for x in s))
def test_what_is_not_seen_reaches_nothing_in_larger_calls(shape, form, bad):
    """As below, on the larger calls' kernels: one key's and one query's rows hold infinities or NaN."""
    b, nq, nk, H, Hkv, hd, window, sinks = shape
    note(f"larger window attention unseen {shape} {form} {bad}")
    jbad, rbad = nk - nq + nq // 3, nq // 2

    def spoil(v):
        v["k"][:, jbad], v["v"][:, jbad] = bad, bad
        v["q"][:, rbad], v["do"][:, rbad] = bad, bad

    c, clean = Call(*shape, form, spoil=spoil), Call(*shape, form)
    for x in (c, clean):
        x.forward()
        x.backward()
    got, want = c.read(), clean.want()
    see = visible(nq, nk, nq, nk, window, sinks)
    rows = ~see[:, jbad]
    rows[rbad] = False
    keys = ~see[rbad]
    keys[jbad] = False
    keys &= ~see[see[:, jbad]].any(0)
    assert rows.any()
    for n in ("o", "lse", "dq"):
        want[n], got[n] = want[n][:, rows], got[n][:, rows]
    want["size"], want["edq"], want["edk"] = want["size"][:, rows], want["edq"][:, rows], want["edk"][:, keys]
    for n in ("dk", "dv"):
        want[n], got[n] = want[n][:, keys], got[n][:, keys]
    c.check(got, want, [n for n in ("o", "lse", "dq", "dk", "dv") if want[n].size])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", [(1, 200, 200, 4, 2, 128, 48, 2), (1, 150, 290, 2, 1, 64, 40, 0), (1, 40, 60, 2, 1, 32, 9, 1),
                                   (1, 2, 500, 4, 2, 128, 60, 3), (1, 260, 260, 2, 2, 64, 0, 0)],
                         ids=lambda s: "-".join(str(x) for x in s))
def test_what_is_not_seen_reaches_nothing(shape, form, bad):
    """One key's K and V rows and one query's Q and dO rows hold infinities or NaN: results that do
    not see them are those of a call in which they hold something else."""
    b, nq, nk, H, Hkv, hd, window, sinks = shape
    note(f"window attention unseen {shape} {form} {bad}")
    jbad, rbad = nk - 30 if nq > 30 else nk - 1, nq // 2

    def spoil(v):
        v["k"][:, jbad], v["v"][:, jbad] = bad, bad
        v["q"][:, rbad], v["do"][:, rbad] = bad, bad

    c = Call(*shape, form, spoil=spoil)
    clean = Call(*shape, form)
    c.forward()
    c.backward()
    got, want = c.read(), clean.want()
    see = visible(nq, nk, nq, nk, window, sinks)
    rows = ~see[:, jbad]
    rows[rbad] = False
    keys = ~see[rbad]
    keys[jbad] = False
    # a key that is seen together with a spoilt row or by a row that sees the spoilt key has no clean gradient
    keys &= ~see[see[:, jbad]].any(0)
    assert rows.any() or nq == 2
    for n in ("o", "lse", "dq"):
        want[n], got[n] = want[n][:, rows], got[n][:, rows]
    want["size"], want["edq"], want["edk"] = want["size"][:, rows], want["edq"][:, rows], want["edk"][:, keys]
    for n in ("dk", "dv"):
        want[n], got[n] = want[n][:, keys], got[n][:, keys]
    c.check(got, want, [n for n in ("o", "lse", "dq", "dk", "dv") if want[n].size])
    full = c.read()
    if bad != -np.inf:
        assert np.isnan(full["o"][:, see[:, jbad]]).all()  # and what sees it says so


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_rows_whose_scores_are_all_minus_infinity(form):
    """Every key that row 0 sees has a score of -inf: O = 0, LSE = -inf, no gradient, as for a row that
    sees no key."""
    def spoil(v):
        v["q"][0, 0] = 1.0
        v["k"][0, 0] = -np.inf

    c = Call(1, 70, 70, 2, 1, 64, 1, 0, form, spoil=spoil)
    c.forward()
    c.backward()
    got, want = c.read(), Call(1, 70, 70, 2, 1, 64, 1, 0, form).want()
    assert np.isneginf(got["lse"][0, 0]).all()
    for n in ("o", "dq", "dk", "dv"):
        assert not got[n][0, 0].any(), n
        want[n][0, 0] = 0
    want["lse"][0, 0] = -np.inf
    c.check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fp32", "bf16-fp32"])
def test_large_scores(form):
    """Scores of thousands: the maximum carries them (P is 0 or 1 but for ties)."""
    def spoil(v):
        for n in ("q", "k"):
            v[n][:] = np.sign(v[n]) * 16.0

    c = Call(1, 140, 140, 2, 1, 128, 60, 2, form, spoil=spoil)
    c.forward()
    c.backward()
    c.check(c.read(), c.want())


@pytest.mark.gpu
def test_gradients_against_differences():
    """sum(dO O) moves with q, k and v as dQ, dK and dV say (steps of 2^-5: truncation of about 2^-10,
    rounding of fp32 outputs over the step)."""
    shape, h = (1, 40, 55, 4, 2, 64, 17, 3), 2.0 ** -5
    c = Call(*shape, "fp32")
    c.forward()
    c.backward()
    got, rng = c.read(), np.random.default_rng(1)

    def loss(n, at, step):
        def move(v):
            v[n][at] += step

        m = Call(*shape, "fp32", spoil=move)
        m.forward()
        return float((m.read()["o"] * c.vals["do"]).sum())

    for n in ("q", "k", "v"):
        for _ in range(5):
            at = tuple(int(rng.integers(0, s)) for s in c.vals[n].shape)
            num = (loss(n, at, h) - loss(n, at, -h)) / (2 * h)
            size = np.abs(c.vals["do"]).sum()
            assert abs(num - got["d" + n][at]) <= 4 * U * size / (2 * h) + 4 * h * h, (n, at)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_without_window_or_sinks_it_is_the_causal_attention(form):
    """Against the framework's dense entry point on the same call."""
    from valkyr_amd import kernels as K

    b, n, H, Hkv, hd = 2, 200, 4, 2, 128
    c = Call(b, n, n, H, Hkv, hd, 0, 0, form)
    c.forward()
    o, lse = (dev(np.zeros(b * n * H * w, np.float32)) for w in (hd, 1))
    K.fa_forward(K.attn_params(n, n, H, Hkv, hd, True, b, int(c.bf)), c.up["q"], c.up["k"], c.up["v"], o, lse)
    got = c.read()
    assert rel_l2(host(o), got["o"]) <= (2e-5 if form == "fp32" else 2 * U16 + c.bar("o"))
    assert np.abs(host(lse).reshape(b, n, H) - got["lse"]).max() <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("form,shape", [("bf16", (2, 300, 300, 8, 2, 128, 100, 4)), ("fp32", (1, 260, 260, 4, 1, 64, 90, 2)),
                                        ("bf16", (3, 1, 3000, 8, 2, 128, 1500, 4)), ("fp32", (1, 2, 2000, 8, 8, 64, 0, 0))])
def test_same_bits_every_time_with_any_workspace(form, shape):
    """The caller's workspace, the library's scratch, another stream: the same results bit for bit."""
    from valkyr_amd.device import Stream, synchronize

    c, st, seen = Call(*shape, form), Stream(), []
    need = max(16, c.K.fa_window_forward_workspace_bytes(c.p), c.K.fa_window_backward_workspace_bytes(c.p))
    ws = dev(np.full(need // 4 + 4, np.nan, np.float32))
    synchronize()
    for kw in ({}, dict(workspace=ws), dict(stream=st), dict(stream=st, workspace=ws), {}):
        c.out = {n: c.empty(n) for n in c.out}
        synchronize()
        c.forward(**kw)
        c.backward(**kw)
        seen.append(c.read())
    for s in seen[1:]:
        for n in s:
            assert np.array_equal(s[n], seen[0][n]), n
    c.check(seen[0], c.want())


@pytest.mark.gpu
@pytest.mark.parametrize("own_ws", [False, True], ids=["no-workspace", "workspace"])
@pytest.mark.parametrize("form,shape", [("bf16", (2, 1, 2000, 8, 2, 128, 900, 4)), ("bf16", (1, 333, 333, 4, 2, 64, 60, 1)),
                                        ("fp32", (1, 200, 200, 4, 1, 128, 60, 1)), ("bf16", (1, 50, 2000, 4, 2, 64, 1700, 1)),
                                        ("fp32", (2, 40, 600, 4, 2, 64, 500, 2))])
def test_on_a_captured_stream_with_lengths_that_grow(form, shape, own_ws):
    """A step recorded once is replayed while the lengths on the device change."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    b, nq, nk = shape[:3]
    note(f"captured window attention {form} {shape} {own_ws}")
    lens = lambda i: ([nq] * b, [nk * (i + 1) // 5 + 13 * x for x in range(b)])  # noqa: E731
    c, st = Call(*shape, form, lens=lens(0)), Stream()
    need = max(16, c.K.fa_window_forward_workspace_bytes(c.p), c.K.fa_window_backward_workspace_bytes(c.p))
    kw = dict(workspace=dev(np.zeros(need // 4 + 4, np.float32))) if own_ws else {}
    now = [0]

    def run(stream, **kw):
        c.forward(stream=stream, **kw)
        c.backward(stream=stream, **kw)

    def check():
        c.ql, c.kl = (np.array(x) for x in lens(now[0]))
        c.ql, c.kl = np.minimum(c.ql, nq), np.minimum(c.kl, nk)
        c.check(c.read(), c.want())

    def between():
        now[0] += 1
        c.lens["kv_len"].upload(np.array(lens(now[0])[1], np.uint32))
        run(st)
        synchronize()
        for n, buf in c.out.items():
            x = host(c.empty(n), dtype=np.uint16 if c.obf else np.float32)
            buf.upload(x)

    synchronize()
    _replays(lib(), st, lambda: run(st, **kw), check, between)


@pytest.mark.gpu
def test_a_cache_past_two_to_the_31_bytes():
    """One new token against the end of a bf16 cache of 2.1e9 bytes (2^20 + 5 rows of 1024): offsets pass
    31 bits; the keys seen are the sinks and the last ones."""
    from valkyr_amd import kernels as K
    from valkyr_amd.device import BF16, DeviceBuffer, f32_to_bf16_bits, synchronize  # noqa: F401

    nk, H, Hkv, hd, window, sinks = (1 << 20) + 5, 16, 8, 128, 300, 3
    rng = np.random.default_rng(2)
    note("window attention on a cache of 2 GiB")
    cache = [DeviceBuffer.zeros(nk * Hkv * hd * 2) for _ in range(2)]
    rows = {}
    for x, buf in zip("kv", cache):
        for lo, n in ((0, sinks), (nk - window, window)):
            bits = f32_to_bf16_bits(rng.standard_normal((n, Hkv * hd)).astype(np.float32))
            from valkyr_amd._lib import check, lib

            check(lib().vkh_memcpy_h2d(buf.offset(lo * Hkv * hd * 2), bits.ctypes.data, bits.nbytes))
            rows.setdefault(x, []).append((bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64))
    k, v = (np.concatenate(rows[x]).reshape(-1, Hkv, hd) for x in "kv")
    bq, q = bf16_dev(rng.standard_normal((1, H * hd)))
    o, lse = dev(np.zeros(H * hd, np.float32)), dev(np.zeros(H, np.float32))
    p = K.window_params(1, nk, H, Hkv, hd, window, sinks, dtype=K.BF16, out_dtype=K.F32)
    K.fa_window_forward(p, bq, *cache, o, lse)
    q = np.asarray(q, np.float64).reshape(1, H, hd)
    ref = attention64(q, k, v, np.zeros_like(q), np.ones((1, len(k)), bool), 1 / math.sqrt(hd))
    assert rel_l2(ref["o"], host(o)) <= U16
    assert np.abs(host(lse) - ref["lse"][0]).max() <= 2e-5


@pytest.mark.gpu
def test_rows_at_the_end_of_a_cache_past_two_to_the_31_bytes():
    """The last 100 rows of a bf16 sequence of 2^20 + 5 keys, forward and backward: offsets of K, V and their
    gradients pass 31 bits, and keys that no row sees get gradients of zero."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, f32_to_bf16_bits

    nq, nk, H, Hkv, hd, window, sinks = 100, (1 << 20) + 5, 16, 8, 128, 300, 3
    rng, row = np.random.default_rng(3), Hkv * hd * 2
    note("window attention at the end of 2 GiB")
    at = np.concatenate([np.arange(sinks), np.arange(nk - window - nq, nk)])  # the keys that count
    cache, vals = [DeviceBuffer.zeros(nk * row) for _ in range(2)], []
    for buf in cache:
        bits = f32_to_bf16_bits(rng.standard_normal((len(at), Hkv * hd)).astype(np.float32))
        for lo, part in ((0, bits[:sinks]), (nk - window - nq, bits[sinks:])):
            part = np.ascontiguousarray(part)
            check(lib().vkh_memcpy_h2d(buf.offset(lo * row), part.ctypes.data, part.nbytes))
        vals.append((bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64).reshape(-1, Hkv, hd))
    (bq, q), (bdo, do) = (bf16_dev(rng.standard_normal((nq, H * hd))) for _ in range(2))
    q, do = (np.asarray(x, np.float64).reshape(nq, H, hd) for x in (q, do))
    f32 = lambda n: dev(np.zeros(n, np.float32))  # noqa: E731
    o, dq, lse, d = f32(nq * H * hd), f32(nq * H * hd), f32(nq * H), f32(nq * H)
    grads = [DeviceBuffer.zeros(nk * row * 2) for _ in range(2)]  # fp32: past 2^32 bytes
    unseen, sevens = (sinks, 1 << 18, nk // 2, nk - window - nq - 64), np.full((64, Hkv * hd), 7.0, np.float32)
    for buf in grads:
        for lo in unseen:
            check(lib().vkh_memcpy_h2d(buf.offset(lo * row * 2), sevens.ctypes.data, sevens.nbytes))
    p = K.window_params(nq, nk, H, Hkv, hd, window, sinks, dtype=K.BF16, out_dtype=K.F32)
    K.fa_window_forward(p, bq, *cache, o, lse)
    K.fa_window_backward(p, bq, *cache, o, bdo, lse, d, dq, *grads)
    t = np.arange(nk - nq, nk)[:, None]
    see = (at <= t) & ((at > t - window) | (at < sinks))
    ref = attention64(q, *vals, do, see, 1 / math.sqrt(hd))
    assert rel_l2(ref["o"], host(o)) <= U16
    assert rel_l2(ref["dq"], host(dq)) <= 2 * U16
    for n, buf in zip(("dk", "dv"), grads):
        for lo, part in ((0, ref[n][:sinks]), (nk - window - nq, ref[n][sinks:])):
            got = np.empty(part.shape, np.float32)
            check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset(lo * row * 2), got.nbytes))
            assert rel_l2(part, got) <= 2 * U16, n
        for lo in unseen:
            got = np.ones((64, Hkv * hd), np.float32)
            check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset(lo * row * 2), got.nbytes))
            assert not got.any(), (n, lo)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Calls of few rows and a training pass that both split their work, queued on two streams without
    workspaces: the results of the same calls alone."""
    from valkyr_amd.device import Stream, synchronize

    calls = [Call(2, 1, 3000, 8, 2, 128, 1500, 4, "bf16"), Call(1, 300, 300, 4, 2, 64, 90, 2, "bf16", seed=1)]
    alone = []
    for c in calls:
        c.forward()
        c.backward()
        alone.append(c.read())
    streams = [Stream(), Stream()]
    for c in calls:
        c.out = {n: c.empty(n) for n in c.out}
    synchronize()
    for _ in range(5):
        for c, st in zip(calls, streams):
            c.forward(stream=st)
            c.backward(stream=st)
    synchronize()
    for c, want in zip(calls, alone):
        got = c.read()
        for n in want:
            assert np.array_equal(got[n], want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fp32", "bf16"])
def test_the_operators_as_a_layer_runs_them(form):
    """q|k|v rows of a projection -> norm and rotation -> windowed attention, and backward to the rows and
    the gains, all through the fused rows' strides, against the chain in 64 bits (numeric gradients of
    the norm and rotation are their own tests': here each stage feeds the next)."""
    from test_rotary import frequencies, norm64, plan_of, turn
    from valkyr_amd import kernels as K
    from valkyr_amd.device import DeviceBuffer

    note(f"layer chain {form}")
    b, n, H, Hkv, hd, window, sinks, eps = 2, 150, 4, 2, 64, 40, 2, 1e-6
    rng, T, N = np.random.default_rng(3), 300, (4 + 4) * 64
    d, es = (1, 2) if form == "bf16" else (0, 4)
    x = rng.standard_normal((T, N)).astype(np.float32)  # the projection's fp32 rows
    w = [rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2)]
    do = rng.standard_normal((T, H * hd)).astype(np.float32)
    plan, (f, a) = plan_of(hd, scaling="yarn", factor=4.0, orig_len=4096), frequencies(hd, 1e4, "yarn", 4.0, 4096)
    bx, bw = dev(x), [dev(v) for v in w]
    at = lambda buf, col, size: buf.offset(col * size)  # noqa: E731
    rows = DeviceBuffer.zeros(T * N * es)  # what the attention reads: q, k normed and turned, v as it is
    if form == "bf16":
        K.cast_f32_to_bf16(bx, rows, T * N)
        bdo, do64 = bf16_dev(do)
    else:
        K.scale(bx, rows, T * N, 1.0)
        bdo, do64 = dev(do), do
    p = K.rotary_params(T, H, Hkv, hd, seq_len=n, eps=eps, y_dtype=d, ld_xq=N, ld_xk=N, ld_yq=N, ld_yk=N,
                        ld_dyq=N, ld_dyk=N, ld_dxq=N, ld_dxk=N)
    K.qk_norm_rotary_forward(p, plan, *bw, at(bx, 0, 4), at(rows, 0, es), at(bx, H * hd, 4), at(rows, H * hd, es))
    kc, vc = H * hd, (H + Hkv) * hd
    wp = K.window_params(n, n, H, Hkv, hd, window, sinks, n_batch=b, dtype=d, out_dtype=K.F32, ld_q=N, ld_k=N, ld_v=N,
                         ld_dq=N, ld_dk=N, ld_dv=N)
    o, lse, dd = (DeviceBuffer.zeros(T * H * k * 4) for k in (hd, 1, 1))
    g, dx = DeviceBuffer.zeros(T * N * 4), DeviceBuffer.zeros(T * N * 4)
    qkv = [at(rows, c, es) for c in (0, kc, vc)]
    K.fa_window_forward(wp, *qkv, o, lse)
    K.fa_window_backward(wp, *qkv, o, bdo, lse, dd, *(at(g, c, 4) for c in (0, kc, vc)))
    dw = [DeviceBuffer.zeros(hd * 4) for _ in range(2)]
    K.qk_norm_rotary_backward(p, plan, *bw, at(bx, 0, 4), at(bx, kc, 4), at(g, 0, 4), at(g, kc, 4), at(dx, 0, 4), at(dx, kc, 4), *dw)
    # the same in 64 bits
    x64, pos = x.astype(np.float64), np.arange(T) % n
    parts = [x64[:, :kc].reshape(T, H, hd), x64[:, kc:vc].reshape(T, Hkv, hd)]
    v64 = x64[:, vc:].reshape(b, n, Hkv, hd)
    turned = [turn(norm64(z, v.astype(np.float64), eps, 0)[0] * v, pos, f, a, 0) for z, v in zip(parts, w)]
    q64, k64 = (z.reshape(b, n, -1, hd) for z in turned)
    do64 = np.asarray(do64, np.float64).reshape(b, n, H, hd)
    ref = [attention64(q64[i], k64[i], v64[i], do64[i], visible(n, n, n, n, window, sinks), 1 / math.sqrt(hd)) for i in range(b)]
    # fp32: the fp32 bar through three stages; bf16: q, k, v, P, dS and O's share of D rounded once each
    tol = 3e-5 if form == "fp32" else 6 * U16
    assert rel_l2(np.concatenate([r["o"] for r in ref]).reshape(T, -1), host(o)) <= tol
    got_dx = host(dx).reshape(T, N)
    assert rel_l2(np.concatenate([r["dv"] for r in ref]).reshape(T, -1), host(g).reshape(T, N)[:, vc:]) <= tol
    for side, (z, v, name, lo) in enumerate(((parts[0], w[0], "dq", 0), (parts[1], w[1], "dk", kc))):
        xh, r, _ = norm64(z, v.astype(np.float64), eps, 0)
        gr = turn(np.concatenate([q[name] for q in ref]), pos, f, a, 0, True)
        gw = gr * v
        want = r * (gw - xh * (gw * xh).mean(-1, keepdims=True))
        assert rel_l2(want.reshape(T, -1), got_dx[:, lo:lo + z.shape[1] * hd]) <= tol
        assert rel_l2((gr * xh).sum((0, 1)), host(dw[side])) <= tol


class Long:
    """A call of `b` sequences of n tokens, whose operands are zeros but for some sequences' rows."""

    def __init__(self, b, n, H, Hkv, hd, window, sinks, bf, some, seed=0):
        from valkyr_amd import kernels as K
        from valkyr_amd._lib import check, lib
        from valkyr_amd.device import DeviceBuffer

        self.n, self.H, self.Hkv, self.hd, self.es, self.some = n, H, Hkv, hd, 2 if bf else 4, some
        rng = np.random.default_rng(seed)
        self.p = K.window_params(n, n, H, Hkv, hd, window, sinks, n_batch=b, dtype=int(bf))
        self.heads = dict(q=H, k=Hkv, v=Hkv, do=H, o=H, dq=H, dk=Hkv, dv=Hkv)
        self.buf = {name: DeviceBuffer.zeros(b * n * h * hd * self.es) for name, h in self.heads.items()}
        self.lse, self.d = (DeviceBuffer.zeros(b * n * H * 4) for _ in range(2))
        self.vals = []
        for i in some:
            v = {}
            for name in ("q", "k", "v", "do"):
                x = rng.standard_normal((n, self.heads[name], hd))
                up, w = bf16_dev(x) if bf else (dev(x.astype(np.float32)), x.astype(np.float32))
                raw = host(up, dtype=np.uint16 if bf else np.float32)
                check(lib().vkh_memcpy_h2d(self.at(name, i), raw.ctypes.data, raw.nbytes))
                v[name] = np.asarray(w, np.float64).reshape(x.shape)
            self.vals.append(v)
        u = self.buf
        K.fa_window_forward(self.p, u["q"], u["k"], u["v"], u["o"], self.lse)
        K.fa_window_backward(self.p, u["q"], u["k"], u["v"], u["o"], u["do"], self.lse, self.d, u["dq"], u["dk"], u["dv"])

    def at(self, name, i):
        return self.buf[name].offset(i * self.n * self.heads[name] * self.hd * self.es)

    def rows(self, name, i):
        from valkyr_amd._lib import check, lib
        from valkyr_amd.device import bf16_bits_to_f32

        x = np.empty((self.n, self.heads[name], self.hd), np.uint16 if self.es == 2 else np.float32)
        check(lib().vkh_memcpy_d2h(x.ctypes.data, self.at(name, i), x.nbytes))
        return (bf16_bits_to_f32(x) if self.es == 2 else x).astype(np.float64)

    def log_sums(self, i):
        from valkyr_amd._lib import check, lib

        x = np.empty((self.n, self.H), np.float32)
        check(lib().vkh_memcpy_d2h(x.ctypes.data, self.lse.offset(i * self.n * self.H * 4), x.nbytes))
        return x.astype(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,H,Hkv,hd,window,sinks,bf", [
    ((1 << 16) + 3, 1024, 1, 1, 4, 3, 1, False),  # 2^26 rows and more, a wave each
    ((1 << 13) + 1, 4096, 2, 1, 6, 2, 0, True),
    ((1 << 24) + 5, 1, 1, 1, 64, 1, 0, True),     # more tiles than a launch takes
    ((1 << 24) + 5, 1, 1, 1, 64, 0, 0, False),
    ((1 << 23) + 3, 1, 1, 1, 64, 1, 0, True),     # forward and dQ would fit, dK/dV would not
], ids=lambda x: str(x))
def test_more_rows_than_one_axis_of_a_launch_holds(b, n, H, Hkv, hd, window, sinks, bf):
    note(f"window attention {b} x {n}, {H} / {Hkv} heads of {hd}")
    some = (0, (1 << 24) // n if n > 1 else 1 << 22, b // 2 + 1, b - 1)
    c = Long(b, n, H, Hkv, hd, window, sinks, bf, some)
    see = visible(n, n, n, n, window, sinks)
    for i, v in zip(some, c.vals):
        want = attention64(v["q"], v["k"], v["v"], v["do"], see, 1 / math.sqrt(hd))
        off = np.abs(c.log_sums(i) - want["lse"])
        assert np.all(off <= (hd / 16 + 8) * U * want["size"] + 8 * U * (1 + np.abs(want["lse"])))
        for name in ("o", "dq", "dk", "dv"):
            bar = 1e-5 if not bf else (2 if name == "o" else 3) * U16
            slack = np.linalg.norm(want["e" + name]) if "e" + name in want else 0.0
            assert np.linalg.norm(c.rows(name, i) - want[name]) <= bar * np.linalg.norm(want[name]) + slack, (i, name)
    for i in (1, b // 3, b - 2):  # sequences of zeros
        assert np.abs(c.log_sums(i)[:, 0] - np.log(see.sum(1))).max() <= 8 * U * (1 + np.log(n))
        assert not any(c.rows(name, i).any() for name in ("o", "dq", "dk", "dv")), i


def test_the_backward_asks_for_a_bounded_workspace():
    """Partial sums of at most 256 MiB, whatever the batch; many sequences need none."""
    from valkyr_amd import kernels as K

    for dtype in (K.F32, K.BF16):
        for hd in (64, 128):
            for b in (1, 3, 16, 64, 256, 512, 4096, 1 << 15):
                for n in (1, 100, 256, 1024, 5000):
                    for heads, kv in ((1, 1), (16, 8), (48, 16)):
                        for window, sinks in ((64, 4), (256, 100), (900, 300), (0, 0)):
                            p = K.window_params(n, n, heads, kv, hd, window, sinks, n_batch=b, dtype=dtype)
                            assert K.fa_window_backward_workspace_bytes(p) <= 256 << 20, (dtype, hd, b, n, heads, kv, window)
    for b, n, window in ((512, 256, 64), (4096, 256, 64), (512, 512, 256)):
        assert K.fa_window_backward_workspace_bytes(K.window_params(n, n, 16, 8, 128, window, 4, n_batch=b, dtype=K.BF16)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", [(1, 400, 400, 4, 2, 128, 0, 0), (1, 400, 400, 3, 1, 64, 300, 2), (8, 300, 300, 32, 16, 64, 40, 3),
                                   (1, 90, 120, 2, 1, 40, 0, 0)], ids=lambda s: "-".join(str(x) for x in s))
def test_queries_of_minus_infinity_have_no_gradient(shape, form):
    """A query of -inf against keys over 0: all of its scores are -inf, so O = 0, LSE = -inf, and neither it nor
    any key has a gradient from it, also where all rows beside it see the same keys."""
    b, nq, nk, H, Hkv, hd, window, sinks = shape
    rbad = nq * 3 // 4
    note(f"window attention -inf query {shape} {form}")

    def spoil(v):
        v["k"][:] = np.abs(v["k"]) + 0.01
        v["q"][:, rbad] = -np.inf

    c = Call(*shape, form, spoil=spoil)
    c.forward()
    c.backward()
    got = c.read()
    see = visible(nq, nk, nq, nk, window, sinks)
    see[rbad] = False
    each = [attention64(*(c.vals[n][i] for n in ("q", "k", "v", "do")), see, c.scale) for i in range(b)]
    c.check(got, {n: np.stack([e[n] for e in each]) for n in each[0]})


# ── each row by itself ───────────────────────────────────────────────────

def row_bounds(c, want):
    """How far each head row of a bf16 call's O, dQ, dK and dV may be off, as 2-norms.  P (dS) is rounded
    once for its products, u = 2^-8 of itself at most: a sum of n such terms T_j x_j is off by sum u |T_j|
    |x_j| at the very most, and roundings that do not conspire stay within 8 u sqrt(sum T_j^2 |x_j|^2) (a mean
    of at most one such root, and bounded differences leave 7 more a chance of e^-24).  O's own error, bf16 or
    not, moves D, and with it dQ along P K, and dK by that share of each row.  bf16 results are rounded once
    more; 1e-5 of the terms covers the sums and the exponentials in 32 bits (of scores under 64)."""
    b, nq, nk, H, Hkv, hd, window, sinks = c.shape
    out = {n: np.zeros(want[n].shape[:3]) for n in ("o", "dq", "dk", "dv")}
    g, f32 = H // Hkv, 1e-5
    norm = lambda x: np.linalg.norm(x, axis=-1)  # noqa: E731
    sure = lambda t, x, ax: np.minimum(8 * U16 * np.sqrt((t * t) @ (x * x)) if ax else 8 * U16 * np.sqrt((t * t).T @ (x * x)),  # noqa: E731
                                       (U16 * np.abs(t) @ x) if ax else (U16 * np.abs(t).T @ x))
    for i in range(b):
        see = visible(nq, nk, c.ql[i], c.kl[i], window, sinks)
        k, v = (np.where(see.any(0)[:, None, None], c.vals[n][i], 0) for n in ("k", "v"))
        q, do = (np.where(see.any(1)[:, None, None], c.vals[n][i], 0) for n in ("q", "do"))
        live = see.any(1)
        for h in range(H):
            kh, vh, qh, gh = k[:, h // g], v[:, h // g], q[:, h], do[:, h]
            s = np.where(see, qh @ kh.T * c.scale, -np.inf)
            p = np.where(live[:, None], np.exp(s - np.where(live, want["lse"][i][:, h], 0)[:, None]), 0)
            dd = (gh * want["o"][i][:, h]).sum(-1)
            ds = p * (gh @ vh.T - dd[:, None]) * c.scale
            eo = sure(p, norm(vh), True) + f32 * (p @ norm(vh)) + (U16 * norm(want["o"][i][:, h]) if c.obf else 0)
            out["o"][i][:, h] = eo
            ed = norm(gh) * eo
            out["dq"][i][:, h] = (sure(ds, norm(kh), True) + f32 * (np.abs(ds) @ norm(kh)) + ed * norm(p @ kh) * c.scale +
                                  norm(want["edq"][i][:, h]) + (U16 * norm(want["dq"][i][:, h]) if c.obf else 0))
            t = p * (ed * norm(qh))[:, None] * c.scale
            out["dk"][i][:, h // g] += (sure(ds, norm(qh), False) + f32 * (np.abs(ds).T @ norm(qh)) +
                                        np.minimum(8 * np.sqrt((t * t).sum(0)), t.sum(0)))
            out["dv"][i][:, h // g] += sure(p, norm(gh), False) + f32 * (p.T @ norm(gh))
    out["dk"] += norm(want["edk"])
    if c.obf:
        for n in ("dk", "dv"):
            out[n] += U16 * norm(want[n])
    return out


def check_rows(c):
    got, want = c.read(), c.want()
    c.check(got, want)
    for n, most in row_bounds(c, want).items():
        off = np.linalg.norm(got[n] - want[n], axis=-1)
        worst = np.unravel_index(np.argmax(off - most), off.shape)
        assert np.all(off <= most), (n, worst, off[worst], most[worst], int((off > most).sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["bf16", "bf16-fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s))
def test_each_row_of_bf16_calls(shape, form):
    note(f"window attention rows {shape} {form}")
    c = Call(*shape, form, seed=7)
    c.forward()
    c.backward()
    check_rows(c)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LARGER, ids=lambda s: "-".join(str(x) for x in s))
def test_each_row_of_larger_bf16_calls(shape):
    note(f"larger window attention rows {shape}")
    c = Call(*shape, "bf16", seed=7)
    c.forward()
    c.backward()
    check_rows(c)


# more key blocks than CUs, few sinks: the pairs of a sink and a row past its window have blocks of their own,
# here with several query heads on a KV head, an odd number of them, and slices of 16 and of 32 sinks
FAR = [
    (8, 300, 300, 32, 16, 64, 40, 3),
    (8, 300, 300, 48, 16, 128, 60, 40),
    (6, 420, 420, 64, 16, 64, 30, 100),
    (8, 290, 290, 32, 16, 128, 50, 17),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("form", ["bf16", "bf16-fp32"])
@pytest.mark.parametrize("shape", FAR, ids=lambda s: "-".join(str(x) for x in s))
def test_sinks_of_several_heads_apart(shape, form, ragged):
    note(f"window attention far pairs {shape} {form} {ragged}")
    b, n = shape[:2]
    lens = ([n - 31 * i for i in range(b)],) * 2 if ragged else None

    def spoil(v):
        for i in range(b if ragged else 0):
            v["k"][i, lens[1][i]:] = v["v"][i, lens[1][i]:] = np.nan
            v["q"][i, lens[0][i]:] = v["do"][i, lens[0][i]:] = np.inf

    c = Call(*shape, form, lens=lens, seed=8, spoil=spoil)
    c.forward()
    c.backward()
    check_rows(c)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 300, 4, 2, 128, 64, 4), (3, 1, 3000, 8, 2, 128, 1500, 4), (1, 4, 900, 6, 2, 64, 0, 0),
                                   (1, 13, 1200, 8, 1, 64, 500, 2), (1, 50, 2000, 4, 2, 64, 1700, 1)],
                         ids=lambda s: "-".join(str(x) for x in s))
def test_few_rows_of_bf16_operands_lose_nothing_to_p(shape):
    """O in fp32 of a few rows: P is held as two bf16 terms, off by 2^-16 of itself at most, beside the fp32
    bar for the sums."""
    note(f"window attention few rows {shape}")
    c = Call(*shape, "bf16-fp32", seed=9)
    c.forward()
    got, want = c.read(), c.want()
    assert np.linalg.norm(got["o"] - want["o"]) <= (2.0 ** -16 + 1e-5) * np.linalg.norm(want["o"])


def test_lengths_that_are_not_aligned_are_refused():
    from valkyr_amd import kernels as K

    p, args = K.window_params(4, 4, 2, 1, 64, 2, 1), [256] * 10
    for kw in (dict(q_len=258), dict(kv_len=257), dict(q_len=256, kv_len=254)):
        assert refused(K.fa_window_forward, p, *args[:4], **kw) == "InvalidArgument"
        assert refused(K.fa_window_backward, p, *args, **kw) == "InvalidArgument"
