"""The gated linear recurrence, forward and backward, through the C ABI against its formulas in 64 bits:
refusals on the CPU, the kernels on the GPU.

Tolerances count roundings (U = 2^-24 is half a step of fp32, U16 = 2^-8 of bf16).  A sigmoid and one minus it are
within 8 U of their size (the exponential 4, the sum, the quotient and a product); a step of the recurrence,
however its rows are grouped, gives every way of a value through the rows one factor's product, one sum's and one
of joining stretches: with the gate's own, 12 U.  So with M_t = |a| M_{t-1} + |u| (how large the terms are),
    E_t = |a| E_{t-1} + 12 U (|a| M_{t-1} + |u|)
bounds the state's error, and the same from the other end the gradient's.
"""
import numpy as np
import pytest

from helpers import dev, host, note
from test_rotary import U, U16, down, filled, refused, up


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g))


def formulas(x, g, h0=None, sig=True, coupled=False, dh=None, dlast=None, length=None):
    """x, g, dh [batch, rows, dim] in 64 bits: each output and how far off fp32 may be."""
    b, n, d = x.shape
    length = [n] * b if length is None else [min(int(v), n) for v in length]
    zero = np.zeros((b, d))
    h0, dlast = (zero if h0 is None else h0), (zero if dlast is None else dlast)
    a = sigmoid(g) if sig else g
    rest = sigmoid(-g) if sig else 1 - g
    out = {k: [np.zeros((b, n, d)), np.zeros((b, n, d))] for k in ("h", "dx", "dg")}
    out["last"], out["dh0"] = [h0.copy(), 0 * h0], [dlast.copy(), 0 * dlast]
    for i in range(b):
        m = length[i]
        H, M, E = h0[i], np.abs(h0[i]), 0 * h0[i]
        before, err = [], []
        for t in range(m):
            before.append(H)
            err.append(E)
            u = rest[i, t] * x[i, t] if coupled else x[i, t]
            A = np.abs(a[i, t])
            E = A * E + 12 * U * (A * M + np.abs(u))
            M = A * M + np.abs(u)
            H = a[i, t] * H + u
            out["h"][0][i, t], out["h"][1][i, t] = H, E
        out["last"][0][i], out["last"][1][i] = H, E
        if dh is None:
            continue
        R, M, E = dlast[i], np.abs(dlast[i]), 0 * h0[i]
        for t in reversed(range(m)):
            G, size, e = dh[i, t] + R, np.abs(dh[i, t]) + M, E + 2 * U * (np.abs(dh[i, t]) + M)
            A = np.abs(a[i, t])
            E = A * e + 12 * U * A * size
            M = A * size
            R = a[i, t] * G
            hp = before[t] - (x[i, t] if coupled else 0)
            da, ea = G * hp, e * (np.abs(hp) + err[t]) + np.abs(G) * (err[t] + U * (np.abs(before[t]) + np.abs(x[i, t]) * coupled))
            slope = a[i, t] * rest[i, t] if sig else 1.0
            out["dg"][0][i, t], out["dg"][1][i, t] = da * slope, (ea + 24 * U * np.abs(da)) * slope
            r = rest[i, t] if coupled else 1.0
            out["dx"][0][i, t], out["dx"][1][i, t] = r * G, np.abs(r) * (e + 12 * U * np.abs(G))
        out["dh0"][0][i], out["dh0"][1][i] = R, E
    if dh is None:
        out = {k: out[k] for k in ("h", "last")}
    return out


# ── the formulas and the refusals (no GPU) ───────────────────────────────

@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("sig", [False, True])
def test_formulas_gradients_against_differences(sig, coupled):
    rng = np.random.default_rng(2)
    x, g, dh = (rng.standard_normal((2, 5, 3)) for _ in range(3))
    g = g if sig else sigmoid(g)
    h0, dl = (rng.standard_normal((2, 3)) for _ in range(2))
    length = [5, 3]

    def f(x, g, h0):
        o = formulas(x, g, h0, sig, coupled, length=length)
        return (o["h"][0] * dh).sum() + (o["last"][0] * dl).sum()

    out = formulas(x, g, h0, sig, coupled, dh, dl, length)
    for n, i in (("dx", 0), ("dg", 1), ("dh0", 2)):
        at = (x, g, h0)[i]
        want = np.zeros_like(at)
        for j in np.ndindex(at.shape):
            v = []
            for s in (1e-6, -1e-6):
                a = [x, g, h0]
                a[i] = at.copy()
                a[i][j] += s
                v.append(f(*a))
            want[j] = (v[0] - v[1]) / 2e-6
        assert np.allclose(out[n][0], want, rtol=1e-6, atol=1e-8), n


def test_refusals():
    """Arguments are checked before any device work (the addresses here are not memory)."""
    from valkyr_amd import kernels as K

    ok = K.scan_params(4, 64)
    fw = lambda p, *a, **kw: refused(K.gated_scan_forward, p, *(a or (256, 256, 256)), **kw)  # noqa: E731
    bw = lambda p, *a, **kw: refused(K.gated_scan_backward, p, *(a or (256, 256, 256, 256, 256, 512)), **kw)  # noqa: E731
    for p, why in ((K.scan_params(4, 0), "InvalidArgument"), (K.scan_params(4, 64, gate=2), "InvalidArgument"),
                   (K.scan_params(4, 64, dtype=2, out_dtype=0), "InvalidArgument"), (K.scan_params(4, 64, out_dtype=2), "InvalidArgument"),
                   (K.scan_params(1 << 30, 64), "Unsupported"), (K.scan_params(4, 1 << 24), "Unsupported"),
                   (K.scan_params(4, 64, n_batch=1 << 16), "Unsupported")):
        assert fw(p) == why and bw(p) == why
        assert K.gated_scan_states_floats(p) == 0 and K.gated_scan_workspace_bytes(p) == 0
    for n in ("x", "g", "h", "dh", "dx", "dg"):
        assert fw(K.scan_params(4, 64, **{f"ld_{n}": 63})) == "InvalidArgument"
    for i in range(3):
        for bad in (None, 258):
            a = [256] * 3
            a[i] = bad
            assert fw(ok, *a) == "InvalidArgument"
    for i in range(6):
        for bad in (None, 258):
            a = [256] * 5 + [512]
            a[i] = bad
            assert bw(ok, *a) == "InvalidArgument"
    for n in ("h0", "h_last", "states", "length"):
        assert fw(ok, **{n: 258}) == "InvalidArgument"
    for n in ("dh_last", "dh0", "length"):
        assert bw(ok, **{n: 258}) == "InvalidArgument"
    assert bw(ok, 256, 256, 256, 256, 512, 512) == "InvalidArgument"  # one place for two gradients
    long = K.scan_params(100000, 64)
    if K.gated_scan_workspace_bytes(long):
        assert fw(long, workspace=264) == "InvalidArgument"
    assert K.gated_scan_states_floats(K.scan_params(1, 64, n_batch=3)) >= 3 * 64


# ── the kernels ──────────────────────────────────────────────────────────

class Call:
    """Rows of `pad` more values than the operator's, which have to stay as they are; rows behind a sequence's
    end are NaN."""

    def __init__(self, b, n, d, types="ff", sig=True, coupled=False, state=True, lens=None, pad=0, seed=4, mean=2.0):
        from valkyr_amd import kernels as K

        rng = np.random.default_rng(seed)
        self.K, self.b, self.n, self.d, self.pad, self.sig, self.coupled = K, b, n, d, pad, sig, coupled
        self.bin, self.bout = (c == "b" for c in types)
        ld = d + pad if pad else 0
        self.p = K.scan_params(n, d, b, 0 if sig else 1, coupled, int(self.bin), int(self.bout), ld, ld, ld, ld, ld, ld)
        self.lens = lens
        live = np.ones((b, n), bool) if lens is None else np.arange(n) < np.minimum(lens, n)[:, None]
        logits = rng.standard_normal((b, n, d)) * 2 + mean
        self.live = live
        self.x, self.X = self.rows_up(rng.standard_normal((b, n, d)))
        self.g, self.G = self.rows_up(logits if sig else sigmoid(logits) * rng.choice([1, 1, 1, -1], (b, n, d)))
        self.dh, self.DH = self.rows_up(rng.standard_normal((b, n, d)))
        self.H0, self.DL = (rng.standard_normal((b, d)).astype(np.float32) if state else None for _ in range(2))
        self.h0, self.dl = (None if v is None else dev(v) for v in (self.H0, self.DL))
        self.length = None if lens is None else dev(np.asarray(lens, np.uint32))
        self.out = {k: filled(b * n, d + pad, self.bout) for k in ("h", "dx", "dg")}
        self.out.update(last=filled(b, d, False), dh0=filled(b, d, False))
        self.states = dev(np.full(max(1, K.gated_scan_states_floats(self.p)), np.nan, np.float32))

    def rows_up(self, x):
        full = np.full((self.b, self.n, self.d + self.pad), np.nan)
        full[:, :, :self.d] = np.where(self.live[..., None], x, np.nan)
        b, v = up(full, self.bin)
        return b, np.where(self.live[..., None], v.reshape(full.shape)[:, :, :self.d], 0.0)

    def forward(self, **kw):
        o = self.out
        self.K.gated_scan_forward(self.p, self.x, self.g, o["h"], self.h0, o["last"], self.states, self.length, **kw)

    def backward(self, **kw):
        o = self.out
        self.K.gated_scan_backward(self.p, self.x, self.g, self.states, self.dh, o["dx"], o["dg"], self.dl, o["dh0"], self.length, **kw)

    def run(self, stream=None, **kw):
        self.forward(stream=stream, **kw)
        self.backward(stream=stream, **kw)

    def read(self):
        out = {k: host(self.out[k]).reshape(self.b, self.d).astype(np.float64) for k in ("last", "dh0")}
        for k in ("h", "dx", "dg"):
            full = down(self.out[k], (self.b, self.n, self.d + self.pad), self.bout)
            assert np.all(full[..., self.d:] == 7.0)
            out[k] = full[..., :self.d]
        return out

    def want(self):
        f64 = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
        return formulas(self.X, self.G, f64(self.H0), self.sig, self.coupled, self.DH, f64(self.DL), self.lens)

    def check(self, got=None, want=None):
        got, want = got or self.read(), want or self.want()
        for k, (ref, off) in want.items():
            stored = U16 + U if self.bout and k in ("h", "dx", "dg") else U
            assert np.all(np.abs(got[k] - ref) <= off + stored * (np.abs(ref) + off) + 1e-37), k


# sequences, rows, channels, lengths, pad
SHAPES = [(1, 1, 1, None, 0), (3, 1, 64, None, 0), (2, 2, 130, None, 2), (1, 15, 33, None, 1), (2, 16, 128, None, 0),
          (1, 17, 256, None, 8), (3, 127, 96, [127, 1, 0], 0), (2, 128, 64, [128, 64], 0), (1, 129, 65, None, 0),
          (2, 300, 190, [17, 300], 6), (1, 1000, 1, None, 0), (1, 777, 129, None, 0), (4, 513, 130, [513, 0, 400, 9999], 2),
          (1, 4100, 64, None, 0), (2, 2049, 258, [2049, 1300], 0), (1, 2000, 1030, None, 0), (9, 260, 70, None, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ff", "bb", "fb", "bf"])
@pytest.mark.parametrize("b,n,d,lens,pad", SHAPES)
def test_scan_matches_the_formula(b, n, d, lens, pad, types):
    k = b + n + d
    sig, coupled, state = k % 3 != 0, k % 2 == 0, k % 5 != 0
    for coupled in (coupled, not coupled):
        note(f"scan {b} x {n} x {d} {types} {lens} pad {pad} sigmoid {sig} coupled {coupled} state {state}")
        c = Call(b, n, d, types, sig, coupled, state, lens, pad)
        c.run()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("sig,coupled", [(True, True), (False, False)])
@pytest.mark.parametrize("n,d", [(40, 64), (700, 64), (2000, 640)])
def test_optional_outputs_and_states_in_place(n, d, sig, coupled):
    """h_last over h0 and dh0 over dh_last; without h_last, states or dh0; h over x or g and dx, dg over the
    inputs: the same bits."""
    note(f"scan in place {n} {d} {sig} {coupled}")
    make = lambda: Call(2, n, d, "bb", sig, coupled)  # noqa: E731
    c = make()
    c.run()
    want = c.read()
    c.check(want)
    c = make()
    c.K.gated_scan_forward(c.p, c.x, c.g, c.out["h"], c.h0, c.h0, c.states)
    c.K.gated_scan_backward(c.p, c.x, c.g, c.states, c.dh, c.out["dx"], c.out["dg"], c.dl, c.dl)
    c.out.update(last=c.h0, dh0=c.dl)
    assert all(np.array_equal(v, want[k]) for k, v in c.read().items())
    shape = (2, n, d)
    for over in ("x", "g"):
        c = make()
        c.K.gated_scan_forward(c.p, c.x, c.g, getattr(c, over), c.h0)
        assert np.array_equal(down(getattr(c, over), shape, True), want["h"])
    for dx, dg in (("x", "g"), ("dh", "x"), ("g", "dh")):
        c = make()
        c.forward()
        c.K.gated_scan_backward(c.p, c.x, c.g, c.states, c.dh, getattr(c, dx), getattr(c, dg), c.dl)
        assert np.array_equal(down(getattr(c, dx), shape, True), want["dx"])
        assert np.array_equal(down(getattr(c, dg), shape, True), want["dg"])


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ff", "bb"])
@pytest.mark.parametrize("sig", [False, True])
def test_gates_at_their_ends(sig, types):
    """Gates that keep everything for thousands of rows, that reset (also logits of minus infinity and of the type's
    lowest value), and logits far past where the exponential ends."""
    note(f"scan gates {sig} {types}")
    n, d = 1500, 64
    for coupled in (False, True):
        c = Call(1, n, d, types, sig, coupled, mean=0)
        g = c.G.copy()
        g[0, :, 0], g[0, :, 1] = (200.0, 30.0) if sig else (1.0, -1.0)
        g[0, 700, 2:9] = -np.inf if sig else 0.0
        g[0, 701, 2:9] = -3e38 if sig else 0.0
        g[0, 100:900, 9] = 3e38 if sig else 1.0
        g[0, ::3, 10], g[0, 1::3, 10] = (-90.0, 95.0) if sig else (0.0, 1.0)
        c.g, c.G = up(g, c.bin)
        c.G = np.asarray(c.G, np.float64).reshape(g.shape)
        c.run()
        c.check()


@pytest.mark.gpu
def test_what_is_not_finite_stays_in_its_channel():
    note("scan of NaN and infinities")
    n, d = 900, 130
    for types in ("ff", "bb"):
        c = Call(1, n, d, types)
        c.run()
        good = c.read()
        x, g, dh = c.X.copy(), c.G.copy(), c.DH.copy()
        x[0, 300, 5], x[0, 10, 77], g[0, 400, 6], dh[0, 500, 7] = np.nan, np.inf, np.nan, np.nan
        for k, v in (("x", x), ("g", g), ("dh", dh)):
            setattr(c, k, up(v, c.bin)[0])
        c.run()
        got = c.read()
        rest = np.setdiff1d(np.arange(d), [5, 6, 7, 77])
        for k in got:
            assert np.array_equal(got[k][..., rest], good[k][..., rest]), k
        assert np.array_equal(got["h"][:, :300, 5], good["h"][:, :300, 5]) and not np.isfinite(got["h"][:, 300:, 5]).any()
        assert np.array_equal(got["h"][:, :400, 6], good["h"][:, :400, 6]) and not np.isfinite(got["h"][:, 400:, 6]).any()
        assert np.array_equal(got["dx"][:, 501:, 7], good["dx"][:, 501:, 7]) and not np.isfinite(got["dx"][:, :501, 7]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ff", "bb"])
def test_a_nan_whose_bits_are_all_ones(types):
    """The word that a split call's tiles hold before they are published is such a NaN; one among the values is passed
    on as another."""
    note(f"scan of a NaN of ones {types}")
    n, d = 1500, 66
    c = Call(1, n, d, types)
    c.run()
    good = c.read()
    word = np.uint16 if c.bin else np.uint32
    for k, row, ch in (("x", 200, 3), ("g", 700, 4), ("dh", 900, 5)):
        buf = getattr(c, k)
        bits = buf.to_numpy(word).reshape(n, d)
        bits[row, ch] = np.iinfo(word).max
        buf.upload(bits)
    h0 = c.h0.to_numpy(np.uint32)
    h0[6] = 0xFFFFFFFF
    c.h0.upload(h0)
    c.run()
    got = c.read()
    rest = np.setdiff1d(np.arange(d), [3, 4, 5, 6])
    for k in got:
        assert np.array_equal(got[k][..., rest], good[k][..., rest]), k
    assert np.isnan(got["h"][0, 200:, 3]).all() and np.isnan(got["h"][0, 700:, 4]).all() and np.isnan(got["h"][0, :, 6]).all()
    assert np.isnan(got["dx"][0, :901, 5]).all() and np.isnan(got["last"][0, [3, 4, 6]]).all()


@pytest.mark.gpu
def test_no_rows():
    """The states go through."""
    c = Call(2, 1, 70)
    p = c.K.scan_params(0, 70, 2)
    c.K.gated_scan_forward(p, None, None, None, c.h0, c.out["last"])
    c.K.gated_scan_backward(p, None, None, None, None, None, None, c.dl, c.out["dh0"])
    assert np.array_equal(host(c.out["last"]), host(c.h0)) and np.array_equal(host(c.out["dh0"]), host(c.dl))
    c = Call(2, 40, 70, lens=[0, 0])
    c.run()
    got = c.read()
    assert np.array_equal(got["last"], c.H0) and np.array_equal(got["dh0"], c.DL)
    assert not got["h"].any() and not got["dx"].any() and not got["dg"].any()


@pytest.mark.gpu
def test_a_sequence_in_pieces_and_token_by_token():
    """A prompt in two calls and then single tokens: what one call gives, up to the steps counted above."""
    note("scan in pieces")
    n, d, b = 400, 192, 3
    c = Call(b, n, d, "fb", True, True)
    c.forward()
    want = formulas(c.X, c.G, c.H0.astype(np.float64), True, True)
    state, h, K = c.h0, np.zeros((b, n, d)), c.K
    for lo, hi in [(0, 250), (250, 389)] + [(t, t + 1) for t in range(389, n)]:
        p = K.scan_params(hi - lo, d, b, coupled=True, out_dtype=K.BF16)
        x, g = (dev(np.ascontiguousarray(v[:, lo:hi], np.float32)) for v in (c.X, c.G))
        out = filled(b * (hi - lo), d, True)
        K.gated_scan_forward(p, x, g, out, state, state)
        h[:, lo:hi] = down(out, (b, hi - lo, d), True)
    ref, off = want["h"]
    assert np.all(np.abs(h - ref) <= off + (U16 + U) * (np.abs(ref) + off))
    ref, off = want["last"]
    assert np.all(np.abs(host(state).reshape(b, d) - ref) <= off + U * np.abs(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,d,lens", [(1, 5000, 192, None), (2, 1500, 66, [1500, 700]), (3, 5, 64, None), (1, 3000, 2050, None)])
def test_the_same_every_time_on_two_streams_and_replayed(b, n, d, lens):
    """Two calls at once, each with a workspace, then captured ones (with one, and without) replayed between
    eager calls while the lengths on the device change."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    note(f"scan streams and graph {b} {n} {d}")
    cs, st = [Call(b, n, d, "bb", lens=lens, seed=s) for s in (7, 8)], [Stream(), Stream()]
    synchronize()
    seen = []
    for _ in range(3):
        for c, s in zip(cs, st):
            c.run(s)
        synchronize()
        seen.append(cs[0].read())
    for c in cs:
        c.check()
    assert all(np.array_equal(s[k], seen[0][k]) for s in seen for k in s)
    c = cs[0]
    ws = dev(np.full(max(4, c.K.gated_scan_workspace_bytes(c.p) // 4), np.nan, np.float32))
    whole = c.X, c.G, c.DH  # the rows of the longest lengths, which come first
    for kw in ({"workspace": ws}, {}):
        now = [-1]

        def shrink():
            now[0] += 1
            if lens is not None:
                c.lens = [max(0, v - 200 * now[0]) for v in lens]
                c.length.upload(np.array(c.lens, np.uint32))
                live = (np.arange(n) < np.array(c.lens)[:, None])[..., None]
                c.X, c.G, c.DH = (np.where(live, v, 0.0) for v in whole)

        def check():
            c.check()

        def between():
            shrink()
            c.run(st[0])
            synchronize()
            for k, buf in c.out.items():
                buf.upload(np.full(buf.nbytes // 2, 0x4040, np.uint16))

        shrink()
        _replays(lib(), st[0], lambda: c.run(st[0], **kw), check, between)


@pytest.mark.gpu
@pytest.mark.parametrize("types,b,n,d,lens", [("bb", 1, 4000, 192, None), ("ff", 2, 1001, 130, [1001, 400]), ("fb", 3, 640, 64, [640, 0, 513])])
def test_split_and_whole_sequences_give_the_same_bits(types, b, n, d, lens):
    """A call on a captured stream without a workspace takes each sequence in one block."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    note(f"scan split and whole {types} {b} {n} {d}")
    c, st = Call(b, n, d, types, coupled=True, lens=lens), Stream()
    assert c.K.gated_scan_workspace_bytes(c.p) > 0
    synchronize()
    c.run(st)
    want = c.read()
    c.check(want)

    def check():
        got = c.read()
        assert all(np.array_equal(got[k], want[k]) for k in want)

    _replays(lib(), st, lambda: c.run(st), check, lambda: None)


@pytest.mark.gpu
def test_rows_past_two_to_the_31_bytes():
    """A bf16 sequence of 2.1e9 bytes: zeros but for its first rows and its last."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    n, d, m = (1 << 20) + 77, 1024, 40
    note("scan of 2 GiB")
    rng, row = np.random.default_rng(6), d * 2
    x, g, dh, out, dg = (DeviceBuffer.zeros(n * row) for _ in range(5))
    vals = {}
    for at in (0, n - m):
        for k, buf in (("x", x), ("g", g), ("dh", dh)):
            bits = f32_to_bf16_bits(rng.standard_normal((m, d)).astype(np.float32))
            check(lib().vkh_memcpy_h2d(buf.offset(at * row), bits.ctypes.data, bits.nbytes))
            vals[k, at] = bf16_bits_to_f32(bits).astype(np.float64).reshape(1, m, d)
    p = K.scan_params(n, d, dtype=K.BF16)
    states = filled(1, K.gated_scan_states_floats(p), False)

    def rows_at(buf, at):
        got = np.empty((m, d), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset(at * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(1, m, d)

    K.gated_scan_forward(p, x, g, out, states=states)
    for at in (0, n - m):  # gates of zero logits between them halve the state: nothing is left of it
        ref, off = formulas(vals["x", at], vals["g", at])["h"]
        assert np.all(np.abs(rows_at(out, at) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), at
    K.gated_scan_backward(p, x, g, states, dh, out, dg)
    for at in (0, n - m):
        w = formulas(vals["x", at], vals["g", at], dh=vals["dh", at])
        for k, buf in (("dx", out), ("dg", dg)):
            ref, off = w[k]
            assert np.all(np.abs(rows_at(buf, at) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), (k, at)


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ff", "bb"])
@pytest.mark.parametrize("n", [1, 5, 16])
@pytest.mark.parametrize("d", [64, 65])
def test_a_few_rows_in_place(n, d, types):
    """Sequences of up to 16 rows, one of them with fewer: states over each other, h over x or g, dx and dg over the
    inputs give the bits of a call with places of its own."""
    note(f"scan of a few rows in place {n} {d} {types}")
    bf, shape = types == "bb", (3, n, d)
    for sig, coupled, lens in ((True, True, None), (False, False, [n, n // 2, 0])):
        make = lambda: Call(3, n, d, types, sig, coupled, lens=lens)  # noqa: E731
        c = make()
        c.run()
        want = c.read()
        c.check(want)
        c = make()
        c.K.gated_scan_forward(c.p, c.x, c.g, c.out["h"], c.h0, c.h0, c.states, c.length)
        c.K.gated_scan_backward(c.p, c.x, c.g, c.states, c.dh, c.out["dx"], c.out["dg"], c.dl, c.dl, c.length)
        c.out.update(last=c.h0, dh0=c.dl)
        assert all(np.array_equal(v, want[k]) for k, v in c.read().items())
        for over in ("x", "g"):
            c = make()
            c.K.gated_scan_forward(c.p, c.x, c.g, getattr(c, over), c.h0, length=c.length)
            assert np.array_equal(down(getattr(c, over), shape, bf), want["h"])
        for dx, dg in (("x", "g"), ("dh", "x"), ("g", "dh"), ("x", "dh"), ("dh", "g"), ("g", "x")):
            c = make()
            c.forward()
            c.K.gated_scan_backward(c.p, c.x, c.g, c.states, c.dh, getattr(c, dx), getattr(c, dg), c.dl, length=c.length)
            assert np.array_equal(down(getattr(c, dx), shape, bf), want["dx"])
            assert np.array_equal(down(getattr(c, dg), shape, bf), want["dg"])


@pytest.mark.gpu
@pytest.mark.parametrize("sig", [True, False])
@pytest.mark.parametrize("coupled", [True, False])
@pytest.mark.parametrize("types,b,n,d,lens", [("bb", 1, 2500, 130, None), ("ff", 2, 900, 64, [900, 515])])
def test_split_and_whole_sequences_give_the_same_bits_for_every_gate(types, b, n, d, lens, sig, coupled):
    same_bits_whole(Call(b, n, d, types, sig, coupled, lens=lens), True)


def same_bits_whole(c, split, want=None):
    """A call, against 64 bits, and the same one on a captured stream without a workspace, where each sequence is one
    block's: the same bits."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    st = Stream()
    if split is not None:
        assert (c.K.gated_scan_workspace_bytes(c.p) > 0) == split
    synchronize()
    c.run(st)
    got = c.read()
    c.check(got, want)

    def check():
        now = c.read()
        assert all(np.array_equal(now[k], got[k]) for k in got)

    def clear():
        for buf in c.out.values():
            buf.upload(np.full(buf.nbytes // 2, 0x40E0, np.uint16))  # (7 in bf16)

    clear()
    _replays(lib(), st, lambda: c.run(st), check, clear, 2)


# 64-channel groups of all sequences: where a sequence's tiles stop being shared between blocks (256 blocks
# are resident in the backward, 512 in the forward), and more groups than there are blocks
@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ff", "bb"])
@pytest.mark.parametrize("b,groups,lens", [(2, 64, None), (3, 43, [400, 31, 300]), (4, 40, None), (1, 256, None), (1, 257, None), (5, 64, [400, 0, 399, 129, 128]),
                                           (10, 60, None)])
def test_groups_around_the_blocks_that_are_resident(b, groups, lens, types):
    n = 400
    d = 64 * groups - (7 if groups % 2 else 0)
    note(f"scan of {b * groups} groups {types} {lens}")
    same_bits_whole(Call(b, n, d, types, coupled=b % 2 == 0, lens=lens), None)


@pytest.mark.gpu
def test_more_groups_than_threads_of_a_launch():
    """65535 bf16 sequences of 17 rows and 65 groups of channels, over 2^22 groups in all, each a block of 1024 threads
    in the backward: more threads than one axis of a launch takes.  Zeros (gates of 1/2) but for some sequences."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    b, n, d = 65535, 17, 64 * 64 + 1
    note(f"scan of {b} x {n} x {d}")
    rng, seq = np.random.default_rng(7), n * d * 2
    x, g, c = (DeviceBuffer.zeros(b * seq) for _ in range(3))  # c: h, and then dh
    some, vals = (0, 32262, 32264, 64526, 64528, b - 1), {}

    def put(k, buf):
        for i in some:
            bits = f32_to_bf16_bits(rng.standard_normal((n, d)).astype(np.float32))
            check(lib().vkh_memcpy_h2d(buf.offset(i * seq), bits.ctypes.data, bits.nbytes))
            vals[k, i] = bf16_bits_to_f32(bits).astype(np.float64).reshape(1, n, d)

    def at(buf, i):
        got = np.empty((n, d), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset(i * seq), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(1, n, d)

    put("x", x)
    put("g", g)
    p = K.scan_params(n, d, b, dtype=K.BF16)
    states = DeviceBuffer.zeros(K.gated_scan_states_floats(p) * 4)
    K.gated_scan_forward(p, x, g, c, states=states)
    for i in some:
        ref, off = formulas(vals["x", i], vals["g", i])["h"]
        assert np.all(np.abs(at(c, i) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), i
        assert not at(c, min(i + 1, b - 2)).any()
    c.fill_zero()
    put("dh", c)
    K.gated_scan_backward(p, x, g, states, c, c, g)
    for i in some:
        w = formulas(vals["x", i], vals["g", i], dh=vals["dh", i])
        for k, buf in (("dx", c), ("dg", g)):
            ref, off = w[k]
            assert np.all(np.abs(at(buf, i) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), (k, i)
            assert not at(buf, min(i + 1, b - 2)).any()


@pytest.mark.gpu
def test_a_sequence_whose_words_would_be_too_many():
    """128 groups of a sequence of 1.3 million rows: the words of its tiles would take a GB, so it stays whole.  Zeros
    (gates of 1/2) but for its first rows and its last."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    n, d, m = 128 * 10240 + 77, 64 * 128, 40
    note(f"scan of {n} x {d}")
    p = K.scan_params(n, d, dtype=K.BF16)
    assert K.gated_scan_workspace_bytes(p) == 0 and K.gated_scan_workspace_bytes(K.scan_params(n // 2, d, dtype=K.BF16)) > 0
    rng, row = np.random.default_rng(8), d * 2
    x, g, c = (DeviceBuffer.zeros(n * row) for _ in range(3))  # c: h, and then dh
    vals = {}

    def put(k, buf):
        for at in (0, n - m):
            bits = f32_to_bf16_bits(rng.standard_normal((m, d)).astype(np.float32))
            check(lib().vkh_memcpy_h2d(buf.offset(at * row), bits.ctypes.data, bits.nbytes))
            vals[k, at] = bf16_bits_to_f32(bits).astype(np.float64).reshape(1, m, d)

    def rows_at(buf, at):
        got = np.empty((m, d), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset(at * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(1, m, d)

    put("x", x)
    put("g", g)
    states = DeviceBuffer.zeros(K.gated_scan_states_floats(p) * 4)
    K.gated_scan_forward(p, x, g, c, states=states)
    for at in (0, n - m):  # (gates of 1/2 between them: nothing is left of the state)
        ref, off = formulas(vals["x", at], vals["g", at])["h"]
        assert np.all(np.abs(rows_at(c, at) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), at
    c.fill_zero()
    put("dh", c)
    K.gated_scan_backward(p, x, g, states, c, c, g)
    for at in (0, n - m):
        w = formulas(vals["x", at], vals["g", at], dh=vals["dh", at])
        for k, buf in (("dx", c), ("dg", g)):
            ref, off = w[k]
            assert np.all(np.abs(rows_at(buf, at) - ref) <= off + (U16 + U) * (np.abs(ref) + off) + 1e-37), (k, at)
