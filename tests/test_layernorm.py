"""Layer norm, forward and backward, through the C ABI against its formulas in 64 bits: refusals on the
CPU, the kernels on the GPU.

Tolerances count roundings (U = 2^-24 is half a step of fp32, U16 = 2^-8 of bf16).  A lane adds up at most
dim / 64 values of a row one after the other and 12 partial sums after that, so a mean over a row is within
D U of the mean size, D = dim / 64 + 16 (the quotient and the squares' steps in it).  With m = mean |x|:
    dmu <= D U m,  dr / r <= D U + (dmu r)^2 / 2 + 2 U,  dxh <= r (dmu + 2 U |x - mu|) + |xh| dr / r
    dy  <= |w| dxh + 3 U (|xh w| + |b|)
    g = dy w:  ds <= (D + 1) U mean |g|,  dq <= (D + 3) U mean |g xh| + mean(|g| dxh)
    ddx <= r (3 U |g| + ds + |xh| dq + |q| dxh + 3 U (|s| + |xh q|)) + |dx| (dr / r + U) + U |res|
A gain's gradient adds a block's rows, at most rows / 512 + 4 of them one after the other, and up to 520 partial sums.
"""
import ctypes as C

import numpy as np
import pytest

from helpers import dev, host, note
from test_rotary import U, U16, down, filled, refused, up


def formulas(x, w, b, eps, dy=None, res=None):
    """The outputs in 64 bits and how far off fp32 may be (before the rounding of what is stored)."""
    dim = x.shape[1]
    w, b = (np.ones(dim) if w is None else w), (np.zeros(dim) if b is None else b)
    mu = x.mean(1, keepdims=True)
    c = x - mu
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    xh = c * r
    D = dim / 64 + 16
    dmu = D * U * np.abs(x).mean(1, keepdims=True)
    dr = D * U + (dmu * r) ** 2 / 2 + 2 * U
    dxh = r * (dmu + 2 * U * np.abs(c)) + np.abs(xh) * dr
    out = {"y": (xh * w + b, np.abs(w) * dxh + 3 * U * (np.abs(xh * w) + np.abs(b)))}
    if dy is not None:
        rows = x.shape[0]
        g = dy * w
        s, q = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
        ds = (D + 1) * U * np.abs(g).mean(1, keepdims=True)
        dq = (D + 3) * U * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * dxh).mean(1, keepdims=True)
        dx = r * (g - s - xh * q)
        off = (r * (3 * U * np.abs(g) + ds + np.abs(xh) * dq + np.abs(q) * dxh + 3 * U * (np.abs(s) + np.abs(xh * q))) +
               np.abs(dx) * (dr + U))
        if res is not None:
            dx = dx + res
            off = off + U * (np.abs(res) + np.abs(dx))
        out["dx"] = (dx, off)
        Dr = rows / 512 + 4 + 520
        out["dw"] = ((dy * xh).sum(0), (np.abs(dy) * dxh).sum(0) + Dr * U * np.abs(dy * xh).sum(0))
        out["db"] = (dy.sum(0), Dr * U * np.abs(dy).sum(0))
    return out


def close(got, want, off, bf16=False):
    return np.all(np.abs(got - want) <= off + ((U16 + U) * (np.abs(want) + off) if bf16 else U * np.abs(want)) + 1e-37)


# ── the formulas and the refusals (no GPU) ───────────────────────────────

def test_formulas_gradients_against_differences():
    rng = np.random.default_rng(1)
    x, dy, res = (rng.standard_normal((5, 7)) for _ in range(3))
    w, b = rng.standard_normal(7), rng.standard_normal(7)
    f = lambda x, w, b: (formulas(x, w, b, 1e-3)["y"][0] * dy).sum() + (x * res).sum()  # noqa: E731
    out = formulas(x, w, b, 1e-3, dy, res)
    for n, at, i in (("dx", x, 0), ("dw", w, 1), ("db", b, 2)):
        want = np.zeros_like(at)
        for j in np.ndindex(at.shape):
            a = [x, w, b]
            hi, lo = at.copy(), at.copy()
            hi[j] += 1e-5
            lo[j] -= 1e-5
            a[i] = hi
            up_ = f(*a)
            a[i] = lo
            want[j] = (up_ - f(*a)) / 2e-5
        assert np.allclose(out[n][0], want, rtol=1e-7, atol=1e-8)


def test_refusals():
    """Arguments are checked before any device work (the addresses here are not memory)."""
    from valkyr_amd import kernels as K

    ok = K.layernorm_params(4, 64)
    fw = lambda p, *a: refused(K.layernorm_forward, p, *(a or (256, 256, 256, 256)))  # noqa: E731
    bw = lambda p, *a, **kw: refused(K.layernorm_backward, p, *(a or (256, 256, 256, 256)), **kw)  # noqa: E731
    assert fw(K.layernorm_params(4, 0)) == "InvalidArgument"
    assert fw(K.layernorm_params(1 << 31, 8)) == "Unsupported"
    assert fw(K.layernorm_params(1, 1 << 24)) == "Unsupported"
    for n in ("x", "y", "dy", "dx"):
        assert fw(K.layernorm_params(4, 64, **{f"ld_{n}": 63})) == "InvalidArgument"
        assert bw(K.layernorm_params(4, 64, **{f"{n}_dtype": 2})) == "InvalidArgument"
    assert fw(ok, None, 256, 256, 256) == "InvalidArgument"
    assert fw(ok, 256, 256, 256, None) == "InvalidArgument"
    for i in range(4):
        a = [256] * 4
        a[i] = 258
        assert fw(ok, *a) == "InvalidArgument"
        assert bw(ok, *a) == "InvalidArgument"
    assert fw(K.layernorm_params(4, 64, x_dtype=1), 257, 256, 256, 256) == "InvalidArgument"
    assert bw(ok, 256, 256, 256, None) == "InvalidArgument"
    assert bw(ok, None, 256, 256, 256) == "InvalidArgument"
    assert bw(ok, residual=258) == "InvalidArgument"
    assert bw(ok, dw=258) == "InvalidArgument"
    assert bw(ok, db=258) == "InvalidArgument"
    assert bw(ok, dw=256, workspace=264) == "InvalidArgument"
    assert K.layernorm_backward_workspace_bytes(K.layernorm_params(4, 0)) == 0
    assert K.layernorm_backward_workspace_bytes(ok) >= 2 * 64 * 4


def test_struct_layouts(tmp_path):
    import os
    import subprocess

    from valkyr_amd import _lib as L

    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    structs = {"vkh_layernorm_params": L.LayernormParams, "vkh_scan_params": L.ScanParams, "vkh_grad": L.Grad}
    body = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in c._fields_)
                   for n, c in structs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "vkhip.h"\nint main(void){{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [x for c in structs.values() for x in [C.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]]


# ── the kernels ──────────────────────────────────────────────────────────

class Call:
    """Rows of `pad` more values than the operator's, which have to stay as they are."""

    def __init__(self, rows, dim, types="ffff", w=True, b=True, res=False, pad=0, seed=3, x=None, dy=None, eps=1e-5):
        from valkyr_amd import kernels as K

        rng = np.random.default_rng(seed)
        self.K, self.rows, self.dim, self.pad, self.eps = K, rows, dim, pad, eps
        self.t = dict(zip(("x", "y", "dy", "dx"), (c == "b" for c in types)))
        ld = dim + pad if pad else 0
        self.p = K.layernorm_params(rows, dim, eps, *(int(v) for v in self.t.values()), ld, ld, ld, ld)
        self.x, self.X = self.rows_up(rng.standard_normal((rows, dim)) * 1.5 + 0.4 if x is None else x, self.t["x"])
        self.dy, self.DY = self.rows_up(rng.standard_normal((rows, dim)) if dy is None else dy, self.t["dy"])
        self.res, self.RES = self.rows_up(rng.standard_normal((rows, dim)), self.t["dx"]) if res else (None, None)
        self.W = rng.uniform(0.5, 1.5, dim).astype(np.float32) if w else None
        self.B = rng.standard_normal(dim).astype(np.float32) if b else None
        self.w, self.b = (None if v is None else dev(v) for v in (self.W, self.B))
        self.y, self.dx = (filled(rows, dim + pad, self.t[n]) for n in ("y", "dx"))
        self.dw, self.db = filled(1, dim, False), filled(1, dim, False)

    def rows_up(self, x, bf16):
        full = np.full((self.rows, self.dim + self.pad), np.nan)  # what lies between the rows is not read
        full[:, :self.dim] = x
        b, v = up(full, bf16)
        return b, v.reshape(full.shape)[:, :self.dim]

    def run(self, stream=None, **kw):
        self.K.layernorm_forward(self.p, self.x, self.w, self.b, self.y, stream=stream)
        self.K.layernorm_backward(self.p, self.dy, self.x, self.w, self.dx, self.res, self.dw, self.db, stream=stream, **kw)

    def read(self):
        out = {}
        for n, buf in (("y", self.y), ("dx", self.dx)):
            full = down(buf, (self.rows, self.dim + self.pad), self.t[n])
            assert np.all(full[:, self.dim:] == 7.0)
            out[n] = full[:, :self.dim]
        out["dw"], out["db"] = host(self.dw).astype(np.float64), host(self.db).astype(np.float64)
        return out

    def want(self):
        f64 = lambda v: None if v is None else np.asarray(v, np.float64)  # noqa: E731
        return formulas(self.X, f64(self.W), f64(self.B), self.eps, self.DY, self.RES)

    def check(self, got=None, want=None):
        got, want = got or self.read(), want or self.want()
        for n, (ref, off) in want.items():
            assert close(got[n], ref, off, self.t.get(n, False)), n


SHAPES = [(1, 1), (3, 2), (1, 1024), (5, 7), (9, 64), (33, 65), (257, 128), (64, 777), (7, 1000), (40, 1024), (2050, 1024),
          (3, 1027), (129, 2048), (10, 2560), (5, 4096), (600, 4096), (2, 5000), (3, 8192), (4, 12289), (2, 40001)]


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ffff", "bbbb", "fbff", "bfbf", "fbbb"])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_layernorm_matches_the_formula(rows, dim, types):
    note(f"layernorm {rows} x {dim} {types}")
    c = Call(rows, dim, types, res=dim % 3 != 0, pad=(0, 1, 8)[(rows + dim) % 3])
    c.run()
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("w,b,res", [(False, True, False), (True, False, True), (False, False, False)])
@pytest.mark.parametrize("dim", [96, 333, 4096])
def test_without_gain_bias_or_gradients_of_them(dim, w, b, res):
    note(f"layernorm of {dim} without {w} {b} {res}")
    c = Call(21, dim, w=w, b=b, res=res)
    c.run()
    c.check()
    got = c.read()
    for dw, db in ((None, None), (c.dw, None), (None, c.db)):
        dx, ndw, ndb = filled(21, dim, False), filled(1, dim, False), filled(1, dim, False)
        c.K.layernorm_backward(c.p, c.dy, c.x, c.w, dx, c.res, dw and ndw, db and ndb)
        assert np.array_equal(down(dx, (21, dim), False), got["dx"])
        assert np.array_equal(host(ndw), got["dw"] if dw else np.full(dim, 7.0))
        assert np.array_equal(host(ndb), got["db"] if db else np.full(dim, 7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ffff", "bbbb"])
@pytest.mark.parametrize("dim", [17, 1024, 4096, 20000])
def test_rows_far_from_zero_constant_rows_and_rows_that_are_not_finite(dim, types):
    """A row of 10^4 and more with a spread of 1, constant rows (their variance is 0), rows with infinities and
    NaN: each is its own affair but for the gain's gradients."""
    note(f"layernorm odd rows {dim} {types}")
    rng = np.random.default_rng(5)
    x = rng.standard_normal((8, dim))
    x[1] += 1e4
    x[2] = -3.0
    x[3] = 0.0
    x[4] *= 1e-12
    c = Call(8, dim, types, x=x)
    c.run()
    want = c.want()
    c.check(want=want)
    good = c.read()
    x[5, dim // 2], x[6, 0], x[7, dim - 1] = np.inf, np.nan, -np.inf
    c = Call(8, dim, types, x=x)
    c.run()
    got = c.read()
    for n in ("y", "dx"):
        assert np.array_equal(got[n][:5], good[n][:5])
        assert np.all(np.isnan(got[n][5:]).any(1))


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ffff", "bbbb"])
@pytest.mark.parametrize("rows,dim", [(70, 1024), (3, 333), (5, 4096), (2, 30000)])
def test_in_place(rows, dim, types):
    """y over x, and dx over dy, x or the residual: the bits of a call with rows of its own."""
    note(f"layernorm in place {rows} {dim} {types}")
    c = Call(rows, dim, types, res=True)
    c.run()
    want = c.read()
    for over in ("x", "dy", "res"):
        c = Call(rows, dim, types, res=True)
        if over == "x":
            c.K.layernorm_forward(c.p, c.x, c.w, c.b, c.x)
            assert np.array_equal(down(c.x, (rows, dim), c.t["x"]), want["y"])
            c = Call(rows, dim, types, res=True)
        dx = getattr(c, over)
        c.K.layernorm_backward(c.p, c.dy, c.x, c.w, dx, c.res, c.dw, c.db)
        assert np.array_equal(down(dx, (rows, dim), c.t["dx"]), want["dx"])
        assert np.array_equal(host(c.dw), want["dw"]) and np.array_equal(host(c.db), want["db"])


@pytest.mark.gpu
def test_no_rows():
    c = Call(1, 64)
    p = c.K.layernorm_params(0, 64)
    c.K.layernorm_forward(p, c.x, c.w, c.b, c.y)
    c.K.layernorm_backward(p, c.dy, c.x, c.w, c.dx, dw=c.dw, db=c.db)
    assert np.all(host(c.y) == 7.0) and np.all(host(c.dx) == 7.0) and not host(c.dw).any() and not host(c.db).any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim,types", [(1500, 1024, "fbff"), (300, 4096, "bbbb"), (50, 777, "ffff")])
def test_the_same_every_time_on_two_streams_and_replayed(rows, dim, types):
    """Two calls at once on streams of their own, then a captured one replayed between eager ones."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    note(f"layernorm streams and graph {rows} {dim} {types}")
    cs, st = [Call(rows, dim, types, res=True, seed=s) for s in (7, 8)], [Stream(), Stream()]
    synchronize()
    for _ in range(3):
        for c, s in zip(cs, st):
            c.run(s)
    synchronize()
    for c in cs:
        c.check()
    c = cs[0]
    want = c.read()
    ws = filled(1, c.K.layernorm_backward_workspace_bytes(c.p) // 4, False)
    outs = [c.y, c.dx, c.dw, c.db]
    raw = [host(b, dtype=np.uint16) for b in outs]

    def check():
        got = c.read()
        assert all(np.array_equal(got[n], want[n]) for n in want)
        for b, r in zip(outs, raw):
            b.upload(np.where(np.arange(r.size).reshape(r.shape) < 0, r, 0).astype(np.uint16))

    _replays(lib(), st[0], lambda: c.run(st[0], workspace=ws), check, lambda: c.run(st[0]))
    assert lib().hipStreamBeginCapture(st[0].handle, 0) == 0
    name = refused(c.K.layernorm_backward, c.p, c.dy, c.x, c.w, c.dx, dw=c.dw, stream=st[0])
    graph = C.c_void_p()
    assert lib().hipStreamEndCapture(st[0].handle, C.byref(graph)) == 0 and lib().hipGraphDestroy(graph) == 0
    assert name == "InvalidArgument"


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rows", [(1024, (1 << 20) + 9), (8, (1 << 26) + 37)])
def test_rows_past_two_to_the_31_bytes_and_past_a_launch(dim, rows):
    """bf16 rows whose offsets pass 31 bits, and more rows than one axis of a launch holds: those at both ends hold
    numbers, the others zeros."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    note(f"layernorm of {rows} rows of {dim}")
    rng, n, row = np.random.default_rng(9), 16, dim * 2
    x, dy, out = (DeviceBuffer.zeros(rows * row) for _ in range(3))
    W, B, starts, vals = rng.uniform(0.5, 1.5, dim).astype(np.float32), rng.standard_normal(dim).astype(np.float32), (0, rows // 2, rows - n), []
    for at in starts:
        v = []
        for buf in (x, dy):
            bits = f32_to_bf16_bits(rng.standard_normal((n, dim)).astype(np.float32))
            check(lib().vkh_memcpy_h2d(buf.offset(at * row), bits.ctypes.data, bits.nbytes))
            v.append(bf16_bits_to_f32(bits).astype(np.float64).reshape(n, dim))
        vals.append(v)

    def rows_at(at):
        got = np.empty((n, dim), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, out.offset(at * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(n, dim)

    p = K.layernorm_params(rows, dim, 1e-5, 1, 1, 1, 1)
    for name in ("y", "dx"):
        if name == "y":
            K.layernorm_forward(p, x, dev(W), dev(B), out)
        else:
            K.layernorm_backward(p, dy, x, dev(W), out)
        for at, (X, G) in zip(starts, vals):
            ref, off = formulas(X, W.astype(np.float64), B.astype(np.float64), 1e-5, G)[name]
            assert close(rows_at(at), ref, off, True), (name, at)
        rest = rows_at(rows // 3)
        assert np.all(rest == bf16_bits_to_f32(f32_to_bf16_bits(B)).astype(np.float64)) if name == "y" else not rest.any()


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["ffff", "bbbb"])
@pytest.mark.parametrize("rows,dim", [(700, 5000), (600, 8200), (515, 16384), (530, 16400), (450, 40001)])
def test_more_wide_rows_than_blocks(rows, dim, types):
    """Rows of which a block takes several in turn, the last of them not by every block: up to 256 blocks for these
    widths up to 16384, min(512, 2^23 / dim) beyond them.  A gain's gradient then adds at most 3 rows one after the other and
    up to 256 / 16 + 16 (512 / 16 + 16) partial sums, within what formulas() allows.  The same bits each time."""
    note(f"layernorm of many wide rows {rows} x {dim} {types}")
    c = Call(rows, dim, types, res=True, pad=dim % 2)
    c.run()
    got = c.read()
    c.check(got)
    for n in ("dw", "db"):
        getattr(c, n).upload(np.full(dim, 7.0, np.float32))
    c.run()
    again = c.read()
    assert all(np.array_equal(again[n], got[n]) for n in got)


@pytest.mark.gpu
def test_more_wide_rows_than_threads_of_a_launch():
    """2^22 + 3 bf16 rows of 8200 values, each a block of 1024 threads: more threads than one axis of a launch takes.
    In place; rows at both ends and around 2^21 blocks hold numbers, the others zeros, whose result is the bias."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    rows, dim, n = (1 << 22) + 3, 8200, 4
    row = dim * 2
    note(f"layernorm of {rows} rows of {dim}")
    x, rng = DeviceBuffer.zeros(rows * row), np.random.default_rng(10)
    W, B = rng.uniform(0.5, 1.5, dim).astype(np.float32), rng.standard_normal(dim).astype(np.float32)
    starts, vals = (0, (1 << 21) - 2, rows - n), []
    for at in starts:
        bits = f32_to_bf16_bits(rng.standard_normal((n, dim)).astype(np.float32))
        check(lib().vkh_memcpy_h2d(x.offset(at * row), bits.ctypes.data, bits.nbytes))
        vals.append(bf16_bits_to_f32(bits).astype(np.float64).reshape(n, dim))

    def rows_at(at):
        got = np.empty((n, dim), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, x.offset(at * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(n, dim)

    K.layernorm_forward(K.layernorm_params(rows, dim, 1e-5, 1, 1), x, dev(W), dev(B), x)
    for at, X in zip(starts, vals):
        ref, off = formulas(X, W.astype(np.float64), B.astype(np.float64), 1e-5)["y"]
        assert close(rows_at(at), ref, off, True), at
    for at in (4, rows // 3, rows - 2 * n):
        assert np.all(rows_at(at) == bf16_bits_to_f32(f32_to_bf16_bits(B)).astype(np.float64)), at
