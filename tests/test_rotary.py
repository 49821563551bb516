"""Rotary positions and the Q/K norm with the rotation in the same pass, through the C ABI,
against their formulas in 64 bits: the plan and the refusals on the CPU, the kernels on the GPU.

Tolerances count roundings (u = 2^-24 is half a step of fp32, 2^-8 of bf16).  An angle is within
pi u / 2 (the reduced half turn is rounded once, below 1) and its cosine and sine within two more
steps, 2.6 u + 4 u: with the scale and the two products, 12 u of |a| + |b| bounds a turned pair.  A
norm adds its sum of squares (a lane's 16 terms and up to 6 shuffles, half of which counts behind
the root), the mean, the root, the quotient and two products: 20 u.
"""
import ctypes as C
import math

import numpy as np
import pytest

from helpers import bf16_dev, dev, host, note

U = 2.0 ** -24
U16 = 2.0 ** -8
NAMES = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


def frequencies(r, theta, scaling="none", factor=1.0, orig_len=0):
    i = np.arange(r // 2, dtype=np.float64)
    if scaling == "ntk":
        theta = theta * factor ** (r / (r - 2))
    f = theta ** (-2 * i / r) if r else i
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        lo, hi = (r * math.log(orig_len / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (32, 1))
        lo, hi = math.floor(lo), min(math.ceil(hi), r - 1)
        u = np.clip((i - lo) / (hi - lo), 0, 1)
        return f * (1 - u) + f / factor * u, 0.1 * math.log(factor) + 1
    if scaling == "bands":
        keep = np.clip((orig_len * f / (2 * math.pi) - 1) / 3, 0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    return f, 1.0


def plan_of(r, theta=1e4, layout=0, scaling="none", factor=1.0, orig_len=0, **kw):
    from valkyr_amd import kernels as K

    return K.rotary_plan(r, theta, layout, NAMES[scaling], factor, orig_len, **kw)


def turn(x, pos, f, a, layout, back=False):
    """x [rows, heads, hd] in 64 bits turned by pos * f."""
    r = 2 * len(f)
    ang = pos[:, None, None].astype(np.float64) * f * (-1 if back else 1)
    c, s = np.cos(ang) * a, np.sin(ang) * a
    lo, hi = (slice(0, r // 2), slice(r // 2, r)) if layout == 0 else (slice(0, r, 2), slice(1, r, 2))
    y = x.copy()
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    return y


def pair_size(x, r, layout, a):
    """|a| + |b| of each value's pair (its own size where it is not turned)."""
    z = np.abs(x)
    lo, hi = (slice(0, r // 2), slice(r // 2, r)) if layout == 0 else (slice(0, r, 2), slice(1, r, 2))
    out = z.copy()
    out[..., lo] = out[..., hi] = (z[..., lo] + z[..., hi]) * a
    return out


# ── the plan and the refusals (no GPU) ───────────────────────────────────

@pytest.mark.parametrize("r,theta,scaling,factor,orig_len", [
    (128, 1e6, "none", 1.0, 0), (2, 1e4, "none", 1.0, 0), (0, 1e4, "none", 1.0, 0), (256, 5e5, "linear", 4.0, 0),
    (64, 1e4, "ntk", 8.0, 0), (128, 1e6, "yarn", 4.0, 32768), (32, 1e4, "yarn", 2.5, 2048), (96, 5e5, "bands", 8.0, 8192)])
def test_plan_holds_the_formulas_frequencies(r, theta, scaling, factor, orig_len):
    f, a = frequencies(r, theta, scaling, factor, orig_len)
    for layout in (0, 1):
        p = plan_of(r, theta, layout, scaling, factor, orig_len)
        assert (p.rotary_dim, p.layout) == (r, layout)
        assert abs(p.attn_factor - a) <= 2 * U * a
        got = np.array(p.turns[:r // 2]) * 2 * math.pi
        assert np.all(np.abs(got - f) <= 1e-13 * f)
        assert not any(p.turns[r // 2:])


def test_plan_attn_factor_and_band_limits_of_the_callers():
    p = plan_of(64, 1e6, 0, "yarn", 4.0, 4096, attn_factor=1.5)
    assert p.attn_factor == 1.5
    q = plan_of(64, 1e4, 0, "bands", 4.0, 4096, low_freq=2.0, high_freq=8.0)
    f, _ = frequencies(64, 1e4)
    keep = np.clip((4096 * f / (2 * math.pi) - 2) / 6, 0, 1)
    assert np.allclose(np.array(q.turns[:32]) * 2 * math.pi, f * keep + f / 4 * (1 - keep), rtol=1e-13, atol=0)


@pytest.mark.parametrize("kw", [
    dict(r=7), dict(r=258), dict(theta=1.0), dict(theta=0.0), dict(theta=math.nan), dict(theta=math.inf),
    dict(layout=2), dict(scaling=5), dict(scaling=1, factor=0.0), dict(scaling=1, factor=-2.0),
    dict(scaling=1, factor=math.nan), dict(scaling=2, factor=2.0, r=2), dict(scaling=3, factor=2.0, orig_len=200),
    dict(scaling=3, factor=2.0, orig_len=4096, beta_fast=1.0, beta_slow=1.0), dict(scaling=4, factor=2.0),
    dict(scaling=3, factor=2.0, orig_len=4096, beta_fast=math.nan),
    dict(scaling=4, factor=2.0, orig_len=4096, low_freq=4.0), dict(attn_factor=-1.0), dict(attn_factor=math.nan)])
def test_plan_refusals(kw):
    import valkyr_amd as v
    from valkyr_amd import kernels as K

    kw = dict(r=64, theta=1e4) | kw
    with pytest.raises(v.VkhError) as e:
        K.rotary_plan(kw.pop("r"), kw.pop("theta"), **kw)
    assert e.value.name == "InvalidArgument"


def refused(call, *args, **kw):
    import valkyr_amd as v

    with pytest.raises(v.VkhError) as e:
        call(*args, **kw)
    return e.value.name


def test_call_refusals():
    """Arguments are checked before any device work (the addresses here are not memory)."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import RotaryPlan

    ok, plan = K.rotary_params(4, 2, 1, 64), plan_of(64)
    fw = lambda p, pl=plan, **kw: refused(K.rotary_forward, p, pl, 256, 256, 256, 256, **kw)  # noqa: E731
    assert fw(K.rotary_params(4, 0, 0, 64)) == "InvalidArgument"
    assert fw(K.rotary_params(4, 2, 1, 0)) == "InvalidArgument"
    assert fw(K.rotary_params(4, 2, 1, 258)) == "Unsupported"
    assert fw(K.rotary_params(1 << 31, 2, 1, 64)) == "Unsupported"
    assert fw(K.rotary_params(4, 1 << 16, 1, 64)) == "Unsupported"
    assert fw(K.rotary_params(4, 2, 1, 32)) == "InvalidArgument"  # turns more than the head
    assert fw(K.rotary_params(4, 2, 1, 64, ld_xq=127)) == "InvalidArgument"
    assert fw(K.rotary_params(4, 2, 1, 64, ld_dxk=63)) == "InvalidArgument"
    assert fw(K.rotary_params(4, 2, 1, 64, y_dtype=2)) == "InvalidArgument"
    assert fw(ok, positions=258) == "InvalidArgument"
    bad = RotaryPlan(rotary_dim=9)
    assert fw(ok, bad) == "InvalidArgument"
    assert fw(ok, RotaryPlan(rotary_dim=64, layout=2)) == "InvalidArgument"
    assert refused(K.rotary_forward, ok, plan, 256, None, 256, 256) == "InvalidArgument"
    assert refused(K.rotary_forward, ok, plan, 256, 256) == "InvalidArgument"  # key heads without rows
    assert refused(K.rotary_forward, ok, plan, 258, 256, 256, 256) == "InvalidArgument"
    assert refused(K.rotary_backward, K.rotary_params(4, 2, 1, 64, dy_dtype=K.BF16), plan, 257, 256, 256, 256) == "InvalidArgument"
    assert refused(K.qk_norm_rotary_forward, ok, plan, None, 256, 256, 256, 256, 256) == "InvalidArgument"
    assert refused(K.qk_norm_rotary_forward, ok, plan, 256, 257, 256, 256, 256, 256) == "InvalidArgument"
    back = [256] * 8
    assert refused(K.qk_norm_rotary_backward, ok, plan, *([256] * 5), None, 256, 256) == "InvalidArgument"
    assert refused(K.qk_norm_rotary_backward, ok, plan, *back, 258) == "InvalidArgument"
    assert refused(K.qk_norm_rotary_backward, ok, plan, *back, 256, workspace=260) == "InvalidArgument"
    assert K.qk_norm_rotary_workspace_bytes(K.rotary_params(4, 2, 1, 258)) == 0
    assert K.qk_norm_rotary_workspace_bytes(ok) >= 2 * 64 * 4


def test_struct_layouts(tmp_path):
    import os
    import subprocess

    from valkyr_amd import _lib as L

    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    structs = {"vkh_rotary_spec": L.RotarySpec, "vkh_rotary_plan": L.RotaryPlan, "vkh_rotary_params": L.RotaryParams,
               "vkh_window_params": L.WindowParams}
    body = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in c._fields_)
                   for n, c in structs.items())
    src = tmp_path / "s.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "vkhip.h"\nint main(void){{ {body} return 0; }}\n')
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    want = [x for c in structs.values() for x in [C.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]]
    assert got == want


# ── the kernels ──────────────────────────────────────────────────────────

def up(x, bf16):
    """(device buffer, the values that it holds in 64 bits)."""
    b, w = bf16_dev(x) if bf16 else (dev(np.asarray(x, np.float32)), np.asarray(x, np.float32))
    return b, np.asarray(w, np.float64)


def down(b, shape, bf16):
    from valkyr_amd.device import bf16_bits_to_f32

    x = bf16_bits_to_f32(host(b, dtype=np.uint16)) if bf16 else host(b)
    return x[:int(np.prod(shape))].reshape(shape).astype(np.float64)


def filled(rows, ld, bf16, pattern=7.0):
    """An output buffer whose every value is known: what a call leaves alone stays."""
    x = np.full((rows, ld), pattern, np.float32)
    return bf16_dev(x)[0] if bf16 else dev(x)


# rows, query heads, key heads, head_dim, rotary_dim, layout, scaling, bf16 in, bf16 out, stride past the heads
CASES = [
    (1, 1, 1, 128, 128, 0, "none", False, False, 0),
    (5, 16, 8, 128, 128, 0, "yarn", True, True, 0),
    (9, 3, 1, 128, 64, 1, "linear", False, True, 0),
    (33, 4, 4, 64, 64, 1, "ntk", True, True, 16),
    (257, 4, 2, 96, 96, 0, "bands", False, False, 4),
    (18, 3, 2, 80, 40, 1, "none", True, False, 8),
    (18, 3, 2, 80, 16, 0, "none", False, False, 0),
    (7, 2, 1, 256, 256, 0, "yarn", False, True, 0),
    (7, 2, 1, 256, 128, 1, "none", True, True, 0),
    (4099, 2, 1, 64, 64, 0, "none", False, False, 0),
    (2050, 1, 0, 64, 32, 0, "none", True, True, 0),
    (300, 0, 3, 32, 32, 1, "linear", False, False, 0),
    # per-value kernels: odd widths, spans and strides
    (11, 3, 2, 33, 14, 0, "none", False, False, 3),
    (11, 3, 2, 33, 14, 1, "linear", True, True, 1),
    (6, 2, 1, 250, 250, 0, "none", True, False, 0),
    (6, 2, 1, 128, 128, 0, "none", True, True, 1),
    (9, 2, 2, 20, 0, 0, "none", False, True, 0),
]


def rotated(case, seed=3):
    rows, nq, nk, hd, r, layout, scaling, bin_, bout, pad = case
    rng = np.random.default_rng(seed)
    opt = {} if scaling == "none" else dict(scaling=scaling, factor=4.0, orig_len=4096)
    plan = plan_of(r, 1e4, layout, **opt)
    f, a = frequencies(r, 1e4, **opt)
    pos = rng.integers(0, 200000, rows).astype(np.uint32)
    if rows > 2:
        pos[1] = 400000000  # its whole turns are lost in 32 bits
    xs = [rng.standard_normal((rows, n, hd)) for n in (nq, nk)]
    return plan, f, a, pos, xs


@pytest.mark.gpu
@pytest.mark.parametrize("back", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_rotary_matches_the_formula(case, back):
    from valkyr_amd import kernels as K

    note(f"rotary {case} {'backward' if back else 'forward'}")
    rows, nq, nk, hd, r, layout, scaling, bin_, bout, pad = case
    plan, f, a, pos, xs = rotated(case)
    lds = [n * hd + pad if n else 0 for n in (nq, nk)]
    ins, vals, outs = [], [], []
    for x, n, ld in zip(xs, (nq, nk), lds):
        full = np.zeros((rows, max(1, ld)))
        full[:, :n * hd] = x.reshape(rows, n * hd)
        b, w = up(full, bin_)
        ins.append(b)
        vals.append(w[:, :n * hd].reshape(rows, n, hd))
        outs.append(filled(rows, max(1, ld), bout))
    names = ("dyq", "dyk", "dxq", "dxk") if back else ("xq", "xk", "yq", "yk")
    strides = {f"ld_{n}": lds[i % 2] for i, n in enumerate(names)} if pad else {}
    p = K.rotary_params(rows, nq, nk, hd, x_dtype=int(bin_), y_dtype=int(bout), dy_dtype=int(bin_), dx_dtype=int(bout), **strides)
    (K.rotary_backward if back else K.rotary_forward)(p, plan, ins[0], outs[0], ins[1], outs[1], positions=dev(pos))
    for x, o, n, ld in zip(vals, outs, (nq, nk), lds):
        if not n:
            continue
        got = down(o, (rows, ld), bout)
        assert np.all(got[:, n * hd:] == 7.0)  # between the rows
        ref = turn(x, pos, f, a, layout, back)
        tol = 12 * U * pair_size(x, r, layout, a) + (U16 * np.abs(ref) if bout else 0) + 1e-30
        assert np.all(np.abs(got[:, :n * hd].reshape(ref.shape) - ref) <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp32", "bf16"])
def test_rotary_in_place_out_of_fused_rows_at_running_positions(bf16):
    """q and k as columns of one q|k|v matrix, turned where they are: v keeps its bits; positions
    pos0 + row % seq_len; and the backward turns them back."""
    from valkyr_amd import kernels as K

    rows, nq, nk, hd, seq, pos0 = 45, 4, 2, 64, 15, 1000
    ld, es = (nq + 2 * nk) * hd, 2 if bf16 else 4
    b, x = up(np.random.default_rng(0).standard_normal((rows, ld)), bf16)
    d = int(bf16)
    p = K.rotary_params(rows, nq, nk, hd, seq_len=seq, pos0=pos0, x_dtype=d, y_dtype=d, dy_dtype=d, dx_dtype=d,
                        **{f"ld_{n}": ld for n in ("xq", "xk", "yq", "yk", "dyq", "dyk", "dxq", "dxk")})
    plan, (f, a) = plan_of(hd), frequencies(hd, 1e4)
    q, k = b.offset(0), b.offset(nq * hd * es)
    K.rotary_forward(p, plan, q, q, k, k)
    got = down(b, (rows, ld), bf16)
    z = x[:, :(nq + nk) * hd].reshape(rows, nq + nk, hd)
    ref = turn(z, pos0 + np.arange(rows) % seq, f, a, 0)
    tol = 12 * U * pair_size(z, hd, 0, a) + (U16 * np.abs(ref) if bf16 else 0)
    assert np.all(np.abs(got[:, :(nq + nk) * hd].reshape(ref.shape) - ref) <= tol)
    assert np.array_equal(got[:, (nq + nk) * hd:], x[:, (nq + nk) * hd:])
    K.rotary_backward(p, plan, q, q, k, k)
    again = down(b, (rows, ld), bf16)[:, :(nq + nk) * hd].reshape(z.shape)
    tol2 = 36 * U * pair_size(z, hd, 0, a) + (3 * U16 * pair_size(z, hd, 0, a) if bf16 else 0)
    assert np.all(np.abs(again - z) <= tol2)


def norm64(x, w, eps, quirk):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * r, r, w + (1 if quirk else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("quirk", [False, True], ids=["w", "1+w"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_qk_norm_rotary_matches_the_formula(case, quirk):
    from valkyr_amd import kernels as K

    note(f"qk norm rotary {case} {quirk}")
    rows, nq, nk, hd, r, layout, scaling, bin_, bout, pad = case
    plan, f, a, pos, xs = rotated(case, 4)
    rng = np.random.default_rng(5)
    eps, lds = 1e-5, [n * hd + pad if n else 0 for n in (nq, nk)]
    dpos, bufs = dev(pos), []
    for x, n, ld in zip(xs, (nq, nk), lds):
        full = np.zeros((2, rows, max(1, ld)))
        full[0, :, :n * hd] = 3 * x.reshape(rows, n * hd)
        full[1, :, :n * hd] = 0.1 * rng.standard_normal((rows, n * hd))
        (bx, vx), (bg, vg) = up(full[0], bin_), up(full[1], bout)
        w = rng.uniform(0.5, 1.5, hd).astype(np.float32)
        bufs.append(dict(x=bx, g=bg, w=dev(w), W=w.astype(np.float64), y=filled(rows, max(1, ld), bout),
                         dx=filled(rows, max(1, ld), bin_), dw=filled(1, hd, False),
                         X=vx[:, :n * hd].reshape(rows, n, hd), G=vg[:, :n * hd].reshape(rows, n, hd)))
    strides = {f"ld_{n}{s}": lds[i] for n in ("x", "y", "dy", "dx") for i, s in enumerate("qk")} if pad else {}
    p = K.rotary_params(rows, nq, nk, hd, eps=eps, gemma_quirk=quirk, x_dtype=int(bin_), y_dtype=int(bout),
                        dy_dtype=int(bout), dx_dtype=int(bin_), **strides)
    s, t = bufs
    K.qk_norm_rotary_forward(p, plan, s["w"], t["w"], s["x"], s["y"], t["x"], t["y"], positions=dpos)
    ws = filled(1, max(4, K.qk_norm_rotary_workspace_bytes(p) // 4), False, np.nan)
    K.qk_norm_rotary_backward(p, plan, s["w"], t["w"], s["x"], t["x"], s["g"], t["g"], s["dx"], t["dx"], s["dw"], t["dw"],
                              positions=dpos, workspace=ws)
    for s, n, ld in zip(bufs, (nq, nk), lds):
        if not n:
            assert not host(s["dw"]).any()  # a sum over no heads
            continue
        xh, rs, w = norm64(s["X"], s["W"], eps, quirk)
        y = turn(xh * w, pos, f, a, layout)
        got = down(s["y"], (rows, ld), bout)
        assert np.all(got[:, n * hd:] == 7.0)
        tol = 32 * U * pair_size(xh * w, r, layout, a) + (U16 * np.abs(y) if bout else 0) + 1e-30
        assert np.all(np.abs(got[:, :n * hd].reshape(y.shape) - y) <= tol)
        g = turn(s["G"], pos, f, a, layout, True)
        gs = pair_size(s["G"], r, layout, a)  # bounds |g| and scales its error
        gw = g * w
        dx = rs * (gw - xh * (gw * xh).mean(-1, keepdims=True))
        # rounding: g 12 u of gs, the norm 20 u of each factor, the mean's sum 11 u of its terms
        tol = rs * 64 * U * (gs * np.abs(w) + np.abs(xh) * (gs * np.abs(w * xh)).mean(-1, keepdims=True))
        tol = tol + (U16 * np.abs(dx) if bin_ else 0) + 1e-30
        got = down(s["dx"], (rows, ld), bin_)
        assert np.all(got[:, n * hd:] == 7.0)
        assert np.all(np.abs(got[:, :n * hd].reshape(dx.shape) - dx) <= tol)
        # each term 33 u; a lane adds at most 64 of them, then 32 lane sums, 32 rows and 16 threads
        dw, size = (g * xh).sum((0, 1)), (gs * np.abs(xh)).sum((0, 1))
        assert np.all(np.abs(host(s["dw"]) - dw) <= (33 + 64 + 32 + 32 + 16) * U * size + 1e-30)


@pytest.mark.gpu
def test_qk_norm_rotary_gradient_against_differences():
    """sum(dy y) moves with x and w as the gradients say (central differences of the forward in
    fp32: steps of 2^-6 leave truncation of about 2^-12 and rounding of 2^-24 * 2^6 * |sum|)."""
    from valkyr_amd import kernels as K

    rng = np.random.default_rng(8)
    rows, nq, nk, hd, h = 3, 2, 1, 64, 2.0 ** -6
    plan = plan_of(32, layout=1)
    x = [rng.standard_normal((rows, n * hd)).astype(np.float32) for n in (nq, nk)]
    w = [rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2)]
    g = [rng.standard_normal(a.shape).astype(np.float32) for a in x]
    p = K.rotary_params(rows, nq, nk, hd, pos0=50)

    def loss(x, w):
        y = [filled(rows, n * hd, False) for n in (nq, nk)]
        K.qk_norm_rotary_forward(p, plan, dev(w[0]), dev(w[1]), dev(x[0]), y[0], dev(x[1]), y[1])
        return sum(float((host(b).reshape(c.shape).astype(np.float64) * c).sum()) for b, c in zip(y, g))

    dx = [filled(rows, n * hd, False) for n in (nq, nk)]
    dw = [filled(1, hd, False) for _ in range(2)]
    K.qk_norm_rotary_backward(p, plan, dev(w[0]), dev(w[1]), dev(x[0]), dev(x[1]), dev(g[0]), dev(g[1]), dx[0], dx[1], dw[0], dw[1])
    size = sum(np.abs(a).sum() for a in g) * 3
    for which, grads in ((0, dx), (1, dw)):
        for side in range(2):
            got = host(grads[side]).reshape(-1).astype(np.float64)
            for i in rng.integers(0, got.size, 4):
                lo, hi = [[a.copy() for a in v] for v in (x, w)], [[a.copy() for a in v] for v in (x, w)]
                lo[which][side].reshape(-1)[i] -= h
                hi[which][side].reshape(-1)[i] += h
                num = (loss(*hi) - loss(*lo)) / (2 * h)
                assert abs(num - got[i]) <= 32 * U * size / (2 * h) + 20 * h * h, (which, side, i)


@pytest.mark.gpu
def test_qk_norm_rotary_gain_gradients_are_the_same_every_time():
    from valkyr_amd import kernels as K
    from valkyr_amd.device import Stream

    rng = np.random.default_rng(9)
    rows, nq, nk, hd = 3000, 8, 2, 128
    plan, p = plan_of(hd), K.rotary_params(rows, nq, nk, hd)
    x, g = ([dev(rng.standard_normal((rows, n * hd), dtype=np.float32)) for n in (nq, nk)] for _ in range(2))
    w = [dev(rng.uniform(0.5, 1.5, hd).astype(np.float32)) for _ in range(2)]
    st, seen = Stream(), []
    for stream in (None, st, None, st):
        dx = [filled(rows, n * hd, False) for n in (nq, nk)]
        dw = [filled(1, hd, False) for _ in range(2)]
        K.qk_norm_rotary_backward(p, plan, *w, *x, *g, *dx, *dw, stream=stream)
        seen.append([host(b) for b in dw + dx])
    assert all(np.array_equal(a, b) for s in seen[1:] for a, b in zip(seen[0], s))
    one = filled(1, hd, False)
    K.qk_norm_rotary_backward(p, plan, *w, *x, *g, *dx, None, one)  # one gain's alone
    assert np.array_equal(host(one), seen[0][1])


@pytest.mark.gpu
def test_no_rows():
    from valkyr_amd import kernels as K

    plan, p = plan_of(64), K.rotary_params(0, 2, 1, 64)
    b, dw = filled(1, 64, False), [filled(1, 64, False) for _ in range(2)]
    K.rotary_forward(p, plan, b, b, b, b)
    K.qk_norm_rotary_backward(p, plan, b, b, b, b, b, b, b, b, *dw)
    assert np.all(host(b) == 7.0) and not host(dw[0]).any() and not host(dw[1]).any()


@pytest.mark.gpu
def test_qk_norm_rotary_on_a_captured_stream():
    from test_gpu_kernels import _replays
    from valkyr_amd import kernels as K
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    rng = np.random.default_rng(10)
    rows, nq, nk, hd = 700, 4, 2, 64
    plan, p = plan_of(hd), K.rotary_params(rows, nq, nk, hd)
    x, g = ([dev(rng.standard_normal((rows, n * hd), dtype=np.float32)) for n in (nq, nk)] for _ in range(2))
    w = [dev(rng.uniform(0.5, 1.5, hd).astype(np.float32)) for _ in range(2)]
    out = [filled(rows, n * hd, False) for n in (nq, nk) * 2] + [filled(1, hd, False) for _ in range(2)]
    ws, st = filled(1, K.qk_norm_rotary_workspace_bytes(p) // 4, False), Stream()

    def run(stream):
        K.qk_norm_rotary_forward(p, plan, *w, x[0], out[0], x[1], out[1], stream=stream)
        K.qk_norm_rotary_backward(p, plan, *w, *x, *g, *out[2:], workspace=ws, stream=stream)

    synchronize()
    run(st)
    want = [host(b) for b in out]

    def check():
        for b, r in zip(out, want):
            assert np.array_equal(host(b), r)
            b.upload(np.zeros_like(r))

    _replays(lib(), st, lambda: run(st), check, lambda: run(st))
    assert lib().hipStreamBeginCapture(st.handle, 0) == 0
    name = refused(K.qk_norm_rotary_backward, p, plan, *w, *x, *g, *out[2:], stream=st)
    graph = C.c_void_p()
    assert lib().hipStreamEndCapture(st.handle, C.byref(graph)) == 0 and lib().hipGraphDestroy(graph) == 0
    assert name == "InvalidArgument"


@pytest.mark.gpu
def test_rows_past_two_to_the_31_bytes():
    """The last rows of bf16 matrices of 2.2e9 bytes: norm and rotation in place, and their backward in place
    of the gradient; the rows before them are zeros and stay so."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    rows, n, nh, hd, pos0 = 270_000, 16, 32, 128, 77
    rng, row = np.random.default_rng(8), nh * hd * 2
    note("rotary on 2.2e9 bytes")

    def make():
        buf, bits = DeviceBuffer.zeros(rows * row), f32_to_bf16_bits(rng.standard_normal((n, nh * hd)).astype(np.float32))
        check(lib().vkh_memcpy_h2d(buf.offset((rows - n) * row), bits.ctypes.data, bits.nbytes))
        return buf, bf16_bits_to_f32(bits).astype(np.float64).reshape(n, nh, hd)

    def last(buf):
        got = np.empty((n, nh * hd), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, buf.offset((rows - n) * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(n, nh, hd)

    (x, vx), (dy, vdy) = make(), make()
    w = rng.uniform(0.5, 1.5, hd).astype(np.float32)
    p = K.rotary_params(rows, nh, 0, hd, pos0=pos0, x_dtype=1, y_dtype=1, dy_dtype=1, dx_dtype=1)
    plan, (f, a), dw = plan_of(hd), frequencies(hd, 1e4), dev(np.zeros(hd, np.float32))
    pos = pos0 + np.arange(rows - n, rows)
    xh, r, g = norm64(vx, w.astype(np.float64), 1e-6, False)
    K.qk_norm_rotary_backward(p, plan, dev(w), None, x, None, dy, None, dy, None, dw)
    t = turn(vdy, pos, f, a, 0, True)
    ref = r * (t * g - xh * (t * g * xh).mean(-1, keepdims=True))
    assert np.linalg.norm(last(dy) - ref) <= (U16 + 100 * U) * np.linalg.norm(ref)
    dref = (t * xh).sum((0, 1))
    assert np.linalg.norm(host(dw) - dref) <= 1e-5 * np.linalg.norm(dref)
    K.qk_norm_rotary_forward(p, plan, dev(w), None, x, x)
    ref = turn(xh * g, pos, f, a, 0)
    assert np.linalg.norm(last(x) - ref) <= (U16 + 100 * U) * np.linalg.norm(ref)
    for buf in (x, dy):
        some = np.ones((64, nh * hd), np.uint16)
        for at in (0, rows // 2, rows - n - 64):
            check(lib().vkh_memcpy_d2h(some.ctypes.data, buf.offset(at * row), some.nbytes))
            assert not (some & 0x7fff).any()


# nothing turned, on chunks of 8 and of 4 values a lane
UNTURNED = [
    (5, 4, 2, 64, 0, 0, "none", False, False, 0),
    (5, 4, 2, 64, 0, 1, "none", True, True, 0),
    (33, 3, 1, 128, 0, 0, "none", True, True, 16),
    (7, 2, 1, 256, 0, 0, "none", False, True, 0),
    (9, 3, 2, 72, 0, 0, "none", False, False, 0),
    (9, 3, 2, 72, 0, 1, "none", True, True, 0),
    (1030, 2, 1, 64, 0, 0, "none", True, False, 0),
    (2050, 1, 0, 128, 0, 0, "none", False, False, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("back", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("case", UNTURNED, ids=lambda c: "-".join(str(x) for x in c))
def test_rotary_that_turns_nothing(case, back):
    test_rotary_matches_the_formula(case, back)


@pytest.mark.gpu
@pytest.mark.parametrize("case", UNTURNED, ids=lambda c: "-".join(str(x) for x in c))
def test_qk_norm_that_turns_nothing(case):
    test_qk_norm_rotary_matches_the_formula(case, False)


@pytest.mark.gpu
@pytest.mark.parametrize("back", [False, True], ids=["forward", "backward"])
@pytest.mark.parametrize("bf16", [False, True], ids=["fp32", "bf16"])
@pytest.mark.parametrize("hd,r,layout", [(128, 64, 0), (128, 32, 1), (72, 24, 0), (72, 24, 1), (64, 0, 0), (33, 14, 0)])
def test_values_behind_the_turned_ones_keep_their_bits(hd, r, layout, bf16, back):
    """Infinities, NaN and zeros of both signs among the values that are not turned stay where they are, and
    reach no other value."""
    from valkyr_amd import kernels as K

    note(f"rotary rest {hd} {r} {layout} {bf16} {back}")
    rows, nq, nk = 6, 3, 2
    plan, (f, a), rng = plan_of(r, layout=layout), frequencies(r, 1e4), np.random.default_rng(11)
    pos = rng.integers(0, 5000, rows).astype(np.uint32)
    odd, ins, vals, outs = [np.nan, np.inf, -np.inf, -0.0, 0.0, 1.5], [], [], []
    for n in (nq, nk):
        x = rng.standard_normal((rows, n, hd))
        for e in range(r, hd):
            x[:, :, e] = np.where(rng.random((rows, n)) < 0.5, x[:, :, e], odd[e % 6])
        b, w = up(x.reshape(rows, -1), bf16)
        ins.append(b)
        vals.append(w.reshape(rows, n, hd))
        outs.append(filled(rows, n * hd, bf16))
    d = int(bf16)
    p = K.rotary_params(rows, nq, nk, hd, x_dtype=d, y_dtype=d, dy_dtype=d, dx_dtype=d)
    (K.rotary_backward if back else K.rotary_forward)(p, plan, ins[0], outs[0], ins[1], outs[1], positions=dev(pos))
    for x, o, n in zip(vals, outs, (nq, nk)):
        got = down(o, x.shape, bf16)
        rest, want = got[..., r:], x[..., r:]
        assert np.array_equal(np.isnan(rest), np.isnan(want))
        nan = np.isnan(want)
        assert np.array_equal(rest[~nan], want[~nan]) and np.array_equal(np.signbit(rest[~nan]), np.signbit(want[~nan]))
        ref = turn(x[..., :r], pos, f, a, layout, back)
        tol = 12 * U * pair_size(x[..., :r], r, layout, a) + (U16 * np.abs(ref) if bf16 else 0) + 1e-30
        assert np.all(np.abs(got[..., :r] - ref) <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp32", "bf16"])
@pytest.mark.parametrize("hd,r", [(128, 64), (72, 24), (64, 0), (33, 14)])
def test_an_infinite_gradient_behind_the_turned_values_reaches_its_own_gain_only(hd, r, bf16):
    from valkyr_amd import kernels as K

    note(f"qk norm infinite gradient {hd} {r} {bf16}")
    rows, n, rng, d = 9, 3, np.random.default_rng(14), int(bf16)
    (f, a), pos, w, at = frequencies(r, 1e4), np.arange(9), rng.uniform(0.5, 1.5, hd).astype(np.float32), hd - 3
    x, X = up(rng.standard_normal((rows, n * hd)), bf16)
    g = rng.standard_normal((rows, n * hd))
    g[4, hd + at] = np.inf  # of the middle head
    g, G = up(g, bf16)
    p = K.rotary_params(rows, n, 0, hd, x_dtype=d, y_dtype=d, dy_dtype=d, dx_dtype=d)
    dw = filled(1, hd, False)
    K.qk_norm_rotary_backward(p, plan_of(r), dev(w), None, x, None, g, None, filled(rows, n * hd, bf16), None, dw)
    xh, _, _ = norm64(X.reshape(rows, n, hd), w.astype(np.float64), 1e-6, False)
    G = np.delete(G.reshape(rows, n, hd), at, -1)
    xh = np.delete(xh, at, -1)
    want, size = (turn(G, pos, f, a, 0, True) * xh).sum((0, 1)), (pair_size(G, r, 0, a) * np.abs(xh)).sum((0, 1))
    got = host(dw)
    assert not np.isfinite(got[at])
    assert np.all(np.abs(np.delete(got, at) - want) <= (33 + 64 + 32 + 32 + 16) * U * size + 1e-30)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nq,nk,hd,r", [(3, 1, 64, 64), (5, 2, 128, 64), (1, 1, 256, 0), (9, 3, 32, 32), (3, 2, 33, 14)])
def test_gain_gradients_without_an_eps(nq, nk, hd, r, bf16):
    """eps = 0, and fewer heads than the rows' lanes hold at a time: lanes without a head add nothing."""
    from valkyr_amd import kernels as K

    note(f"qk norm without eps {nq} {nk} {hd} {r} {bf16}")
    rows, rng = 19, np.random.default_rng(12)
    plan, (f, a), pos = plan_of(r), frequencies(r, 1e4), np.arange(19)
    p = K.rotary_params(rows, nq, nk, hd, eps=0.0, x_dtype=int(bf16), y_dtype=int(bf16), dy_dtype=int(bf16), dx_dtype=int(bf16))
    w = [rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2)]
    (x, X), (g, G) = (tuple(zip(*(up(rng.standard_normal((rows, n * hd)), bf16) for n in (nq, nk)))) for _ in range(2))
    dx, dw = [filled(rows, n * hd, bf16) for n in (nq, nk)], [filled(1, hd, False) for _ in range(2)]
    K.qk_norm_rotary_backward(p, plan, dev(w[0]), dev(w[1]), *x, *g, *dx, *dw)
    for i, n in enumerate((nq, nk)):
        xh, _, _ = norm64(X[i].reshape(rows, n, hd), w[i].astype(np.float64), 0.0, False)
        gi = G[i].reshape(rows, n, hd)
        want = (turn(gi, pos, f, a, 0, True) * xh).sum((0, 1))
        size = (pair_size(gi, r, 0, a) * np.abs(xh)).sum((0, 1))
        # as in the test of the formula above: 33 u a term, and the sums' own steps
        assert np.all(np.abs(host(dw[i]) - want) <= (33 + 64 + 32 + 32 + 16) * U * size + 1e-30)


def test_more_head_rows_than_a_launch_takes_are_refused():
    from valkyr_amd import kernels as K

    p, plan = K.rotary_params(1 << 30, 1 << 9, 1, 64), plan_of(64)
    assert refused(K.rotary_forward, p, plan, 256, 256, 256, 256) == "Unsupported"
    assert refused(K.rotary_backward, p, plan, 256, 256, 256, 256) == "Unsupported"
    assert refused(K.qk_norm_rotary_backward, p, plan, *([256] * 8)) == "Unsupported"
    assert K.qk_norm_rotary_workspace_bytes(p) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("nh,hd,rows", [(1, 8, (1 << 26) + 37), (2, 6, (1 << 25) + 40)], ids=["chunks", "values"])
def test_more_rows_than_one_axis_of_a_launch_holds(nh, hd, rows):
    """2^26 head rows and a few: more than 2^32 lanes.  Rows at both ends and about the axis' end hold
    numbers, the others zeros, which stay zeros."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

    note(f"rotary and norm on {rows} rows of {nh} x {hd}")
    rng, n, row = np.random.default_rng(15), 16, nh * hd * 2
    starts = (0, (1 << 24) - 8, rows // 2, (1 << 26) // nh - 8, rows - n)
    pos0, (f, a), w = 5, frequencies(hd, 1e4), rng.uniform(0.5, 1.5, hd).astype(np.float32)
    x, y, vals = DeviceBuffer.zeros(rows * row), DeviceBuffer.zeros(rows * row), []
    for at in starts:
        bits = f32_to_bf16_bits(rng.standard_normal((n, nh * hd)).astype(np.float32))
        check(lib().vkh_memcpy_h2d(x.offset(at * row), bits.ctypes.data, bits.nbytes))
        vals.append(bf16_bits_to_f32(bits).astype(np.float64).reshape(n, nh, hd))
    p = K.rotary_params(rows, nh, 0, hd, seq_len=1000003, pos0=pos0, x_dtype=1, y_dtype=1, dy_dtype=1, dx_dtype=1)

    def rows_at(at, count=n):
        got = np.empty((count, nh * hd), np.uint16)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, y.offset(at * row), got.nbytes))
        return bf16_bits_to_f32(got).astype(np.float64).reshape(count, nh, hd)

    for op in ("forward", "backward", "norm"):
        if op == "norm":
            K.qk_norm_rotary_forward(p, plan_of(hd), dev(w), None, x, y)
        else:
            (K.rotary_forward if op == "forward" else K.rotary_backward)(p, plan_of(hd), x, y)
        for at, v in zip(starts, vals):
            pos = pos0 + (at + np.arange(n)) % 1000003
            z = norm64(v, w.astype(np.float64), 1e-6, False)[0] * w if op == "norm" else v
            ref = turn(z, pos, f, a, 0, op == "backward")
            assert np.all(np.abs(rows_at(at) - ref) <= 32 * U * pair_size(z, hd, 0, a) + U16 * np.abs(ref) + 1e-30), (op, at)
        assert not rows_at(rows // 3, 64).any() and not rows_at((1 << 24) + 64, 64).any()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,nq,nk,hd,r", [(3000, 16, 4, 128, 64), (700, 5, 3, 96, 96), (11, 3, 2, 33, 14)])
def test_qk_norm_rotary_backward_in_place_of_x(rows, nq, nk, hd, r, bf16):
    """dx over x, or over dy: the bits of a call with rows of its own."""
    from valkyr_amd import kernels as K

    note(f"qk norm backward over x {rows} {nq} {nk} {hd} {r} {bf16}")
    rng, d = np.random.default_rng(13), int(bf16)
    plan, p = plan_of(r), K.rotary_params(rows, nq, nk, hd, x_dtype=d, y_dtype=d, dy_dtype=d, dx_dtype=d)
    X, G = ([rng.standard_normal((rows, n * hd)) for n in (nq, nk)] for _ in range(2))
    w = [dev(rng.uniform(0.5, 1.5, hd).astype(np.float32)) for _ in range(2)]
    seen = []
    for over in (None, "x", "dy"):
        x, g = ([up(z, bf16)[0] for z in zs] for zs in (X, G))
        dx = {None: [filled(rows, n * hd, bf16) for n in (nq, nk)], "x": x, "dy": g}[over]
        dw = [filled(1, hd, False) for _ in range(2)]
        K.qk_norm_rotary_backward(p, plan, *w, *x, *g, *dx, *dw)
        seen.append([down(b, (rows, n * hd), bf16) for b, n in zip(dx, (nq, nk))] + [host(b) for b in dw])
    for s in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(seen[0], s))
