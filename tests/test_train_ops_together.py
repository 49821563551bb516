"""Layer norm, the gated scan and gradient clipping as a training step uses them: in the Runner's own step, and in a
recurrent layer that is put together from the library's calls (norm, projections, scan, projection; back; clip; Adam).

Tolerances of the Runner's tests: a step without an effect of clipping gives the bits of one that is not clipped, and a
clipped one those of the calls by hand.  Those of the layer: each fp32 product of K terms is within 2 sqrt(K) U of its
terms' root mean square sum, the norm, the scan and their backward within 64 U of theirs (their own tests count the
steps); a dozen such stages follow one another, so 1e-5 relative in the 2-norm bounds a gradient of any of them.
"""
import math

import numpy as np
import pytest

from helpers import dev, host, note, rel_l2, zeros
from test_gated_scan import formulas as scan64
from test_gpu_runner import build_pair, lora_keys, tensor_keys
from test_rotary import U
from valkyr_amd.runner import ADAM_M, ADAM_V, GRAD, PARAM

SHAPES = {"tied fp32": dict(tied_embeddings=1), "untied bf16": dict(precision=1, tied_embeddings=0),
          "lora fp32": dict(lora_targets=0x7F, lora_rank=4, lora_alpha=16.0, lora_lr_b_scale=2.0),
          "lora bf16": dict(precision=1, lora_targets=0xF, lora_rank=4, lora_alpha=16.0, lora_lr_b_scale=2.0),
          "four layers bf16": dict(precision=1, n_layers=4)}


def keys_of(cfg):
    return lora_keys(cfg) if cfg["lora_targets"] else tensor_keys(cfg)


def all_of(r, cfg):
    return {(kind, k): r.get(kind, *k) for kind in (PARAM, GRAD, ADAM_M, ADAM_V) for k in keys_of(cfg)}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", list(SHAPES))
def test_a_runner_step_below_the_norm_is_an_unclipped_step(shape):
    note(f"runner clipping without effect: {shape}")
    seen = []
    for clip in (0.0, 1e30, math.inf):
        m, r, tok, tgt, cfg = build_pair(**SHAPES[shape])
        r.set_grad_clip(clip)
        for _ in range(3):
            r.step(tok, tgt)
        seen.append(all_of(r, cfg))
        if clip:
            want = math.sqrt(sum(float((r.get(GRAD, *k).astype(np.float64) ** 2).sum()) for k in keys_of(cfg)))
            assert abs(r.last_grad_norm() - want) <= 1.001 * U * want
        r.close()
    for s in seen[1:]:
        for k in s:
            assert np.array_equal(s[k], seen[0][k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("tick", [False, True], ids=["step", "tick"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_a_clipped_runner_step_is_the_calls_by_hand(shape, tick):
    from valkyr_amd import kernels as K

    note(f"runner clipping: {shape} tick {tick}")
    m, r, tok, tgt, cfg = build_pair(**SHAPES[shape])
    keys = keys_of(cfg)
    r.forward_backward(tok, tgt)
    grads = {k: r.get(GRAD, *k) for k in keys}
    params = {k: r.get(PARAM, *k) for k in keys}
    norm = math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads.values()))
    limit = float(np.float32(norm / 3))
    r.set_grad_clip(limit)
    t = r.step_t
    if tick:
        r.upload_train_batch(tok, tgt)
        assert r.tick_frame_train(steps=1).steps_completed == 1
        r.synchronize()
    else:
        r.step(tok, tgt)
    assert abs(r.last_grad_norm() - norm) <= 1.001 * U * norm
    bufs = {k: dev(g) for k, g in grads.items()}
    K.grad_clip(K.grad_list([(bufs[k], grads[k].size, K.F32) for k in keys]), limit)
    for k in keys:
        g = host(bufs[k])
        assert np.array_equal(g, r.get(GRAD, *k)), k
        p, mm, vv = dev(params[k]), zeros(g.size), zeros(g.size)
        lr = cfg["lr"] * (cfg["lora_lr_b_scale"] if cfg["lora_targets"] and k[1] % 2 else 1.0)
        K.adam_step(p, bufs[k], mm, vv, g.size, lr, cfg["beta1"], cfg["beta2"], cfg["eps_adam"], t)
        assert np.array_equal(host(p), r.get(PARAM, *k)) and np.array_equal(host(mm), r.get(ADAM_M, *k)), k
    r.set_grad_clip(0.0)
    r.step(tok, tgt)  # and back to the step that is not clipped
    assert r.last_grad_norm() == pytest.approx(norm, rel=1e-6)
    r.close()


@pytest.mark.gpu
def test_runner_clipping_refusals():
    import valkyr_amd as v

    m, r, tok, tgt, cfg = build_pair()
    for bad in (-1.0, math.nan):
        with pytest.raises(v.VkhError) as e:
            r.set_grad_clip(bad)
        assert e.value.name == "InvalidArgument"
    with pytest.raises(v.VkhError) as e:
        r.last_grad_norm()
    assert e.value.name == "InvalidArgument"
    r.close()


# ── a recurrent layer out of the library's calls ─────────────────────────

class Layer:
    """y = x + scan(xn Wx^T, xn Wg^T) Wo^T, xn = layer norm of x, for b sequences of n rows."""

    NAMES = ("w", "b", "wx", "wg", "wo")

    def __init__(self, b, n, d, c, seed=3):
        from valkyr_amd import kernels as K

        rng = np.random.default_rng(seed)
        self.K, self.b, self.n, self.d, self.c, self.T = K, b, n, d, c, b * n
        shape = dict(w=(d,), b=(d,), wx=(c, d), wg=(c, d), wo=(d, c))
        self.val = {k: (rng.standard_normal(s) / math.sqrt(s[-1] if len(s) > 1 else 4) + (k == "w")).astype(np.float32)
                    for k, s in shape.items()}
        self.p = {k: dev(v) for k, v in self.val.items()}
        self.g = {k: zeros(v.size) for k, v in self.val.items()}
        self.m, self.v = ({k: zeros(v.size) for k, v in self.val.items()} for _ in range(2))
        self.ln = K.layernorm_params(self.T, d)
        self.sp = K.scan_params(n, c, b, coupled=True)
        T = self.T
        self.buf = {k: zeros(T * w) for k, w in dict(xn=d, u=c, z=c, h=c, y=d, dh=c, du=c, dz=c, dn=d, dn2=d, dx=d).items()}
        self.states = zeros(max(1, K.gated_scan_states_floats(self.sp)))
        self.list = K.grad_list([(self.g[k], self.val[k].size, K.F32) for k in self.NAMES])
        self.norm = zeros(1)

    def step(self, x, dy, limit, t):
        K, b, p, g = self.K, self.buf, self.p, self.g
        T, d, c = self.T, self.d, self.c
        K.layernorm_forward(self.ln, x, p["w"], p["b"], b["xn"])
        K.matmul_nt(b["xn"], p["wx"], b["u"], T, c, d)
        K.matmul_nt(b["xn"], p["wg"], b["z"], T, c, d)
        K.gated_scan_forward(self.sp, b["u"], b["z"], b["h"], states=self.states)
        K.matmul_nt(b["h"], p["wo"], b["y"], T, d, c)
        K.add_in_place(b["y"], x, T * d)
        # back: dy is the gradient of y
        K.linear_backward_dx(dy, p["wo"], b["dh"], T, d, c)
        K.linear_backward_dw(dy, b["h"], g["wo"], T, d, c)
        K.gated_scan_backward(self.sp, b["u"], b["z"], self.states, b["dh"], b["du"], b["dz"])
        K.linear_backward_dw(b["du"], b["xn"], g["wx"], T, c, d)
        K.linear_backward_dw(b["dz"], b["xn"], g["wg"], T, c, d)
        K.linear_backward_dx(b["du"], p["wx"], b["dn"], T, c, d)
        K.linear_backward_dx(b["dz"], p["wg"], b["dn2"], T, c, d)
        K.add_in_place(b["dn"], b["dn2"], T * d)
        K.layernorm_backward(self.ln, b["dn"], x, p["w"], b["dx"], residual=dy, dw=g["w"], db=g["b"])
        K.grad_clip(self.list, limit, self.norm)
        for k in self.NAMES:
            K.adam_step(p[k], g[k], self.m[k], self.v[k], self.val[k].size, 1e-2, 0.9, 0.999, 1e-8, t)


def layer64(val, x, dy, b, n):
    """y, dx and the weights' gradients in 64 bits."""
    v = {k: a.astype(np.float64) for k, a in val.items()}
    d, c = v["wo"].shape
    mu = x.mean(1, keepdims=True)
    r = 1 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + 1e-5)
    xh = (x - mu) * r
    xn = xh * v["w"] + v["b"]
    u, z = xn @ v["wx"].T, xn @ v["wg"].T
    three = lambda a: a.reshape(b, n, -1)  # noqa: E731
    dh = dy @ v["wo"]
    s = scan64(three(u), three(z), coupled=True, dh=three(dh))
    h, du, dz = (s[k][0].reshape(b * n, c) for k in ("h", "dx", "dg"))
    dn = du @ v["wx"] + dz @ v["wg"]
    gn = dn * v["w"]
    dx = r * (gn - gn.mean(1, keepdims=True) - xh * (gn * xh).mean(1, keepdims=True)) + dy
    return dict(y=x + h @ v["wo"].T, dx=dx, w=(dn * xh).sum(0), b=dn.sum(0), wx=du.T @ xn, wg=dz.T @ xn, wo=dy.T @ h)


def test_layer_gradients_against_differences():
    rng = np.random.default_rng(4)
    b, n, d, c = 2, 4, 3, 5
    val = {k: rng.standard_normal(s).astype(np.float32) for k, s in dict(w=(d,), b=(d,), wx=(c, d), wg=(c, d), wo=(d, c)).items()}
    x, dy = (rng.standard_normal((b * n, d)) for _ in range(2))
    out = layer64(val, x, dy, b, n)
    for k in list(val) + ["dx"]:
        at = x if k == "dx" else val[k].astype(np.float64)
        want = np.zeros(at.shape)
        for j in np.ndindex(at.shape):
            f = []
            for e in (1e-6, -1e-6):
                a = at.copy()
                a[j] += e
                o = layer64({**val, **({} if k == "dx" else {k: a})}, a if k == "dx" else x, dy, b, n)
                f.append((o["y"] * dy).sum())
            want[j] = (f[0] - f[1]) / 2e-6
        assert np.allclose(out[k], want, rtol=1e-6, atol=1e-7), k


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,d,c", [(1, 300, 64, 96), (2, 129, 100, 68), (3, 7, 32, 32)])
def test_a_recurrent_layers_training_steps(b, n, d, c):
    note(f"recurrent layer {b} x {n}, {d} -> {c}")
    rng = np.random.default_rng(5)
    layer = Layer(b, n, d, c)
    x, dy = (rng.standard_normal((b * n, d)).astype(np.float32) for _ in range(2))
    bx, bdy = dev(x), dev(dy)
    for t in (1, 2, 3):
        val = {k: host(layer.p[k]).reshape(layer.val[k].shape) for k in layer.NAMES}
        want = layer64(val, x.astype(np.float64), dy.astype(np.float64), b, n)
        norm = math.sqrt(sum(float((want[k] ** 2).sum()) for k in layer.NAMES))
        layer.step(bx, bdy, norm / 2, t)
        assert rel_l2(want["y"], host(layer.buf["y"])) <= 1e-5 and rel_l2(want["dx"], host(layer.buf["dx"])) <= 1e-5
        assert abs(float(host(layer.norm)[0]) - norm) <= 1e-5 * norm
        for k in layer.NAMES:
            assert rel_l2(want[k] / 2, host(layer.g[k])) <= 2e-5, k


@pytest.mark.gpu
def test_a_recurrent_layers_step_replayed():
    """Captured with workspaces of its own, and replayed between eager steps that leave other gradients behind."""
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    note("recurrent layer in a graph")
    b, n, d, c = 2, 700, 64, 64
    layer, rng = Layer(b, n, d, c), np.random.default_rng(6)
    K, B, p, g = layer.K, layer.buf, layer.p, layer.g
    x, dy = (dev(rng.standard_normal((b * n, d)).astype(np.float32)) for _ in range(2))
    ws = [dev(np.zeros(max(4, k // 4), np.float32)) for k in (K.layernorm_backward_workspace_bytes(layer.ln),
                                                             K.gated_scan_workspace_bytes(layer.sp), K.grad_clip_workspace_bytes(layer.list))]
    st = Stream()

    def run():
        K.layernorm_forward(layer.ln, x, p["w"], p["b"], B["xn"], stream=st)
        K.gated_scan_forward(layer.sp, B["xn"], x, B["h"], states=layer.states, workspace=ws[1], stream=st)
        K.gated_scan_backward(layer.sp, B["xn"], x, layer.states, dy, B["dn"], B["dn2"], workspace=ws[1], stream=st)
        K.layernorm_backward(layer.ln, B["dn"], x, p["w"], B["dx"], dw=g["w"], db=g["b"], workspace=ws[0], stream=st)
        K.grad_clip(layer.list, 0.5, layer.norm, workspace=ws[2], stream=st)

    names = [(B, k) for k in ("xn", "h", "dn", "dn2", "dx")] + [(g, "w"), (g, "b")]
    synchronize()
    run()
    want = [host(o[k]) for o, k in names] + [host(layer.norm)]

    def check():
        got = [host(o[k]) for o, k in names] + [host(layer.norm)]
        assert all(np.array_equal(u, v) for u, v in zip(got, want))

    def between():
        run()
        synchronize()
        for o, k in names:
            o[k].fill_zero()

    _replays(lib(), st, run, check, between)


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [0.0, 1e-3])
@pytest.mark.parametrize("precision", [0, 1])
def test_a_lora_steps_loss_is_there_before_its_update_is(precision, clip):
    """An asynchronous step's loss is known when its forward and backward are: with 400 M adapter values, whose update
    moves 11 GB (1.4 ms at 8 TB/s), the step goes on for a millisecond and more once last_loss() has come back."""
    import time

    import valkyr_amd as v
    from valkyr_amd.device import Stream

    note(f"loss ahead of Adam: precision {precision} clip {clip}")
    T = 64
    r = v.Runner(v.make_config(dim=1024, n_heads=8, n_kv_heads=8, head_dim=128, ff_dim=1024, n_pos=T, n_layers=28, vocab_size=512,
                               rotary_dim=128, qk_norm=1, lora_targets=0x7F, lora_rank=1024, lora_alpha=16.0, precision=precision))
    r.init_random(seed=3, std=0.02, lora_std=0.02)
    assert r.param_count() == 28 * 14 * 1024 * 1024
    r.set_grad_clip(clip)
    rng, st = np.random.default_rng(1), Stream()
    tok, tgt = (rng.integers(0, 512, T).astype(np.uint32) for _ in range(2))
    r.step(tok, tgt)
    rest = []
    for _ in range(5):
        r.step_async(tok, tgt, stream=st)
        assert math.isfinite(r.last_loss())
        t = time.perf_counter()
        r.synchronize()
        rest.append(time.perf_counter() - t)
    note(f"  the step ends {[round(1e6 * t) for t in rest]} us after its loss")
    assert sorted(rest)[2] > 1e-3
    r.close()
