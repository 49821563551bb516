"""The operators of a recurrent layer's training step, as measurable cases.

A case is a dict of plain values; `kind` names its operator:

  layernorm   layer norm of rows, forward, and with `train` backward too: the gradient of its input
              (added to the residual path's where there is one) and of its gain and bias
  scan        a gated linear recurrence h_t = a_t h_{t-1} + u_t of each channel over a sequence: gates
              given as they are or as the logits of a sigmoid, u = x or (1 - a) x; forward, and with
              `train` backward too
  clip        the norm of all gradients of a step, a list of tensors of many sizes, and the gradients
              scaled down to a largest norm

Types: "fp32" holds everything in 32 bits; "bf16" activations and their gradients in bf16 and sums,
statistics, states, gains and their gradients in 32 bits; "mixed" reads fp32 and writes bf16 (a projection's
output on its way into a bf16 product; layer norm's dx stays in the residual stream's 32 bits; a list
of gradients has tensors of both).
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# ── the cases ────────────────────────────────────────────────────────────

def listed():
    return [
        # One token on its way into a layer: launch and latency.
        dict(kind="layernorm", name="layernorm_bf16_1", form="bf16", rows=1, dim=1024, bias=True, train=False),
        # The headline step's batch (4 sequences of 512 tokens), fp32 residual stream, bf16 products.
        dict(kind="layernorm", name="layernorm_mixed_train_2048", form="mixed", rows=2048, dim=1024, bias=True,
             residual=True, train=True),
        # An odd-sized batch in the reference's precision, a width of no whole vectors, no bias.
        dict(kind="layernorm", name="layernorm_fp32_train_1001", form="fp32", rows=1001, dim=777, bias=False,
             residual=False, train=True),
        # The largest: a long-context step's tokens at the 8B model's width.
        dict(kind="layernorm", name="layernorm_bf16_train_16384", form="bf16", rows=16384, dim=4096, bias=True,
             residual=True, train=True),
        # One new token of each of 32 sequences, their states at hand.
        _scan("scan_bf16_step_32", form="bf16", b=32, n=1, dim=4096, state=True, train=False),
        # A chunk of prompts of different lengths behind what came before.
        _scan("scan_mixed_chunk_777", form="mixed", b=3, n=777, dim=2560, state=True, ragged=True, train=False),
        # A padded batch of two odd-sized documents in the reference's precision, decays as they are.
        _scan("scan_fp32_train_1001", form="fp32", b=2, n=1001, dim=1155, gate="decay", ragged=True, train=True),
        # The headline step's batch, the gate also scaling what comes in.
        _scan("scan_mixed_train_512", form="mixed", b=4, n=512, dim=1024, coupled=True, train=True),
        # The largest: one long sequence at the 8B model's width.
        _scan("scan_bf16_train_16384", form="bf16", b=1, n=16384, dim=4096, coupled=True, state=True, train=True),
        # Adapters of rank 16 on four projections of 28 layers.
        dict(kind="clip", name="clip_fp32_adapters", form="fp32", sizes="adapters", tensors=224, most=32768,
             share=0.25, gap=0),
        # Gradients of both types and of every size, few of them where a vector could start.
        dict(kind="clip", name="clip_mixed_61", form="mixed", sizes="spread", tensors=61, most=3000001, share=0.5,
             gap=3),
        # The largest: all gradients of the headline model (28 layers of 11 tensors, the embedding).
        dict(kind="clip", name="clip_fp32_model", form="fp32", sizes="model", tensors=310, most=155582464, share=0.1,
             gap=0),
    ]


def _scan(name, **kw):
    c = dict(kind="scan", name=name, gate="sigmoid", coupled=False, state=False, ragged=False)
    c.update(kw)
    return c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layernorm", "scan", "scan", "clip"])
    form = rng.choice(["fp32", "bf16", "mixed"])
    if kind == "clip":
        sizes = rng.choice(["spread", "spread", "adapters"])
        most = _log(rng, 1, 4000000) if sizes == "spread" else 1024 * rng.randint(1, 64)
        return dict(kind=kind, form=form, sizes=sizes, tensors=_log(rng, 1, 300), most=most,
                    share=rng.choice([0.1, 0.5, 0.9, 2.0]), gap=rng.choice([0, 0, 1, 3]))
    dim = rng.choice([_log(rng, 1, 8192), 64 * rng.randint(1, 80), 8 * rng.randint(1, 200)])
    if kind == "layernorm":
        c = dict(kind=kind, form=form, dim=dim, rows=min(_log(rng, 1, 16384), (16384 * 4096) // (dim * (1 if form == "bf16" else 2))),
                 bias=rng.random() < 0.7, train=rng.random() < 0.6)
        if c["train"]:
            c["residual"] = rng.random() < 0.5
        return c
    c = _scan("", form=form, b=rng.choice([1, 1, 2, 3, 4, 8]), dim=dim, gate=rng.choice(["sigmoid", "sigmoid", "decay"]),
              coupled=rng.random() < 0.4, state=rng.random() < 0.5, ragged=rng.random() < 0.4)
    del c["name"]
    use = rng.choice(["step", "chunk", "train", "train"])
    c["train"] = use == "train"
    room = (16384 * 4096) // (c["b"] * dim * (1 if form == "bf16" else 2))
    c["n"] = rng.choice([1, 1, 4]) if use == "step" else max(1, min(_log(rng, 8, 16384), room))
    if use == "step":
        c.update(b=_log(rng, 1, 64), state=True)
    return c


# ── what a pass cannot do without ────────────────────────────────────────

def _types(form):
    """What is read and what is written."""
    return {"fp32": (F32, F32), "bf16": (BF16, BF16), "mixed": (F32, BF16)}[form]


def _size(t):
    return 2 if t == BF16 else 4


def _dx_type(c):
    """Layer norm's dx and the residual path's gradient."""
    return BF16 if c["form"] == "bf16" else F32


def _lens(c):
    """The sequences' rows: in a ragged batch between a 16th of the room and all of it, and none of the
    third sequence's."""
    n, b = c["n"], c["b"]
    if not c["ragged"]:
        return [n] * b
    lo = max(1, n // 16)
    return [0 if i == 2 else n if b == 1 else lo + (n - lo) * (7 * i % b) // (b - 1) for i in range(b)]


def _tensors(c):
    """Each gradient's (size, is bf16): the same for every seed."""
    k = c["tensors"]
    if c["sizes"] == "adapters":  # pairs of factors
        n = [c["most"] // (1, 2)[i % 2] for i in range(k)]
    elif c["sizes"] == "model":  # a vocabulary's rows, then each layer's
        layer = [1024, 2048 * 1024, 1024 * 1024, 1024 * 1024, 2048 * 1024, 1024, 3 << 20, 3 << 20, 3 << 20, 128, 128]
        n = ([c["most"], 1024] + layer * (k // len(layer)))[:k]
    else:  # every size from one value up
        n = [max(1, int(c["most"] ** ((7 * i % k) / max(1, k - 1)))) for i in range(k)]
    return [(v, c["form"] == "bf16" or (c["form"] == "mixed" and i % 3 != 0)) for i, v in enumerate(n)]


def work(case):
    c = case
    if c["kind"] == "clip":
        n = _tensors(c)
        return {"bytes": sum(2 * v * (2 if h else 4) for v, h in n) + 4, "flops": 3.0 * sum(v for v, _ in n)}
    r, w = (_size(t) for t in _types(c["form"]))
    if c["kind"] == "layernorm":
        n = c["rows"] * c["dim"]
        if not c["train"]:
            return {"bytes": n * (r + w) + 8 * c["dim"], "flops": 7.0 * n}
        d = _size(_dx_type(c))
        return {"bytes": n * (2 * r + w + d * (2 if c["residual"] else 1)) + 16 * c["dim"], "flops": 22.0 * n}
    n, s = sum(_lens(c)) * c["dim"], 4 * c["b"] * c["dim"]
    if not c["train"]:
        return {"bytes": n * (2 * r + w) + s * (2 if c["state"] else 1), "flops": 8.0 * n}
    # x, the gates and dh in; h, dx and the gates' gradients out; the states before and behind and their gradients
    return {"bytes": n * (3 * r + 3 * w) + s * (4 if c["state"] else 1), "flops": 22.0 * n}


# ── inputs ───────────────────────────────────────────────────────────────

def _inputs(c, seed):
    """The numbers that a case starts from, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std=1.0, mean=0.0, dtype=F32):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = {}
    if c["kind"] == "clip":  # one stretch of memory for each type, with gaps between the tensors
        where, end = [], {True: 0, False: 0}
        for n, h in _tensors(c):
            where.append((h, end[h], n))
            end[h] += n + c["gap"]
        s["where"] = where
        s["flat"] = {h: normal((n,), 0.01, 0.0, BF16 if h else F32) for h, n in end.items() if n}
        for h, o, n in where:  # nothing between them
            if c["gap"]:
                s["flat"][h][o + n:o + n + c["gap"]] = 0
        # the largest norm allowed: `share` of what such gradients have
        s["max"] = c["share"] * 0.01 * math.sqrt(sum(n for _, _, n in where))
        return s
    read, _ = _types(c["form"])
    d = c["dim"]
    if c["kind"] == "layernorm":
        s["x"] = normal((c["rows"], d), 1.5, 0.3, read)  # a residual stream is not centred
        s["w"] = normal((d,), 0.1, 1.0)
        if c["bias"]:
            s["b"] = normal((d,), 0.1)
        if c["train"]:
            s["dy"] = normal((c["rows"], d), 0.1, 0.0, read)
            if c["residual"]:
                s["res"] = normal((c["rows"], d), 0.1, 0.0, _dx_type(c))
        return s
    rows = c["b"] * c["n"]
    s["x"] = normal((rows, d), 1.0, 0.0, read)
    logits = normal((rows, d), 2.0, 2.5)  # from gates that forget at once to such that keep for long
    s["g"] = (logits if c["gate"] == "sigmoid" else torch.sigmoid(logits)).to(read)
    if c["state"]:
        s["h0"] = normal((c["b"], d))
    if c["train"]:
        s["dh"] = normal((rows, d), 0.1, 0.0, read)
        if c["state"]:
            s["dlast"] = normal((c["b"], d), 0.1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "scan":
        s["len"] = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
    if own:
        _handles(s)
    return s


# ── the plain forms ──────────────────────────────────────────────────────

def _plain_layernorm(s):
    c = s["case"]
    to = _types(c["form"])[1]
    x = s["x"].float()
    x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)
    x = x * r
    y = x * s["w"]
    out = dict(y=(y + s["b"] if c["bias"] else y).to(to))
    if c["train"]:
        dy = s["dy"].float()
        g = dy * s["w"]
        dx = (g - g.mean(-1, keepdim=True) - x * (g * x).mean(-1, keepdim=True)) * r
        if c["residual"]:
            dx = dx + s["res"].float()
        out.update(dx=dx.to(_dx_type(c)), dw=(dy * x).sum(0))
        if c["bias"]:
            out["db"] = dy.sum(0)
    return out


def _doubled(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, from h = 0: spans of twice the length in each pass."""
    d = 1
    while d < a.shape[1]:
        u = torch.cat([u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return u


def _plain_scan(s):
    c = s["case"]
    b, n, d = c["b"], c["n"], c["dim"]
    to = _types(c["form"])[1]
    x, g = s["x"].view(b, n, d).float(), s["g"].view(b, n, d).float()
    live = (torch.arange(n, device=x.device) < s["len"][:, None])[..., None]
    # of the gate: a and 1 - a
    a, rest = (torch.sigmoid(g), torch.sigmoid(-g)) if c["gate"] == "sigmoid" else (g, 1 - g)
    h0 = s["h0"] if c["state"] else torch.zeros(b, d, device=x.device)
    u = rest * x if c["coupled"] else x
    a, u = torch.where(live, a, 1.0), torch.where(live, u, 0.0)  # behind the end the state stays
    u = torch.cat([u[:, :1] + a[:, :1] * h0[:, None], u[:, 1:]], 1)
    h = _doubled(a, u)
    last = h[:, -1]
    out = dict(h=torch.where(live, h, 0.0).to(to).view(b * n, d), last=last)
    if not c["train"]:
        return out
    dh = torch.where(live, s["dh"].view(b, n, d).float(), 0.0)
    if c["state"]:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dlast"][:, None]], 1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)  # a_{t+1}
    G = _doubled(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    da = G * (before - x) if c["coupled"] else G * before
    if c["gate"] == "sigmoid":
        da = da * a * rest
    dx = G * rest if c["coupled"] else G
    out.update(dx=torch.where(live, dx, 0.0).to(to).view(b * n, d), dg=torch.where(live, da, 0.0).to(to).view(b * n, d))
    if c["state"]:
        out["dh0"] = a[:, 0] * G[:, 0]
    return out


def _plain_clip(s):
    total = torch.zeros((), device="cuda", dtype=F64)
    for h, o, n in s["where"]:
        total = total + s["flat"][h][o:o + n].float().square().sum(dtype=F64)
    norm = total.sqrt()
    scale = torch.where((norm > s["max"]) & norm.isfinite(), s["max"] / norm, 1.0).float()
    out = {h: torch.zeros_like(f) for h, f in s["flat"].items()}
    for h, o, n in s["where"]:
        out[h][o:o + n] = s["flat"][h][o:o + n].float() * scale
    return dict(norm=norm.float().view(1), **{"bf16" if h else "fp32": f for h, f in out.items()})


# ── the framework's calls ────────────────────────────────────────────────

class _Stream:
    """torch's current stream, as the entry points take one."""

    @property
    def handle(self):
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _handles(s):
    """Parameters, workspace and output buffers, as a program keeps them."""
    from valkyr_amd import kernels as K

    c = s["case"]
    dt = {F32: K.F32, BF16: K.BF16}
    s["K"] = K

    def new(shape, dtype=F32):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if c["kind"] == "clip":
        flat = {h: torch.zeros_like(f) for h, f in s["flat"].items()}
        s["list"] = K.grad_list([(s["flat"][h].data_ptr() + (2 if h else 4) * o, n, K.BF16 if h else K.F32,
                                  flat[h].data_ptr() + (2 if h else 4) * o) for h, o, n in s["where"]])
        out = dict(norm=new((1,)), **{"bf16" if h else "fp32": f for h, f in flat.items()})
        need = K.grad_clip_workspace_bytes(s["list"])
    else:
        read, write = _types(c["form"])
        d = c["dim"]
        if c["kind"] == "layernorm":
            back = _dx_type(c)
            s["p"] = K.layernorm_params(c["rows"], d, eps=1e-5, x_dtype=dt[read], y_dtype=dt[write], dy_dtype=dt[read],
                                        dx_dtype=dt[back])
            out = dict(y=new((c["rows"], d), write))
            need = 0
            if c["train"]:
                out.update(dx=new((c["rows"], d), back), dw=new((d,)))
                if c["bias"]:
                    out["db"] = new((d,))
                need = K.layernorm_backward_workspace_bytes(s["p"])
        else:
            s["p"] = K.scan_params(c["n"], d, n_batch=c["b"], coupled=c["coupled"], dtype=dt[read], out_dtype=dt[write],
                                   gate={"sigmoid": K.SCAN_SIGMOID, "decay": K.SCAN_DECAY}[c["gate"]])
            out = dict(h=new((c["b"] * c["n"], d), write), last=new((c["b"], d)))
            if c["train"]:
                out.update(dx=new((c["b"] * c["n"], d), write), dg=new((c["b"] * c["n"], d), write))
                if c["state"]:
                    out["dh0"] = new((c["b"], d))
                s["states"] = new((K.gated_scan_states_floats(s["p"]),))
            need = K.gated_scan_workspace_bytes(s["p"])
    s["out"] = out
    s["ws"] = torch.empty(max(16, need), device="cuda", dtype=torch.uint8)
    s["ptr"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    s["to"] = {k: v.data_ptr() for k, v in out.items()}
    s["stream"] = _Stream()


def _own(s):
    c, K, at, to, st = s["case"], s["K"], s["ptr"], s["to"], s["stream"]
    if c["kind"] == "clip":
        K.grad_clip(s["list"], s["max"], to["norm"], workspace=at["ws"], stream=st)
    elif c["kind"] == "layernorm":
        K.layernorm_forward(s["p"], at["x"], at["w"], at.get("b"), to["y"], stream=st)
        if c["train"]:
            K.layernorm_backward(s["p"], at["dy"], at["x"], at["w"], to["dx"], residual=at.get("res"), dw=to["dw"],
                                 db=to.get("db"), workspace=at["ws"], stream=st)
    else:
        length = at["len"] if c["ragged"] else None
        K.gated_scan_forward(s["p"], at["x"], at["g"], to["h"], h0=at.get("h0"), h_last=to["last"],
                             states=at.get("states"), length=length, workspace=at["ws"], stream=st)
        if c["train"]:
            K.gated_scan_backward(s["p"], at["x"], at["g"], at["states"], at["dh"], to["dx"], to["dg"],
                                  dh_last=at.get("dlast"), dh0=to.get("dh0"), length=length, workspace=at["ws"], stream=st)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"layernorm": _plain_layernorm, "scan": _plain_scan, "clip": _plain_clip}[state["case"]["kind"]](state)


# ── the same in 64 bits ──────────────────────────────────────────────────

def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["kind"] == "clip":
        wide = {h: f.double() for h, f in s["flat"].items()}  # (zeros between the tensors)
        norm = torch.cat([f.norm().view(1) for f in wide.values()]).norm()
        if norm.item() > s["max"]:
            wide = {h: f.mul_(s["max"] / norm.item()) for h, f in wide.items()}
        return dict(norm=norm.view(1), **{"bf16" if h else "fp32": f for h, f in wide.items()})
    if c["kind"] == "layernorm":
        step, parts = max(1, (1 << 26) // c["dim"]), []
        w = s["w"].double().requires_grad_()
        b = (s["b"] if c["bias"] else torch.zeros_like(s["w"])).double().requires_grad_()
        for r in range(0, c["rows"], step):
            x = s["x"][r:r + step].double().requires_grad_()
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            y = (x - mean) / (var + 1e-5).sqrt() * w + b
            if c["train"]:
                dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"][r:r + step].double())
                if c["residual"]:
                    dx = dx + s["res"][r:r + step].double()
                parts.append((y.detach(), dx, dw, db))
            else:
                parts.append((y.detach(),))
        out = dict(y=torch.cat([p[0] for p in parts]))
        if c["train"]:
            out.update(dx=torch.cat([p[1] for p in parts]), dw=sum(p[2] for p in parts))
            if c["bias"]:
                out["db"] = sum(p[3] for p in parts)
        return out
    b, n, d = c["b"], c["n"], c["dim"]
    h = torch.zeros(b, n, d, device="cuda", dtype=F64)
    last, dx, dg = torch.zeros(b, d, device="cuda", dtype=F64), None, None
    if c["train"]:
        dx, dg, dh0 = torch.zeros_like(h), torch.zeros_like(h), torch.zeros_like(last)
    for i, m in enumerate(_lens(c)):  # one sequence after the other, row by row
        x, g = (s[k].view(b, n, d)[i, :m].double() for k in ("x", "g"))
        a = 1 / (1 + torch.exp(-g)) if c["gate"] == "sigmoid" else g
        rest = 1 / (1 + torch.exp(g)) if c["gate"] == "sigmoid" else 1 - g
        now = start = s["h0"][i].double() if c["state"] else torch.zeros(d, device="cuda", dtype=F64)
        u = rest * x if c["coupled"] else x
        for t in range(m):
            now = torch.addcmul(u[t], a[t], now)
            h[i, t] = now
        last[i] = now
        if c["train"]:
            G = torch.empty_like(x)
            carry = s["dlast"][i].double() if c["state"] else torch.zeros(d, device="cuda", dtype=F64)
            for t in reversed(range(m)):
                G[t] = s["dh"].view(b, n, d)[i, t].double() + carry
                carry = a[t] * G[t]
            dh0[i] = carry
            da = G * torch.cat([start[None], h[i, :max(0, m - 1)]])[:m]
            if c["coupled"]:
                da = da - G * x
            dg[i, :m] = da * a * rest if c["gate"] == "sigmoid" else da
            dx[i, :m] = rest * G if c["coupled"] else G
    out = dict(h=h.view(b * n, d), last=last)
    if c["train"]:
        out.update(dx=dx.view(b * n, d), dg=dg.view(b * n, d))
        if c["state"]:
            out["dh0"] = dh0
    return out
