"""The operators between a layer's projections and its attention output, as measurable cases.

A case is a dict of plain values; `kind` names its operator:

  rotary   rotary positions: pairs (i, i + r/2) or (2i, 2i + 1) of the first r of a head's values,
           any positions, frequencies scaled for long contexts; one direction per case
  qknorm   RMSNorm of each query and key head and the rotation in one pass, forward, and with
           `train` backward too, gain gradients included
  window   attention in which a query sees the last `window` keys up to its own and the first
           `sinks` keys; forward, and with `train` backward too

Types: "fp32" holds everything in 32 bits, "bf16" activations in bf16 and sums, gains, their
gradients and the log-sum-exp in 32 bits, "mixed" reads fp32 and writes bf16 (the projection's output
on its way to a bf16 attention, and back).
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# ── the cases ────────────────────────────────────────────────────────────

_PLAIN = dict(scaling="none", factor=1.0, orig_len=0, theta=1e6)


def listed():
    return [
        # One new token of each of 8 sequences, far into texts of up to four times the length
        # that the frequencies were made for.  Launch and latency.
        dict(kind="rotary", name="rotary_bf16_8", form="bf16", rows=8, seq=0, heads=32, kv_heads=8,
             head_dim=128, rotary=128, layout="half", scaling="yarn", factor=4.0, orig_len=32768,
             theta=1e6, backward=False),
        # A long batch, neighbouring pairs, only half of each head turned.
        dict(kind="rotary", name="rotary_bf16_16384", form="bf16", rows=16384, seq=4096, heads=32,
             kv_heads=8, head_dim=128, rotary=64, layout="interleaved", backward=False, **_PLAIN),
        # Gradients of one odd-sized document in the reference's precision, 96-wide heads.
        dict(kind="rotary", name="rotary_fp32_back_1001", form="fp32", rows=1001, seq=0, heads=12,
             kv_heads=4, head_dim=96, rotary=96, layout="half", scaling="linear", factor=4.0,
             orig_len=4096, theta=1e4, backward=True),
        # One token on its way into a bf16 attention, the headline step's heads.
        dict(kind="qknorm", name="qknorm_mixed_1", form="mixed", rows=1, seq=0, heads=16, kv_heads=8,
             head_dim=128, rotary=128, layout="half", train=False, **_PLAIN),
        # The headline step's batch (4 sequences of 512 tokens), read out of its fused q|k|v rows.
        dict(kind="qknorm", name="qknorm_mixed_train_2048", form="mixed", rows=2048, seq=512, heads=16,
             kv_heads=8, head_dim=128, rotary=128, layout="half", train=True, fused=True, **_PLAIN),
        # A long-context step's tokens, activations in bf16, frequencies scaled by wavelength.
        dict(kind="qknorm", name="qknorm_bf16_train_16384", form="bf16", rows=16384, seq=16384,
             heads=32, kv_heads=8, head_dim=128, rotary=128, layout="half", train=True,
             scaling="bands", factor=8.0, orig_len=8192, theta=5e5),
        # One new token of one sequence: latency.
        _window("window_bf16_step_1", form="bf16", b=1, n_q=1, n_kv=4096, heads=16, kv_heads=8,
                head_dim=128, window=1024, train=False),
        # One new token of each of 32 sequences of any length up to 32k.
        _window("window_bf16_step_32", form="bf16", b=32, n_q=1, n_kv=32768, heads=32, kv_heads=8,
                head_dim=128, window=4096, ragged=True, train=False),
        # A chunk of a long prompt against what came before it, 64-wide heads.
        _window("window_bf16_chunk_777", form="bf16", b=2, n_q=777, n_kv=5001, heads=16, kv_heads=4,
                head_dim=64, window=1000, train=False),
        # A padded batch of two odd-sized documents in the reference's precision.
        _window("window_fp32_train_1001", form="fp32", b=2, n_q=1001, n_kv=1001, heads=16, kv_heads=4,
                head_dim=64, window=256, sinks=1, ragged=True, train=True),
        # The attention of a fine-tune of four 2048-token sequences, out of fused q|k|v rows.
        _window("window_bf16_train_2048", form="bf16", b=4, n_q=2048, n_kv=2048, heads=16, kv_heads=8,
                head_dim=128, window=512, fused=True, train=True),
        # The largest: one long-context step's attention.
        _window("window_bf16_train_16384", form="bf16", b=1, n_q=16384, n_kv=16384, heads=32, kv_heads=8,
                head_dim=128, window=2048, train=True),
    ]


def _window(name, **kw):
    c = dict(kind="window", name=name, sinks=4, ragged=False, fused=False)
    c.update(kw)
    return c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4]), kv


def draw(rng):
    kind = rng.choices(["rotary", "qknorm", "window"], [2, 2, 3])[0]
    heads, kv = _draw_heads(rng)
    if kind != "window":
        hd = rng.choice([64, 80, 96, 128, 128, 256])
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        rows = _log(rng, 1, 16384)
        c = dict(kind=kind, form=rng.choice(["fp32", "bf16"] if kind == "rotary" else ["fp32", "mixed", "bf16"]),
                 rows=rows, seq=rng.choice([0, max(1, rows // 3)]), heads=heads, kv_heads=kv, head_dim=hd,
                 rotary=hd // rng.choice([1, 1, 2, 4]), layout=rng.choice(["half", "interleaved"]),
                 scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                 orig_len=rng.choice([2048, 8192, 32768]), theta=rng.choice([1e4, 5e5, 1e6]))
        c["backward" if kind == "rotary" else "train"] = rng.random() < 0.5
        return c
    form = rng.choice(["bf16", "bf16", "fp32"])
    c = _window("", form=form, b=rng.choice([1, 2, 3, 4]), heads=heads, kv_heads=kv,
                head_dim=rng.choice([64, 128]), sinks=rng.choice([0, 1, 4, 16]), ragged=rng.random() < 0.4)
    del c["name"]
    use = rng.choice(["step", "chunk", "train", "train"])
    c["train"] = use == "train"
    if use == "step":
        c.update(n_q=rng.choice([1, 1, 4]), n_kv=_log(rng, 64, 32768), window=_log(rng, 16, 8192))
    elif use == "chunk":
        c["n_kv"] = _log(rng, 64, (16384 if form == "bf16" else 2048) // c["b"])
        c.update(n_q=max(1, c["n_kv"] // rng.choice([2, 3, 8])), window=_log(rng, 16, 4096))
    else:
        n = _log(rng, 16, (16384 if form == "bf16" else 2048) // c["b"])
        c.update(n_q=n, n_kv=n, window=_log(rng, 8, 2048), fused=rng.random() < 0.3)
    return c


# ── what a pass cannot do without ────────────────────────────────────────

def _sizes(form):
    """Bytes of a value as it is read and as it is written (of a gradient: the other way round)."""
    return {"fp32": (4, 4), "bf16": (2, 2), "mixed": (4, 2)}[form]


def _lens(c):
    """The sequences' query rows and keys: in a ragged batch between a 16th of the room and all of it."""
    n, lo = c["n_kv"], max(c["n_q"] if c["n_q"] < c["n_kv"] else 1, c["n_kv"] // 16)
    kv = [n if not c["ragged"] else lo + (n - lo) * (7 * i % c["b"]) // max(1, c["b"] - 1) if c["b"] > 1 else n
          for i in range(c["b"])]
    return [min(c["n_q"], v) if c["n_q"] == c["n_kv"] else c["n_q"] for v in kv], kv


def _seen(c):
    """(query, key) pairs of one head over all sequences, and the keys that any query sees."""
    pairs = keys = 0
    w, ns = c["window"], c["sinks"]
    for nq, nk in zip(*_lens(c)):
        first, last = nk - nq, nk - 1  # positions

        def upto(t):  # sum over positions 0..t of min(position + 1, w), and of the sinks before the window
            full = max(0, t + 1 - w)
            inside = (t + 1 - full) * (t + 2 - full) // 2 if t < w else w * (w + 1) // 2
            before = max(0, t + 1 - w)  # positions t >= w see min(ns, t - w + 1) sinks more
            short = min(before, ns)
            return inside + full * w + short * (short + 1) // 2 + max(0, before - ns) * ns

        pairs += upto(last) - (upto(first - 1) if first > 0 else 0)
        start = max(0, first - w + 1)
        keys += nk - start + min(ns, start)
    return pairs, keys


def work(case):
    c = case
    r, w = _sizes(c["form"])
    if c["kind"] == "window":
        pairs, keys = _seen(c)
        rows = sum(_lens(c)[0])
        q, kv = rows * c["heads"] * c["head_dim"], keys * c["kv_heads"] * c["head_dim"]
        lse = 4 * rows * c["heads"]
        if not c["train"]:
            return {"bytes": r * (q + 2 * kv) + w * q + lse, "flops": 4.0 * pairs * c["heads"] * c["head_dim"]}
        # q, k, v and dO in; O, the log-sum-exp, dQ, dK and dV out
        return {"bytes": r * (2 * q + 2 * kv) + w * (2 * q + 2 * kv) + lse,
                "flops": 14.0 * pairs * c["heads"] * c["head_dim"]}
    n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
    if c["kind"] == "rotary":
        return {"bytes": n * (r + w) + 4 * c["rows"], "flops": 3.0 * n}
    if not c["train"]:
        return {"bytes": n * (r + w) + 4 * c["rows"] + 8 * c["head_dim"], "flops": 8.0 * n}
    # x and dy in, y and dx out
    return {"bytes": 2 * n * (r + w) + 4 * c["rows"] + 16 * c["head_dim"], "flops": 24.0 * n}


# ── inputs ───────────────────────────────────────────────────────────────

def _normal(g, shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _projected(c, g, rows, nh, nkv, dtype):
    """Query and key (and value) rows: of a fused q|k|v matrix, or each on its own."""
    hd = c["head_dim"]
    if c.get("fused"):
        x = _normal(g, (rows, (nh + 2 * nkv) * hd), 1.0, dtype)
        return x[:, :nh * hd], x[:, nh * hd:(nh + nkv) * hd], x[:, (nh + nkv) * hd:]
    return tuple(_normal(g, (rows, n * hd), 1.0, dtype) for n in (nh, nkv, nkv))


def _inputs(c, seed):
    """The numbers that a case starts from, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    read = BF16 if c["form"] == "bf16" else F32
    if c["kind"] == "window":
        q = _projected(c, g, c["b"] * c["n_q"], nh, nkv, read)
        kv = q if c["n_q"] == c["n_kv"] else _projected(c, g, c["b"] * c["n_kv"], 0, nkv, read)
        s = dict(q=q[0], k=kv[1], v=kv[2])
        if c["train"]:
            s["do"] = _normal(g, (c["b"] * c["n_q"], nh * hd), 0.1, read)
        return s
    n = c["rows"]
    s = {}
    s["q"], s["k"], _ = _projected(c, g, n, nh, nkv, read)
    # sequences of `seq` tokens from position 0 on; without it, rows anywhere in a long text
    s["pos"] = (torch.arange(n, device="cuda") % c["seq"] if c["seq"] else
                torch.randint(0, max(2, 4 * c["orig_len"], 4096), (n,), generator=g, device="cuda")).to(torch.int32)
    if c["kind"] == "qknorm":
        s["wq"], s["wk"] = 1.0 + _normal(g, (hd,), 0.1), 1.0 + _normal(g, (hd,), 0.1)
        if c["train"]:
            write = F32 if c["form"] == "fp32" else BF16
            dy = F32 if c["form"] == "mixed" else write  # fp32 gradients from the attention
            s["dq"], s["dk"] = _normal(g, (n, nh * hd), 0.1, dy), _normal(g, (n, nkv * hd), 0.1, dy)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "window":
        nq, nk = _lens(case)
        s["nq"], s["nk"] = (torch.tensor(v, device="cuda", dtype=torch.int32) for v in (nq, nk))
    else:
        s["freq"], s["scale"] = _frequencies(case)
        s["freq"] = torch.tensor(s["freq"], device="cuda", dtype=F64)
    if own:
        _handles(s)
    return s


# ── the plain forms ──────────────────────────────────────────────────────

def _frequencies(c):
    """Radians a position for each pair, and what the rotated values are multiplied by."""
    r, theta, s = c["rotary"], c["theta"], c["factor"]
    base = theta * s ** (r / (r - 2)) if c["scaling"] == "ntk" else theta
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    if c["scaling"] == "linear":
        return [x / s for x in f], 1.0
    if c["scaling"] == "yarn":  # pairs of over 32 turns in the original length stay, of under one are stretched
        lo, hi = (r * math.log(c["orig_len"] / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32, 1))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / ((hi - lo) or 1e-3))) for i in range(r // 2)]
        return [x * (1 - t) + x / s * t for x, t in zip(f, ramp)], 0.1 * math.log(s) + 1
    if c["scaling"] == "bands":  # between one and four turns in the original length
        t = [min(1.0, max(0.0, (c["orig_len"] * x / (2 * math.pi) - 1) / 3)) for x in f]
        return [x * u + x / s * (1 - u) for x, u in zip(f, t)], 1.0
    return f, 1.0


def _angles(s):
    a = s["pos"].to(F64)[:, None, None] * s["freq"]  # a far position times a frequency: not in 32 bits
    return (a.cos() * s["scale"]).float(), (a.sin() * s["scale"]).float()


def _rotate(c, x, cos, sin):
    """x [rows, heads, hd] in 32 bits."""
    r = c["rotary"]
    if c["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)


def _heads(c, x):
    return x.float().unflatten(-1, (-1, c["head_dim"]))


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    sin = -sin if c["backward"] else sin
    to = F32 if c["form"] == "fp32" else BF16
    return {n: _rotate(c, _heads(c, s[n]), cos, sin).flatten(-2).to(to) for n in ("q", "k")}


def _plain_qknorm(s):
    c = s["case"]
    cos, sin = _angles(s)
    to = F32 if c["form"] == "fp32" else BF16

    def one(x, w, dy):
        x = _heads(c, x)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        x = x * r
        y = _rotate(c, x * w, cos, sin).flatten(-2).to(to)
        if dy is None:
            return y, None, None
        g = _rotate(c, _heads(c, dy), cos, -sin)
        gw = g * w
        return y, ((gw - x * (gw * x).mean(-1, keepdim=True)) * r).flatten(-2).to(to), (g * x).sum((0, 1))

    q, dq, dwq = one(s["q"], s["wq"], s.get("dq"))
    k, dk, dwk = one(s["k"], s["wk"], s.get("dk"))
    return dict(q=q, k=k, dq=dq, dk=dk, dwq=dwq, dwk=dwk) if c["train"] else dict(q=q, k=k)


def _plain_window(s):
    """Blocks of about `window` queries against the keys that any of them may see: the sinks, then
    the window's, gathered."""
    c = s["case"]
    b, nq, nk, nh, nkv, hd = (c[n] for n in ("b", "n_q", "n_kv", "heads", "kv_heads", "head_dim"))
    w, ns, grp = min(c["window"], nk), min(c["sinks"], nk), nh // nkv
    size = min(nq, max(64, w))
    nb = -(-nq // size)
    dev = s["q"].device
    row = torch.arange(nb * size, device=dev).view(nb, size)
    pos = row + (s["nk"] - s["nq"]).view(b, 1, 1)  # [b, nb, size]
    live = (row < s["nq"].view(b, 1, 1)) & (pos >= 0)
    start = (s["nk"] - s["nq"]).view(b, 1) + torch.arange(nb, device=dev) * size - (w - 1)  # [b, nb]
    key = torch.cat([torch.arange(ns, device=dev).expand(b, nb, ns),
                     start[..., None] + torch.arange(w + size - 1, device=dev)], -1)  # [b, nb, cols]
    sink = torch.arange(key.shape[-1], device=dev) < ns
    t, j = pos[..., None], key[:, :, None, :]
    see = (j >= 0) & (j < s["nk"].view(b, 1, 1, 1)) & (j <= t) & torch.where(sink, j <= t - w, j > t - w)
    see = (see & live[..., None])[:, :, None, None]  # [b, nb, 1, 1, size, cols]
    at = key.clamp(0, nk - 1) + torch.arange(b, device=dev).view(b, 1, 1) * nk

    def rows(x):  # [b * nq, nh * hd] -> [b, nb, nkv, grp, size, hd]
        x = torch.nn.functional.pad(x.reshape(b, nq, nkv, grp, hd).float(), (0, 0, 0, 0, 0, 0, 0, nb * size - nq))
        return x.view(b, nb, size, nkv, grp, hd).permute(0, 1, 3, 4, 2, 5).contiguous()

    def keys(x):  # [b * nk, nkv * hd] -> [b, nb, nkv, 1, cols, hd]
        return x.view(-1, nkv, hd)[at].float().permute(0, 1, 3, 2, 4).unsqueeze(3).contiguous()

    def unrows(x):
        return x.permute(0, 1, 4, 2, 3, 5).reshape(b, nb * size, nh * hd)[:, :nq].reshape(b * nq, nh * hd).to(to)

    def unkeys(x):  # each block's share of a key's gradient added to the others'
        x = x.permute(0, 1, 3, 2, 4).reshape(-1, nkv * hd)
        return torch.zeros(b * nk, nkv * hd, device=dev).index_add_(0, at.reshape(-1), x).to(to)

    to = F32 if c["form"] == "fp32" else BF16
    scale = 1.0 / math.sqrt(hd)
    q, k, v = rows(s["q"]), keys(s["k"]), keys(s["v"])
    z = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~see, -math.inf)
    top = z.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    o = torch.matmul(p, v)
    lse = (top + total.log()).squeeze(-1).permute(0, 1, 4, 2, 3).reshape(b, nb * size, nh)[:, :nq].reshape(-1, nh)
    out = dict(o=unrows(o), lse=lse)
    if c["train"]:
        do = rows(s["do"])
        dv = torch.matmul(p.transpose(-1, -2), do).sum(3)
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out.update(dq=unrows(torch.matmul(ds, k)), dk=unkeys(torch.matmul(ds.transpose(-1, -2), q).sum(3)), dv=unkeys(dv))
    return out


# ── the framework's calls ────────────────────────────────────────────────

class _Stream:
    """torch's current stream, as the entry points take one."""

    @property
    def handle(self):
        return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _handles(s):
    """Parameters, plan, workspace and output buffers, as a program keeps them."""
    from valkyr_amd import kernels as K

    c = s["case"]
    dt = {F32: K.F32, BF16: K.BF16}
    write = F32 if c["form"] == "fp32" else BF16
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    s["K"] = K

    def new(n, w, dtype=write):
        return torch.empty(n, w, device="cuda", dtype=dtype)

    if c["kind"] == "window":
        rows, keys = c["b"] * c["n_q"], c["b"] * c["n_kv"]
        s["p"] = K.window_params(c["n_q"], c["n_kv"], nh, nkv, hd, c["window"], c["sinks"], n_batch=c["b"],
                                 dtype=dt[s["q"].dtype], out_dtype=dt[write], ld_q=s["q"].stride(0),
                                 ld_k=s["k"].stride(0), ld_v=s["v"].stride(0))
        out = s["out"] = dict(o=new(rows, nh * hd), lse=new(rows, nh, F32))
        need = K.fa_window_forward_workspace_bytes(s["p"])
        if c["train"]:
            out.update(dq=new(rows, nh * hd), dk=new(keys, nkv * hd), dv=new(keys, nkv * hd))
            s["d"] = new(rows, nh, F32)
            need = max(need, K.fa_window_backward_workspace_bytes(s["p"]))
    else:
        n = c["rows"]
        s["plan"] = K.rotary_plan(
            c["rotary"], c["theta"], layout={"half": K.ROTARY_HALF, "interleaved": K.ROTARY_INTERLEAVED}[c["layout"]],
            scaling={"none": K.ROTARY_UNSCALED, "linear": K.ROTARY_LINEAR, "ntk": K.ROTARY_NTK,
                     "yarn": K.ROTARY_YARN, "bands": K.ROTARY_BANDS}[c["scaling"]],
            factor=c["factor"], orig_len=c["orig_len"])
        read = dt[s["q"].dtype]
        back = dt[s["dq"].dtype] if "dq" in s else read
        s["p"] = K.rotary_params(n, nh, nkv, hd, eps=1e-6, x_dtype=read, y_dtype=dt[write], dy_dtype=back,
                                 dx_dtype=dt[write], ld_xq=s["q"].stride(0), ld_xk=s["k"].stride(0))
        out = s["out"] = dict(q=new(n, nh * hd), k=new(n, nkv * hd))
        need = 0
        if c.get("train"):
            out.update(dq=new(n, nh * hd), dk=new(n, nkv * hd), dwq=new(1, hd, F32)[0], dwk=new(1, hd, F32)[0])
            need = K.qk_norm_rotary_workspace_bytes(s["p"])
    s["ws"] = torch.empty(max(16, need), device="cuda", dtype=torch.uint8)
    s["ptr"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    s["to"] = {k: v.data_ptr() for k, v in out.items()}
    s["stream"] = _Stream()


def _own(s):
    c, K, p, at, to, st = s["case"], s["K"], s["p"], s["ptr"], s["to"], s["stream"]
    if c["kind"] == "rotary":
        call = K.rotary_backward if c["backward"] else K.rotary_forward
        call(p, s["plan"], at["q"], to["q"], at["k"], to["k"], positions=at["pos"], stream=st)
    elif c["kind"] == "qknorm":
        K.qk_norm_rotary_forward(p, s["plan"], at["wq"], at["wk"], at["q"], to["q"], at["k"], to["k"],
                                 positions=at["pos"], stream=st)
        if c["train"]:
            K.qk_norm_rotary_backward(p, s["plan"], at["wq"], at["wk"], at["q"], at["k"], at["dq"], at["dk"],
                                      to["dq"], to["dk"], to["dwq"], to["dwk"], positions=at["pos"],
                                      workspace=at["ws"], stream=st)
    else:
        lens = dict(q_len=at["nq"], kv_len=at["nk"]) if c["ragged"] else {}
        K.fa_window_forward(p, at["q"], at["k"], at["v"], to["o"], to["lse"], workspace=at["ws"], stream=st, **lens)
        if c["train"]:
            K.fa_window_backward(p, at["q"], at["k"], at["v"], to["o"], at["do"], to["lse"], at["d"], to["dq"],
                                 to["dk"], to["dv"], workspace=at["ws"], stream=st, **lens)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "qknorm": _plain_qknorm, "window": _plain_window}[state["case"]["kind"]](state)


# ── the same in 64 bits ──────────────────────────────────────────────────

def _turned(c, x, pos, sign):
    """x [rows, heads, hd] in 64 bits, its pairs as complex numbers turned by position times frequency."""
    f, a = _frequencies(c)
    r = c["rotary"]
    turn = torch.polar(torch.full((1,), a, device=x.device, dtype=F64),
                       sign * pos.double()[:, None] * torch.tensor(f, device=x.device, dtype=F64))[:, None]
    y = x.clone()
    lo, hi = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(x[..., lo].contiguous(), x[..., hi].contiguous()) * turn
    y[..., lo], y[..., hi] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    hd = c["head_dim"]
    if c["kind"] == "rotary":
        sign = -1 if c["backward"] else 1
        return {n: _turned(c, s[n].double().unflatten(-1, (-1, hd)), s["pos"], sign).flatten(-2) for n in ("q", "k")}
    if c["kind"] == "qknorm":
        out = {}
        for n, w in (("q", "wq"), ("k", "wk")):
            x = s[n].double().unflatten(-1, (-1, hd)).contiguous().requires_grad_()
            g = s[w].double().requires_grad_()
            u = x / (x.square().sum(-1, keepdim=True) / hd + 1e-6).sqrt() * g
            out[n] = _turned(c, u.detach(), s["pos"], 1).flatten(-2)
            if c["train"]:  # the rotation's transpose turns back
                du = _turned(c, s["d" + n].double().unflatten(-1, (-1, hd)), s["pos"], -1)
                dx, out["dw" + n] = torch.autograd.grad(u, (x, g), du)
                out["d" + n] = dx.flatten(-2)
        return out
    b, nh, nkv = c["b"], c["heads"], c["kv_heads"]
    o = torch.zeros(b, c["n_q"], nh, hd, device="cuda", dtype=F64)
    lse = torch.full((b, c["n_q"], nh), -math.inf, device="cuda", dtype=F64)
    q, do = (s[n].reshape(b, c["n_q"], nh, hd) if n in s else None for n in ("q", "do"))
    k, v = (s[n].reshape(b, c["n_kv"], nkv, hd) for n in ("k", "v"))
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(b, c["n_kv"], nkv, hd, device="cuda", dtype=F64) for _ in range(2))
    for i, (lq, lk) in enumerate(zip(*_lens(c))):
        for r0 in range(0, lq, 2048):  # the rows of one piece and every key up to its last
            r1 = min(lq, r0 + 2048)
            t = torch.arange(r0, r1, device="cuda")[:, None] + (lk - lq)
            lo = max(0, r0 + lk - lq - c["window"] + 1)
            j = torch.cat([torch.arange(min(c["sinks"], lo), device="cuda"), torch.arange(lo, r1 + lk - lq, device="cuda")])
            hidden = (j > t) | ((t - j >= c["window"]) & (j >= c["sinks"]))
            for h in range(nh):
                kh = h // (nh // nkv)
                x, y, z = (a.double() for a in (q[i, r0:r1, h], k[i, j, kh], v[i, j, kh]))
                sc = (x @ y.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                lse[i, r0:r1, h] = torch.logsumexp(sc, 1)
                p = torch.softmax(sc, 1)
                o[i, r0:r1, h] = p @ z
                if c["train"]:
                    g = do[i, r0:r1, h].double()
                    dv[i, :, kh].index_add_(0, j, p.T @ g)
                    dp = g @ z.T
                    ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(hd)
                    dq[i, r0:r1, h] = ds @ y
                    dk[i, :, kh].index_add_(0, j, ds.T @ x)
    out = dict(o=o.view(-1, nh * hd), lse=lse.view(-1, nh))
    if c["train"]:
        out.update(dq=dq.view(-1, nh * hd), dk=dk.view(-1, nkv * hd), dv=dv.view(-1, nkv * hd))
    return out
