"""The norm of a list of gradients and their clipping, through the C ABI against the formulas in 64 bits:
refusals on the CPU, the kernels on the GPU.

Squares and their sums are in 64 bits (2^-53 a step, far below fp32's): a norm is off by its own rounding, U =
2^-24 of it, and a clipped gradient by one more, or by fp32's and bf16's (U16 = 2^-8) in turn.
"""
import ctypes as C
import math

import numpy as np
import pytest

from helpers import bf16_dev, dev, host, note
from test_rotary import U, U16, refused


def test_refusals():
    """Arguments are checked before any device work (the addresses here are not memory)."""
    from valkyr_amd import kernels as K

    ok = K.grad_list([(256, 16, K.F32), (512, 16, K.BF16)])
    clip = lambda g, m=1.0, norm=4096, **kw: refused(K.grad_clip, g, m, norm, **kw)  # noqa: E731
    assert refused(K.grad_norm, ok, None) == "InvalidArgument"
    assert refused(K.grad_norm, ok, 258) == "InvalidArgument"
    assert clip(ok, norm=258) == "InvalidArgument"
    assert clip(ok, workspace=264) == "InvalidArgument"
    for m in (-1.0, math.nan, -math.inf):
        assert clip(ok, m) == "InvalidArgument"
    for bad in ((None, 16, K.F32), (258, 16, K.F32), (257, 16, K.BF16), (256, 16, 2), (256, 16, K.F32, 514)):
        assert clip(K.grad_list([bad])) == "InvalidArgument"
    assert clip(K.grad_list([(256, 1 << 40, K.F32)])) == "Unsupported"
    assert clip(K.grad_list([(256 + (i << 42), (1 << 40) - 1, K.F32) for i in range(4)] + [(256, 4, K.F32)])) == "Unsupported"
    # outputs on top of each other, of another's gradient, or of a shifted own one
    for tensors in ([(256, 16, K.F32), (256, 16, K.F32)], [(256, 16, K.F32), (300, 16, K.F32)],
                    [(512, 16, K.BF16), (256, 16, K.F32, 540)], [(256, 16, K.F32, 1024), (512, 16, K.F32, 1084)],
                    [(256, 16, K.F32, 260)], [(256, 16, K.F32, 252)], [(4096, 64, K.F32, 256), (512, 8, K.F32), (300, 4, K.F32, 8192)]):
        assert clip(K.grad_list(tensors)) == "InvalidArgument", tensors


SIZES = {"one": [1], "few": [3, 1, 1024, 0, 17], "odd": [1, 4095, 4096, 4097, 100001, 7, 0, 255], "large": [3000001, 12, 1 << 20],
         "many": [(37 * i) % 501 + (i % 7 == 0) * 9000 for i in range(300)], "ones": [1] * 250}


class Grads:
    """Tensors one behind the other (with `gap` values between them) in a stretch of memory for each type."""

    def __init__(self, sizes, form, gap=0, seed=1, scale=1.0, shift=0, inplace=False):
        from valkyr_amd import kernels as K

        rng = np.random.default_rng(seed)
        self.K, where, end = K, [], [shift, shift]
        for i, n in enumerate(sizes):
            t = {"f": 0, "b": 1, "m": i % 3 != 0}[form] + 0
            where.append((t, end[t], n))
            end[t] += n + gap
        vals = [np.full(n + 1, 7.0, np.float32) for n in end]
        for t, o, n in where:
            vals[t][o:o + n] = rng.standard_normal(n).astype(np.float32) * np.float32(scale)
        self.where, self.inplace = where, inplace
        self.src, self.val = [None, None], [None, None]
        self.src[0], self.val[0] = dev(vals[0]), vals[0].astype(np.float64)
        self.src[1], v = bf16_dev(vals[1])
        self.val[1] = v.astype(np.float64)
        self.out = self.src if inplace else [dev(np.full(end[0] + 1, 7.0, np.float32)), bf16_dev(np.full(end[1] + 1, 7.0))[0]]
        at = lambda b, t, o: b[t].addr + o * (2 if t else 4)  # noqa: E731
        self.list = K.grad_list([(at(self.src, t, o), n, t) + (() if inplace else (at(self.out, t, o),)) for t, o, n in where])
        self.norm = dev(np.full(3, 7.0, np.float32))

    def read(self):
        from valkyr_amd.device import bf16_bits_to_f32

        return [host(self.out[0]).astype(np.float64), bf16_bits_to_f32(host(self.out[1], dtype=np.uint16)).astype(np.float64)]

    def true_norm(self):
        return math.sqrt(sum(float((self.val[t][o:o + n] ** 2).sum()) for t, o, n in self.where))

    def check(self, max_norm):
        want = self.true_norm()
        norm = host(self.norm)
        assert np.all(norm[1:] == 7.0)
        assert abs(float(norm[0]) - want) <= 1.0001 * U * want if want < 3.4e38 else np.isinf(norm[0])
        c = max_norm / want if want > max_norm else 1.0
        used = [np.zeros(v.shape, bool) for v in self.val]
        for t, o, n in self.where:
            used[t][o:o + n] = True
        for t, got in enumerate(self.read()):
            ref = self.val[t] * c
            off = np.abs(ref) * ((U16 + 1.01 * U if t else 1.01 * U) if c != 1.0 else 0.0) + (1e-40 if c != 1.0 and t else 2e-45 if c != 1.0 else 0)
            assert np.all(np.abs(got - ref)[used[t]] <= off[used[t]] if c != 1.0 else got[used[t]] == ref[used[t]])
            assert np.all(got[~used[t]] == 7.0)  # between the tensors


@pytest.mark.gpu
@pytest.mark.parametrize("inplace", [False, True], ids=["apart", "in-place"])
@pytest.mark.parametrize("form", ["f", "b", "m"])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_clip_matches_the_formula(sizes, form, inplace):
    for k, (gap, share) in enumerate(((0, 0.37), (3, 5.0), (1, 0.0), (0, math.inf))):
        note(f"clip {sizes} {form} gap {gap} share {share} in place {inplace}")
        g = Grads(SIZES[sizes], form, gap, seed=k, shift=k, inplace=inplace)
        norm = g.true_norm()
        m = float(np.float32(share * norm if math.isfinite(share) else share))
        g.K.grad_norm(g.list, g.norm)
        assert abs(float(host(g.norm)[0]) - norm) <= 1.0001 * U * norm
        assert np.array_equal(g.read()[0], g.val[0] if inplace else np.full_like(g.val[0], 7.0))  # the norm alone writes no gradient
        g.K.grad_clip(g.list, m, g.norm)
        g.check(m)


@pytest.mark.gpu
@pytest.mark.parametrize("scale,m", [(1e25, 1.0), (1e-30, 1e-30), (1e-38, 1.0), (3e38, 1e-3), (1e38, 1e38)])
def test_gradients_near_the_ends_of_fp32(scale, m):
    """Squares past fp32's range, a norm past it, gradients whose squares vanish in it."""
    note(f"clip of {scale}")
    rng = np.random.default_rng(3)
    g = Grads([4096, 999], "f", scale=1.0)
    v = np.clip(rng.standard_normal(g.val[0].size) * scale, -3.3e38, 3.3e38).astype(np.float32)
    v[-1] = 7.0
    g.src[0].upload(v)
    g.val[0] = v.astype(np.float64)
    m = float(np.float32(m))
    g.K.grad_clip(g.list, m, g.norm)
    g.check(m)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_leaves_the_gradients(bad):
    note(f"clip of {bad}")
    for inplace in (False, True):
        g = Grads([5000, 33, 200], "m", inplace=inplace)
        t, o, n = g.where[2]
        val = host(g.src[t], dtype=np.uint16 if t else np.float32)
        val[o + 11] = {math.inf: 0x7F80, -math.inf: 0xFF80}.get(bad, 0x7FC0)
        g.src[t].upload(val)
        before = [host(b, dtype=np.uint16) for b in g.src]
        g.K.grad_clip(g.list, 0.5, g.norm)
        assert not np.isfinite(host(g.norm)[0])
        for b, r in zip(g.out, before):
            got = host(b, dtype=np.uint16)
            assert inplace and np.array_equal(got, r) or np.array_equal(got[:-2], r[:-2])


@pytest.mark.gpu
def test_empty_lists_and_empty_tensors():
    g = Grads([0, 0], "f")
    for lst in (g.list, g.K.grad_list([]), g.K.grad_list([(None, 0, 0)])):
        g.norm.upload(np.full(3, 7.0, np.float32))
        g.K.grad_clip(lst, 1.0, g.norm)
        assert np.array_equal(host(g.norm), [0, 7, 7])
        g.K.grad_clip(lst, 1.0)
        g.norm.upload(np.full(3, 7.0, np.float32))
        g.K.grad_norm(lst, g.norm)
        assert np.array_equal(host(g.norm), [0, 7, 7])


@pytest.mark.gpu
def test_the_same_every_time_on_two_streams_and_replayed():
    from test_gpu_kernels import _replays
    from valkyr_amd import lib
    from valkyr_amd.device import Stream, synchronize

    note("clip on streams and in a graph")
    gs, st = [Grads(SIZES["many"] + [700001], "m", seed=s) for s in (5, 6)], [Stream(), Stream()]
    m = float(np.float32(0.5 * gs[0].true_norm()))  # (the call takes an fp32)
    synchronize()
    for _ in range(3):
        for g, s in zip(gs, st):
            g.K.grad_clip(g.list, m, g.norm, stream=s)
    synchronize()
    for g in gs:
        g.check(m)
    g = gs[0]
    fresh = [np.full(g.out[0].nbytes // 4, 7.0, np.float32), np.full(g.out[1].nbytes // 2, 0x40E0, np.uint16)]
    want = [host(b, dtype=np.uint16) for b in g.out] + [host(g.norm)]
    ws = dev(np.full(g.K.grad_clip_workspace_bytes(g.list) // 4, np.nan, np.float32))

    def check():
        for b, r in zip(g.out + [g.norm], want):
            assert np.array_equal(host(b, dtype=r.dtype), r)
        for b, r in zip(g.out, fresh):
            b.upload(r)

    _replays(lib(), st[0], lambda: g.K.grad_clip(g.list, m, g.norm, workspace=ws, stream=st[0]), check,
             lambda: g.K.grad_clip(g.list, m, g.norm, stream=st[0]))
    assert lib().hipStreamBeginCapture(st[0].handle, 0) == 0
    name = refused(g.K.grad_clip, g.list, m, g.norm, stream=st[0])
    graph = C.c_void_p()
    assert lib().hipStreamEndCapture(st[0].handle, C.byref(graph)) == 0 and lib().hipGraphDestroy(graph) == 0
    assert name == "InvalidArgument"


@pytest.mark.gpu
def test_a_tensor_past_two_to_the_32_bytes():
    """2^30 + 5 fp32 values, zeros but for both ends."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer

    note("clip of 4 GiB")
    n = (1 << 30) + 5
    big, norm = DeviceBuffer.zeros(n * 4), dev(np.zeros(1, np.float32))
    ends = np.arange(1, 101, dtype=np.float32)
    for at in (0, n - 100):
        check(lib().vkh_memcpy_h2d(big.offset(at * 4), ends.ctypes.data, ends.nbytes))
    want = math.sqrt(2 * float((ends.astype(np.float64) ** 2).sum()))
    K.grad_clip(K.grad_list([(big, n, K.F32)]), 2.0, norm)
    assert abs(float(host(norm)[0]) - want) <= 1.0001 * U * want
    for at in (0, n - 100):
        got = np.empty_like(ends)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, big.offset(at * 4), got.nbytes))
        ref = ends.astype(np.float64) * 2.0 / want
        assert np.all(np.abs(got - ref) <= 1.01 * U * ref)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 61, 200])
def test_tensors_far_from_each_other(n):
    """Every other tensor 9 GiB behind the one before it: more than 32 bits of an address apart."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer

    note(f"clip of {n} tensors 9 GiB apart")
    far, step, size = 9 << 30, 4096, 777
    big, norm = DeviceBuffer(far + (n + 1) * step), dev(np.zeros(1, np.float32))
    rng = np.random.default_rng(2)
    at = [(i % 2) * far + i * step + 4 * (i % 5) for i in range(n)]
    vals = [rng.standard_normal(size).astype(np.float32) for _ in at]
    for o, v in zip(at, vals):
        check(lib().vkh_memcpy_h2d(big.offset(o), v.ctypes.data, v.nbytes))
    want = math.sqrt(sum(float((v.astype(np.float64) ** 2).sum()) for v in vals))
    grads = K.grad_list([(big.offset(o), size, K.F32) for o in at])
    K.grad_norm(grads, norm)
    assert abs(float(host(norm)[0]) - want) <= 1.0001 * U * want
    K.grad_clip(grads, 1.5, norm)
    assert abs(float(host(norm)[0]) - want) <= 1.0001 * U * want
    for o, v in zip(at, vals):
        got = np.empty_like(v)
        check(lib().vkh_memcpy_d2h(got.ctypes.data, big.offset(o), got.nbytes))
        ref = v.astype(np.float64) * (1.5 / want)
        assert np.all(np.abs(got - ref) <= 1.01 * U * np.abs(ref) + 2e-45)


@pytest.mark.gpu
def test_a_norm_does_not_depend_on_where_the_tensors_lie():
    """200 tensors of 64 chunks (8192 values), each list of the same values at three places: all tensors one behind the
    other, one of them 9 GiB behind the rest, and outputs that far from each other.

    A chunk that holds 2^24, 2^12, 2^12 and 1, whose squares add up to m^2, m = 2^24 + 1, is followed by one whose eight
    values at one lane's first place have squares of 0.029 and are all that lane adds to the 2^48 there if one block
    takes both chunks: each is under half a step of 2^48 in 64 bits (2^-5), so the norm is m, halfway between two fp32
    numbers, and rounds to 2^24.  Where two blocks take them, the second's sum (0.23) counts and the norm rounds to
    2^24 + 2.  Which blocks take them follows from the sizes alone, so the three places give the same bits."""
    from valkyr_amd import kernels as K
    from valkyr_amd._lib import check, lib
    from valkyr_amd.device import DeviceBuffer

    note("norm of near and far tensors")
    chunk, chunks, n, far = 8192, 64, 200, 9 << 30
    size = chunk * chunks
    whole, apart = DeviceBuffer.zeros(n * size * 4), DeviceBuffer(far + n * size * 4)
    norm = dev(np.zeros(1, np.float32))
    near = [(whole.offset(i * size * 4), size, K.F32) for i in range(n)]
    moved = 100
    check(lib().vkh_memset(apart.offset(far), 0, size * 4))
    distant = list(near)
    distant[moved] = (apart.offset(far), size, K.F32)
    outs = [(g, k, t, apart.offset(i * size * 4 + (far if i % 2 else 0))) for i, (g, k, t) in enumerate(near)]
    lists = [K.grad_list(v) for v in (near, distant, outs)]
    big, small, none = (np.zeros(chunk, np.float32) for _ in range(3))
    big[:4] = 2.0**24, 2.0**12, 2.0**12, 1.0
    small[::1024] = 0.17
    seen = set()
    for at in range(64 * 3 + 5, 64 * n - 1, 197):
        if at % 64 == 63 or at // 64 == moved:  # (both chunks in one tensor)
            continue
        check(lib().vkh_memcpy_h2d(whole.offset(at * chunk * 4), big.ctypes.data, big.nbytes))
        check(lib().vkh_memcpy_h2d(whole.offset((at + 1) * chunk * 4), small.ctypes.data, small.nbytes))
        got = []
        for lst in lists[:2]:
            K.grad_norm(lst, norm)
            got.append(float(host(norm)[0]))
        for lst in lists[2:]:
            K.grad_clip(lst, 1e9, norm)
            got.append(float(host(norm)[0]))
        assert got == got[:1] * 3, (at, got)
        seen.add(got[0])
        for k in (at, at + 1):
            check(lib().vkh_memcpy_h2d(whole.offset(k * chunk * 4), none.ctypes.data, none.nbytes))
    assert seen == {2.0**24, 2.0**24 + 2}  # (both kinds of pairs were among them)


class Spread:
    """Tensors at given places of a stretch of memory, outputs at the same places of another."""

    def __init__(self, places, span, seed):
        from valkyr_amd import kernels as K
        from valkyr_amd._lib import check, lib
        from valkyr_amd.device import DeviceBuffer, bf16_bits_to_f32, f32_to_bf16_bits

        self.K, self.lib, self.check, self.places = K, lib(), check, places
        self.src, self.out = DeviceBuffer(span), DeviceBuffer(span)
        rng, self.val = np.random.default_rng(seed), []
        for at, n, t in places:
            v = rng.standard_normal(n, dtype=np.float32)
            raw = f32_to_bf16_bits(v) if t else v
            check(self.lib.vkh_memcpy_h2d(self.src.offset(at), raw.ctypes.data, raw.nbytes))
            self.val.append((bf16_bits_to_f32(raw) if t else v).astype(np.float64))
        self.norm = dev(np.zeros(1, np.float32))
        self.want = math.sqrt(sum(float((v ** 2).sum()) for v in self.val))

    def clip(self, limit, inplace):
        self.K.grad_clip(self.K.grad_list([(self.src.offset(at), n, t) + (() if inplace else (self.out.offset(at),))
                                           for at, n, t in self.places]), limit, self.norm)
        assert abs(float(host(self.norm)[0]) - self.want) <= 1.0001 * U * self.want
        return self.src if inplace else self.out

    def check_scaled(self, buf, c):
        from valkyr_amd.device import bf16_bits_to_f32

        for (at, n, t), v in zip(self.places, self.val):
            got = np.empty(n, np.uint16 if t else np.float32)
            self.check(self.lib.vkh_memcpy_d2h(got.ctypes.data, buf.offset(at), got.nbytes))
            ref = v * c
            off = np.abs(ref) * (U16 + 1.01 * U if t else 1.01 * U) + (1e-40 if t else 2e-45)
            assert np.all(np.abs((bf16_bits_to_f32(got) if t else got) - ref) <= off), (at, n, t)


@pytest.mark.gpu
def test_more_than_the_last_cache_holds_in_both_types():
    """410 MB at odd places, which are read past the caches, with whole chunks and rests of each type."""
    note("clip of 410 MB, both types")
    sizes, places, at = [(50000001, 1), (3, 0), (40000011, 0), (8192, 1), (12345, 0), (70000000, 1), (1, 1), (2 * 8192 + 5, 0)], [], 4
    for n, t in sizes:
        at += 2 if t else -at % 4
        places.append((at, n, t))
        at += n * (2 if t else 4) + 2
    assert sum(n * (2 if t else 4) for n, t in sizes) > 256 << 20
    g = Spread(places, at, 11)
    limit = float(np.float32(g.want / 3))
    g.check_scaled(g.clip(limit, False), limit / g.want)
    g.check_scaled(g.clip(limit, True), limit / g.want)


@pytest.mark.gpu
def test_both_types_far_from_each_other():
    """Tensors of both types in turn 9 GiB behind each other, more of them than one launch takes."""
    note("clip of both types, 9 GiB apart")
    far, places = 9 << 30, []
    for i in range(230):
        n = 1 + (53 * i) % 9001
        places.append(((i % 3 % 2) * far + i * 40000 + 4 * (i % 7) + 2 * (i % 2), n, i % 2))
    places = [(at - at % (2 if t else 4), n, t) for at, n, t in places]
    g = Spread(places, far + 230 * 40000 + 40000, 12)
    limit = float(np.float32(g.want / 5))
    g.check_scaled(g.clip(limit, False), limit / g.want)
    g.check_scaled(g.clip(limit, True), limit / g.want)
