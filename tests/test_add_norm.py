"""add_norm: the HIP kernel (clarus_hip_add_norm) against the formula in 64 bits.

Tolerance, u = 2^-24, m the additions that a lane and the tree over lanes make in a row (8 octets of 8 and 8 steps at
most: 72). A norm of values v off by e each (e 0 for inputs):
  difference from the mean: u of itself for the first mean, as much for the second; the second mean's own error is m u
  of the mean difference (at most the deviation s): (m + 4) u s in all, and 2 e
  deviation: relative (m + 4) u / 2 + 2 u of the root and its reciprocal, and 2 e / s
  normed: at most ((m + 8) u + 4 e / s) (1 + |v^|); with v^ 0 where s is 0 (equal values, whose mean is off by 2^-46 of them)
The sum: post's error times |scale gate pw|, two roundings of it, three of |scale gate| |pb|, one of the sum.
The outputs are rounded once more: 2^-8 (bf16) or u of themselves.
"""
from __future__ import annotations

import math

import pytest
import torch

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

U = 2.0 ** -24
M = 72


def _rows(t, c):
    return t.double().reshape(-1, 1, c)


def norm64(v, e, kind, eps):
    """(normed, its error) of values off by e."""
    if not kind:
        return v, e
    mean = v.mean(-1, keepdim=True) if kind is True else torch.zeros_like(v[..., :1])
    s = torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    out = (v - mean) / s
    e = e.amax(-1, keepdim=True)
    return out, ((M + 8) * U + 4 * e / s + 2.0 ** -46 * v.abs() / s) * (1 + out.abs())


def plain64(x, y=None, gate=None, scale=1.0, post=False, post_weight=None, post_bias=None, ln=True, weight=None, bias=None,
            eps=1e-6):
    """(sum, its error, norm, its error) before their roundings, [N, rows, C] float64."""
    n, c = x.shape[0], x.shape[-1]
    r = x.double().reshape(n, -1, c)
    e = torch.zeros_like(r)
    if y is not None:
        a, ea = norm64(y.double().reshape(r.shape), torch.zeros_like(r), post, eps)
        f = torch.ones(1, 1, 1, dtype=torch.float64, device=x.device) * scale
        f = f if gate is None else f * _rows(gate, c)
        pw = 1.0 if post_weight is None else _rows(post_weight, c)
        pb = torch.zeros_like(f) if post_bias is None else _rows(post_bias, c)
        r = r + f * (a * pw + pb)
        e = (f * pw).abs() * (ea + 4 * U * a.abs()) + 4 * U * (f * pb).abs() + U * r.abs()
    if not ln:
        return r, e, None, None
    h, eh = norm64(r, e, ln, eps)
    w = torch.ones(1, 1, 1, dtype=torch.float64, device=x.device) if weight is None else _rows(weight, c)
    b = torch.zeros_like(w) if bias is None else _rows(bias, c)
    return r, e, h * w + b, w.abs() * eh + 2 * U * (h * w).abs() + U * b.abs()


def check(got, x, y=None, what="", **kw):
    total, norm = got
    r, er, h, eh = plain64(x, y, **kw)
    pairs = [("sum", total, r, er)] if y is not None else []
    assert (norm is None) == (h is None), what
    pairs += [("norm", norm, h, eh)] if h is not None else []
    for name, t, ref, e in pairs:
        assert t.shape == x.shape and t.is_contiguous(), f"{what} {name}"
        t = t.reshape(ref.shape)
        tol = e + (2.0 ** -8 if t.dtype == torch.bfloat16 else U) * (ref.abs() + e)
        assert torch.isfinite(t).all(), f"{what} {name}"
        off = (t.double() - ref).abs()
        assert (off <= tol).all(), f"{what} {name}: max|d| {off.max().item():.3e}, {(off - tol).max().item():.3e} past the tolerance"


def rand(*shape, dt=torch.float32, dev="cpu", seed=0, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + shift).to(dt).to(dev)


# ------------------------------------------------------------------ CPU
def cpu_hip(dtype=torch.float32):
    from clarus_amd.hip_ops import HipOps
    h = HipOps.__new__(HipOps)
    h.dtype, h.device, h.dev, h._cache, h._plans = dtype, torch.device("cpu"), torch.device("cpu"), {}, {}
    h.lib = _lib.load()
    return h


def test_refusals():
    h, z = cpu_hip(), torch.zeros
    x = z(2, 5, 64)
    cases = [
        ((z(2, 5, 60),), {}), ((z(64),), {}), ((z(2, 1, 16392),), {}), ((x.half(),), {}), ((x, x.half()), {}), ((x, z(2, 4, 64)), {}),
        ((x, z(1, 5, 64)), {}), ((x,), {"out_dtype": torch.float16}), ((x,), {"ln": "layer"}), ((x,), {"ln": 1}), ((x,), {"ln": None}),
        ((x, x), {"post": "x"}), ((x, x), {"post": 1.0}), ((x, x), {"gate": z(32)}), ((x, x), {"gate": z(1, 64)}),
        ((x, x), {"gate": z(2, 5, 64)}), ((x, x), {"post_weight": z(64, dtype=torch.int32)}), ((x,), {"weight": z(2, 1, 64)}),
        ((x,), {"bias": z(3, 64)}), ((x,), {"eps": -1e-6}), ((x,), {"eps": math.nan}), ((x,), {"eps": 1e39}),
        ((x, x), {"scale": math.inf}), ((x, x), {"scale": 1e39}), ((x, x), {"scale": math.nan}),
        ((z(2, 64, 5).transpose(1, 2),), {}), ((z(2, 5, 66)[..., :64],), {}), ((x, z(2, 5, 66)[..., :64]), {}), ((z(2, 5, 65)[..., 1:],), {}),
        ((x.clone().requires_grad_(),), {}), ((x, x.clone().requires_grad_()), {}), ((x, x), {"gate": z(64).requires_grad_()}),
        ((z(1, 1, 8).expand(1 << 23, 1, 8),), {}), ((z(1, 1, 8).expand(1, 1 << 31, 8),), {}),
    ]
    for i, (args, kw) in enumerate(cases):
        with pytest.raises(Unsupported):
            h.add_norm(*args, **kw)
            pytest.fail(f"case {i} was accepted")
    total, norm = h.add_norm(z(2, 0, 64), z(2, 0, 64))
    assert total.shape == norm.shape == (2, 0, 64)
    assert h.add_norm(x, ln=False) == (x, None)  # nothing to do


def test_c_entry_refuses_before_launch():
    import ctypes
    lib = _lib.load()
    assert lib.clarus_hip_add_norm(None, None) == _lib.EINVAL
    base = dict(x=1 << 20, y=1 << 21, sum=1 << 22, norm=1 << 23, n=2, rows=6, c=64, x_bstride=384, ldx=64, y_bstride=384, ldy=64,
                post=1, pre=1, scale=1.0, eps=1e-6)
    for kw in (dict(x=None), dict(sum=None), dict(y=None, norm=None), dict(n=0), dict(rows=0), dict(c=0), dict(c=60), dict(c=16392),
               dict(n=1 << 23, rows=1), dict(n=1 << 62, rows=4), dict(n=2, rows=1 << 30), dict(rows=1 << 62), dict(x_dtype=2), dict(y_dtype=-1),
               dict(sum_dtype=2), dict(norm_dtype=7), dict(post=2), dict(pre=5), dict(eps=-1.0), dict(eps=math.nan), dict(scale=math.inf),
               dict(x=(1 << 20) + 8), dict(y=(1 << 21) + 4), dict(sum=(1 << 22) + 8), dict(norm=(1 << 23) + 8), dict(ldx=66), dict(ldy=-64),
               dict(x_bstride=2), dict(gate=8), dict(w=4), dict(b=8), dict(post_w=8), dict(post_b=8), dict(w_bstride=-64), dict(gate_bstride=2)):
        assert lib.clarus_hip_add_norm(ctypes.byref(_lib.AddNormArgs(**{**base, **kw})), None) == _lib.EINVAL, kw
        assert b"add_norm" in lib.clarus_hip_last_error()


KINDS = [(False, True), (True, "rms"), ("rms", True), ("rms", False), (True, True), (False, False)]


@pytest.mark.parametrize("post,ln", KINDS)
def test_plain_forms(post, ln):
    """The oracle's form and the torch backend's, and the latter's gradients against differences."""
    from clarus_amd.spatial_torch import TorchSpatialOps
    from oracle.torch_ref import TorchRef
    x, y = rand(2, 3, 4, 40, scale=2.0, shift=1.0), rand(2, 3, 4, 40, seed=1)
    kw = dict(gate=rand(2, 40, seed=2), scale=0.5, post=post, post_weight=rand(40, seed=3), post_bias=rand(2, 40, seed=4), ln=ln,
              weight=rand(40, seed=5), bias=rand(2, 40, seed=6))
    check(TorchRef(torch.float32, "cpu").add_norm(x, y, **kw), x, y, **kw)
    ops = TorchSpatialOps(torch.float32, torch.device("cpu"))
    check(ops.add_norm(x, y, **kw), x, y, **kw)
    leaves = [t.clone().requires_grad_() for t in (x, y, kw["gate"], kw["weight"])]
    gx, gy = rand(*x.shape, seed=7), rand(*x.shape, seed=8)

    def loss(x, y, gate, weight):
        total, norm = ops.add_norm(x, y, **{**kw, "gate": gate, "weight": weight})
        return (total * gx).sum() + (0 if norm is None else (norm * gy).sum())
    loss(*leaves).backward()

    def loss64(x, y, gate, weight):
        r, _, h, _ = plain64(x, y, **{**kw, "gate": gate, "weight": weight})
        return (r * gx.reshape(r.shape)).sum() + (0 if h is None else (h * gy.reshape(r.shape)).sum())
    doubles = [t.detach().double() for t in leaves]
    for i, t in enumerate(leaves):
        step = rand(*t.shape, seed=9 + i).double()
        up, down = ([d + s * 1e-4 * step if j == i else d for j, d in enumerate(doubles)] for s in (1, -1))
        want = (loss64(*up) - loss64(*down)).item() / 2e-4
        got = 0.0 if t.grad is None else (t.grad.double() * step).sum().item()
        # fp32 sums of a thousand terms and a second-order difference
        assert abs(got - want) <= 1e-4 * (abs(want) + 30), i


def test_the_torch_form_refuses_flags_that_only_equal_true():
    """What HipOps.add_norm hands on: 1, 1.0 and numpy's truth values are neither LayerNorm nor RMS (1 == True, but 1 is no True)."""
    import numpy as np
    from clarus_amd.spatial_torch import TorchSpatialOps
    ops, h = TorchSpatialOps(torch.float32, torch.device("cpu")), cpu_hip()
    x = rand(2, 5, 64)
    for bad in (1, 0, 1.0, 0.0, np.True_, np.False_, None, "layer", torch.tensor(True)):
        for kw in ({"ln": bad}, {"post": bad}):
            for form in (h, ops):
                with pytest.raises(Unsupported):
                    form.add_norm(x, x, **kw)
                    pytest.fail(f"{form.name} accepted {kw}")


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


SHAPES = [(1, 1, 8), (2, 5, 8), (3, 7, 24), (1, 300, 64), (2, 33, 96), (1, 4, 360), (2, 129, 512), (1, 65, 520), (2, 9, 1024), (1, 17, 1544),
          (2, 3, 4096), (1, 3, 4104), (2, 2, 10000), (1, 5, 16384), (1, 20011, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("xdt,ydt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32, torch.float32),
                                     (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n,rows,c", SHAPES)
def test_shapes(n, rows, c, xdt, ydt, hips, gpu_device):
    dev = gpu_device
    x, y = rand(n, rows, c, dt=xdt, dev=dev, scale=2.0, shift=3.0), rand(n, rows, c, dt=ydt, dev=dev, seed=1)
    for i, (post, ln) in enumerate(KINDS):
        kw = dict(post=post, ln=ln)
        if i % 2 == 0:
            kw.update(gate=rand(n, c, dev=dev, seed=2), scale=0.3, post_weight=rand(c, dev=dev, seed=3), weight=rand(n, c, dev=dev, seed=5),
                      bias=rand(c, dev=dev, seed=6))
        if i % 3 == 0:
            kw.update(post_bias=rand(n, c, dev=dev, seed=4), eps=1e-3)
        print(f"[add_norm] {n} {rows} {c} {xdt} {ydt} {sorted(kw)}", flush=True)
        got = hips[ydt].add_norm(x, y, **kw)
        assert got[0].dtype == xdt and (got[1] is None or got[1].dtype == ydt)
        check(got, x, y, what=f"{post} {ln}", **kw)
        if ln:
            total, norm = hips[ydt].add_norm(x, ln=ln, weight=kw.get("weight"), out_dtype=xdt)
            assert total is x and norm.dtype == xdt
            check((total, norm), x, ln=ln, weight=kw.get("weight"), what="first")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt, hips, gpu_device):
    hip, wide = hips[dt], rand(4, 6, 9, 3 * 40, dt=dt, dev=gpu_device)
    x = rand(4, 6, 9, 40, dt=dt, dev=gpu_device, seed=1)
    w = rand(80, 8, dev=gpu_device, seed=2)
    for what, a, b, kw in (
            ("slices", wide[..., 40:80], wide[..., 80:], {}), ("images", wide[::2, ..., :40], x[1::2], {}),
            ("rows", wide[:, 1:4, :, :40], x[:, 2:5], {}), ("one for all", x[:1].expand(4, 6, 9, 40), x, {}),
            ("vectors with strides", x, x, {"gate": w[:40, 0], "weight": w[:, 1].reshape(2, 40)[:1].expand(4, 40), "bias": w[::2, 2]}),
            ("vectors of other types", x, x, {"weight": w[40:, 3].to(torch.bfloat16), "bias": w[40:, 3].double()}),
            ("a vector inside another", x, x, {"weight": w.reshape(-1)[3:43], "post_weight": w.reshape(-1)[1:41], "post": True}),
            ("rows of [N, C]", wide[:, 2, 3, :40], x[:, 0, 0], {})):
        print(f"[add_norm] {what}", flush=True)
        check(hip.add_norm(a, b, **kw), a, b, what=what, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [8, 96, 512, 1024, 4096, 12000])
def test_values_of_any_size(c, hips, gpu_device):
    """Rows far from zero, equal, zero, as small and as large as documented (2^60)."""
    hip = hips[torch.float32]
    x = rand(1, 7, c, dev=gpu_device)
    for what, v in (("far", x + 1e4), ("equal", torch.full_like(x, 0.1)), ("zero", torch.zeros_like(x)), ("small", x * 2.0 ** -60),
                    ("large", (x / 8).clamp(-1, 1) * 2.0 ** 59)):
        for ln in (True, "rms"):
            for eps in (1e-6, 1e-5):
                check(hip.add_norm(v, ln=ln, eps=eps), v, ln=ln, eps=eps, what=f"{what} {ln}")
            check(hip.add_norm(x, v, post=ln, ln=False), x, v, post=ln, ln=False, what=f"post {what} {ln}")


@pytest.mark.gpu
def test_what_is_not_finite_stays_in_its_row(hips, gpu_device):
    hip = hips[torch.float32]
    for c in (40, 512, 4096, 8192):
        x, y = rand(2, 9, c, dev=gpu_device), rand(2, 9, c, dev=gpu_device, seed=1)
        want = hip.add_norm(x, y, post="rms")
        bad = y.clone()
        bad[0, 3, 5], bad[1, 8, c - 1] = math.nan, math.inf
        got = hip.add_norm(x, bad, post="rms")
        for g, w in zip(got, want):
            assert torch.isnan(g[0, 3]).all() and torch.isnan(g[1, 8, c - 1])
            g[0, 3], g[1, 8] = w[0, 3], w[1, 8]
            assert torch.equal(g, w)


@pytest.mark.gpu
def test_offsets_past_32_bits(hips, gpu_device):
    """Rows 2^21 elements apart, and more than 2^31 elements in all."""
    hip = hips[torch.bfloat16]
    x = rand(1, 1100, 64, dt=torch.bfloat16, dev=gpu_device)
    buf = torch.empty(1, 1100, 1 << 21, dtype=torch.bfloat16, device=gpu_device)
    buf[..., 8:72] = x
    want = hip.add_norm(x, x)
    assert all(torch.equal(a, b) for a, b in zip(hip.add_norm(buf[..., 8:72], buf[..., 8:72]), want))
    del buf
    big = x[:, None].expand(1, 31000, 1100, 64).reshape(1, -1, 64)
    total, norm = hip.add_norm(big, big)
    assert total.numel() > 1 << 31
    for i in (0, 15000, 30999):
        at = slice(i * 1100, (i + 1) * 1100)
        assert torch.equal(total[:, at], want[0]) and torch.equal(norm[:, at], want[1])


@pytest.mark.gpu
def test_c_entry_in_place(gpu_device):
    """The sum over x itself, for rows in one wave and in four."""
    import ctypes
    lib = _lib.load()
    for c in (64, 512, 4096, 6000):
        x, y = rand(2, 19, c, dev=gpu_device), rand(2, 19, c, dev=gpu_device, seed=1)
        s, h = x.clone(), torch.empty_like(x)
        args = _lib.AddNormArgs(x=s.data_ptr(), y=y.data_ptr(), sum=s.data_ptr(), norm=h.data_ptr(), n=2, rows=19, c=c, x_bstride=19 * c,
                                ldx=c, y_bstride=19 * c, ldy=c, post=1, pre=3, scale=0.5, eps=1e-6)
        _lib.check(lib.clarus_hip_add_norm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "add_norm")
        check((s, h), x, y, scale=0.5, post=True, ln="rms")


@pytest.mark.gpu
def test_streams_and_graph(hips, gpu_device):
    hip = hips[torch.bfloat16]
    w = rand(2, 512, dev=gpu_device, seed=4)
    a, b = ([rand(2, 700, 512, dt=torch.bfloat16, dev=gpu_device, seed=s + i) for i in (0, 1)] for s in (1, 5))

    def call(t):
        return hip.add_norm(*t, gate=w, post="rms", weight=w)
    ref = [call(t) for t in (a, b)]
    torch.cuda.synchronize()
    s, outs = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(4):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                outs.append(call(t))
    torch.cuda.synchronize()
    assert all(torch.equal(o[j], ref[i % 2][j]) for i, o in enumerate(outs) for j in (0, 1))
    st = [t.clone() for t in a]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(st)
    for i in range(4):
        for dst, src in zip(st, (a, b)[i % 2]):
            dst.copy_(src)
        graph.replay()
        eager = call(b)
        torch.cuda.synchronize()
        assert all(torch.equal(y[j], ref[i % 2][j]) and torch.equal(eager[j], ref[1][j]) for j in (0, 1))


@pytest.mark.gpu
def test_the_chain_falls_through_for_gradients(gpu_device):
    from clarus_amd import spatial_torch  # noqa: F401
    ops = Ops(["hip", "torch"], torch.float32, gpu_device, log=print)
    x, leaf = rand(1, 6, 7, 64, dev=gpu_device), rand(1, 6, 7, 64, dev=gpu_device, seed=1).requires_grad_()
    ops.add_norm(x, leaf)[1].sum().backward()
    assert leaf.grad is not None
    ops.add_norm(x, x)
    assert ops.report()["ops"]["add_norm"] == {"hip": 1, "torch": 1}
