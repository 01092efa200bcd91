"""rotary: the HIP kernel (clarus_hip_rotary) against the formula in 64 bits.

Tolerance, u = 2^-24: the fraction of a turn is rounded once to fp32 (2^-27 of a turn at most: 0.8 u as an angle), after
roundings of 2^-53 of the turns in the 64-bit product and frequency (as many in the reference: 2^-50 of the turns, as
an angle 6.3 times that); sincospi is within 2 ulp (2 u): cos and sin off by e = 3 u + 2^-47 |turns|. The turned pair: e (|a| + |b|)
and two roundings of u (|a| + |b|); the output once: 2^-8 (bf16) or u of itself.
"""
from __future__ import annotations

import math

import pytest
import torch

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

U = 2.0 ** -24


def plain64(x, heads, sections, positions=None, base=10000.0, pairs="adjacent"):
    """(out, tolerance before the output's rounding), float64."""
    n, d = x.shape[0], x.shape[-1] // heads
    y = x.double().reshape(n, -1, heads, d)
    l, p = y.shape[1], sum(sections)
    if positions is None:
        grid = torch.meshgrid(*[torch.arange(s, device=x.device) for s in x.shape[1:-1]], indexing="ij")
        positions = torch.stack([g.reshape(-1) for g in grid], -1)
    out, tol = y.clone(), torch.zeros_like(y)
    j = 0
    for a, s in enumerate(sections):
        for i in range(s):
            t = positions[..., a].double().reshape(-1, l, 1) * base ** (-i / s)
            ca, cb = (2 * j, 2 * j + 1) if pairs == "adjacent" else (j, p + j)
            u, v = y[..., ca], y[..., cb]
            out[..., ca], out[..., cb] = u * t.cos() - v * t.sin(), u * t.sin() + v * t.cos()
            tol[..., ca] = tol[..., cb] = (5 * U + 2.0 ** -47 * t.abs() / math.tau) * (u.abs() + v.abs())
            j += 1
    return out.reshape(x.shape), tol.reshape(x.shape)


def check(got, x, heads, sections, positions=None, base=10000.0, pairs="adjacent", what=""):
    ref, tol = plain64(x, heads, sections, positions, base, pairs)
    assert got.shape == x.shape and got.is_contiguous(), what
    assert torch.isfinite(got).all(), what
    tol = tol + (2.0 ** -8 if got.dtype == torch.bfloat16 else U) * (ref.abs() + tol)
    off = (got.double() - ref).abs()
    assert (off <= tol).all(), f"{what}: max|d| {off.max().item():.3e}, {(off - tol).max().item():.3e} past the tolerance"


def rand(*shape, dt=torch.float32, dev="cpu", seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(dev)


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
    pos = z(5, 1)
    cases = [
        ((z(2, 5, 60), 5, [3]), {}), ((x, 3, [4]), {}), ((x, 0, [4]), {}), ((x, 2.0, [4]), {}), ((z(2, 5, 264), 1, [4]), {}),
        ((x, 2, [17]), {}), ((x, 2, []), {}), ((x, 2, [0]), {}), ((x, 2, [-1]), {}), ((x, 2, [4.0]), {}), ((x, 2, [4, 4]), {}),
        ((z(2, 2, 2, 2, 2, 2, 64), 2, [1] * 5), {}), ((z(64), 2, [4]), {}), ((x.half(), 2, [4]), {}),
        ((x, 2, [4]), {"out_dtype": torch.float16}), ((x, 2, [4]), {"pairs": "other"}), ((x, 2, [4]), {"base": 0.0}),
        ((x, 2, [4]), {"base": math.nan}), ((x, 2, [4]), {"base": math.inf}), ((x, 2, [4]), {"base": None}),
        ((x, 2, [4]), {"positions": z(4, 1)}), ((x, 2, [4]), {"positions": z(5)}), ((x, 2, [4]), {"positions": z(1, 5, 1)}),
        ((x, 2, [4]), {"positions": pos.double()}), ((x, 2, [4, 2]), {"positions": z(2, 5).t()}),
        ((x, 2, [4]), {"positions": z(5, 2)}),
        ((z(2, 64, 5).transpose(1, 2), 2, [4]), {}), ((z(2, 5, 66)[..., :64], 2, [4]), {}), ((z(2, 5, 65)[..., 1:], 2, [4]), {}),
        ((x.clone().requires_grad_(), 2, [4]), {}), ((x, 2, [4]), {"positions": pos.clone().requires_grad_()}),
        ((z(1, 1, 8).expand(1, 1 << 28, 8), 1, [4]), {}),
    ]
    for i, (args, kw) in enumerate(cases):
        with pytest.raises(Unsupported):
            h.rotary(*args, **kw)
            pytest.fail(f"case {i} was accepted")
    assert h.rotary(z(2, 0, 64), 2, [4]).shape == (2, 0, 64)


def test_c_entry_refuses_before_launch():
    import ctypes
    lib = _lib.load()
    assert lib.clarus_hip_rotary(None, None) == _lib.EINVAL

    def call(sections=(4,), grid=(6,), turn=0.1, **kw):
        base = dict(x=1 << 20, out=1 << 21, n=2, l=6, heads=2, d=32, x_bstride=384, ldx=64, axes=1)
        a = _lib.RotaryArgs(**{**base, **kw})
        for i, s in enumerate(sections):
            a.sections[i] = s
        for i, s in enumerate(grid):
            a.grid[i] = s
        for i in range(128):
            a.turn[i] = turn
        return lib.clarus_hip_rotary(ctypes.byref(a), None)
    for kw in (dict(x=None), dict(out=None), dict(n=0), dict(l=0), dict(heads=0), dict(d=0), dict(d=12), dict(d=264), dict(axes=0),
               dict(axes=5), dict(dtype=2), dict(o_dtype=3), dict(pairs_mode=2), dict(pos_kind=4), dict(pos_kind=1), dict(x=(1 << 20) + 8),
               dict(ldx=66), dict(ldx=-64), dict(x_bstride=2), dict(grid=(5,)), dict(grid=(7,)), dict(grid=(0,)), dict(sections=(17,)),
               dict(sections=(0,)), dict(sections=(-1,)), dict(sections=(1 << 62,)), dict(turn=math.nan), dict(turn=math.inf),
               dict(n=1 << 62, l=4, grid=(4,)), dict(n=1, l=1 << 28, grid=(1 << 28,)), dict(heads=1 << 60), dict(pos_bstride=-1),
               dict(axes=2, grid=(6, 0), sections=(2, 2)), dict(axes=3, grid=(1 << 62, 4, 6), sections=(2, 2, 2))):
        assert call(**kw) == _lib.EINVAL, kw
        assert b"rotary" in lib.clarus_hip_last_error()


CASES = [((1, 16, 24), 8, 32, (8, 8), "adjacent"), ((2, 1), 1, 8, (4,), "adjacent"), ((2, 3, 5, 7), 3, 72, (8, 14, 14), "adjacent"),
         ((1, 33), 5, 64, (20,), "halves"), ((2, 17, 3), 2, 48, (5, 7), "halves"), ((1, 300), 40, 64, (16,), "halves"),
         ((3, 4, 4, 4), 1, 16, (1, 0, 2), "adjacent"), ((1, 130), 2, 256, (128,), "halves"), ((1, 2, 3, 4, 5), 2, 40, (1, 2, 3, 4), "halves"),
         ((2, 61), 12, 128, (3,), "adjacent"), ((1, 9), 1, 8, (1,), "halves")]


@pytest.mark.parametrize("shape,heads,d,sections,pairs", CASES)
def test_plain_forms(shape, heads, d, sections, pairs):
    """The oracle's form and the torch backend's, and the latter's gradient: a rotation's, which turns back."""
    from clarus_amd.spatial_torch import TorchSpatialOps
    from oracle.torch_ref import TorchRef
    x = rand(*shape, heads * d)
    check(TorchRef(torch.float32, "cpu").rotary(x, heads, sections, pairs=pairs), x, heads, sections, pairs=pairs)
    ops = TorchSpatialOps(torch.float32, torch.device("cpu"))
    pos = torch.randint(-50, 5000, (shape[0], math.prod(shape[1:]), len(sections)), generator=torch.Generator().manual_seed(1))
    leaf = x.clone().requires_grad_()
    y = ops.rotary(leaf, heads, sections, pos, pairs=pairs)
    check(y.detach(), x, heads, sections, pos, pairs=pairs)
    g = rand(*x.shape, seed=2)
    y.backward(g)
    check(leaf.grad, g, heads, sections, -pos, pairs=pairs)


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,heads,d,sections,pairs", CASES)
def test_shapes(shape, heads, d, sections, pairs, dt, hips, gpu_device):
    x = rand(*shape, heads * d, dt=dt, dev=gpu_device)
    print(f"[rotary] {shape} {heads} {d} {sections} {pairs} {dt}", flush=True)
    for odt in (torch.bfloat16, torch.float32):
        got = hips[dt].rotary(x, heads, sections, pairs=pairs, out_dtype=odt)
        print(f"[rotary] {_lib.last_kernel()}", flush=True)
        assert got.dtype == odt
        check(got, x, heads, sections, pairs=pairs, what=str(odt))
    # the other order of the pairs, positions as a tensor, another base
    other = "halves" if pairs == "adjacent" else "adjacent"
    l = math.prod(shape[1:])
    for kind in (torch.int32, torch.int64, torch.float32):
        pos = torch.randint(-3000, 1 << 20, (shape[0], l, len(sections)), generator=torch.Generator().manual_seed(3)).to(kind).to(gpu_device)
        if kind == torch.float32:
            pos = pos / 8 + 0.1
        for p in (pos, pos[0]):
            check(hips[dt].rotary(x, heads, sections, p, base=500.0, pairs=other), x, heads, sections, p, 500.0, other, str(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt, hips, gpu_device):
    """Slices of wider rows, rows of images, an image shared by stride 0, positions with strides, one token of [N, C]."""
    hip, wide = hips[dt], rand(4, 6, 9, 3 * 96, dt=dt, dev=gpu_device)
    at = torch.arange(3 * 60 * 4, device=gpu_device, dtype=torch.int32).reshape(3, 60, 4)
    for what, x, sections, pos in (
            ("slice", wide[..., 96:192], (4, 4), None), ("every other image", wide[::2, ..., 192:], (8, 8), None),
            ("rows", wide[:, 1:4, :, :96], (4, 12), None), ("a column", wide[:, :, 3:4, :96], (3, 1), None),
            ("one for all", wide[:1, ..., :96].expand(3, 6, 9, 96), (8, 4), None),
            ("positions' slice", wide[:3, ..., :96], (8, 4), at[:, 2:56, 1:3]), ("shared positions", wide[..., :96], (8,), at[1, 3:57, 2:3]),
            ("expanded positions", wide[..., :96], (8, 2), at[:1, :1, 2:].expand(4, 54, 2)),
            ("one token", wide[:, 2, 3, :96], (8,), at[2, :1, :1])):
        print(f"[rotary] {what}", flush=True)
        check(hip.rotary(x, 3, sections, pos), x, 3, sections, pos, what=what)


@pytest.mark.gpu
def test_far_positions(hips, gpu_device):
    """Positions whose angles fp32 does not hold: up to 2^40 radians of the fastest pair, in 64 bits right to a 2^-47 of the turns."""
    x = rand(1, 64, 4 * 32, dev=gpu_device)
    pos = (torch.arange(64, device=gpu_device, dtype=torch.int64) * ((1 << 34) + 12345) - (1 << 39))[:, None]
    check(hips[torch.float32].rotary(x, 4, (16,), pos), x, 4, (16,), pos)


@pytest.mark.gpu
def test_what_is_not_finite_stays_where_it_is(hips, gpu_device):
    x = rand(1, 5, 2 * 32, dev=gpu_device)
    want = hips[torch.float32].rotary(x, 2, (8,))
    bad = x.clone()
    bad[0, 2, 3], bad[0, 3, 20] = math.nan, math.inf
    got = hips[torch.float32].rotary(bad, 2, (8,))
    assert torch.isnan(got[0, 2, 2:4]).all() and got[0, 3, 20] == math.inf
    got[0, 2, 2:4], got[0, 3, 20] = want[0, 2, 2:4], want[0, 3, 20]
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_offsets_past_32_bits(hips, gpu_device):
    """Rows 2^21 elements apart (the last ones past 2^31), and an output of more than 2^31 elements."""
    buf = torch.empty(1, 1100, 1 << 21, dtype=torch.bfloat16, device=gpu_device)
    x = rand(1, 1100, 64, dt=torch.bfloat16, dev=gpu_device)
    buf[..., 64:128] = x
    assert torch.equal(hips[torch.bfloat16].rotary(buf[..., 64:128], 2, (16,)), hips[torch.bfloat16].rotary(x, 2, (16,)))
    del buf
    pos = torch.arange(1100, device=gpu_device)[None, :, None].repeat(1, 1, 1)
    big = x.repeat(1, 1, 64)[:, None].expand(1, 480, 1100, 4096).reshape(1, -1, 4096)
    got = hips[torch.bfloat16].rotary(big, 128, (16,), pos.repeat(1, 480, 1))
    want = hips[torch.bfloat16].rotary(x, 2, (16,)).repeat(1, 1, 64)
    assert got.numel() > 1 << 31 and all(torch.equal(got[:, i * 1100:(i + 1) * 1100], want) for i in (0, 200, 479))


@pytest.mark.gpu
def test_streams_and_graph(hips, gpu_device):
    hip = hips[torch.bfloat16]
    a, b = (rand(2, 40, 50, 256, dt=torch.bfloat16, dev=gpu_device, seed=s) for s in (1, 2))
    ref = [hip.rotary(t, 4, (8, 24)) for t in (a, b)]
    torch.cuda.synchronize()
    s, outs = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(4):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                outs.append(hip.rotary(t, 4, (8, 24)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i % 2]) for i, o in enumerate(outs))
    st = a.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hip.rotary(st, 4, (8, 24))
    for i in range(4):
        st.copy_((a, b)[i % 2])
        graph.replay()
        eager = hip.rotary(b, 4, (8, 24))
        torch.cuda.synchronize()
        assert torch.equal(y, ref[i % 2]) and torch.equal(eager, ref[1])


@pytest.mark.gpu
def test_c_entry_in_place(gpu_device):
    import ctypes
    lib = _lib.load()
    for pairs in ("adjacent", "halves"):
        x = rand(2, 37, 3 * 32, dev=gpu_device)
        y = x.clone()
        turn = [10000.0 ** (-i / 12) / math.tau for i in range(12)]
        args = _lib.RotaryArgs(x=y.data_ptr(), out=y.data_ptr(), n=2, l=37, heads=3, d=32, x_bstride=37 * 96, ldx=96, axes=1,
                               pairs_mode=int(pairs == "halves"), grid=(ctypes.c_int64 * 4)(37), sections=(ctypes.c_int64 * 4)(12),
                               turn=(ctypes.c_double * 128)(*turn))
        _lib.check(lib.clarus_hip_rotary(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "rotary")
        check(y, x, 3, (12,), pairs=pairs)


@pytest.mark.gpu
def test_the_chain_falls_through_for_gradients(gpu_device):
    from clarus_amd import spatial_torch  # noqa: F401
    ops = Ops(["hip", "torch"], torch.float32, gpu_device, log=print)
    x = rand(1, 6, 7, 64, dev=gpu_device)
    leaf = x.clone().requires_grad_()
    ops.rotary(leaf, 2, (8, 4)).sum().backward()
    assert leaf.grad is not None
    ops.rotary(x, 2, (8, 4))
    assert ops.report()["ops"]["rotary"] == {"hip": 1, "torch": 1}
