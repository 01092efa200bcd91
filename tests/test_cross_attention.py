"""cross_attention: the HIP kernels (clarus_hip_cross_attention) against the formula in 64 bits.

Tolerances, per output, with p the exact weights and u = 2^-24:
  scores     d + 8 roundings, each at most u of scale |q| . |k|: a weight moves by (d + 8) u A relative, A the
             row's largest scale |q| . |k|, in the numerator and in the sum: 2 (d + 8) u A (p @ |v|)
  sums       at most lk + 16 additions, u of (p @ |v|) each, in the numerator and in the sum
  bf16       each weight rounded once, 2^-8 of itself: 2^-8 (p @ |v|); the output once: 2^-8 |o|
"""
from __future__ import annotations

import math

import pytest
import torch

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

U = 2.0 ** -24


def plain64(q, k, v, heads, kv_heads=None, mask=None, scale=None):
    """(o, p @ |v|, A), float64, each of q's shape (A per row and head)."""
    kv_heads = kv_heads or heads
    n, d, rep = q.shape[0], q.shape[-1] // heads, heads // kv_heads
    lq, lk = math.prod(q.shape[1:-1]), math.prod(k.shape[1:-1])
    qh = q.double().reshape(n, lq, heads, d).permute(0, 2, 1, 3).contiguous()
    kh, vh = (t.double().reshape(n, lk, kv_heads, d).permute(0, 2, 1, 3).repeat_interleave(rep, 1) for t in (k, v))
    keep = torch.ones(n, 1, lq, lk, dtype=torch.bool, device=q.device)
    if mask is not None:
        keep = (mask[:, None, None] if mask.dim() == 2 else mask[:, None]).expand(n, 1, lq, lk)
        if mask.dim() == 2:
            kh, vh = (t.masked_fill(~mask[:, None, :, None], 0) for t in (kh, vh))
    sc = d ** -0.5 if scale is None else scale
    kt = kh.transpose(-1, -2).contiguous()
    s = (qh @ kt) * sc
    big = ((qh.abs() @ kt.abs()) * sc * keep).amax(-1, keepdim=True)
    s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    def back(t):
        return t.permute(0, 2, 1, 3).reshape(q.shape)
    return back(p @ vh), back(p @ vh.abs()), back(big.expand(n, heads, lq, d))


def check(got, q, k, v, heads, kv_heads=None, mask=None, scale=None, what=""):
    ref, pv, big = plain64(q, k, v, heads, kv_heads, mask, scale)
    assert got.shape == q.shape and got.is_contiguous(), what
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    d, lk = q.shape[-1] // heads, math.prod(k.shape[1:-1])
    tol = (2 * (d + 8) * U * big + 2 * (lk + 16) * U + (2.0 ** -8 if q.dtype == torch.bfloat16 else 0)) * pv
    tol = tol + (2.0 ** -8 if got.dtype == torch.bfloat16 else U) * ref.abs()
    off = (got.double() - ref).abs()
    worst = (off - tol).max().item()
    assert worst <= 0, f"{what}: max|d| {off.max().item():.3e}, {worst:.3e} past the tolerance"


def inputs(n, lq, lk, heads, kv_heads, d, dt, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(n, lq, heads * d, generator=g) * 1.5).to(dt)
    k, v = (torch.randn(n, lk, kv_heads * d, generator=g).to(dt) for _ in range(2))
    return q.to(dev), k.to(dev), v.to(dev)


def make_mask(kind, n, lq, lk, dev, seed=0):
    """none / keys (ragged prompts, scattered holes, the last image without any) / pairs (random, some rows
    empty, some with one key)."""
    g = torch.Generator().manual_seed(seed + 1)
    if kind == "none":
        return None
    if kind == "keys":
        m = torch.rand(n, lk, generator=g) < 0.7
        for i in range(n):
            m[i, lk - lk * i // n:] = False
        if n > 1:
            m[-1] = False
        return m.to(dev)
    m = torch.rand(n, lq, lk, generator=g) < 0.5
    m[:, ::3] = False
    m[:, ::6, lk // 2] = True
    return m.to(dev)


# ------------------------------------------------------------------ CPU
def cpu_hip(dtype=torch.float32):
    from clarus_amd.hip_ops import HipOps
    h = HipOps.__new__(HipOps)
    h.dtype, h.device, h.dev, h._cache, h._plans = dtype, torch.device("cpu"), torch.device("cpu"), {}, {}
    h.lib = _lib.load()
    return h


def test_refusals():
    h = cpu_hip()
    z = torch.zeros
    q, k = z(2, 5, 64), z(2, 7, 64)
    cases = [
        ((z(2, 5, 60), z(2, 7, 60), z(2, 7, 60), 5), {}),               # head width 12
        ((z(2, 5, 136), z(2, 7, 136), z(2, 7, 136), 1), {}),            # 136
        ((q, k, k, 3), {}), ((q, k, k, 0), {}), ((q, k, k, 2.0), {}),
        ((q, k, k, 4), {"kv_heads": 3}), ((q, k, k, 4), {"kv_heads": 2}),
        ((q, k, z(2, 8, 64), 4), {}), ((q, z(1, 7, 64), z(1, 7, 64), 4), {}), ((q, z(2, 7, 32), z(2, 7, 32), 4), {}),
        ((q, k, k, 4), {"scale": 0.0}), ((q, k, k, 4), {"scale": -1.0}), ((q, k, k, 4), {"scale": math.inf}),
        ((q, k, k, 4), {"scale": math.nan}), ((q, k, k, 4), {"out_dtype": torch.float16}),
        ((q.half(), k.half(), k.half(), 4), {}), ((q, k.bfloat16(), k.bfloat16(), 4), {}),
        ((q, k, k, 4), {"mask": z(2, 7)}), ((q, k, k, 4), {"mask": z(5, 7, dtype=torch.bool)}),
        ((q, k, k, 4), {"mask": z(2, 1, 7, dtype=torch.bool)}),
        ((q, k, k, 4), {"mask": z(7, 2, dtype=torch.bool).t()}),
        ((z(2, 64, 5).transpose(1, 2), k, k, 4), {}),
        ((q, z(2, 3, 4, 64).transpose(1, 2), z(2, 4, 3, 64), 4), {}),
        ((z(2, 5, 66)[..., 1:65], k, k, 4), {}), ((q, z(2, 7, 66)[..., :64], k, 4), {}),
        ((z(64), k, k, 4), {}),
        ((q.clone().requires_grad_(), k, k, 4), {}), ((q, k, k.clone().requires_grad_(), 4), {}),
    ]
    for i, (args, kw) in enumerate(cases):
        with pytest.raises(Unsupported):
            h.cross_attention(*args, **kw)
            pytest.fail(f"case {i} was accepted")


def test_refused_sizes():
    h = cpu_hip()
    q, k = torch.zeros(1, 1, 64).expand(1, 1 << 20, 64), torch.zeros(1, 1, 64).expand(1, 1 << 18, 64)
    cases = [((q, k, k, 2), {"mask": torch.ones(1, 1, 1, dtype=torch.bool).expand(1, 1 << 20, 1 << 18)}),
             ((q[:, :4], k[:, :4], k[:, :4], 2), {"scale": 2.1e38}),
             ((torch.zeros(1, 1, 64).expand(1 << 16, 1, 64), *[torch.zeros(1, 1, 64).expand(1 << 16, 1, 64)] * 2, 1), {})]
    for args, kw in cases:
        with pytest.raises(Unsupported):
            h.cross_attention(*args, **kw)


def test_refused_launches():
    """A launch of 2^32 threads (two for a row) is declined, just below it is not."""
    import ctypes
    h, z = cpu_hip(torch.bfloat16), torch.zeros(1, 1, 8, dtype=torch.bfloat16)
    for heads, lq in ((16, 1 << 27), (1, (1 << 31) - 4097), (2, 1 << 30), (128, (1 << 24) - 40)):
        with pytest.raises(Unsupported):
            h.cross_attention(z.expand(1, 1, 8).repeat(1, 1, heads).expand(1, lq, 8 * heads), *[z.repeat(1, 1, heads)] * 2, heads)
    for heads, lq in ((16, (1 << 27) - 512), (1, (1 << 31) - 4352), (2, (1 << 30) - 2304)):
        q, kv = torch.zeros(1, 1, 8 * heads, dtype=torch.bfloat16).expand(1, lq, 8 * heads), torch.zeros(1, 1, 8 * heads, dtype=torch.bfloat16)
        h._cross_plan(q, kv, kv, heads, heads, None, None, torch.bfloat16)
    lib = _lib.load()
    for kw in (dict(lq=1 << 28, heads=16, kv_heads=16), dict(lq=1 << 23, n=256, heads=8, kv_heads=1), dict(lq=1, heads=1 << 31, kv_heads=2)):
        base = dict(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, n=1, lk=200, d=8, ldq=128, ldk=128, ldv=128, dtype=1, o_dtype=1,
                    mask_mode=0, scale=0.2)
        args = _lib.CrossArgs(**{**base, **kw})
        assert lib.clarus_hip_cross_attention(ctypes.byref(args), 1 << 30, 1 << 40, None) == _lib.EINVAL, kw
        assert b"too large" in lib.clarus_hip_last_error()


def test_a_refusal_does_not_depend_on_earlier_calls():
    h = cpu_hip()
    q, k = torch.zeros(2, 5, 64), torch.zeros(2, 0, 64)
    for ok, bad in (((4,), (4.0,)), ((4, 2), (4, 2.0)), ((4, 2), (4.0, 2))):
        kv = k[..., :32] if len(ok) == 2 else k
        assert h.cross_attention(q, kv, kv, *ok).shape == q.shape
        with pytest.raises(Unsupported):
            h.cross_attention(q, kv, kv, *bad)


def test_tangents_are_declined():
    """A forward-mode tangent would be lost, with gradients enabled or not; outside its level there is none."""
    from torch.autograd import forward_ad
    h, q, k = cpu_hip(), torch.zeros(2, 5, 64), torch.zeros(2, 0, 64)
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(Unsupported, match="tangent"):
            h.cross_attention(dual, k, k, 4)
        with pytest.raises(Unsupported, match="tangent"):
            h.cross_attention(q, k, forward_ad.make_dual(k, k + 1), 4)
        assert h.cross_attention(q, k, k, 4).shape == q.shape
    assert h.cross_attention(dual, k, k, 4).shape == q.shape


def test_scales_that_fp32_does_not_hold_are_declined():
    h, q, k = cpu_hip(), torch.zeros(1, 5, 64), torch.zeros(1, 7, 64)
    for scale in (1e-46, 7e-46, 1e39, math.nextafter(2e38, 0.0)):  # 0, 0, inf, above 2e38 as fp32
        with pytest.raises(Unsupported):
            h.cross_attention(q, k, k, 4, scale=scale)


def test_workspaces_are_sized_with_the_backends_device_current(monkeypatch):
    """The splits and chunks go by the current device's compute units: the query runs where the launch will."""
    h, on, asked = cpu_hip(), [0], []
    h.dev = torch.device("cuda", 1)

    class Current:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            on.append(self.dev.index)

        def __exit__(self, *exc):
            on.pop()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: on[-1])
    monkeypatch.setattr(torch.cuda, "device", Current)

    class Lib:
        def clarus_hip_cross_attention_workspace(self, *args):
            asked.append(on[-1])
            return 0
        clarus_hip_group_norm_workspace = clarus_hip_cross_attention_workspace
    h.lib, x = Lib(), torch.zeros(1, 5, 64)
    h._cross_plan(x, x, x, 4, 4, None, None, torch.float32)
    h._group_norm_plan(x, 8, None, None, None, torch.float32)
    assert asked == [1, 1] and on == [0]


def test_sizes_whose_products_overflow_are_refused():
    """Products of the C entry's sizes that wrap around 64 bits do not pass for small ones."""
    import ctypes
    lib = _lib.load()
    base = dict(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, n=1, lq=4, lk=64, heads=4, kv_heads=1, d=8, ldq=32, ldk=32, ldv=32,
                dtype=1, o_dtype=1, mask_mode=0, scale=0.2)
    for kw in (dict(heads=1 << 62), dict(n=1 << 62, kv_heads=4), dict(n=1 << 60, kv_heads=16, heads=16), dict(kv_heads=1 << 62, heads=1 << 62),
               dict(n=1 << 61, lq=8, mask_mode=2, mask=16), dict(heads=1 << 33, kv_heads=4, lq=1 << 31)):
        assert lib.clarus_hip_cross_attention(ctypes.byref(_lib.CrossArgs(**{**base, **kw})), 1 << 30, 1 << 40, None) == _lib.EINVAL, kw
        assert b"too large" in lib.clarus_hip_last_error(), kw
    assert lib.clarus_hip_cross_attention_workspace(1, 1 << 62, 1, 100000, 4, 4, 8, 0) == 0
    assert lib.clarus_hip_cross_attention_workspace(1, 1, 4, 100000, 1 << 62, 1, 8, 0) == 0
    assert lib.clarus_hip_group_norm_workspace(1 << 62, 100000, 64, 8) == 0
    assert lib.clarus_hip_group_norm_workspace(1, 1 << 62, 64, 8) == 0


def test_nothing_to_attend_or_to_ask_cpu():
    h = cpu_hip()
    assert h.cross_attention(torch.zeros(2, 0, 64), torch.zeros(2, 3, 64), torch.zeros(2, 3, 64), 4).shape == (2, 0, 64)
    assert not h.cross_attention(torch.ones(2, 3, 64), torch.zeros(2, 0, 64), torch.zeros(2, 0, 64), 4).any()


def test_c_entry_refuses_before_launch():
    import ctypes
    lib = _lib.load()

    def call(scratch=1 << 30, size=1 << 30, **kw):
        base = dict(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, n=1, lq=64, lk=64, heads=4, kv_heads=2, d=32, ldq=128,
                    ldk=64, ldv=64, dtype=0, o_dtype=0, mask_mode=0, scale=0.2)
        return lib.clarus_hip_cross_attention(ctypes.byref(_lib.CrossArgs(**{**base, **kw})), scratch, size, None)
    assert lib.clarus_hip_cross_attention(None, None, 0, None) == _lib.EINVAL
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(n=0), dict(lq=0), dict(lk=0), dict(heads=0),
               dict(kv_heads=0), dict(kv_heads=3), dict(d=0), dict(d=12), dict(d=136), dict(dtype=2), dict(o_dtype=-1),
               dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(ldq=130), dict(q=(1 << 20) + 8), dict(ldk=-64),
               dict(k_bstride=2), dict(mask_mode=1), dict(mask_mode=3, mask=16), dict(lk=1 << 31), dict(lq=1 << 31),
               dict(n=1 << 15), dict(lq=1, lk=100000, size=16), dict(lq=1, lk=100000, scratch=None)):
        assert call(**kw) == _lib.EINVAL, kw
        assert b"cross_attention" in lib.clarus_hip_last_error()
    assert lib.clarus_hip_cross_attention_workspace(0, 1, 1, 100000, 4, 2, 32, 0) > 0
    assert lib.clarus_hip_cross_attention_workspace(0, 1, 1, 100000, 4, 3, 32, 0) == 0


@pytest.mark.parametrize("kind", ["none", "keys", "pairs"])
def test_oracle(kind):
    from oracle.torch_ref import TorchRef
    q, k, v = inputs(3, 9, 11, 4, 2, 16, torch.float32, "cpu")
    mask = make_mask(kind, 3, 9, 11, "cpu")
    check(TorchRef(torch.float32, "cpu").cross_attention(q, k, v, 4, 2, mask), q, k, v, 4, 2, mask)


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 77, 4, 4, 32), (1, 48, 77, 4, 4, 32), (2, 130, 65, 2, 2, 40), (1, 33, 64, 3, 1, 64),
          (2, 257, 129, 8, 2, 80), (1, 128, 63, 2, 2, 96), (1, 200, 300, 2, 2, 128), (3, 5, 1000, 4, 1, 64),
          (1, 1, 5000, 8, 2, 128), (2, 16, 3001, 2, 2, 48), (1, 300, 2, 1, 1, 16), (1, 31, 32, 6, 2, 24), (2, 97, 640, 1, 1, 112),
          (1, 2000, 257, 2, 2, 64), (4, 3, 31, 32, 1, 128), (1, 129, 1025, 5, 5, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["none", "keys", "pairs"])
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d", SHAPES)
def test_shapes(n, lq, lk, heads, kv_heads, d, kind, dt, hips, gpu_device):
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, dt, gpu_device, seed=lq + lk)
    mask = make_mask(kind, n, lq, lk, gpu_device)
    print(f"[xa] {n} {lq} {lk} {heads} {kv_heads} {d} {kind} {dt}", flush=True)
    got = hips[dt].cross_attention(q, k, v, heads, kv_heads, mask)
    print(f"[xa] {_lib.last_kernel()}", flush=True)
    assert got.dtype == dt
    check(got, q, k, v, heads, kv_heads, mask, what=f"{(n, lq, lk, heads, kv_heads, d)} {kind}")
    if kind == "keys" and n > 1:
        assert not got[-1].any()
    if kind == "pairs":
        assert not got[:, 3::6].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq,lk", [(70, 150), (1, 2000)])
def test_masked_keys_may_hold_anything(lq, lk, dt, hips, gpu_device):
    n, heads, d = 3, 2, 48
    q, k, v = inputs(n, lq, lk, heads, heads, d, dt, gpu_device)
    mask = make_mask("keys", n, lq, lk, gpu_device)
    want = hips[dt].cross_attention(q, k, v, heads, mask=mask)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dt).min):
        kb, vb = (t.masked_fill(~mask[..., None], bad) for t in (k, v))
        assert torch.equal(hips[dt].cross_attention(q, kb, vb, heads, mask=mask), want), bad
    # masked pairs: K may hold anything that no kept pair reads
    pairs = mask[:, None].expand(n, lq, lk)
    kb = k.masked_fill(~mask[..., None], float("nan"))
    assert torch.equal(hips[dt].cross_attention(q, kb, v, heads, mask=pairs), hips[dt].cross_attention(q, k, v, heads, mask=pairs))
    # a NaN that counts stays in its image and head
    kb = k.clone()
    kb[0, mask[0].nonzero()[0, 0], 3] = float("nan")
    got = hips[dt].cross_attention(q, kb, v, heads, mask=mask)
    assert torch.isnan(got[0, :, :d]).all() and torch.equal(got[0, :, d:], want[0, :, d:]) and torch.equal(got[1:], want[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt, hips, gpu_device):
    """NHWC queries and keys, slices of wider rows, images or keys shared by stride 0, masks with strides."""
    g = torch.Generator().manual_seed(2)
    hip, heads, d = hips[dt], 2, 32
    c = heads * d
    wide = torch.randn(4, 6, 9, 3 * c, generator=g).to(dt).to(gpu_device)
    kv = torch.randn(2, 5, 7, 2 * c + 8, generator=g).to(dt).to(gpu_device)
    k, v = kv[..., :c], kv[..., c:2 * c]
    ctx = torch.randn(1, 35, 2 * c, generator=g).to(dt).to(gpu_device).expand(2, 35, 2 * c)
    big = torch.rand(4, 60, 80, generator=g).to(gpu_device) < 0.6
    for what, args, mask in (
            ("NHWC slices", (wide[::2, ..., c:2 * c], k, v), None),
            ("rows of images", (wide[:2, 1:4, :, :c], k, v), None),
            ("one column", (wide[2:, :, 3:4, 2 * c:], k, v), big[::2, 0, :35]),
            ("shared states", (wide[:2, ..., :c], ctx[..., :c], ctx[..., c:]), big[:1, 3, 5:40].expand(2, 35)),
            ("pair mask slice", (wide[:2, ..., :c], k, v), big[1:3, 3:57, 3:38]),
            ("pair mask of one row", (wide[:2, ..., :c], k, v), big[1:3, :1, 7:42].expand(2, 54, 35))):
        print(f"[xa] {what}", flush=True)
        check(hip.cross_attention(*args, heads, mask=mask, scale=0.3), *args, heads, mask=mask, scale=0.3, what=what)
    q = wide[:2, ..., :c].contiguous()
    for odt in (torch.bfloat16, torch.float32):
        got = hip.cross_attention(q, k, v, heads, out_dtype=odt)
        assert got.dtype == odt
        check(got, q, k, v, heads, what=str(odt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_extreme_scores(dt, hips, gpu_device):
    """Equal scores average; a score far above the others takes all; far below, none; either end of the keys."""
    lk, heads, d = 200, 2, 64
    q, k, v = inputs(1, 40, lk, heads, heads, d, dt, gpu_device)
    same = k[:, :1].expand(1, lk, heads * d)
    check(hips[dt].cross_attention(q, same, v, heads), q, same, v, heads, what="equal")
    for at in (0, 77, lk - 1):
        for big in (1e3, -1e3):
            kk = torch.zeros_like(k)
            qq = torch.ones_like(q)
            kk[:, at] = big
            want = v[:, at:at + 1] if big > 0 else (v.double().sum(1, keepdim=True) - v[:, at:at + 1].double()) / (lk - 1)
            got = hips[dt].cross_attention(qq, kk, v, heads).double()
            tol = (2.0 ** -7 if dt == torch.bfloat16 else 4 * lk * U) * v.double().abs().max()
            assert (got - want.double()).abs().max() <= tol, (at, big)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq,lk", [(70, 100), (3, 3001), (6200, 700)])
def test_scores_of_any_size(lq, lk, dt, hips, gpu_device):
    """Scores up to 2^60 (exact products, equal ones among them, everything else far below): the largest alone count, in
    equal parts. Their weights are 1 and their sum exact up to the mean's rounding: 2^-8 of the largest value in bf16; in
    fp32 sums of up to 31 values and two roundings, under 64 * 2^-24 of it. Rows of ordinary scores among them too."""
    heads, d = 8, 32
    q0, _, v = inputs(1, lq, lk, heads, heads, d, dt, gpu_device)
    for size in (2.0 ** 14, 2.0 ** 17, 2.0 ** 30):
        for sign in (1, -1):
            q = torch.zeros(1, lq, heads, d, device=gpu_device)
            q[..., 3] = sign * size * (1 + torch.arange(lq, device=gpu_device) % 7 / 8.)[None, :, None]
            k = torch.zeros(1, lk, heads, d, device=gpu_device)
            level = 1 + (torch.arange(lk, device=gpu_device) * 37 % 100) / 128.
            k[..., 3] = size * level[None, :, None]
            best = level == (level.max() if sign > 0 else level.min())
            want = v[:, best].double().mean(1, keepdim=True)
            q, k = q.flatten(2).to(dt), k.flatten(2).to(dt)
            tol = (2.0 ** -8 if dt == torch.bfloat16 else 64 * U) * v.double().abs().max()
            for mask in (None, torch.ones(1, lk, dtype=torch.bool, device=gpu_device), best[None, None].expand(1, lq, lk)):
                got = hips[dt].cross_attention(q, k, v, heads, mask=mask)
                assert (got.double() - want).abs().max() <= tol, (size, sign, mask is None or mask.dim())
            # the other rows of a wave keep their accuracy
            qm = torch.where((torch.arange(lq, device=gpu_device) % 3 == 0)[None, :, None], q, q0 / size)
            got = hips[dt].cross_attention(qm, k, v, heads)[:, 1::3].contiguous()
            check(got, qm[:, 1::3], k, v, heads, what="beside far rows")


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 300])
def test_offsets_past_32_bits(lq, hips, gpu_device):
    """Keys and values in rows 2^19 elements apart: the last ones lie past 2^31 elements."""
    lk, heads, d = 4200, 2, 32
    buf = torch.empty(1, lk, 1 << 19, dtype=torch.bfloat16, device=gpu_device)
    q, k, v = inputs(1, lq, lk, heads, heads, d, torch.bfloat16, gpu_device)
    buf[..., :64], buf[..., 128:192] = k, v
    got = hips[torch.bfloat16].cross_attention(q, buf[..., :64], buf[..., 128:192], heads)
    assert torch.equal(got, hips[torch.bfloat16].cross_attention(q, k, v, heads))
    check(got, q, k, v, heads)


@pytest.mark.gpu
def test_a_mask_of_billions_of_pairs(hips, gpu_device):
    """4.4e9 bytes of mask: more words than one launch of the bits kernel makes."""
    lq, lk, d = (1 << 20) + 1000, 4200, 8
    q, k, v = inputs(1, 1000, lk, 1, 1, d, torch.bfloat16, gpu_device)
    row, key = torch.arange(1024, device=gpu_device)[:, None], torch.arange(lk, device=gpu_device)
    at = torch.arange(lq, device=gpu_device)
    mask = ((row * 7 + key) % 1024 < 40)[at % 1024][None]
    got = hips[torch.bfloat16].cross_attention(q[:, at % 1000], k, v, 1, mask=mask)
    for at in (0, lq // 2 // 1000 * 1000, lq // 1000 * 1000 - 1000):
        check(got[:, at:at + 1000].contiguous(), q, k, v, 1, mask=mask[:, at:at + 1000], what=str(at))


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [(200, 300), (2, 3001)])
def test_repeatable_streams_and_graph(lq, lk, hips, gpu_device):
    hip = hips[torch.bfloat16]
    a = inputs(2, lq, lk, 4, 2, 64, torch.bfloat16, gpu_device)
    b = inputs(2, lq, lk, 4, 2, 64, torch.bfloat16, gpu_device, seed=5)
    mask = make_mask("keys", 2, lq, lk, gpu_device)
    ref = [hip.cross_attention(*t, 4, 2, mask) for t in (a, b)]
    for _ in range(3):
        assert torch.equal(hip.cross_attention(*a, 4, 2, mask), ref[0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                outs.append(hip.cross_attention(*t, 4, 2, mask))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i % 2]) for i, o in enumerate(outs))
    # two graphs, each with its own inputs, replayed in turn with eager calls between
    made = []
    for t in (a, b):
        st = [x.clone() for x in t]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = hip.cross_attention(*st, 4, 2, mask)
        made.append((graph, st, y))
    for i in range(6):
        graph, st, y = made[i % 2]
        t = (a, b)[(i // 2) % 2]
        for dst, src in zip(st, t):
            dst.copy_(src)
        graph.replay()
        eager = hip.cross_attention(*b, 4, 2, mask)
        torch.cuda.synchronize()
        assert torch.equal(y, ref[(i // 2) % 2]) and torch.equal(eager, ref[1]), i


# whole keys of an image in LDS at its limit, the widest heads
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d", [(1, 40, 128, 2, 2, 128), (2, 300, 127, 2, 1, 128), (1, 700, 100, 1, 1, 96),
                                                      (1, 5000, 128, 3, 3, 64), (3, 1, 128, 16, 2, 120)])
def test_keys_that_fit(n, lq, lk, heads, kv_heads, d, dt, hips, gpu_device):
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, dt, gpu_device, seed=lk)
    for kind in ("none", "keys", "pairs"):
        mask = make_mask(kind, n, lq, lk, gpu_device)
        print(f"[xa] {n} {lq} {lk} {heads} {kv_heads} {d} {kind} {dt}", flush=True)
        check(hips[dt].cross_attention(q, k, v, heads, kv_heads, mask), q, k, v, heads, kv_heads, mask, what=kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d", [(1, 6000, 128, 8, 8, 128), (1, 6000, 128, 8, 8, 96), (2, 3000, 97, 4, 4, 72),
                                                      (2, 3000, 128, 4, 2, 80), (1, 6000, 128, 4, 4, 104), (1, 6000, 75, 4, 4, 112),
                                                      (1, 2000, 128, 8, 8, 112), (2, 2000, 65, 8, 8, 80)])
def test_many_rows_on_keys_that_fit(n, lq, lk, heads, kv_heads, d, dt, hips, gpu_device):
    """Rows enough that the keys stay in LDS, up to 128 KB of them, for every width over 64 that the kernels tell apart."""
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, dt, gpu_device, seed=lk)
    for kind in ("none", "keys", "pairs"):
        mask = make_mask(kind, n, lq, lk, gpu_device)
        print(f"[xa] {n} {lq} {lk} {heads} {kv_heads} {d} {kind} {dt}", flush=True)
        got = hips[dt].cross_attention(q, k, v, heads, kv_heads, mask)
        assert "xa_resident_kernel" in _lib.last_kernel()
        check(got, q, k, v, heads, kv_heads, mask, what=kind)


@pytest.mark.gpu
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d", [(1, 40, 128, 2, 2, 128), (2, 300, 127, 2, 1, 128), (1, 700, 100, 1, 1, 96), (3, 1, 128, 16, 2, 120)])
def test_few_rows_of_wide_fp32_heads_split_keys_that_would_fit(n, lq, lk, heads, kv_heads, d, hips, gpu_device):
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, torch.float32, gpu_device, seed=lk)
    for kind in ("none", "keys", "pairs"):
        mask = make_mask(kind, n, lq, lk, gpu_device)
        got = hips[torch.float32].cross_attention(q, k, v, heads, kv_heads, mask)
        assert "xa_kernel" in _lib.last_kernel() and not _lib.last_kernel().endswith("splits=1")
        check(got, q, k, v, heads, kv_heads, mask, what=kind)


def stretches(what, lq, lk, dev):
    """Masks over thousands of keys in one pass: stretches of whole tiles that nothing keeps."""
    key, row = torch.arange(lk, device=dev), torch.arange(lq, device=dev)[:, None]
    if what == "none":
        return None
    if what == "last keys":
        return (key >= lk - 150)[None]
    if what == "both ends":
        return ((key < 70) | (key >= lk - 37))[None]
    if what == "one key":
        return (key == lk - 1)[None]
    if what == "no key":
        return (key < 0)[None]
    if what == "bands":  # each row its own 90 keys, every seventh none
        return ((key - row * (lk - 90) // lq).clamp(-1, 90).remainder(90) > 0)[None] & (row % 7 != 3)[None]
    if what == "late rows":  # only the last rows keep anything, and only the last keys
        return ((row >= lq - 50) & (key >= lk - 200))[None]
    return ((key < 40) | (key >= lk - 33) | (key // 500 == row // 400))[None]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["none", "last keys", "both ends", "one key", "no key", "bands", "late rows", "regions"])
def test_long_passes(what, dt, hips, gpu_device):
    """Enough rows that no split happens, more keys than 64 tiles (4096 in bf16, 2048 in fp32)."""
    lq, lk, heads, d = 4205, 4501, 8, 32
    q, k, v = inputs(1, lq, lk, heads, heads, d, dt, gpu_device, seed=11)
    mask = stretches(what, lq, lk, gpu_device)
    print(f"[xa] {what} {dt}", flush=True)
    got = hips[dt].cross_attention(q, k, v, heads, mask=mask)
    assert "xa_kernel" in _lib.last_kernel() and _lib.last_kernel().endswith("splits=1")
    check(got, q, k, v, heads, mask=mask, what=what)
    if mask is not None:
        assert not got[:, ~mask.expand(1, lq, lk)[0].any(-1) if mask.dim() == 3 else slice(0, 0 if mask.any() else lq)].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["none", "last keys", "both ends", "one key", "no key", "bands", "late rows", "regions", "scattered keys",
                                  "scattered pairs"])
def test_long_parts(what, dt, hips, gpu_device):
    """Keys split into parts of more than 64 tiles each: the second part's masks past its first 64 tiles."""
    n, lq, lk, heads, d = 2, 700, 8450, 17, 32
    q, k, v = inputs(n, lq, lk, heads, heads, d, dt, gpu_device, seed=13)
    if what.startswith("scattered"):
        mask = make_mask(what.split()[1], n, lq, lk, gpu_device)
    else:
        mask = stretches(what, lq, lk, gpu_device)
        mask = mask if mask is None else mask.expand(n, *mask.shape[1:])
    print(f"[xa] {what} {dt}", flush=True)
    got = hips[dt].cross_attention(q, k, v, heads, mask=mask)
    assert _lib.last_kernel().endswith("splits=2")
    check(got, q, k, v, heads, mask=mask, what=what)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["none", "last keys", "both ends", "one key", "no key"])
def test_long_passes_of_many_rows(what, hips, gpu_device):
    """Enough rows for workgroups of eight waves, the last of them without rows, more keys than 64 tiles."""
    lq, lk, heads, kv_heads, d = 6200, 4501, 16, 4, 40
    q, k, v = inputs(1, lq, lk, heads, kv_heads, d, torch.bfloat16, gpu_device, seed=12)
    mask = stretches(what, lq, lk, gpu_device)
    print(f"[xa] {what}", flush=True)
    got = hips[torch.bfloat16].cross_attention(q, k, v, heads, kv_heads, mask=mask)
    assert "waves=8" in _lib.last_kernel()
    check(got, q, k, v, heads, kv_heads, mask=mask, what=what)
    assert mask is None or mask.any() or not got.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq", [54, 26000])
def test_layouts_of_long_keys(lq, dt, hips, gpu_device):
    """Masks and keys with strides where the keys stream by, split (54 queries) and whole."""
    g = torch.Generator().manual_seed(4)
    hip, heads, d, lk = hips[dt], 2, 32, 9 * 37
    c = heads * d
    q = torch.randn(2, lq // 2, 2, 3 * c, generator=g).to(dt).to(gpu_device)[..., c:2 * c]
    kv = torch.randn(2, 9, 37, 2 * c + 8, generator=g).to(dt).to(gpu_device)
    k, v = kv[..., :c], kv[..., c:2 * c]
    ctx = torch.randn(1, lk, 2 * c, generator=g).to(dt).to(gpu_device).expand(2, lk, 2 * c)
    few = torch.rand(4, 7, 380, generator=g).to(gpu_device) < 0.6
    big = torch.rand(3, lq + 3, 341, generator=g).to(gpu_device) < 0.4
    for what, args, mask in (
            ("keys", (q, k, v), None),
            ("unaligned keys", (q, k, v), few[::2, 0, 5:5 + lk]),
            ("one row for both images", (q, ctx[..., :c], ctx[..., c:]), few[:1, 3, 7:7 + lk].expand(2, lk)),
            ("pair slice", (q, k, v), big[1:, 3:, 3:3 + lk]),
            ("pairs of both images", (q, k, v), big[:1, 1:lq + 1, 8:8 + lk].expand(2, lq, lk)),
            ("pairs of all queries", (q, k, v), few[2:, 6:, 1:1 + lk].expand(2, lq, lk)),
            ("pairs of everything", (q, k, v), few[:1, :1, 47:47 + lk].expand(2, lq, lk))):
        print(f"[xa] {what} {lq} {dt}", flush=True)
        got = hip.cross_attention(*args, heads, mask=mask)
        assert _lib.last_kernel().endswith("splits=1") == (lq > 54)
        check(got, *args, heads, mask=mask, what=what)


@pytest.mark.gpu
@pytest.mark.parametrize("lk", [50, 130, 2000])
def test_any_byte_but_zero_keeps(lk, hips, gpu_device):
    q, k, v = inputs(2, 20, lk, 2, 2, 32, torch.bfloat16, gpu_device)
    byte = torch.randint(0, 256, (2, 20, lk), generator=torch.Generator().manual_seed(6), dtype=torch.uint8).to(gpu_device)
    byte[..., ::3] = 0
    for b in (byte, byte[:, 0].contiguous()):
        got = hips[torch.bfloat16].cross_attention(q, k, v, 2, mask=b.view(torch.bool))
        assert torch.equal(got, hips[torch.bfloat16].cross_attention(q, k, v, 2, mask=b != 0))


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [(150, 900), (40, 60)])
def test_pair_masks_on_streams_and_in_graphs(lq, lk, hips, gpu_device):
    """Each call's bits of its mask are its own: two streams at once, two graphs in turn, eager calls between."""
    hip = hips[torch.bfloat16]
    q, k, v = inputs(2, lq, lk, 4, 2, 64, torch.bfloat16, gpu_device)
    masks = [make_mask("pairs", 2, lq, lk, gpu_device, seed=s) for s in (1, 2)]
    ref = [hip.cross_attention(q, k, v, 4, 2, m) for m in masks]
    assert not torch.equal(*ref)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(s[i]):
                outs.append(hip.cross_attention(q, k, v, 4, 2, masks[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i % 2]) for i, o in enumerate(outs))
    made = []
    for m in masks:
        st = m.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = hip.cross_attention(q, k, v, 4, 2, st)
        made.append((graph, st, y))
    for i in range(6):
        graph, st, y = made[i % 2]
        st.copy_(masks[(i // 2) % 2])
        graph.replay()
        eager = hip.cross_attention(q, k, v, 4, 2, masks[1])
        torch.cuda.synchronize()
        assert torch.equal(y, ref[(i // 2) % 2]) and torch.equal(eager, ref[1]), i


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq,lk", [(9, 20), (9, 2500), (40000, 150)])
def test_output_types_and_flat_queries(lq, lk, dt, hips, gpu_device):
    """Either output type from each form (keys in LDS, split, whole passes), and one query per image as [N, C]."""
    q, k, v = inputs(2, lq, lk, 4, 2, 40, dt, gpu_device)
    for odt in (torch.bfloat16, torch.float32):
        got = hips[dt].cross_attention(q, k, v, 4, 2, out_dtype=odt)
        assert got.dtype == odt
        check(got, q, k, v, 4, 2, what=str(odt))
    one = hips[dt].cross_attention(q[:, 3], k, v, 4, 2, make_mask("pairs", 2, 1, lk, gpu_device, seed=4))
    assert one.shape == (2, 160)
    check(one, q[:, 3], k, v, 4, 2, make_mask("pairs", 2, 1, lk, gpu_device, seed=4))


@pytest.mark.gpu
def test_threads(hips, gpu_device):
    """Calls from several host threads, each on a stream of its own, sizes that share and do not share plans."""
    import threading
    hip = hips[torch.bfloat16]
    cases = [inputs(1, 70 + 30 * (i % 2), 400, 4, 4, 32, torch.bfloat16, gpu_device, seed=i) for i in range(4)]
    refs = [hip.cross_attention(*c, 4) for c in cases]
    torch.cuda.synchronize()
    bad, done = [], []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [hip.cross_attention(*cases[i], 4) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            bad.extend(i for o in outs if not torch.equal(o, refs[i]))
        done.append(i)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert sorted(done) == [0, 1, 2, 3] and not bad


@pytest.mark.gpu
def test_a_scale_is_read_with_every_call(hips, gpu_device):
    q, k, v = inputs(1, 30, 40, 2, 2, 32, torch.float32, gpu_device)
    scale = torch.tensor(0.25)
    for value in (0.25, 0.5):
        scale.fill_(value)
        got = hips[torch.float32].cross_attention(q, k, v, 2, scale=scale)
        check(got, q, k, v, 2, scale=value)


@pytest.mark.gpu
def test_no_keys_and_no_queries(hips, gpu_device):
    for hip in hips.values():
        q, k, v = inputs(2, 3, 5, 2, 2, 32, hip.dtype, gpu_device)
        assert not hip.cross_attention(q, k[:, :0], v[:, :0], 2).any()
        assert hip.cross_attention(q[:, :0], k, v, 2).shape == (2, 0, 64)
        assert not hip.cross_attention(q, k, v, 2, mask=torch.zeros(2, 5, dtype=torch.bool, device=gpu_device)).any()


@pytest.mark.gpu
def test_conditioning_block(gpu_device):
    """The operators as a block uses them: x + linear(cross_attention(linear(group_norm(x)), linear(context))),
    each prompt padded, against the oracle (fp32, 1e-5 of the output's scale)."""
    from _tol import assert_fp32
    from oracle.torch_ref import TorchRef
    g = torch.Generator().manual_seed(3)
    c, cc, heads = 96, 64, 3
    t = {"x": torch.randn(2, 24, 37, c, generator=g), "ctx": torch.randn(2, 1, 77, cc, generator=g),
         "gw": torch.rand(c, generator=g) + 0.5, "gb": torch.randn(c, generator=g) * 0.2,
         "wq": torch.randn(c, c, generator=g) * c ** -0.5, "wkv": torch.randn(cc, 2 * c, generator=g) * cc ** -0.5,
         "wo": torch.randn(c, c, generator=g) * c ** -0.5, "bo": torch.randn(c, generator=g) * 0.1}
    mask = torch.arange(77)[None] < torch.tensor([[77], [20]])

    def block(o, t, mask):
        q = o.linear(o.group_norm(t["x"], 32, t["gw"], t["gb"]), t["wq"])
        kv = o.linear(t["ctx"], t["wkv"])
        y = o.cross_attention(q, kv[..., :c], kv[..., c:], heads, mask=mask)
        return o.linear(y, t["wo"], t["bo"], residual=t["x"])
    want = block(TorchRef(torch.float32, "cpu"), t, mask)
    ops = Ops(["hip"], torch.float32, gpu_device, log=print)
    got = block(ops, {k: v.to(gpu_device) for k, v in t.items()}, mask.to(gpu_device))
    assert_fp32(got.cpu(), want, what="conditioning block")
    ops = Ops(["hip"], torch.bfloat16, gpu_device, log=print)
    low = block(ops, {k: v.to(gpu_device).to(torch.bfloat16 if k in ("x", "ctx", "wq", "wkv", "wo") else torch.float32)
                      for k, v in t.items()}, mask.to(gpu_device))
    # nine roundings to bf16 on the path (five operands, four results), each 2^-8 of values of the output's scale at most
    assert (low.double().cpu() - want.double()).abs().max() <= 9 * 2.0 ** -8 * want.abs().max()
