"""group_norm: the HIP kernels (clarus_hip_group_norm) against the formula in 64 bits.

Tolerances. fp32: the sums of a thread are at most 64 values in a row, joined a few times, so the mean is
off by at most 80 * 2^-24 of the largest |x| and the variance by as much of itself; y moves by that times
|weight| / std plus a few roundings of y and of the activation: STAT * (max|x - 0| / std) * max|weight| with
STAT = 80 * 2^-24, and 16 * 2^-24 of y's scale. bf16 outputs add one rounding, 2^-8 of the value.
"""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

EPS = 1e-5
STAT = 80 * 2.0 ** -24


def plain64(x, groups, weight=None, bias=None, eps=EPS, act=None):
    """(y, the value that STAT multiplies) in float64."""
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
    rstd = torch.rsqrt(var + eps)
    w = torch.ones(1, 1, c, dtype=torch.float64, device=x.device) if weight is None else weight.double().reshape(-1, 1, c)
    y = ((v - mean) * rstd).reshape(n, -1, c) * w
    if bias is not None:
        y = y + bias.double().reshape(-1, 1, c)
    slack = (v.abs().amax((1, 3), keepdim=True) * rstd).expand(n, 1, groups, c // groups).reshape(n, 1, c) * w.abs()
    slack = (slack + y.abs().amax(1, keepdim=True)).expand(y.shape)
    if act == "silu":
        y = F.silu(y)
    elif act == "gelu":
        y = F.gelu(y)
    return y.reshape(x.shape), 1.2 * slack.reshape(x.shape)  # |act'| <= 1.2


def check(got, x, groups, weight=None, bias=None, eps=EPS, act=None, what=""):
    ref, slack = plain64(x, groups, weight, bias, eps, act)
    assert got.shape == x.shape and got.is_contiguous(), what
    d = (got.double() - ref).abs()
    tol = STAT * slack + (2.0 ** -8 * ref.abs() if got.dtype == torch.bfloat16 else 0)
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    worst = (d - tol).max().item()
    assert worst <= 0, f"{what}: max|d| {d.max().item():.3e}, {worst:.3e} past the tolerance"


def inputs(shape, dt, dev, seed=0, per_image=False, affine=True):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(*shape, generator=g) * (0.5 + torch.randn(c, generator=g).abs()) + torch.randn(c, generator=g)).to(dt)
    ab = (shape[0], c) if per_image else (c,)
    w = torch.randn(*ab, generator=g) * 0.3 + 1 if affine else None
    b = torch.randn(*ab, generator=g) * 0.3 if affine else None
    return x.to(dev), *(t if t is None else t.to(dev) for t in (w, b))


# ------------------------------------------------------------------ CPU
def cpu_hip(dtype=torch.float32):
    """HipOps' argument checks without a device: what passes them fails before anything is launched."""
    from clarus_amd.hip_ops import HipOps
    h = HipOps.__new__(HipOps)
    h.dtype, h.device, h.dev, h._cache, h._plans = dtype, torch.device("cpu"), torch.device("cpu"), {}, {}
    h.lib = _lib.load()
    return h


@pytest.mark.parametrize("shape,groups,kw", [
    ((2, 4, 4, 12), 4, {}),                       # channels no multiple of 8
    ((2, 4, 4, 16), 3, {}),                       # nor of the groups
    ((2, 4, 4, 16), 0, {}),
    ((2, 4, 4, 16), 2.0, {}),
    ((2, 4, 4, 16), 4, {"act": "relu"}),
    ((2, 4, 4, 16), 4, {"out_dtype": torch.float16}),
    ((1, 2, 2, 4096), 1, {}),                     # a group wider than 2048 channels
    ((1, 2, 2, 8 * 257), 8, {}),                  # 257 channels a group: 8 * 257 to whole octets
    ((2, 4, 4, 16), 4, {"weight": torch.ones(8)}),
    ((2, 4, 4, 16), 4, {"bias": torch.ones(3, 16)}),
    ((2, 4, 4, 16), 4, {"weight": torch.ones(16, dtype=torch.int64)}),
    ((16,), 4, {}),
])
def test_refusals(shape, groups, kw):
    with pytest.raises(Unsupported):
        cpu_hip().group_norm(torch.zeros(shape), groups, **kw)


@pytest.mark.parametrize("kw", [{"act": "relu"}, {"act": True}, {"groups": 3}, {"groups": 0}, {"groups": 2.0}, {"weight": torch.ones(16, 2)},
                                {"weight": torch.ones(32)}, {"bias": torch.ones(1, 1, 16)}, {"bias": torch.ones(16, dtype=torch.int64)},
                                {"eps": -1.0}, {"eps": float("nan")}, {"out_dtype": torch.int32}])
def test_what_no_backend_answers_is_declined_by_all(kw):
    """The torch form of the chain declines too what is no group norm, instead of answering something else."""
    from clarus_amd.spatial_torch import TorchSpatialOps
    args = {"groups": 4, **kw}
    for be in (cpu_hip(), TorchSpatialOps(torch.float32, "cpu")):
        with pytest.raises(Unsupported):
            be.group_norm(torch.zeros(2, 4, 4, 16), **args)
    with pytest.raises(Unsupported):
        TorchSpatialOps(torch.float32, "cpu").group_norm(torch.zeros(16), 4)


def test_refused_layouts_and_gradients():
    h = cpu_hip()
    for x in (torch.zeros(2, 4, 4, 32)[..., ::2], torch.zeros(2, 16, 4, 4).permute(0, 2, 3, 1),
              torch.zeros(2, 4, 6, 16)[:, :, :4], torch.zeros(2, 4, 4, 20)[..., 2:18], torch.zeros(1, 1, 1, 16).expand(2, 4, 4, 16),
              torch.zeros(2, 4, 4, 16, dtype=torch.float16), torch.zeros(2, 4, 4, 16, requires_grad=True)):
        with pytest.raises(Unsupported):
            h.group_norm(x, 4)
    with pytest.raises(Unsupported):
        h.group_norm(torch.zeros(2, 4, 4, 16), 4, weight=torch.ones(16, requires_grad=True))


def test_refused_values():
    h = cpu_hip()
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(Unsupported):
            h.group_norm(torch.zeros(2, 4, 4, 16), 4, eps=eps)
    with pytest.raises(Unsupported):
        h.group_norm(torch.zeros(1, 1, 1 << 19), 1 << 16)
    lib = _lib.load()
    for kw in (dict(eps=-1.0), dict(eps=float("nan")), dict(c=1 << 19, ldx=1 << 19)):
        kw = {**dict(eps=1e-5, c=64, ldx=64), **kw}
        assert lib.clarus_hip_group_norm(1 << 20, 0, 0, kw["ldx"], None, 0, None, 0, 1 << 24, 0, 1, 4, kw["c"], kw["c"] // 8,
                                         kw["eps"], 0, None, 0, None) == _lib.EINVAL, kw


def test_a_refusal_does_not_depend_on_earlier_calls():
    h, x = cpu_hip(), torch.zeros(2, 0, 4, 16)
    assert h.group_norm(x, 4).shape == x.shape
    with pytest.raises(Unsupported):
        h.group_norm(x, 4.0)


def test_tangents_go_to_the_torch_form():
    from torch.autograd import forward_ad
    from clarus_amd.spatial_torch import TorchSpatialOps
    h, be, x, w = cpu_hip(), TorchSpatialOps(torch.float32, "cpu"), torch.randn(2, 4, 4, 16), torch.ones(16)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for args in ((dual, 4, w), (x, 4, forward_ad.make_dual(w, w))):
            with pytest.raises(Unsupported, match="tangent"):
                h.group_norm(*args)
            assert forward_ad.unpack_dual(be.group_norm(*args)).tangent is not None


def test_an_eps_that_fp32_does_not_hold_is_declined():
    for eps in (1e39, 3.5e38, -1e-50):
        with pytest.raises(Unsupported):
            cpu_hip().group_norm(torch.zeros(2, 4, 4, 16), 4, eps=eps)


def test_refused_launches():
    """As many strips of channels as a launch has no workgroups for."""
    with pytest.raises(Unsupported):
        cpu_hip().group_norm(torch.zeros(1, 1, 1 << 18).expand(65535, 1, 1 << 18), 1 << 8)
    cpu_hip()._group_norm_plan(torch.zeros(1, 1, 1 << 18).expand(65000, 1, 1 << 18), 1 << 8, None, None, None, torch.float32)


def test_c_entry_refuses_before_launch():
    lib = _lib.load()

    def call(x=1 << 20, xdt=0, xbs=0, ldx=64, wbs=0, out=1 << 24, odt=0, n=1, p=100, c=64, g=8, act=0, scratch=1 << 28, size=1 << 20):
        return lib.clarus_hip_group_norm(x, xdt, xbs, ldx, None, wbs, None, 0, out, odt, n, p, c, g, 1e-5, act, scratch, size, None)
    for kw in (dict(x=None), dict(out=None), dict(p=100000, scratch=None), dict(n=0), dict(p=0), dict(c=60, g=4), dict(g=7), dict(g=0),
               dict(xdt=2), dict(odt=5), dict(act=2), dict(ldx=56), dict(ldx=66), dict(x=(1 << 20) + 4), dict(out=(1 << 24) + 8),
               dict(wbs=8), dict(p=100000, size=8), dict(n=1 << 16), dict(p=1 << 31), dict(c=4096, g=1, ldx=4096), dict(n=2, xbs=-64)):
        assert call(**kw) == _lib.EINVAL, kw
        assert b"group_norm" in lib.clarus_hip_last_error()
    assert lib.clarus_hip_group_norm_workspace(1, 100, 60, 4) == 0
    assert lib.clarus_hip_group_norm_workspace(2, 100000, 64, 8) > 0


@pytest.mark.parametrize("per_image", [False, True])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_torch_form_and_oracle(act, per_image):
    from clarus_amd import spatial_torch
    from oracle.torch_ref import TorchRef
    x, w, b = inputs((2, 5, 7, 24), torch.float32, "cpu", per_image=per_image)
    for be in (spatial_torch.TorchSpatialOps(torch.float32, "cpu"), TorchRef(torch.float32, "cpu")):
        check(be.group_norm(x, 3, w, b, eps=EPS, act=act), x, 3, w, b, act=act, what=be.name)


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


SHAPES = [((1, 1, 1, 8), 1), ((2, 1, 1, 64), 32), ((2, 7, 13, 96), 32), ((1, 5, 9, 48), 16), ((3, 16, 24, 512), 32),
          ((1, 173, 251, 128), 32), ((2, 33, 64), 16), ((5, 40), 5), ((1, 64, 64, 2048), 8), ((1, 9, 9, 4096), 32),
          ((2, 3, 5, 2056), 257), ((1, 11, 3, 2400), 32), ((1, 7, 3, 40), 2), ((2, 50, 70, 192), 32), ((70, 3, 3, 64), 1),
          ((2, 300, 301, 32), 8), ((1, 4, 4, 1320), 11), ((1, 90, 160, 512), 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_shapes(shape, groups, dt, hips, gpu_device):
    for i, act in enumerate((None, "silu", "gelu")):
        x, w, b = inputs(shape, dt, gpu_device, seed=i, per_image=i == 1, affine=i != 2)
        print(f"[gn] {shape} {groups} {dt} {act}", flush=True)
        got = hips[dt].group_norm(x, groups, w, b, eps=EPS, act=act)
        assert got.dtype == dt
        check(got, x, groups, w, b, act=act, what=f"{shape} {groups} {act}")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,groups", [((130, 42, 50, 64), 8), ((700, 41, 51, 32), 8), ((37, 30, 40, 264), 33), ((3, 70, 60, 2400), 12),
                                          ((200, 3, 5, 512), 64)])
def test_many_images_and_strips(shape, groups, dt, hips, gpu_device):
    """Fewer chunks of an image than XCDs, several strips of channels."""
    x, w, b = inputs(shape, dt, gpu_device, per_image=True)
    print(f"[gn] {shape} {groups} {dt}", flush=True)
    got = hips[dt].group_norm(x, groups, w, b, eps=EPS, act="silu")
    print(f"[gn] {_lib.last_kernel()}", flush=True)
    check(got, x, groups, w, b, act="silu", what=str(shape))


@pytest.mark.gpu
def test_types_of_operands(hips, gpu_device):
    x, w, b = inputs((2, 12, 17, 64), torch.float32, gpu_device)
    for xdt in (torch.bfloat16, torch.float32):
        for odt in (torch.bfloat16, torch.float32):
            xx = x.to(xdt)
            got = hips[torch.bfloat16].group_norm(xx, 16, w.bfloat16(), b, act="silu", out_dtype=odt)
            assert got.dtype == odt
            check(got, xx, 16, w.bfloat16(), b, act="silu", what=f"{xdt} -> {odt}")
    check(hips[torch.float32].group_norm(x, 16, w), x, 16, w)
    check(hips[torch.float32].group_norm(x, 16, bias=b), x, 16, None, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_strides(dt, hips, gpu_device):
    wide, w, b = inputs((4, 12, 17, 96), dt, gpu_device)
    w, b = w[:32], b[:32]
    for what, x in (("channel slice", wide[..., 32:64]), ("image slice", wide[1::2, ..., :32]), ("rows", wide[:, 3:7, :, 64:]),
                    ("one row", wide[:, 2:3, 4:9, :32]), ("one column", wide[:1, :, 5:6, :32]), ("image twice", wide[:1, ..., :32].expand(3, 12, 17, 32))):
        print(f"[gn] {what}", flush=True)
        check(hips[dt].group_norm(x, 8, w, b, act="silu"), x, 8, w, b, act="silu", what=what)


@pytest.mark.gpu
def test_hard_values(hips, gpu_device):
    """Means far from zero, one huge value, a constant group, and NaN or inf in another group or image."""
    hip = hips[torch.float32]
    x, w, b = inputs((2, 40, 50, 64), torch.float32, gpu_device)
    check(hip.group_norm(x + 1000, 8, w, b), x + 1000, 8, w, b, what="offset")
    y = x.clone()
    y[0, 0, 0, 0] = 1e4
    y[1, 39, 49, 63] = -3e4
    check(hip.group_norm(y, 8, w, b), y, 8, w, b, what="outlier")
    z = torch.full_like(x, 3.25)
    assert torch.equal(hip.group_norm(z, 8, w, b), b.expand(x.shape))
    base = hip.group_norm(x, 8, w, b)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[1, 3, 4, 20] = bad  # group 2 of image 1
        got = hip.group_norm(y, 8, w, b)
        assert torch.equal(got[0], base[0]) and not torch.isfinite(got[1, ..., 16:24]).any()
        assert torch.equal(got[1, ..., :16], base[1, ..., :16]) and torch.equal(got[1, ..., 24:], base[1, ..., 24:])


# one launch and three, an octet in one group and in several, several strips of channels
FORMS = [((2, 20, 30, 64), 8), ((2, 9, 11, 96), 32), ((1, 120, 130, 64), 8), ((2, 70, 90, 96), 32), ((3, 40, 50, 2400), 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,groups", FORMS)
def test_values_whose_square_overflows(shape, groups, dt, hips, gpu_device):
    """Values around 1e20, whose squares fp32 does not hold, with a variance that it does."""
    noise = torch.randn(*shape, generator=torch.Generator().manual_seed(8))
    _, w, b = inputs(shape, dt, gpu_device)
    for size in (1e20, -1e20):
        x = (size * (1 + 1e-3 * noise)).to(dt).to(gpu_device)
        check(hips[dt].group_norm(x, groups, w, b), x, groups, w, b, what=f"{size}")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,groups", FORMS)
def test_equal_values(shape, groups, dt, hips, gpu_device):
    """A group of one value, its mantissa full, has that mean and no variance: the bias comes out."""
    _, w, b = inputs(shape, dt, gpu_device)
    for value in (1000.1, 0.1, -100.3, 1e-30, 3e36):
        x = torch.full(shape, value, dtype=dt, device=gpu_device)
        assert torch.equal(hips[dt].group_norm(x, groups, w, b), b.to(dt).expand(shape)), value


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", FORMS)
def test_what_is_not_finite_stays_in_its_group(shape, groups, hips, gpu_device):
    """First and last values of a group among them: what other values are taken relative to."""
    hip, size = hips[torch.float32], shape[-1] // groups
    x, w, b = inputs(shape, torch.float32, gpu_device)
    base = hip.group_norm(x, groups, w, b)
    g = groups // 2
    inside = slice(g * size, (g + 1) * size)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for at in ((0, 0, g * size), (shape[1] - 1, shape[2] - 1, (g + 1) * size - 1), (shape[1] // 2, 3, g * size + size // 2)):
            y = x.clone()
            y[(shape[0] - 1, *at)] = bad
            got = hip.group_norm(y, groups, w, b)
            assert torch.equal(got[:-1], base[:-1]) and not torch.isfinite(got[-1, ..., inside]).any(), (bad, at)
            assert torch.equal(got[-1, ..., :g * size], base[-1, ..., :g * size]), (bad, at)
            assert torch.equal(got[-1, ..., (g + 1) * size:], base[-1, ..., (g + 1) * size:]), (bad, at)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,groups", FORMS)
def test_c_entry_in_place(shape, groups, dt, hips, gpu_device):
    """out may be x itself."""
    hip = hips[dt]
    x, w, b = inputs(shape, dt, gpu_device)
    want = hip.group_norm(x, groups, w, b, act="silu")
    n, p, c, code = shape[0], shape[1] * shape[2], shape[-1], _lib.dtype_code(dt)
    need = hip.lib.clarus_hip_group_norm_workspace(n, p, c, groups)
    scratch = torch.empty(max(need, 8), dtype=torch.uint8, device=gpu_device)
    _lib.check(hip.lib.clarus_hip_group_norm(x.data_ptr(), code, p * c, c, w.data_ptr(), 0, b.data_ptr(), 0, x.data_ptr(), code, n, p, c,
                                             groups, EPS, _lib.ACT_SILU, scratch.data_ptr(), need,
                                             torch.cuda.current_stream().cuda_stream), "group_norm")
    assert torch.equal(x, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("shape", [(1, 20, 30, 64), (1, 120, 130, 64)])
def test_activations_over_their_range(shape, act, dt, hips, gpu_device):
    """Values from -60 to 60: the tails go to 0 and x. In bf16, beside the general check, the values of the tail
    themselves, down to -5.4 (below, they are under 2^-21): 2^-8 of the value for the rounding and as much for the
    formula, and what y may be off by times the activation's slope there (its curvature times the square is nothing)."""
    x, _, _ = inputs(shape, torch.float32, gpu_device)
    for w, b in ((1.0, 0.0), (1.0, -3.0), (0.5, -5.0), (12.0, 5.0), (0.25, 50.0), (0.25, -50.0)):
        wt, bt = (torch.full((shape[-1],), t, device=gpu_device) for t in (w, b))
        got = hips[dt].group_norm(x, 8, wt, bt, act=act, out_dtype=dt)
        check(got, x, 8, wt, bt, act=act, what=f"{act} {w} {b}")
        if dt == torch.bfloat16:
            y, slack = plain64(x, 8, wt, bt)
            y.requires_grad_()
            ref = F.silu(y) if act == "silu" else F.gelu(y)
            slope, = torch.autograd.grad(ref.sum(), y)
            tol = 2 * 2.0 ** -8 * ref.abs() + STAT * slack * slope.abs()
            off = torch.where(y > -5.4, (got.double() - ref).abs() - tol, torch.zeros_like(ref))
            assert off.max() <= 0, (w, b, off.max().item())


@pytest.mark.gpu
def test_a_weight_is_read_with_every_call(hips, gpu_device):
    """A weight of another type that changes outside autograd's sight, and one used on another stream."""
    x, w, b = inputs((1, 9, 7, 64), torch.float32, gpu_device)
    hip = hips[torch.float32]
    wb = w.bfloat16()
    for i in range(3):
        wb.data.copy_((w * (i + 1)).bfloat16())
        check(hip.group_norm(x, 8, wb, b), x, 8, wb, b, what=str(i))
    with torch.inference_mode():
        wi = w.bfloat16()
        check(hip.group_norm(x, 8, wi, b), x, 8, wi, b, what="inference")


@pytest.mark.gpu
def test_offsets_past_32_bits(hips, gpu_device):
    """2.2e9 elements: 33 copies of one map, whose statistics are the map's."""
    x, w, b = inputs((1, 1 << 20, 64), torch.bfloat16, gpu_device)
    got = hips[torch.bfloat16].group_norm(x.repeat(1, 33, 1), 16, w, b)
    ref, slack = plain64(x, 16, w, b)
    for i in (0, 15, 31, 32):
        d = (got[:, i << 20:(i + 1) << 20].double() - ref).abs()
        assert (d <= STAT * slack + 2.0 ** -8 * ref.abs()).all(), (i, d.max().item())


@pytest.mark.gpu
def test_empty_repeatable_streams_and_graph(hips, gpu_device):
    hip = hips[torch.bfloat16]
    assert hip.group_norm(torch.zeros(0, 4, 4, 16, device=gpu_device), 4).shape == (0, 4, 4, 16)
    assert hip.group_norm(torch.zeros(2, 0, 4, 16, device=gpu_device), 4).shape == (2, 0, 4, 16)
    x, w, b = inputs((2, 90, 77, 96), torch.bfloat16, gpu_device)
    x2, _, _ = inputs((2, 90, 77, 96), torch.bfloat16, gpu_device, seed=9)
    ref, ref2 = hip.group_norm(x, 32, w, b, act="silu"), hip.group_norm(x2, 32, w, b, act="silu")
    for _ in range(3):
        assert torch.equal(hip.group_norm(x, 32, w, b, act="silu"), ref)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        for s, v in ((s1, x), (s2, x2)):
            with torch.cuda.stream(s):
                outs.append(hip.group_norm(v, 32, w, b, act="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref2 if i % 2 else ref) for i, o in enumerate(outs))
    static = x.clone()
    wb = w.bfloat16()  # converted inside the graph: nothing of a capture is kept for eager calls
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hip.group_norm(static, 32, wb, b, act="silu")
    want = hip.group_norm(x, 32, wb, b, act="silu"), hip.group_norm(x2, 32, wb, b, act="silu")
    for i in range(4):
        static.copy_((x, x2)[i % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i % 2]), i
        assert torch.equal(hip.group_norm(x, 32, w, b, act="silu"), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 12, 17, 64), 16), ((2, 60, 70, 64), 16), ((1, 50, 60, 96), 12)])
def test_output_types_and_graphs_of_each_form(shape, groups, hips, gpu_device):
    hip = hips[torch.bfloat16]
    x, w, b = inputs(shape, torch.float32, gpu_device)
    for xdt in (torch.bfloat16, torch.float32):
        for odt in (torch.bfloat16, torch.float32):
            got = hip.group_norm(x.to(xdt), groups, w, b, act="gelu", out_dtype=odt)
            check(got, x.to(xdt), groups, w, b, act="gelu", what=f"{xdt} -> {odt}")
    a = [x.bfloat16(), x.flip(0, 1).mul(2).bfloat16()]
    want = [hip.group_norm(t, groups, w, b, act="silu") for t in a]
    made = []
    for t in a:
        st = t.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = hip.group_norm(st, groups, w, b, act="silu")
        made.append((graph, st, y))
    for i in range(6):
        graph, st, y = made[i % 2]
        st.copy_(a[(i // 2) % 2])
        graph.replay()
        eager = hip.group_norm(a[1], groups, w, b, act="silu")
        torch.cuda.synchronize()
        assert torch.equal(y, want[(i // 2) % 2]) and torch.equal(eager, want[1]), i


@pytest.mark.gpu
def test_chain_serves_gradients_on_torch(gpu_device):
    """An input that needs its gradient goes to the torch form of the chain, which has it."""
    from clarus_amd import spatial_torch  # noqa: F401
    ops = Ops(["hip", "torch"], torch.float32, gpu_device, log=print)
    x, w, b = inputs((1, 6, 5, 32), torch.float32, gpu_device)
    ops.group_norm(x, 4, w, b)
    x.requires_grad_()
    y = ops.group_norm(x, 4, w, b)
    assert y.requires_grad and ops.report()["ops"]["group_norm"] == {"hip": 1, "torch": 1}
    with torch.no_grad():
        ops.group_norm(x, 4, w, b)
    assert ops.report()["ops"]["group_norm"] == {"hip": 2, "torch": 1}
