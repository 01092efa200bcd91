"""linear_attention: the HIP kernels (clarus_hip_linear_attention) against the sums over all pairs of tokens in 64 bits.

Tolerance, u = 2^-24; A the sum of the same terms' sizes (of an output: scale e^{g (i - j)} sum|q||k| |v|, and of the state that
goes in). A term is rounded in its products and factors (10 u: exponents g n are off by 2 u of themselves, x e^-x of which
is below u) and once for each addition behind it: dk in q . k, at most a quarter of the tokens (sixteen, or two in fp32,
go into a state at once, a chunk's sum into the next one's, a segment's into the state; counted with room), 64 within a
chunk: (l / 4 + dk + 150) u A in all. bf16: q . k of tokens in one chunk rounded once (2^-8 of the terms up to 64 tokens
away), the state and its values in parts of 2^-16 (for outputs only). The outputs' own rounding: 2^-8 (bf16), u.
"""
from __future__ import annotations

import math

import pytest
import torch

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

U = 2.0 ** -24


def plain64(q, k, v, log_decay, heads, kv_heads=None, state=None, scale=None):
    """(out, A, A of tokens within 64, state, A of the state), float64."""
    kv_heads = kv_heads or heads
    n, rep, dk, dv = q.shape[0], heads // kv_heads, q.shape[-1] // heads, v.shape[-1] // kv_heads
    qh = q.double().reshape(n, -1, heads, dk).permute(0, 2, 1, 3).contiguous() * (dk ** -0.5 if scale is None else scale)
    l = qh.shape[2]
    kh, vh = (t.double().reshape(n, l, kv_heads, -1).permute(0, 2, 1, 3).contiguous() for t in (k, v))
    g = log_decay.double().clamp_min(-1e9)[:, None, None]
    at = torch.arange(l, device=q.device, dtype=torch.float64)
    gap = at[:, None] - at[None]
    w = torch.where(gap >= 0, torch.exp(g * gap), torch.zeros_like(gap)).repeat_interleave(rep, 0)
    near = w * (gap < 64)
    kt = kh.repeat_interleave(rep, 1).transpose(-1, -2).contiguous()
    vr = vh.repeat_interleave(rep, 1)
    s0 = torch.zeros(n, kv_heads, dk, dv, dtype=torch.float64, device=q.device) if state is None else state.double()
    since = torch.exp(g * (at[:, None] + 1)).repeat_interleave(rep, 0)
    out = (qh @ kt * w) @ vr + since * (qh @ s0.repeat_interleave(rep, 1))
    size = qh.abs() @ kt.abs()
    big = (size * w) @ vr.abs() + since * (qh.abs() @ s0.abs().repeat_interleave(rep, 1))
    left = torch.exp(g * (l - 1 - at[:, None]))
    last = (kh * left).transpose(-1, -2).contiguous() @ vh + torch.exp(g * l) * s0
    slast = (kh.abs() * left).transpose(-1, -2).contiguous() @ vh.abs() + torch.exp(g * l) * s0.abs()

    def back(t):
        return t.permute(0, 2, 1, 3).reshape(*q.shape[:-1], heads * dv)
    return back(out), back(big), back((size * near) @ vr.abs()), last, slast


def check(got, q, k, v, log_decay, heads, kv_heads=None, state=None, scale=None, what=""):
    out, last = got
    ref, big, near, rlast, slast = plain64(q, k, v, log_decay, heads, kv_heads, state, scale)
    l, dk = math.prod(q.shape[1:-1]), q.shape[-1] // heads
    assert out.shape == ref.shape and out.is_contiguous() and last.shape == rlast.shape and last.dtype == torch.float32, what
    assert torch.isfinite(out).all() and torch.isfinite(last).all(), what
    m = (l / 4 + dk + 150) * U
    tol = m * big + (2.0 ** -8 * near + 2.0 ** -14 * big if q.dtype == torch.bfloat16 else 0)
    tol = tol + (2.0 ** -8 if out.dtype == torch.bfloat16 else U) * (ref.abs() + tol)
    for name, t, r, e in (("out", out, ref, tol), ("state", last, rlast, m * slast)):
        off = (t.double() - r).abs()
        assert (off <= e).all(), f"{what} {name}: max|d| {off.max().item():.3e}, {(off - e).max().item():.3e} past the tolerance"


def inputs(n, l, heads, kv_heads, dk, dv, dt, dev, seed=0, carried=True):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(n, l, h * d, generator=g).to(dt).to(dev) for h, d in ((heads, dk), (kv_heads, dk), (kv_heads, dv)))
    return q, k, v, (torch.randn(n, kv_heads, dk, dv, generator=g) * 3).to(dev) if carried else None


def decays(kv_heads, dev):
    return torch.tensor([-1 / 16, 0.0, -0.5, -1e-3, -8.0, -math.inf, -1 / 64, -100.0])[:kv_heads].to(dev)


# ------------------------------------------------------------------ CPU
def cpu_hip(dtype=torch.float32):
    from clarus_amd.hip_ops import HipOps
    h = HipOps.__new__(HipOps)
    h.dtype, h.device, h.dev, h._cache, h._plans = dtype, torch.device("cpu"), torch.device("cpu"), {}, {}
    h.lib = _lib.load()
    return h


def test_refusals():
    h, z = cpu_hip(), torch.zeros
    q, k, g, s = z(2, 5, 64), z(2, 5, 32), z(2), z(2, 2, 16, 16)
    cases = [
        ((q, k, k, g, 3), {}), ((q, k, k, g, 4), {}), ((q, k, k, g, 4, 3), {}), ((q, k, k, g, 4.0, 2), {}), ((q, k, k, g, 4, 2.0), {}),
        ((q, k, k, g, 0, 0), {}), ((z(2, 6, 64), k, k, g, 4, 2), {}), ((q, k, z(2, 4, 32), g, 4, 2), {}), ((q, z(1, 5, 32), k, g, 4, 2), {}),
        ((z(2, 5, 48), z(2, 5, 24), k, g, 4, 2), {}), ((z(2, 5, 544), z(2, 5, 272), k, g, 4, 2), {}), ((q, k, z(2, 5, 24), g, 4, 2), {}),
        ((q, k, z(2, 5, 272), g, 4, 2), {}), ((q, k, k, z(3), 4, 2), {}), ((q, k, k, z(2, 1), 4, 2), {}), ((q, k, k, z(2).long(), 4, 2), {}),
        ((q.half(), k.half(), k.half(), g, 4, 2), {}), ((q, k.bfloat16(), k, g, 4, 2), {}), ((q, k, k, g, 4, 2), {"out_dtype": torch.float16}),
        ((q, k, k, g, 4, 2), {"scale": math.inf}), ((q, k, k, g, 4, 2), {"scale": math.nan}), ((q, k, k, g, 4, 2), {"scale": 1e39}),
        ((q, k, k, g, 4, 2), {"state": z(2, 2, 16, 8)}), ((q, k, k, g, 4, 2), {"state": s.double()}),
        ((q, k, k, g, 4, 2), {"state": s.transpose(-1, -2)}), ((q, k, k, g, 4, 2), {"state_out": z(1, 2, 16, 16)}),
        ((q, k, k, g, 4, 2), {"state_out": s.bfloat16()}), ((z(2, 64, 5).transpose(1, 2), k, k, g, 4, 2), {}),
        ((z(2, 5, 66)[..., :64], k, k, g, 4, 2), {}), ((q, z(2, 5, 33)[..., 1:], k, g, 4, 2), {}), ((z(64), z(32), z(32), g, 4, 2), {}),
        ((q.clone().requires_grad_(), k, k, g, 4, 2), {}), ((q, k, k, g.clone().requires_grad_(), 4, 2), {}),
        ((q, k, k, g, 4, 2), {"state": s.clone().requires_grad_()}),
        ((z(1, 1, 64).expand(1 << 20, 1, 64), z(1, 1, 32).expand(1 << 20, 1, 32), z(1, 1, 32).expand(1 << 20, 1, 32), g, 4, 2), {}),
        ((q, z(2 * 5 * (1 << 24)).as_strided((2, 5, 32), (0, 1 << 24, 1)), k, g, 4, 2), {}),
    ]
    for i, (args, kw) in enumerate(cases):
        with pytest.raises(Unsupported):
            h.linear_attention(*args, **kw)
            pytest.fail(f"case {i} was accepted")


def test_no_tokens_keep_the_state():
    h, z = cpu_hip(), torch.zeros
    s = torch.randn(2, 2, 16, 8)
    args = z(2, 0, 64), z(2, 0, 32), z(2, 0, 16), z(2), 4, 2
    out, last = h.linear_attention(*args, state=s)
    assert out.shape == (2, 0, 32) and torch.equal(last, s) and last is not s
    assert not h.linear_attention(*args)[1].any()
    t = torch.ones_like(s)
    assert h.linear_attention(*args, state=s, state_out=t)[1] is t and torch.equal(t, s)
    assert h.linear_attention(*args, state=s, state_out=s)[1] is s


def test_c_entry_refuses_before_launch():
    import ctypes
    lib = _lib.load()
    assert lib.clarus_hip_linear_attention(None, None, 0, None) == _lib.EINVAL

    def call(scratch=1 << 30, size=1 << 30, **kw):
        base = dict(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, log_decay=1 << 24, state_out=1 << 25, n=1, l=64, heads=4, kv_heads=2,
                    dk=32, dv=16, ldq=128, ldk=64, ldv=32, scale=0.2)
        return lib.clarus_hip_linear_attention(ctypes.byref(_lib.LinearArgs(**{**base, **kw})), scratch, size, None)
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(log_decay=None), dict(state_out=None), dict(n=0), dict(l=0),
               dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dk=0), dict(dk=12), dict(dk=136), dict(dv=4), dict(dv=136),
               dict(dtype=2), dict(o_dtype=-1), dict(scale=math.nan), dict(scale=math.inf), dict(q=(1 << 20) + 8), dict(ldq=130),
               dict(ldk=-64), dict(v_bstride=2), dict(ldq=1 << 24), dict(ldk=1 << 24), dict(ldv=1 << 24), dict(state_in=8), dict(state_out=8), dict(log_decay=2),
               dict(n=1 << 19), dict(n=1 << 62), dict(n=1 << 60, kv_heads=16, heads=16), dict(heads=1 << 62), dict(l=1 << 31),
               dict(scratch=None), dict(size=16), dict(scratch=8)):
        assert call(**kw) == _lib.EINVAL, kw
        assert b"linear_attention" in lib.clarus_hip_last_error()
    assert lib.clarus_hip_linear_attention_workspace(1, 1, 1000, 4, 2, 32, 32) > 0
    assert lib.clarus_hip_linear_attention_workspace(1, 1, 1, 4, 2, 32, 32) == 0
    assert lib.clarus_hip_linear_attention_workspace(1, 1 << 62, 1000, 4, 4, 32, 32) == 0


def test_oracle():
    from oracle.torch_ref import TorchRef
    q, k, v, s = inputs(2, 37, 6, 3, 16, 24, torch.float32, "cpu")
    check(TorchRef(torch.float32, "cpu").linear_attention(q, k, v, decays(3, "cpu"), 6, 3, s), q, k, v, decays(3, "cpu"), 6, 3, s)


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


SHAPES = [(1, 1, 1, 1, 8, 8), (64, 1, 16, 8, 128, 128), (3, 2, 4, 4, 64, 64), (1, 5, 4, 2, 48, 96), (2, 16, 8, 2, 128, 40), (1, 17, 2, 2, 32, 32),
          (2, 31, 1, 1, 64, 8), (1, 32, 3, 3, 96, 64), (1, 33, 4, 4, 128, 128), (2, 63, 6, 2, 64, 64), (1, 64, 2, 1, 40, 72), (3, 65, 2, 2, 64, 96),
          (1, 127, 8, 8, 16, 128), (1, 128, 2, 2, 128, 32), (2, 129, 2, 2, 24, 24), (1, 300, 8, 8, 64, 64), (2, 501, 4, 1, 80, 112),
          (1, 1537, 3, 3, 64, 64), (1, 2200, 1, 1, 128, 128), (5, 70, 8, 8, 56, 120), (9, 11, 2, 2, 32, 32), (64, 20, 16, 8, 128, 64), (128, 21, 8, 8, 128, 128),
          (8200, 40, 8, 4, 24, 8), (34, 600, 8, 8, 32, 64), (1 << 16, 24, 4, 4, 8, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,l,heads,kv_heads,dk,dv", SHAPES)
def test_shapes(n, l, heads, kv_heads, dk, dv, dt, hips, gpu_device):
    q, k, v, s = inputs(n, l, heads, kv_heads, dk, dv, dt, gpu_device, seed=l)
    g = decays(kv_heads, gpu_device)
    for state in (None, s):
        for odt in (torch.bfloat16, torch.float32):
            print(f"[la] {n} {l} {heads} {kv_heads} {dk} {dv} {dt} {odt}", flush=True)
            got = hips[dt].linear_attention(q, k, v, g, heads, kv_heads, state, out_dtype=odt)
            torch.cuda.synchronize()
            print(f"[la] {_lib.last_kernel()}", flush=True)
            assert got[0].dtype == odt
            check(got, q, k, v, g, heads, kv_heads, state, what=f"{odt}")


def in_pieces64(q, k, v, log_decay, heads, kv_heads, state, size=1000, before=63):
    """plain64 of a long sequence, a piece at a time from the state of the piece before (and the size of it)."""
    zero = torch.zeros(q.shape[0], kv_heads, q.shape[-1] // heads, v.shape[-1] // kv_heads, dtype=torch.float64, device=q.device)
    s, a = (zero, zero) if state is None else (state.double(), state.double().abs())
    outs = []
    for i in range(0, q.shape[1], size):
        at = slice(i, i + size)
        out, _, _, s, _ = plain64(q[:, at], k[:, at], v[:, at], log_decay, heads, kv_heads, s)
        big, _, _, a, _ = plain64(q[:, at].abs(), k[:, at].abs(), v[:, at].abs(), log_decay, heads, kv_heads, a)
        m = min(i, before)  # the tokens within 64 of the piece's first ones
        wide = slice(i - m, i + size)
        near = plain64(q[:, wide], k[:, wide], v[:, wide], log_decay, heads, kv_heads)[2][:, m:]
        outs.append((out, big, near))
    return [torch.cat(t, 1) for t in zip(*outs)] + [s, a]


def test_pieces_are_the_whole():
    q, k, v, s = inputs(2, 301, 4, 2, 16, 24, torch.float32, "cpu")
    for state in (None, s):
        for a, b in zip(in_pieces64(q, k, v, decays(2, "cpu"), 4, 2, state, 90), plain64(q, k, v, decays(2, "cpu"), 4, 2, state)):
            assert (a - b).abs().max() <= 1e-12 * b.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,l,heads,kv_heads,dk,dv,segments", [(1, 5003, 4, 4, 40, 40, 79), (1, 20011, 4, 4, 40, 40, 209), (1, 20011, 1, 1, 64, 96, 313),
                                                               (2, 6031, 8, 4, 48, 32, 95), (1, 40013, 2, 1, 128, 24, 626)])
def test_many_segments(n, l, heads, kv_heads, dk, dv, segments, dt, hips, gpu_device):
    """More segments than 64, which groups of threads chain together, and more than 128, which they take in several rounds; none a
    multiple of 128, and lengths that are padded in front."""
    q, k, v, s = inputs(n, l, heads, kv_heads, dk, dv, dt, gpu_device, seed=l)
    g = torch.tensor([0.0, -1e-4, -1 / 64, -0.5])[:kv_heads].to(gpu_device)
    for state in (None, s):
        out, last = hips[dt].linear_attention(q, k, v, g, heads, kv_heads, state, out_dtype=torch.float32)
        torch.cuda.synchronize()
        print(f"[la] {l} {dt} {_lib.last_kernel()}", flush=True)
        assert f"segments={segments} " in _lib.last_kernel()
        ref, big, near, rlast, slast = in_pieces64(q, k, v, g, heads, kv_heads, state)
        m = (l / 4 + dk + 150) * U
        tol = m * big + (2.0 ** -8 * near + 2.0 ** -14 * big if dt == torch.bfloat16 else 0) + U * ref.abs()
        for name, t, r, e in (("out", out, ref, tol), ("state", last, rlast, m * slast)):
            off = (t.double() - r).abs()
            assert (off <= e).all(), f"{name}: max|d| {off.max().item():.3e}, {(off - e).max().item():.3e} past the tolerance"
        again = hips[dt].linear_attention(q, k, v, g, heads, kv_heads, state, out_dtype=torch.float32)
        assert torch.equal(again[0], out) and torch.equal(again[1], last)
    held = s.clone()
    over, same = hips[dt].linear_attention(q, k, v, g, heads, kv_heads, held, state_out=held, out_dtype=torch.float32)
    assert same is held and torch.equal(held, last) and torch.equal(over, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_in_pieces(dt, hips, gpu_device):
    """A sequence in pieces, the state written over itself, against the whole."""
    heads, kv, dk, dv = 4, 2, 64, 48
    q, k, v, s = inputs(2, 400, heads, kv, dk, dv, dt, gpu_device)
    g = decays(kv, gpu_device)
    state, outs, at = s.clone(), [], 0
    for size in (1, 100, 3, 200, 0, 64, 1, 31):
        sl = slice(at, at + size)
        out, same = hips[dt].linear_attention(q[:, sl], k[:, sl], v[:, sl], g, heads, kv, state, state_out=state)
        assert same is state
        outs.append(out)
        at += size
    check((torch.cat(outs, 1), state), q, k, v, g, heads, kv, s)


@pytest.mark.gpu
def test_a_state_does_not_drift(hips, gpu_device):
    """Twenty thousand single tokens under a decay that fp32 rounds: a state only scaled, then against exp in 64 bits. Each
    step rounds once, up or down; the factor's own rounding (up to 2^-25 each step, 6e-4 in all) would show."""
    g = torch.tensor([-1.0 / 30000], device=gpu_device)
    state = torch.linspace(1, 2, 64, device=gpu_device).reshape(1, 1, 8, 8).contiguous()
    first = state.double()
    z = torch.zeros(1, 1, 8, device=gpu_device)
    for _ in range(20000):
        hips[torch.float32].linear_attention(z, z, z, g, 1, state=state, state_out=state)
    want = first * torch.exp(20000 * g.double())
    # 20000 roundings of half a step at most, of signs that the values decide: within 16 standard deviations (of 0.29 steps each)
    assert ((state.double() - want).abs() <= 16 * 0.29 * math.sqrt(20000) * 2 * U * first).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,d,l", [(2100, 8, 20000), (520, 128, 10000)])
def test_a_segment_does_not_drift(n, d, l, dt, hips, gpu_device):
    """States only scaled, chunk after chunk of one segment: the last token's outputs against exp in 64 bits. Each chunk rounds a
    state, up or down as its value decides, so the mean over n d states (16 800 or more, 625 roundings of 0.29 steps each) is off by 0.6 u
    at 5 deviations; its factor must not round to the same side again and again. Left are a step of the factors together,
    2 u |x| a chunk of the exponent x and, with bf16, the state's two parts (2^-17, as random: 2 u at 5 deviations)."""
    z = torch.zeros(1, l, d, dtype=dt, device=gpu_device)
    q = z.clone()
    q[:, -1, 0] = 1
    state = torch.linspace(1, 2, n * d * d, device=gpu_device).reshape(n, 1, d, d).contiguous()
    for time in (45000, 30000, 7000):
        g = torch.tensor([-1.0 / time], device=gpu_device)
        out, _ = hips[dt].linear_attention(q.expand(n, l, d), z.expand(n, l, d), z.expand(n, l, d), g, 1, state=state, scale=1.0, out_dtype=torch.float32)
        assert "segments=1 " in _lib.last_kernel()
        want = state[:, 0, 0].double() * torch.exp(l * g.double())
        off = ((out[:, -1].double() - want) / want).mean().abs().item()
        assert off <= (4 + 2 * l / time) * U, f"{time}: {off / U:.1f} u"


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("l", [3, 54])
def test_layouts(l, dt, hips, gpu_device):
    """Slices of wider rows, NHWC rows, images shared by stride 0, one token of [N, C], decays of another type."""
    heads, d = 3, 32
    c = heads * d
    wide = torch.randn(4, l, 9, 4 * c, generator=torch.Generator().manual_seed(1)).to(dt).to(gpu_device)
    g = decays(heads, gpu_device)
    hip = hips[dt]
    for what, q, k, v in (("slices", wide[..., :c], wide[..., c:2 * c], wide[..., 2 * c:3 * c]),
                          ("images", wide[::2, ..., c:2 * c], wide[1::2, ..., :c], wide[2:, ..., 3 * c:]),
                          ("a column", wide[:, :, 4, :c], wide[:, :, 2, c:2 * c], wide[:, :, 7, :c]),
                          ("shared", wide[..., :c], wide[:1, ..., c:2 * c].expand(4, l, 9, c), wide[:1, ..., :c].expand(4, l, 9, c)),
                          ("one token", wide[:, 0, 0, :c], wide[:, 0, 1, :c], wide[:, 1, 0, c:2 * c])):
        print(f"[la] {what} {l} {dt}", flush=True)
        check(hip.linear_attention(q, k, v, g, heads), q, k, v, g, heads, what=what)
        check(hip.linear_attention(q, k, v, g.to(torch.float64), heads, scale=-0.3), q, k, v, g, heads, scale=-0.3, what=what)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_what_is_not_finite_stays_behind(dt, hips, gpu_device):
    """A query that is not finite stays in its row; a key that is not, behind its token; a head's, in its head."""
    heads, d, l = 2, 64, 200
    q, k, v, s = inputs(1, l, heads, heads, d, d, dt, gpu_device)
    g = decays(heads, gpu_device)
    want, wlast = hips[dt].linear_attention(q, k, v, g, heads, state=s)
    qb = q.clone()
    qb[0, 77, 5] = math.nan
    got, last = hips[dt].linear_attention(qb, k, v, g, heads, state=s)
    assert torch.isnan(got[0, 77, :d]).all() and torch.equal(last, wlast)
    got[0, 77, :d] = want[0, 77, :d]
    assert torch.equal(got, want)
    kb = k.clone()
    kb[0, 90, d + 3] = math.inf
    got, last = hips[dt].linear_attention(q, kb, v, g, heads, state=s)
    assert torch.equal(got[..., :d], want[..., :d]) and torch.equal(got[:, :90], want[:, :90]) and torch.equal(last[:, 0], wlast[:, 0])
    assert not torch.isfinite(got[0, 90:, d:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 104, 128])
def test_a_value_that_is_not_finite_stays_behind_its_token(d, dt, hips, gpu_device):
    """No output before it sees it, also in the chunk that holds it; from it on that column's are not finite."""
    heads, kv_heads, l = 4, 2, 333
    q, k, v, s = inputs(1, l, heads, kv_heads, d, d, dt, gpu_device)
    g = torch.tensor([-1 / 16, 0.0], device=gpu_device)
    want, wlast = hips[dt].linear_attention(q, k, v, g, heads, kv_heads, state=s)
    for token, column, value in ((0, 3, math.nan), (200, d - 1, math.inf), (331, 17, -math.inf), (332, 0, math.nan), (301, d + 5, math.inf)):
        vb = v.clone()
        vb[0, token, column] = value
        got, last = hips[dt].linear_attention(q, k, vb, g, heads, kv_heads, state=s)
        h, c = divmod(column, d)
        hit = torch.zeros(l, heads, d, dtype=torch.bool, device=gpu_device)
        hit[token:, 2 * h:2 * h + 2, c] = True
        assert torch.equal(torch.isfinite(got).view(l, heads, d), ~hit), (token, column, value)
        assert torch.equal(got.view(l, heads, d)[~hit], want.view(l, heads, d)[~hit]), (token, column, value)
        other = torch.ones(kv_heads, d, dtype=torch.bool, device=gpu_device)
        other[h, c] = False
        assert torch.equal(torch.isfinite(last[0]), other[:, None].expand(kv_heads, d, d)), (token, column, value)
        assert torch.equal(last[0].transpose(1, 2)[other], wlast[0].transpose(1, 2)[other])


@pytest.mark.gpu
def test_offsets_past_32_bits(hips, gpu_device):
    """Rows 2^21 elements apart, the last ones past 2^31."""
    l, heads, d = 1100, 2, 32
    q, k, v, s = inputs(1, l, heads, heads, d, d, torch.bfloat16, gpu_device)
    buf = torch.empty(1, l, 1 << 21, dtype=torch.bfloat16, device=gpu_device)
    buf[..., :64], buf[..., 64:128], buf[..., 192:256] = q, k, v
    g = decays(heads, gpu_device)
    got = hips[torch.bfloat16].linear_attention(buf[..., :64], buf[..., 64:128], buf[..., 192:256], g, heads, state=s)
    for a, b in zip(got, hips[torch.bfloat16].linear_attention(q, k, v, g, heads, state=s)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("l", [1, 500])
def test_repeatable_streams_and_graph(l, hips, gpu_device):
    hip, g = hips[torch.bfloat16], decays(4, gpu_device)
    a, b = (inputs(2, l, 4, 4, 64, 64, torch.bfloat16, gpu_device, seed=s) for s in (1, 2))

    def call(t):
        return hip.linear_attention(*t[:3], g, 4, state=t[3])
    ref = [call(t) for t in (a, b)]
    torch.cuda.synchronize()
    s, outs = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(4):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                outs.append(call(t))
    torch.cuda.synchronize()
    assert all(torch.equal(o[j], ref[i % 2][j]) for i, o in enumerate(outs) for j in (0, 1))
    made = []
    for t in (a, b):
        st = [x.clone() for x in t]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(st)
        made.append((graph, st, y))
    for i in range(6):
        graph, st, y = made[i % 2]
        for dst, src in zip(st, (a, b)[(i // 2) % 2]):
            dst.copy_(src)
        graph.replay()
        eager = call(b)
        torch.cuda.synchronize()
        assert all(torch.equal(y[j], ref[(i // 2) % 2][j]) and torch.equal(eager[j], ref[1][j]) for j in (0, 1)), i


@pytest.mark.gpu
def test_served_through_the_chain(gpu_device):
    ops = Ops(["hip"], torch.bfloat16, gpu_device, log=print)
    q, k, v, s = inputs(1, 40, 2, 2, 32, 32, torch.bfloat16, gpu_device)
    check(ops.linear_attention(q, k, v, decays(2, gpu_device), 2, state=s), q, k, v, decays(2, gpu_device), 2, state=s)
    assert ops.report()["ops"]["linear_attention"] == {"hip": 1}
