"""sparse_attention and block_means: the HIP kernels against the definition in 64 bits. The choice of blocks has to be equal
(its scores are 64-bit products; the inputs have no two that close but equal ones, which go to the lowest index). Tolerances of the
attention over the chosen keys, u = 2^-24, p the exact weights: as cross_attention's,
  scores     d + 8 roundings, each at most u of scale |q| . |k|: 2 (d + 8) u A (p @ |v|), A a row's largest scale |q| . |k|
  sums       at most lk + 16 additions, u of (p @ |v|) each, in the numerator and in the sum
  bf16       each weight rounded once, 2^-8 of itself; the output once: 2^-8 |o|
Means: 64-bit sums of at most 2^20 terms (2^-32 of their sizes left), rounded once to fp32: u.
"""
from __future__ import annotations

import math

import pytest
import torch

from clarus_amd import _lib
from clarus_amd.dispatch import Ops, Unsupported

U = 2.0 ** -24


def means64(k, block, mask=None):
    """fp32 means of the kept rows of each block, NaN for none."""
    n, lk, c = k.shape
    nb = -(-lk // block)
    out = torch.full((n, nb, c), math.nan, device=k.device)
    for b in range(nb):
        rows = k[:, b * block:(b + 1) * block].double()
        keep = torch.ones(rows.shape[:2], dtype=torch.bool, device=k.device) if mask is None else mask[:, b * block:(b + 1) * block]
        total = torch.where(keep[..., None], rows, torch.zeros_like(rows)).sum(1)
        out[:, b] = (total / keep.sum(1)[:, None]).float()
    return out


def choice64(q, means, heads, kv_heads, group, top):
    """bool [n, heads, groups, nb]"""
    n, lq, c = q.shape
    d, rep = c // heads, heads // kv_heads
    asks = q.double() if group == 1 else torch.stack([t.double().mean(1) for t in q.split(group, 1)], 1).float().double()
    asks = asks.reshape(n, -1, heads, d).permute(0, 2, 1, 3).contiguous()
    m = means.double().reshape(n, -1, kv_heads, d).permute(0, 2, 3, 1).repeat_interleave(rep, 1).contiguous()
    score = asks @ m
    score = torch.where(score > -math.inf, score, torch.full_like(score, -math.inf))
    order = score.sort(dim=-1, descending=True, stable=True)[1][..., :top]
    return torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True) & (score > -math.inf)


def choice_of_copies(q, means, heads, top):
    """choice64 of a head for each kv head and groups of one, every block's products added in the same order: a large matrix product
    adds in an order that differs from tile to tile, so that copies of a block differ in their last bit."""
    d = q.shape[-1] // heads
    out = []
    for h in range(heads):
        a, m = q[..., h * d:(h + 1) * d].double(), means[..., h * d:(h + 1) * d].double()
        score = torch.cat([(t[:, :, None] * m[:, None]).sum(-1) for t in a.split(256, 1)], 1)
        score = torch.where(score > -math.inf, score, torch.full_like(score, -math.inf))
        order = score.sort(dim=-1, descending=True, stable=True)[1][..., :top]
        out.append(torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True) & (score > -math.inf))
    return torch.stack(out, 1)


def attend64(q, k, v, heads, kv_heads, chosen, block, group, mask=None, scale=None):
    """(o, p @ |v|, A), float64, over the chosen blocks' kept keys."""
    n, lq, c = q.shape
    lk, d, rep = k.shape[1], c // heads, heads // kv_heads
    if mask is not None:
        k, v = (torch.where(mask[..., None], t, torch.zeros_like(t)) for t in (k, v))
    outs = []
    for h in range(heads):
        kv = slice(h // rep * d, h // rep * d + d)
        qh, kt, vh = q[..., h * d:(h + 1) * d].double(), k[..., kv].double().transpose(1, 2).contiguous(), v[..., kv].double()
        see = chosen[:, h].repeat_interleave(group, 1)[:, :lq].repeat_interleave(block, 2)[..., :lk]
        see = see if mask is None else see & mask[:, None]
        sc = d ** -0.5 if scale is None else scale
        s = (qh @ kt * sc).masked_fill(~see, -math.inf)
        big = (qh.abs() @ kt.abs() * sc * see).amax(-1, keepdim=True)
        top = s.amax(-1, keepdim=True)
        p = (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        outs.append((p @ vh, p @ vh.abs(), big.expand(n, lq, d)))
    return [torch.stack(t, 2).reshape(q.shape) for t in zip(*outs)]


def check(hip, q, k, v, heads, top, kv_heads=None, block=64, group=1, mask=None, means=None, scale=None, out_dtype=None, what=""):
    kv = kv_heads or heads
    got, chosen = hip.sparse_attention(q, k, v, heads, top, kv_heads, block, group, mask, means, scale, out_dtype, return_blocks=True)
    torch.cuda.synchronize()
    flat = [t.reshape(t.shape[0], -1, t.shape[-1]) for t in (q, k, v)]
    want = choice64(flat[0], means64(flat[1], block, mask) if means is None else means, heads, kv, group, top)
    assert torch.equal(chosen, want), f"{what}: {(chosen != want).any(-1).sum().item()} choices of {want[..., 0].numel()} differ"
    ref, pv, big = attend64(*flat, heads, kv, want, block, group, mask, scale)
    assert got.shape == q.shape and got.is_contiguous() and torch.isfinite(got).all(), what
    d, lk = q.shape[-1] // heads, flat[1].shape[1]
    tol = (2 * (d + 8) * U * big + 2 * (lk + 16) * U + (2.0 ** -8 if q.dtype == torch.bfloat16 else 0)) * pv
    tol = tol + (2.0 ** -8 if got.dtype == torch.bfloat16 else U) * ref.abs()
    off = (got.reshape(ref.shape).double() - ref).abs()
    assert (off <= tol).all(), f"{what}: max|d| {off.max().item():.3e}, {(off - tol).max().item():.3e} past the tolerance"
    again = hip.sparse_attention(q, k, v, heads, top, kv_heads, block, group, mask, means, scale, out_dtype)
    assert torch.equal(got, again), what
    return got, chosen


def inputs(n, lq, lk, heads, kv_heads, d, dt, dev, seed=0):
    g = torch.Generator().manual_seed(seed)

    def tokens(length, h, size):  # neighbours alike, as along a map
        coarse = (torch.randn(n, -(-length // 40), h * d, generator=g) * size).repeat_interleave(40, 1)[:, :length]
        return (coarse + 0.6 * torch.randn(n, length, h * d, generator=g)).to(dt).to(dev)
    return tokens(lq, heads, 1.2), tokens(lk, kv_heads, 0.8), torch.randn(n, lk, kv_heads * d, generator=g).to(dt).to(dev)


def make_mask(n, lk, dev, seed=0):
    """Ragged keys with holes, the last image without any."""
    g = torch.Generator().manual_seed(seed + 1)
    m = torch.rand(n, lk, generator=g) < 0.7
    for i in range(n):
        m[i, lk - lk * i // n:] = False
    if n > 1:
        m[-1] = False
    return m.to(dev)


# ------------------------------------------------------------------ CPU
def cpu_hip(dtype=torch.float32):
    from clarus_amd.hip_ops import HipOps
    h = HipOps.__new__(HipOps)
    h.dtype, h.device, h.dev, h._cache, h._plans = dtype, torch.device("cpu"), torch.device("cpu"), {}, {}
    h.lib = _lib.load()
    return h


def test_refusals():
    h, z = cpu_hip(), torch.zeros
    q, k = z(2, 5, 64), z(2, 7, 64)
    cases = [
        ((z(2, 5, 60), z(2, 7, 60), z(2, 7, 60), 5, 1), {}), ((z(2, 5, 136), z(2, 7, 136), z(2, 7, 136), 1, 1), {}), ((q, k, k, 3, 1), {}),
        ((q, k, k, 0, 1), {}), ((q, k, k, 2.0, 1), {}), ((q, k, k, 4, 1), {"kv_heads": 3}), ((q, k, k, 4, 1), {"kv_heads": 2}),
        ((q, k, z(2, 8, 64), 4, 1), {}), ((q, z(1, 7, 64), z(1, 7, 64), 4, 1), {}), ((q, k, k, 4, 0), {}), ((q, k, k, 4, 1.0), {}),
        ((q, k, k, 4, 1), {"block": 32}), ((q, k, k, 4, 1), {"block": 100}), ((q, k, k, 4, 1), {"block": 64.0}),
        ((q, k, k, 4, 1), {"block": 1 << 20}), ((q, k, k, 4, 1), {"group": 0}), ((q, k, k, 4, 1), {"group": 1.0}),
        ((q, k, k, 4, 1), {"scale": 0.0}), ((q, k, k, 4, 1), {"scale": math.inf}), ((q, k, k, 4, 1), {"scale": math.nan}),
        ((q, k, k, 4, 1), {"out_dtype": torch.float16}), ((q.half(), k.half(), k.half(), 4, 1), {}), ((q, k.bfloat16(), k.bfloat16(), 4, 1), {}),
        ((q, k, k, 4, 1), {"mask": z(2, 7)}), ((q, k, k, 4, 1), {"mask": z(2, 5, 7, dtype=torch.bool)}),
        ((q, k, k, 4, 1), {"mask": z(7, 2, dtype=torch.bool).t()}), ((q, k, k, 4, 1), {"means": z(2, 2, 64)}),
        ((q, k, k, 4, 1), {"means": z(2, 1, 64).bfloat16()}), ((q, k, k, 4, 1), {"means": z(2, 1, 128)[..., ::2]}),
        ((z(2, 64, 5).transpose(1, 2), k, k, 4, 1), {}), ((q, z(2, 3, 4, 64).transpose(1, 2), z(2, 4, 3, 64), 4, 1), {}),
        ((z(2, 5, 65)[..., 1:], k, k, 4, 1), {}), ((z(64), k, k, 4, 1), {}), ((q.clone().requires_grad_(), k, k, 4, 1), {}),
        ((q, k, k, 4, 1), {"means": z(2, 1, 64).requires_grad_()}),
        ((z(1, 1, 8).expand(1 << 16, 1, 8), z(1, 1, 8).expand(1 << 16, 1, 8), z(1, 1, 8).expand(1 << 16, 1, 8), 1, 1), {}),
        ((z(1, 1, 8), z(1, 1, 8).expand(1, 1 << 27, 8), z(1, 1, 8).expand(1, 1 << 27, 8), 1, 1), {}),
        ((z(1, 1, 8).expand(1, 1 << 24, 8), z(1, 1, 8), z(1, 1, 8), 1, 1), {"group": 2}),
    ]
    for i, (args, kw) in enumerate(cases):
        with pytest.raises(Unsupported):
            h.sparse_attention(*args, **kw)
            pytest.fail(f"case {i} was accepted")
    for args, kw in (((z(2, 7, 60),), {}), ((k, 65), {}), ((k, 64.0), {}), ((k.half(),), {}), ((z(2, 64, 7).transpose(1, 2),), {}),
                     ((k,), {"mask": z(2, 7)}), ((k,), {"mask": z(1, 7, dtype=torch.bool)}), ((z(64),), {}), ((k.clone().requires_grad_(),), {})):
        with pytest.raises(Unsupported):
            h.block_means(*args, **kw)
    assert h.block_means(z(2, 0, 64)).shape == (2, 0, 64)


def test_nothing_to_attend_or_to_ask_cpu():
    h = cpu_hip()
    q, k = torch.ones(2, 3, 64), torch.zeros(2, 0, 64)
    out, blocks = h.sparse_attention(q, k, k, 4, 2, return_blocks=True)
    assert not out.any() and blocks.shape == (2, 4, 3, 0)
    out, blocks = h.sparse_attention(q[:, :0], q, q, 4, 2, group=8, return_blocks=True)
    assert out.shape == (2, 0, 64) and blocks.shape == (2, 4, 0, 1)


def test_c_entry_refuses_before_launch():
    import ctypes
    lib = _lib.load()

    def call(scratch=1 << 30, size=1 << 40, **kw):
        base = dict(q=1 << 20, k=1 << 21, v=1 << 22, out=1 << 23, n=1, lq=64, lk=640, heads=4, kv_heads=2, d=32, top=4, block=64, group=8,
                    ldq=128, ldk=64, ldv=64, dtype=0, o_dtype=0, scale=0.2)
        return lib.clarus_hip_sparse_attention(ctypes.byref(_lib.SparseArgs(**{**base, **kw})), scratch, size, None)
    assert lib.clarus_hip_sparse_attention(None, None, 0, None) == _lib.EINVAL
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(n=0), dict(lq=0), dict(lk=0), dict(heads=0), dict(kv_heads=0),
               dict(kv_heads=3), dict(d=0), dict(d=12), dict(d=136), dict(top=0), dict(top=-1), dict(block=0), dict(block=32), dict(block=96),
               dict(block=1 << 20), dict(group=0), dict(dtype=2), dict(o_dtype=-1), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf),
               dict(ldq=130), dict(q=(1 << 20) + 8), dict(ldk=-64), dict(k_bstride=2), dict(ldv=1 << 24), dict(mask_bstride=-1), dict(means=8),
               dict(chosen=4), dict(lk=1 << 31), dict(lq=1 << 31), dict(n=1 << 15), dict(n=1 << 62), dict(heads=1 << 62), dict(lk=1 << 30),
               dict(n=1 << 60, kv_heads=16, heads=16), dict(scratch=None), dict(size=16), dict(scratch=8)):
        assert call(**kw) == _lib.EINVAL, kw
        assert b"sparse_attention" in lib.clarus_hip_last_error()
    ws = lib.clarus_hip_sparse_attention_workspace
    assert ws(0, 1, 64, 640, 4, 2, 32, 4, 64, 8, 0, 0) > 0 and ws(0, 1, 64, 640, 4, 3, 32, 4, 64, 8, 0, 0) == 0
    assert ws(0, 1 << 62, 64, 640, 4, 4, 32, 4, 64, 8, 0, 0) == 0

    def means(k=1 << 20, dtype=0, kbs=0, ldk=64, mask=None, mbs=0, out=1 << 21, n=1, lk=640, c=64, block=64):
        return lib.clarus_hip_block_means(k, dtype, kbs, ldk, mask, mbs, out, n, lk, c, block, None)
    for kw in (dict(k=None), dict(out=None), dict(n=0), dict(lk=0), dict(c=0), dict(c=12), dict(block=0), dict(dtype=2), dict(k=8), dict(out=8),
               dict(ldk=66), dict(ldk=-64), dict(kbs=2), dict(mbs=-1), dict(n=1 << 23), dict(n=1 << 62), dict(lk=1 << 31), dict(lk=1 << 30),
               dict(c=1 << 20)):
        assert means(**kw) == _lib.EINVAL, kw
        assert b"block_means" in lib.clarus_hip_last_error()


def test_oracle():
    from oracle.torch_ref import TorchRef
    q, k, v = inputs(3, 150, 333, 4, 2, 16, torch.float32, "cpu")
    mask, ref = make_mask(3, 333, "cpu"), TorchRef(torch.float32, "cpu")
    got, chosen = ref.sparse_attention(q, k, v, 4, 2, 2, 64, 8, mask, return_blocks=True)
    want = choice64(q, means64(k, 64, mask), 4, 2, 8, 2)
    assert torch.equal(chosen, want)
    assert (got.double() - attend64(q, k, v, 4, 2, want, 64, 8, mask)[0]).abs().max() < 1e-5


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def hips(gpu_device):
    from clarus_amd.hip_ops import HipOps
    return {dt: HipOps(dt, gpu_device) for dt in (torch.bfloat16, torch.float32)}


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_block_means(dt, hips, gpu_device):
    for n, lk, c, block in ((1, 1, 8, 64), (2, 64, 40, 64), (3, 1000, 512, 128), (2, 333, 2056, 64), (1, 70000, 64, 1024), (2, 129, 24, 4096)):
        k = torch.randn(n, lk, c, generator=torch.Generator().manual_seed(lk)).to(dt).to(gpu_device)
        for mask in (None, make_mask(n, lk, gpu_device)):
            got, want = hips[dt].block_means(k, block, mask), means64(k, block, mask)
            assert torch.equal(got.isnan(), want.isnan())
            off = (got.double() - want.double()).abs()
            assert (off.nan_to_num() <= 2 * U * want.double().abs().nan_to_num() + 2.0 ** -32 * 5).all(), (n, lk, c, block)
            if mask is not None:
                bad = k.masked_fill(~mask[..., None], math.nan)
                assert torch.equal(hips[dt].block_means(bad, block, mask).nan_to_num(-7), got.nan_to_num(-7))


SHAPES = [  # n, lq, lk, heads, kv_heads, d, top, block, group
    (1, 1, 1, 1, 1, 8, 1, 64, 1), (2, 1, 300, 4, 4, 32, 2, 64, 1), (8, 1, 3001, 16, 4, 128, 5, 64, 1), (1, 5, 9000, 8, 2, 64, 7, 128, 1),
    (1, 300, 300, 2, 2, 64, 2, 64, 1), (2, 257, 700, 8, 2, 80, 3, 64, 64), (1, 130, 64, 3, 1, 64, 4, 64, 16), (1, 1000, 1000, 4, 4, 48, 4, 64, 100),
    (3, 97, 640, 1, 1, 112, 3, 128, 8), (1, 2000, 2500, 2, 2, 64, 6, 64, 256), (2, 33, 129, 6, 2, 24, 1, 64, 7), (1, 64, 4200, 4, 1, 96, 40, 64, 2),
    (1, 300, 130, 1, 1, 16, 9, 64, 1000), (4, 3, 31, 32, 1, 128, 1, 64, 1), (1, 700, 5000, 2, 1, 40, 8, 256, 1), (1, 40, 70000, 2, 2, 32, 12, 64, 4), (1, 3001, 3001, 2, 2, 64, 3, 1024, 5000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d,top,block,group", SHAPES)
def test_shapes(n, lq, lk, heads, kv_heads, d, top, block, group, dt, hips, gpu_device):
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, dt, gpu_device, seed=lq + lk)
    for mask in (None, make_mask(n, lk, gpu_device)):
        print(f"[sparse] {n} {lq} {lk} {heads} {kv_heads} {d} {top} {block} {group} {dt} {mask is not None}", flush=True)
        got, chosen = check(hips[dt], q, k, v, heads, top, kv_heads, block, group, mask, what=str(mask is not None))
        print(f"[sparse] {_lib.last_kernel()}", flush=True)
        if mask is not None and n > 1:
            assert not got[-1].any() and not chosen[-1].any()
        means = hips[dt].block_means(k, block, mask)
        check(hips[dt], q, k, v, heads, top, kv_heads, block, group, mask, means, out_dtype=torch.float32, what="kept means")


# Enough rows that every CU has a workgroup without splitting the blocks (more than 256 of rows): 2, 4 and 1 waves, the finished
# rows stored by the kernel itself
UNSPLIT = [  # n, lq, lk, heads, kv_heads, d, top, block, group
    (2, 1201, 4470, 8, 8, 32, 9, 64, 1), (2, 1201, 4470, 8, 8, 64, 20, 64, 64), (2, 2101, 4470, 8, 8, 48, 40, 64, 256),
    (40, 3, 2500, 8, 8, 104, 12, 64, 1), (1, 2301, 70390, 8, 8, 16, 40, 64, 1), (1, 4203, 9000, 4, 4, 72, 17, 128, 1),
    (3, 1003, 4100, 12, 4, 64, 5, 64, 100), (2, 1077, 3000, 8, 8, 128, 33, 64, 7), (1, 5001, 5001, 8, 8, 64, 50, 64, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,lq,lk,heads,kv_heads,d,top,block,group", UNSPLIT)
def test_rows_that_fill_the_gpu(n, lq, lk, heads, kv_heads, d, top, block, group, dt, hips, gpu_device):
    q, k, v = inputs(n, lq, lk, heads, kv_heads, d, dt, gpu_device, seed=lq + lk)
    for mask in (None, make_mask(n, lk, gpu_device)):
        print(f"[sparse] {n} {lq} {lk} {heads} {kv_heads} {d} {top} {block} {group} {dt} {mask is not None}", flush=True)
        got, _ = check(hips[dt], q, k, v, heads, top, kv_heads, block, group, mask, what=str(mask is not None))
        print(f"[sparse] {_lib.last_kernel()}", flush=True)
        assert _lib.last_kernel().endswith("splits=1")
        assert mask is None or n == 1 or not got[-1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,nb", [(16, 70), (16, 300), (64, 1000), (72, 70), (72, 130), (128, 300), (128, 1000)])
def test_choices_of_many_rows(d, nb, dt, hips, gpu_device):
    """528 tiles of 32 rows, for which a wave holds the scores of 256 blocks (heads past 64: 128). Means kept by the caller: copies of
    each other, NaN, infinite, and some that differ in their last bits, a head each; queries of zeros."""
    g = torch.Generator().manual_seed(nb + d)
    heads, lq, lk = 4, 4200, 64 * nb - 13
    q = torch.randn(1, lq, heads * d, generator=g).to(dt)
    means = torch.randn(1, nb, heads, d, generator=g)
    means[:, 5::9, 0] = means[:, 6:7, 0]
    means[:, 3::17, 1] = math.nan
    means[:, 11, 2, 5], means[:, nb - 2, 2, 0] = math.inf, -math.inf
    base = means[:, :1, 3].clone()
    means[:, :, 3] = base + 2.0 ** -22 * torch.randint(-3, 4, (1, nb, d), generator=g) * base.abs()
    q[:, ::50] = 0
    q, means = q.to(gpu_device), means.reshape(1, nb, -1).to(gpu_device)
    k = torch.randn(1, lk, heads * d, generator=g).to(dt).to(gpu_device)
    for top in (1, 16, nb - 1):
        print(f"[sparse] choices {d} {nb} {dt} {top}", flush=True)
        want = choice_of_copies(q, means, heads, top)
        _, chosen = hips[dt].sparse_attention(q, k, k, heads, top, means=means, return_blocks=True)
        assert torch.equal(chosen, want), f"{top}: {(chosen != want).any(-1).sum().item()} choices differ"


@pytest.mark.gpu
@pytest.mark.parametrize("n,lq,nb,heads,kv_heads,group", [(1, 1, 1025, 4, 1, 1), (3, 1, 2100, 6, 2, 1), (1, 130, 4097, 2, 1, 2),
                                                          (2, 3, 8200, 2, 2, 1), (1, 16000, 1100, 2, 1, 1)])
def test_choices_of_many_blocks(n, lq, nb, heads, kv_heads, group, hips, gpu_device):
    """Means kept by the caller, some of them copies, some NaN or infinite; the last shape's scores take two turns."""
    g = torch.Generator().manual_seed(nb)
    d, lk = 8, 64 * nb - 13
    q = torch.randn(n, lq, heads * d, generator=g).to(gpu_device)
    q[:, ::11] = 0
    k, v = (torch.randn(n, lk, kv_heads * d, generator=g).to(torch.bfloat16).float().to(gpu_device) for _ in "kv")
    means = hips[torch.float32].block_means(k)
    means[:, 5::9] = means[:, 700:701]
    means[:, 64:80] = math.nan
    means[:, 130, 0] = -math.inf
    for top in (1, 7, 1000, nb - 1, nb, 1 << 30):
        want = choice64(q, means, heads, kv_heads, group, min(top, nb))
        if lq > 1000 and top > 7:  # the attention over nearly all keys would take its time
            continue
        _, chosen = hips[torch.float32].sparse_attention(q, k, v, heads, top, kv_heads, group=group, means=means, return_blocks=True)
        assert torch.equal(chosen, want), top


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_equal_scores_go_to_the_lowest_index(dt, hips, gpu_device):
    """Blocks that are copies of each other, queries of zeros, keys of zeros, scores of both signs of zero."""
    n, heads, d, lk = 1, 2, 32, 64 * 150
    q, k, v = inputs(n, 90, lk, heads, heads, d, dt, gpu_device)
    k = k.reshape(n, 150, 64, -1)
    k[:, 10::7] = k[:, 3:4]
    k[:, 77] = 0
    k = k.reshape(n, lk, -1)
    q[:, ::3] = 0
    q[:, 1::9] *= -1
    for top in (1, 3, 13, 149, 150, 400):
        for group in (1, 30):
            check(hips[dt], q, k, v, heads, top, group=group, what=f"{top} {group}")
    check(hips[dt], q, torch.zeros_like(k), v, heads, 5, what="zeros")
    check(hips[dt], q, k[:, :64].repeat(1, 150, 1), v, heads, 5, what="all the same")


@pytest.mark.gpu
def test_scores_that_fp32_does_not_tell_apart(hips, gpu_device):
    """Means that differ in their last bit, or whose products cancel to fp32's rounding: the choice is 64 bits'."""
    heads, d, nb, lq = 1, 64, 200, 120
    g = torch.Generator().manual_seed(3)
    base = torch.randn(1, 1, d, generator=g)
    means = (base + 2.0 ** -23 * torch.randint(-3, 4, (1, nb, d), generator=g) * base.abs()).to(gpu_device)
    q = (torch.randn(1, lq, d, generator=g)).to(gpu_device)
    q = q - (q @ means[:, 0, :, None]) / (means[:, 0] ** 2).sum() * means[:, :1]  # nearly at right angles to all of them
    k = means.repeat_interleave(64, 1).contiguous()
    v = torch.randn(1, nb * 64, d, generator=g).to(gpu_device)
    for dt in (torch.bfloat16, torch.float32):
        for group in (1, 5):
            check(hips[dt], q.to(dt), k.to(dt), v.to(dt), heads, 9, means=means, group=group, what=f"{dt} {group}")


@pytest.mark.gpu
@pytest.mark.parametrize("q_size,m_size", [(0, -80), (-80, 0), (-50, -50), (-120, 0), (0, -110), (-100, 60), (60, 60), (64, 0), (0, 70)])
@pytest.mark.parametrize("nb", [50, 200])
def test_choices_whatever_the_size_of_queries_and_means(nb, q_size, m_size, hips, gpu_device):
    """The same near ties at sizes whose squares leave fp32: a power of two changes no choice of 64 bits."""
    heads, d, lq = 1, 64, 120
    g = torch.Generator().manual_seed(4)
    base = torch.randn(1, 1, d, generator=g)
    means = (base + 2.0 ** -20 * torch.randint(-3, 4, (1, nb, d), generator=g) * base.abs()).to(gpu_device)
    q = torch.randn(1, lq, d, generator=g).to(gpu_device)
    q = q - (q @ means[:, 0, :, None]) / (means[:, 0] ** 2).sum() * means[:, :1]
    q[:, ::7] = torch.randn(1, 18, d, generator=g).to(gpu_device)  # and some that leave no doubt
    # small sizes keep all digits: nothing below 2^-126
    q = torch.where(q.abs() < 2.0 ** -4, torch.zeros_like(q), q) * 2.0 ** q_size
    means = torch.where(means.abs() < 2.0 ** -4, torch.zeros_like(means), means) * 2.0 ** m_size
    k = torch.randn(1, nb * 64, d, generator=g).to(gpu_device)
    for top in (1, 9, nb - 3):
        want = choice64(q, means, heads, heads, 1, top)
        _, chosen = hips[torch.float32].sparse_attention(q, k, k, heads, top, means=means, scale=0.1 * 2.0 ** -max(q_size, 0), return_blocks=True)
        assert torch.equal(chosen, want), f"{top}: {(chosen != want).any(-1).sum().item()} choices of {lq} differ"


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq,lk,group", [(70, 350, 1), (3, 3001, 1), (200, 900, 64)])
def test_masked_keys_may_hold_anything(lq, lk, group, dt, hips, gpu_device):
    n, heads, d = 3, 2, 48
    q, k, v = inputs(n, lq, lk, heads, heads, d, dt, gpu_device)
    mask = make_mask(n, lk, gpu_device)
    want = hips[dt].sparse_attention(q, k, v, heads, 3, group=group, mask=mask)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dt).min):
        kb, vb = (t.masked_fill(~mask[..., None], bad) for t in (k, v))
        assert torch.equal(hips[dt].sparse_attention(q, kb, vb, heads, 3, group=group, mask=mask), want), bad


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_scores_that_are_not_finite(dt, hips, gpu_device):
    """A block with a NaN key is not chosen, one whose mean is inf is where its product is inf; the rest as without."""
    heads, d = 2, 32
    q, k, v = inputs(1, 50, 64 * 9, heads, heads, d, dt, gpu_device)
    q = q.abs() + 0.5
    means = hips[dt].block_means(k)
    means[0, 4, 3] = math.nan
    means[0, 7, 5] = math.inf
    means[0, 2, 5] = -math.inf
    got, chosen = check(hips[dt], q, k, v, heads, 3, means=means)
    assert not chosen[:, 0, :, 4].any() and chosen[:, 0, :, 7].all() and not chosen[:, 0, :, 2].any()
    got, chosen = check(hips[dt], q, k, v, heads, 9, means=means)
    assert not chosen[:, 0, :, 4].any() and not chosen[:, 0, :, 2].any() and chosen[:, 1].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lq", [40, 1003, 20000])
def test_a_row_takes_nothing_from_blocks_that_only_others_have_chosen(lq, dt, hips, gpu_device):
    """Queries that are not finite have no block and are 0, whatever their neighbours chose; a product that leaves fp32 in a block
    that only the neighbours chose changes nothing."""
    heads, d, nb, dev = 2, 32, 10, gpu_device
    q, k, v = inputs(1, lq, nb * 64, heads, heads, d, dt, dev, seed=lq)
    masks = (None, torch.rand(1, nb * 64, generator=torch.Generator().manual_seed(1)).to(dev) < 0.8)

    def compare(q, k, mask, what):
        got, chosen = hips[dt].sparse_attention(q, k, v, heads, 2, mask=mask, return_blocks=True, out_dtype=torch.float32)
        want = choice64(q, means64(k, 64, mask), heads, heads, 1, 2)
        assert torch.equal(chosen, want), what
        ref, pv, big = attend64(torch.where(q.isnan(), torch.zeros_like(q), q), k, v, heads, heads, want, 64, 1, mask)
        tol = (2 * (d + 8) * U * big + 2 * (nb * 64 + 16) * U + (2.0 ** -8 if dt == torch.bfloat16 else 0)) * pv + U * ref.abs()
        assert torch.isfinite(got).all(), f"{what}: {(~torch.isfinite(got)).any(-1).sum().item()} rows of {lq} are not finite"
        assert ((got.double() - ref).abs() <= tol).all(), what
        return got, chosen
    for mask in masks:
        bad = q.clone()
        bad[0, 5::17, :d] = math.nan
        bad[0, 7::29, d + 3] = math.nan
        got, chosen = compare(bad, k, mask, "queries")
        assert not got[0, 5::17, :d].any() and not chosen[0, 0, 5::17].any() and not got[0, 7::29, d:].any()
    # queries of 2^100 meet keys of +-2^30 (mean 0) in a block that the others choose
    q, k = (q / 16).view(1, lq, heads, d), k.clone().view(1, nb, 64, heads, d)
    q[..., 0], q[..., 1], k[..., 0], k[..., 1] = 0, 6, 0, 0
    q[:, ::4, :, 0], q[:, ::4, :, 1], k[:, 3, :, :, 0], k[:, 7, :, :, 1] = 2.0 ** 100, -6, 2.0 ** -96, 5
    k[:, 7, ::2, :, 0], k[:, 7, 1::2, :, 0] = 2.0 ** 30, -2.0 ** 30
    q, k = q.view(1, lq, -1), k.view(1, nb * 64, -1)
    mask = torch.ones(1, nb * 64, dtype=torch.bool, device=dev)
    mask[0, 130:140] = mask[0, 450:452] = False  # also two keys of that block, one of each sign
    for m in (None, mask):
        _, chosen = compare(q, k, m, "products")
        assert chosen[0, :, ::4, 3].all() and not chosen[0, :, ::4, 7].any() and chosen[0, :, 1::4, 7].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dt, hips, gpu_device):
    g = torch.Generator().manual_seed(2)
    hip, heads, d = hips[dt], 2, 32
    c = heads * d
    wide = torch.randn(4, 16, 29, 3 * c, generator=g).to(dt).to(gpu_device)
    kv = torch.randn(2, 25, 17, 2 * c + 8, generator=g).to(dt).to(gpu_device)
    k, v = kv[..., :c], kv[..., c:2 * c]
    ctx = torch.randn(1, 425, 2 * c, generator=g).to(dt).to(gpu_device).expand(2, 425, 2 * c)
    big = torch.rand(4, 60, 480, generator=g).to(gpu_device) < 0.6
    for what, args, mask, group in (
            ("NHWC slices", (wide[::2, ..., c:2 * c], k, v), None, 1), ("rows of images", (wide[:2, 1:4, :, :c], k, v), None, 29),
            ("one column", (wide[2:, :, 3:4, 2 * c:], k, v), big[::2, 0, :425], 4),
            ("shared states", (wide[:2, ..., :c], ctx[..., :c], ctx[..., c:]), big[:1, 3, 5:430].expand(2, 425), 1),
            ("flat queries", (wide[:2, 3, 4, :c], k, v), big[:2, 7, 3:428], 1)):
        print(f"[sparse] {what}", flush=True)
        check(hip, *args, heads, 3, mask=mask, group=group, scale=0.3, what=what)


@pytest.mark.gpu
def test_offsets_past_32_bits(hips, gpu_device):
    """Keys and values in rows 2^19 elements apart: the last ones lie past 2^31 elements."""
    lk, heads, d = 4200, 2, 32
    buf = torch.empty(1, lk, 1 << 19, dtype=torch.bfloat16, device=gpu_device)
    for lq, group in ((1, 1), (300, 20)):
        q, k, v = inputs(1, lq, lk, heads, heads, d, torch.bfloat16, gpu_device)
        buf[..., :64], buf[..., 128:192] = k, v
        got = hips[torch.bfloat16].sparse_attention(q, buf[..., :64], buf[..., 128:192], heads, 8, group=group)
        assert torch.equal(got, hips[torch.bfloat16].sparse_attention(q, k, v, heads, 8, group=group))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_the_longest_keys(dt, hips, gpu_device):
    """2^31 - 1 keys (rows of stride 0: all the same), the last block of which ends past 2^31."""
    lk, block, d = (1 << 31) - 1, (1 << 20) - 64, 8
    q, k, v = (torch.randn(1, 1, d, generator=torch.Generator().manual_seed(i)).to(dt).to(gpu_device) for i in range(3))
    means = torch.zeros(1, -(-lk // block), d, device=gpu_device)
    means[:, -1] = q[:, 0]
    mask = torch.zeros(1, lk, dtype=torch.bool, device=gpu_device)
    mask[0, -3000:] = True
    for m in (None, mask):
        got, chosen = hips[dt].sparse_attention(q, k.expand(1, lk, d), v.expand(1, lk, d), 1, 1, block=block, means=means, mask=m, return_blocks=True)
        assert chosen[0, 0, 0].nonzero().flatten().tolist() == [means.shape[1] - 1]
        # equal weights of equal values: what their sums of up to 2^17 terms round
        assert ((got.double() - v.double()).abs() <= (2.0 ** 17 * 2 * U + (2.0 ** -7 if dt == torch.bfloat16 else 0)) * v.double().abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,group", [(400, 700, 1), (2, 3001, 1), (400, 700, 32)])
def test_repeatable_streams_and_graph(lq, lk, group, hips, gpu_device):
    hip = hips[torch.bfloat16]
    a, b = (inputs(2, lq, lk, 4, 2, 64, torch.bfloat16, gpu_device, seed=s) for s in (0, 5))
    mask = make_mask(2, lk, gpu_device)

    def call(t):
        return hip.sparse_attention(*t, 4, 3, 2, group=group, mask=mask)
    ref = [call(t) for t in (a, b)]
    torch.cuda.synchronize()
    s, outs = (torch.cuda.Stream(), torch.cuda.Stream()), []
    for _ in range(4):
        for i, t in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                outs.append(call(t))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i % 2]) for i, o in enumerate(outs))
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
        assert torch.equal(y, ref[(i // 2) % 2]) and torch.equal(eager, ref[1]), i


@pytest.mark.gpu
def test_every_block_is_cross_attention(hips, gpu_device):
    """All blocks chosen: what cross_attention answers, within both tolerances' sum (each output once rounded, weights once)."""
    for dt in (torch.bfloat16, torch.float32):
        q, k, v = inputs(2, 150, 500, 4, 2, 64, dt, gpu_device)
        a, b = hips[dt].sparse_attention(q, k, v, 4, 99, 2), hips[dt].cross_attention(q, k, v, 4, 2)
        assert (a.double() - b.double()).abs().max() <= (4 * 2.0 ** -8 if dt == torch.bfloat16 else 4 * 700 * U) * v.double().abs().max()


@pytest.mark.gpu
def test_served_through_the_chain(gpu_device):
    ops = Ops(["hip"], torch.bfloat16, gpu_device, log=print)
    q, k, v = inputs(1, 40, 200, 2, 2, 32, torch.bfloat16, gpu_device)
    assert torch.equal(ops.sparse_attention(q, k, v, 2, 2, means=ops.block_means(k)), ops.sparse_attention(q, k, v, 2, 2))
    assert ops.report()["ops"] == {"sparse_attention": {"hip": 2}, "block_means": {"hip": 1}}
