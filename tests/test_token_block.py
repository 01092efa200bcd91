"""add_norm, rotary, sparse_attention and linear_attention in a row, as a block over the tokens of a map runs them between
its products: each operator's own tolerance at each step, on what the step before it wrote (slices of the products' rows);
two blocks captured into one graph; and the same tokens in pieces.
"""
from __future__ import annotations

import pytest
import torch

from clarus_amd import spatial_torch  # noqa: F401
from clarus_amd.dispatch import Ops, Unsupported
from test_add_norm import check as check_norm
from test_linear_attention import check as check_linear
from test_rotary import check as check_rotary
from test_sparse_attention import attend64, check as check_sparse

HEADS, KV, D, C = 4, 2, 32, 128
SECTIONS, TOP, GROUP = (8, 8), 3, 17


def weights(dt, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    wide = (HEADS + 2 * KV) * D
    w = {"qkv": torch.randn(C, wide, generator=g) * C ** -0.5, "out": torch.randn(C, C, generator=g) * C ** -0.5,
         "qkv2": torch.randn(C, wide, generator=g) * C ** -0.5, "out2": torch.randn(C, C, generator=g) * C ** -0.5,
         "gate": torch.randn(2, C, generator=g), "ln": torch.rand(C, generator=g) + 0.5, "rms": torch.rand(C, generator=g) + 0.5}
    return {k: t.to(dev) if k in ("gate", "ln", "rms") else t.to(dt).to(dev) for k, t in w.items()} | {
        "decay": torch.tensor([-1 / 32, -0.2], device=dev)}


def split(qkv):
    return qkv[..., :HEADS * D], qkv[..., HEADS * D:(HEADS + KV) * D], qkv[..., (HEADS + KV) * D:]


def block(ops, x, w, state, mask, seen=None):
    """A block of sparse attention and one of linear attention; (tokens, state)."""
    def step(what, got, *args, **kw):
        if seen is not None:
            seen.append((what, got, args, kw))
        return got
    _, h = step("norm", ops.add_norm(x, weight=w["ln"]), x, None, weight=w["ln"])
    q, k, v = split(ops.linear(h, w["qkv"]))
    qr = step("rotary", ops.rotary(q, HEADS, SECTIONS), q, HEADS, SECTIONS)
    kr = step("rotary", ops.rotary(k, KV, SECTIONS), k, KV, SECTIONS)
    kw = dict(kv_heads=KV, group=GROUP, mask=mask)
    a = step("sparse", ops.sparse_attention(qr, kr, v, HEADS, TOP, **kw), qr, kr, v, HEADS, TOP, **kw)
    y = ops.linear(a, w["out"])
    kw = dict(gate=w["gate"], scale=0.5, post="rms", post_weight=w["rms"], weight=w["ln"])
    x, h = step("norm", ops.add_norm(x, y, **kw), x, y, **kw)
    q, k, v = split(ops.linear(h, w["qkv2"]))
    qr = step("rotary", ops.rotary(q, HEADS, SECTIONS, pairs="halves"), q, HEADS, SECTIONS, pairs="halves")
    kr = step("rotary", ops.rotary(k, KV, SECTIONS, pairs="halves"), k, KV, SECTIONS, pairs="halves")
    a, state = step("linear", ops.linear_attention(qr, kr, v, w["decay"], HEADS, KV, state=state), qr, kr, v, w["decay"], HEADS, KV,
                    state=state)
    y = ops.linear(a, w["out2"])
    x, _ = step("norm", ops.add_norm(x, y, gate=w["gate"], ln=False), x, y, gate=w["gate"], ln=False)
    return x, state


def tokens(dt, dev, h, wd, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, h, wd, C, generator=g).to(dt).to(dev)
    mask = torch.rand(2, h * wd, generator=g) < 0.8
    mask[1, h * wd - 40:] = False
    return x, (torch.randn(2, KV, D, D, generator=g)).to(dev), mask.to(dev)


@pytest.fixture(scope="module")
def chains(gpu_device):
    return {dt: Ops(["hip"], dt, gpu_device, log=print) for dt in (torch.bfloat16, torch.float32)}


@pytest.mark.gpu
@pytest.mark.parametrize("h,wd", [(1, 1), (9, 29), (24, 40)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_steps(dt, h, wd, chains, gpu_device):
    ops, w = chains[dt], weights(dt, gpu_device)
    x, state, mask = tokens(dt, gpu_device, h, wd)
    if h * wd == 1:
        mask = None
    seen = []
    block(ops, x, w, state, mask, seen)
    torch.cuda.synchronize()
    for i, (what, got, args, kw) in enumerate(seen):
        print(f"[block] step {i} {what}", flush=True)
        if what == "norm":
            check_norm(got, *args, what=f"step {i}", **kw)
        elif what == "rotary":
            check_rotary(got, *args, what=f"step {i}", **kw)
        elif what == "linear":
            check_linear(got, *args, what=f"step {i}", **kw)
        else:
            again, _ = check_sparse(ops, *args, what=f"step {i}", **kw)
            assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_captured(dt, chains, gpu_device):
    """Two graphs of the block on tokens of other sizes, replayed in turn between eager calls: bitwise the eager results."""
    ops, w = chains[dt], weights(dt, gpu_device)
    made = []
    for h, wd in ((9, 29), (24, 40)):
        sets = [tokens(dt, gpu_device, h, wd, seed) for seed in (1, 2)]
        refs = [block(ops, s[0], w, s[1], s[2]) for s in sets]
        st = [t.clone() for t in sets[0]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = block(ops, st[0], w, st[1], st[2])
        made.append((graph, sets, refs, st, got))
    for i in range(6):
        for graph, sets, refs, st, got in made:
            for dst, src in zip(st, sets[i % 2]):
                dst.copy_(src)
            graph.replay()
            eager = block(ops, sets[1][0], w, sets[1][1], sets[1][2])
            torch.cuda.synchronize()
            for j in (0, 1):
                assert torch.equal(got[j], refs[i % 2][j]) and torch.equal(eager[j], refs[1][j]), i


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_tokens_in_pieces(dt, chains, gpu_device):
    """Rows of a map one after another, with the positions of the whole: rotary, then linear attention from state to state,
    then a last query over all keys with means kept from before; against all the tokens at once."""
    ops = chains[dt]
    g = torch.Generator().manual_seed(3)
    rows, wd = 7, 61
    q, k, v = (torch.randn(2, rows, wd, n * D, generator=g).to(dt).to(gpu_device) for n in (HEADS, KV, KV))
    grid = torch.stack(torch.meshgrid(torch.arange(rows), torch.arange(wd), indexing="ij"), -1).to(gpu_device)
    decay = weights(dt, gpu_device)["decay"]
    qr, kr = ops.rotary(q, HEADS, SECTIONS), ops.rotary(k, KV, SECTIONS)
    state, outs = None, []
    for r in range(rows):
        cuts = [0, wd] if r % 2 else [0, 1, 17, wd]  # single tokens, a step's longest, chunks
        for a, b in zip(cuts, cuts[1:]):
            pos = grid[r, a:b].contiguous()
            pq, pk = (ops.rotary(t[:, r, a:b], n, SECTIONS, positions=pos) for t, n in ((q, HEADS), (k, KV)))
            assert torch.equal(pq, qr[:, r, a:b]) and torch.equal(pk, kr[:, r, a:b])
            out, state = ops.linear_attention(pq, pk, v[:, r, a:b], decay, HEADS, KV, state=state, state_out=state)
            outs.append(out)
    check_linear((torch.cat(outs, 1), state), qr.flatten(1, 2), kr.flatten(1, 2), v.flatten(1, 2), decay, HEADS, KV)
    means = ops.block_means(kr)
    last, chosen = ops.sparse_attention(qr[:, -1, -1:], kr, v, HEADS, TOP, KV, means=means, return_blocks=True)
    whole, every = ops.sparse_attention(qr, kr, v, HEADS, TOP, KV, return_blocks=True)
    assert torch.equal(chosen[:, :, 0], every[:, :, -1])
    flat = [t.flatten(1, 2) for t in (qr[:, -1:, -1:], kr, v)]
    ref, pv, big = attend64(*flat, HEADS, KV, chosen, 64, 1)
    u, lk = 2.0 ** -24, rows * wd
    tol = (2 * (D + 8) * u * big + 2 * (lk + 16) * u + (2.0 ** -8 if dt == torch.bfloat16 else 0)) * pv
    tol = tol + (2.0 ** -8 if dt == torch.bfloat16 else u) * ref.abs()
    for got in (last, whole[:, -1, -1:]):
        assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_gradients_pass_through_the_chain(gpu_device):
    """rotary and add_norm of operands with gradients fall through to their plain forms; the attentions, which have none, refuse."""
    ops = Ops(["hip", "torch"], torch.float32, gpu_device, log=print)
    x = tokens(torch.float32, gpu_device, 3, 5)[0].requires_grad_()
    out = ops.rotary(ops.add_norm(x, x * 0.5, gate=weights(torch.float32, gpu_device)["gate"])[1], HEADS, SECTIONS)
    out.square().sum().backward()
    assert torch.isfinite(x.grad).all() and x.grad.norm().item() > 0
    assert ops.report()["ops"]["rotary"] == ops.report()["ops"]["add_norm"] == {"torch": 1}
    qkv = [t.contiguous() for t in split(torch.zeros(1, 3, 5, (HEADS + 2 * KV) * D, device=gpu_device, requires_grad=True))]
    with pytest.raises((Unsupported, NotImplementedError)):
        ops.linear_attention(*qkv, torch.zeros(KV, device=gpu_device), HEADS, KV)
    with pytest.raises((Unsupported, NotImplementedError)):
        ops.sparse_attention(*qkv, HEADS, 1, KV)
