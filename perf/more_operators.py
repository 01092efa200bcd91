"""Timed calls of the operators around the token mixers of image and video transformers:

  rotary            rotary positions with an axis each for time, height and width on the heads of a projection
  add_norm          a block's output normed, gated, scaled and added to the residual stream, and the norm (with its
                    scale and shift) that the next block reads
  linear_attention  causal linear attention with a decay for each head: whole sequences, and single tokens from a state
  sparse_attention  attention over the blocks of keys that a cheap score selects for each query or group of queries

`run` computes them in a plain form, elementary torch operations in 32 bits (angles, block means and scores in 64)
rounded once at the end; with `own` set it makes the calls of the framework's operator dispatch instead. Forward only, as
the framework is.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
BASE = 10000.0
_handles = {}


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _ops(dtype):
    """The operator dispatch of one compute dtype, made once as a program makes it."""
    if dtype not in _handles:
        from clarus_amd.dispatch import Ops
        _handles[dtype] = Ops(["hip"], dtype, _device(), log=lambda *a: None)
    return _handles[dtype]


# ------------------------------------------------------------------------------- the cases
def _rope(dtype, n, grid, heads, d, sections, pairs="adjacent", given=False, extra=0):
    """grid: sizes of the axes, joined by "x"; sections: pairs of columns of each axis; given: positions as a tensor
    (else the grid's own); extra: columns of the rows that the call leaves out (the values of a joint projection)."""
    return {"op": "rotary", "dtype": dtype, "n": n, "grid": grid, "heads": heads, "d": d, "sections": sections,
            "pairs": pairs, "given": given, "extra": extra}


def _norm(x_dtype, y_dtype, n, rows, c, post, pre, per_image, first=False):
    """x_dtype: of the residual stream; first: no block before (the norm alone)."""
    return {"op": "add_norm", "dtype": y_dtype, "x_dtype": x_dtype, "n": n, "rows": rows, "c": c, "post": post,
            "pre": pre, "per_image": per_image, "first": first}


def _lin(dtype, n, length, heads, kv_heads, dk, dv, carried):
    """carried: a state from before goes in."""
    return {"op": "linear_attention", "dtype": dtype, "n": n, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dk": dk, "dv": dv, "carried": carried}


def _sparse(dtype, n, lq, lk, heads, kv_heads, d, top, block, group, padded=False, kept=False):
    """padded: a mask of keys; kept: the blocks' means are kept from call to call, as keys that stay are."""
    return {"op": "sparse_attention", "dtype": dtype, "n": n, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads,
            "d": d, "top": top, "block": block, "group": group, "padded": padded, "kept": kept}


def listed():
    return [
        # queries and keys of a thumbnail's deepest map, before its attention: launches and latency
        {"name": "rope_bf16_16x24_h8", **_rope("bf16", 1, "16x24", 16, 32, "8,8", extra=256)},
        # queries and keys of a 180 x 320 map, slices of one projection's rows
        {"name": "rope_bf16_180x320_h8", **_rope("bf16", 1, "180x320", 16, 64, "16,16", "halves", extra=512)},
        # two clips of odd size in fp32 with frame times and places of their own, heads of 72
        {"name": "rope_f32_2x5x45x81_h6", **_rope("fp32", 2, "5x45x81", 6, 72, "8,14,14", given=True)},
        # the deepest map of a thumbnail: a block's output added, the next block's norm
        {"name": "an_bf16_384_c512", **_norm("bf16", "bf16", 1, 384, 512, "rms", "ln", True)},
        # the level at which most of a width-64 network's blocks run on a 720p frame, two images, fp32 stream
        {"name": "an_bf16_2x14400_c512", **_norm("fp32", "bf16", 2, 14400, 512, "rms", "ln", True)},
        # one frame's token for each of 64 streams: reading and writing states
        {"name": "la_bf16_64x1_h16_d128", **_lin("bf16", 64, 1, 16, 16, 128, 128, True)},
        # the tokens of a 180 x 320 map in raster order
        {"name": "la_bf16_57600_h8_d64", **_lin("bf16", 1, 57600, 8, 8, 64, 64, False)},
        # two odd sequences in fp32 carried on from a state, two heads to a state, wider values
        {"name": "la_f32_2x5003_h8_d48", **_lin("fp32", 2, 5003, 8, 4, 48, 96, True)},
        # one token for each of eight images over a long context that stays, heads shared by four
        {"name": "sa_bf16_8x1q_30001k", **_sparse("bf16", 8, 1, 30001, 16, 4, 128, 32, 64, 1, kept=True)},
        # a 90 x 160 map over itself, every query with blocks of its own
        {"name": "sa_bf16_14400_each", **_sparse("bf16", 1, 14400, 14400, 8, 8, 64, 16, 64, 1)},
        # a 180 x 320 map over itself, 64 neighbours choosing together: the largest
        {"name": "sa_bf16_57600_g64", **_sparse("bf16", 1, 57600, 57600, 8, 8, 64, 16, 64, 64)},
        # fp32, maps padded to one length, the last one empty, larger blocks
        {"name": "sa_f32_3x3601_pad", **_sparse("fp32", 3, 3601, 3601, 4, 4, 48, 6, 128, 16, padded=True)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "add_norm", "linear_attention", "sparse_attention"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    wide = 2 if dtype == "fp32" else 1
    if op == "rotary":
        axes = rng.choice([1, 2, 2, 3])
        d = rng.choice([16, 32, 48, 64, 64, 72, 96, 128])
        heads = _log_int(rng, 1, 32)
        n = rng.choice([1, 1, 2, 4])
        area = _log_int(rng, 1, max(1, 57600 * 1024 // (n * heads * d * wide)))
        grid = []
        for i in range(axes - 1):
            grid.append(_log_int(rng, 1, max(1, int(area ** (1 / (axes - i))))))
            area //= grid[-1]
        grid.append(max(1, area))
        most = d // 2 if rng.random() < 0.7 else d // 4
        cuts = sorted(rng.sample(range(1, most), axes - 1)) if axes > 1 else []
        sections = [b - a for a, b in zip([0] + cuts, cuts + [most])]
        return _rope(dtype, n, "x".join(map(str, grid)), heads, d, ",".join(map(str, sections)),
                     rng.choice(["adjacent", "halves"]), rng.random() < 0.4, rng.choice([0, 0, heads * d]))
    if op == "add_norm":
        c = rng.choice([32, 48, 96, 128, 192, 256, 320, 384, 512, 512, 768, 1024, 1536, 2048, 4096])
        n = rng.choice([1, 1, 2, 4])
        first = rng.random() < 0.2
        return _norm(rng.choice(["fp32", dtype]), dtype, n, _log_int(rng, 1, max(1, 57600 * 512 // (n * c))), c,
                     rng.choice(["none", "ln", "rms"]), rng.choice(["ln", "ln", "rms"] + ["none"] * (not first)),
                     rng.random() < 0.6, first)
    if op == "linear_attention":
        dk, dv = rng.choice([16, 32, 48, 64, 64, 96, 128]), rng.choice([32, 40, 64, 64, 96, 128])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
        if rng.random() < 0.4:  # single tokens, or a few
            return _lin(dtype, _log_int(rng, 1, max(1, 64 * 16 * 128 * 128 // (kv_heads * dk * dv))), rng.choice([1, 1, 1, 2, 5, 16]),
                        heads, kv_heads, dk, dv, rng.random() < 0.8)
        n = rng.choice([1, 1, 2, 4])
        return _lin(dtype, n, _log_int(rng, 17, max(17, 57600 * 512 // (n * heads * max(dk, dv) * wide))), heads, kv_heads, dk, dv,
                    rng.random() < 0.5)
    d = rng.choice([32, 40, 48, 64, 64, 80, 96, 128, 128])
    block = rng.choice([64, 64, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    n = rng.choice([1, 1, 2, 4])
    padded = rng.random() < 0.3
    top = _log_int(rng, 1, 32)
    if rng.random() < 0.3:
        lq = rng.choice([1, 1, 2, 5, 16])
        lk = _log_int(rng, 64, max(64, 245760 * 512 // (n * kv_heads * d * wide)))
        return _sparse(dtype, n, lq, lk, heads, kv_heads, d, top, block, 1, padded, rng.random() < 0.5)
    group = rng.choice([1, 1, 8, 16, 64, 64, 100, 256])
    lk = _log_int(rng, 1, 57600)
    lq = lk if rng.random() < 0.7 else _log_int(rng, 16, 57600)
    # no more than the largest listed in the products of chosen keys (fp32 a twelfth of it), and a score for each
    # query, or group of them, and block
    most = 57600 * 1024 * 8 * 64 // (1 if dtype == "bf16" else 12)
    while (n * heads * d * lq * min(lk, top * block) > most
           or n * heads * d * -(-lq // group) * (lk / block) > 14400 * 225 * 8 * 64):
        lq, lk = max(1, lq * 3 // 4), max(1, lk * 3 // 4)
    return _sparse(dtype, n, lq, lk, heads, kv_heads, d, top, block, group, padded, rng.random() < 0.2)


# ------------------------------------------------------------------------------- inputs
def _ints(text, by):
    return [int(t) for t in text.split(by)]


def _kept_keys(case):
    """Kept keys of each image where keys are padded: full down to none (one image: three quarters)."""
    n, lk = case["n"], case["lk"]
    return [lk - lk // 4] if n == 1 else [lk * (n - 1 - i) // (n - 1) for i in range(n)]


def _decays(kv_heads, device):
    """Logarithms of the heads' decays: from 1/32 down by a factor of two a head, in 4 octaves at most; the last head
    of several keeps everything."""
    g = -(2.0 ** (-5 - 4 * torch.arange(kv_heads, device=device, dtype=torch.float32) / kv_heads))
    if kv_heads > 2:
        g[-1] = 0.0
    return g


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).add_(shift)
    n = case["n"]
    if case["op"] == "rotary":
        grid = _ints(case["grid"], "x")
        c = case["heads"] * case["d"]
        x = randn(n, *grid, c + case["extra"]).to(dt)[..., :c]
        pos = None
        if case["given"]:  # a clip's frame times (in 90 kHz ticks, far from zero) and places of its own
            at = torch.stack(torch.meshgrid(*[torch.arange(s, device=dev, dtype=torch.float32) for s in grid], indexing="ij"), -1)
            at = at.reshape(1, -1, len(grid)).repeat(n, 1, 1)
            start = torch.randint(0, 5000, (n, 1, 1), generator=g, device=dev)
            at = at + start
            at[..., 0] = (at[..., 0] * 3003.0 / 90.0).round()
            pos = at.contiguous() if case["dtype"] == "fp32" else at.long()
        return {"case": case, "x": x, "sections": _ints(case["sections"], ","), "positions": pos}
    if case["op"] == "add_norm":
        rows, c = case["rows"], case["c"]
        per = (n, c) if case["per_image"] else (c,)
        chan = randn(c)  # residual streams have channels with means and sizes of their own
        x = (randn(n, rows, c) * (0.5 + 2 * randn(c).abs()) + chan).to(DTYPES[case["x_dtype"]])
        return {"case": case, "x": x, "y": None if case["first"] else (randn(n, rows, c) * 1.5).to(dt),
                "gate": randn(*per, scale=0.5), "post_weight": randn(c, scale=0.2, shift=1.0),
                "weight": randn(*per, scale=0.2, shift=1.0), "bias": randn(*per, scale=0.2)}
    if case["op"] == "linear_attention":
        length, kv = case["length"], case["kv_heads"]
        q = randn(n, length, case["heads"] * case["dk"]).to(dt)
        # keys after a positive feature map, values of a projection
        k = (randn(n, length, kv * case["dk"]).abs() * 0.5 + randn(n, length, kv * case["dk"], scale=0.25)).to(dt)
        v = randn(n, length, kv * case["dv"]).to(dt)
        state = randn(n, kv, case["dk"], case["dv"], scale=3.0) if case["carried"] else None
        return {"case": case, "q": q, "k": k, "v": v, "log_decay": _decays(kv, dev), "state": state}
    lq, lk, d = case["lq"], case["lk"], case["d"]

    def tokens(length, heads, size):
        """Neighbours along a map are alike: a coarse field, a value for every 48 tokens, and noise of their own."""
        coarse = randn(n, -(-length // 48), heads * d, scale=size).repeat_interleave(48, 1)[:, :length]
        return (coarse + randn(n, length, heads * d, scale=0.6)).to(dt)
    q, k = tokens(lq, case["heads"], 1.2), tokens(lk, case["kv_heads"], 0.8)
    v = randn(n, lk, case["kv_heads"] * d).to(dt)
    mask = means = None
    if case["padded"]:
        mask = torch.arange(lk, device=dev)[None] < torch.tensor(_kept_keys(case), device=dev)[:, None]
    if case["kept"]:
        means = _plain_means(k, case["block"], mask)
    return {"case": case, "q": q, "k": k, "v": v, "mask": mask, "means": means}


# ------------------------------------------------------------------------------- one pass, plainly
def _plain_rotary(x, heads, sections, positions, pairs):
    n, c = x.shape[0], x.shape[-1]
    d = c // heads
    y = x.reshape(n, -1, heads, d).float()
    if positions is None:
        at = torch.stack(torch.meshgrid(*[torch.arange(s, device=x.device, dtype=torch.float64) for s in x.shape[1:-1]],
                                        indexing="ij"), -1).reshape(1, -1, x.dim() - 2)
    else:
        at = positions.double().reshape(-1, y.shape[1], len(sections))
    angle = torch.cat([at[..., a:a + 1] * BASE ** (-torch.arange(s, device=x.device, dtype=torch.float64) / s)
                       for a, s in enumerate(sections)], -1)[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    p = sum(sections)
    a, b = (y[..., 0:2 * p:2], y[..., 1:2 * p:2]) if pairs == "adjacent" else (y[..., :p], y[..., p:2 * p])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if pairs == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., 2 * p:]], -1).reshape(x.shape).to(x.dtype)


def _plain_norm(x, kind):
    if kind == "none":
        return x
    if kind == "ln":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_add_norm(state, case):
    def rows(t):
        return t if t.dim() == 1 else t[:, None]
    r = state["x"].float()
    if state["y"] is not None:
        y = _plain_norm(state["y"].float(), case["post"])
        if case["post"] != "none":
            y = y * state["post_weight"]
        r = r + y * rows(state["gate"]) * 0.75
    h = None
    if case["pre"] != "none":
        h = (_plain_norm(r, case["pre"]) * rows(state["weight"]) + rows(state["bias"])).to(DTYPES[case["dtype"]])
    return r.to(state["x"].dtype), h


def _plain_linear(q, k, v, log_decay, heads, kv_heads, state, step=512):
    n, length, ck = k.shape
    dk, dv, rep = ck // kv_heads, v.shape[-1] // kv_heads, heads // kv_heads
    qh = q.float().reshape(n, length, kv_heads, rep, dk).permute(0, 2, 3, 1, 4) * dk ** -0.5
    kh, vh = (t.float().reshape(n, length, kv_heads, -1).permute(0, 2, 1, 3).contiguous() for t in (k, v))
    s = torch.zeros(n, kv_heads, dk, dv, device=q.device) if state is None else state
    g = log_decay.double()[:, None, None]
    at = torch.arange(min(step, length), device=q.device, dtype=torch.float64)
    gap = at[:, None] - at[None]
    within = torch.where(gap >= 0, torch.exp(g * gap), torch.zeros_like(gap)).float()  # [kv, i, j]
    since = torch.exp(g[..., 0] * (at + 1)).float()[:, None, :, None]
    out = torch.empty(n, kv_heads, rep, length, dv, device=q.device)
    for a in range(0, length, step):
        b = min(a + step, length)
        m = b - a
        qc = qh[:, :, :, a:b].contiguous()
        kc, vc = kh[:, :, a:b], vh[:, :, a:b]
        inter = (qc * since[:, :, :m]).reshape(n * kv_heads, rep * m, dk) @ s.reshape(n * kv_heads, dk, dv)
        p = qc.reshape(n * kv_heads, rep * m, dk) @ kc.transpose(-1, -2).contiguous().reshape(n * kv_heads, dk, m)
        p = (p.reshape(n, kv_heads, rep, m, m) * within[:, None, :m, :m]).reshape(n * kv_heads, rep * m, m)
        out[:, :, :, a:b] = (inter + p @ vc.reshape(n * kv_heads, m, dv)).reshape(n, kv_heads, rep, m, dv)
        left = torch.exp(g[..., 0] * (m - 1 - at[:m])).float()[:, :, None]
        kt = (kc * left).transpose(-1, -2).contiguous().reshape(n * kv_heads, dk, m)
        s = s * torch.exp(g * m).float() + (kt @ vc.reshape(n * kv_heads, m, dv)).reshape(n, kv_heads, dk, dv)
    return out.permute(0, 3, 1, 2, 4).reshape(n, length, heads * dv).to(q.dtype), s


def _plain_means(k, block, mask):
    """Means of the kept keys of each block, in 64 bits, rounded to 32; NaN for a block that keeps none."""
    n, lk, c = k.shape
    nb = -(-lk // block)
    if mask is not None:
        k = k.masked_fill(~mask[..., None], 0)
    pad = nb * block - lk
    count = (torch.ones(n, lk, device=k.device) if mask is None else mask).double()
    total = torch.nn.functional.pad(k.double(), (0, 0, 0, pad)).reshape(n, nb, block, c).sum(2)
    return (total / torch.nn.functional.pad(count, (0, pad)).reshape(n, nb, block).sum(2)[..., None]).float()


def _plain_chosen(q, means, heads, kv_heads, group, top):
    """[n, heads, groups, top'] blocks in falling order of their scores, ties to the lowest index, and whether
    each is there."""
    n, lq, c = q.shape
    d, rep, nb, groups = c // heads, heads // kv_heads, means.shape[1], -(-lq // group)
    asks = q
    if group > 1:
        size = torch.full((groups,), group, device=q.device, dtype=torch.float64)
        size[-1] = lq - (groups - 1) * group
        pad = torch.nn.functional.pad(q.double(), (0, 0, 0, groups * group - lq))
        asks = (pad.reshape(n, groups, group, c).sum(2) / size[:, None]).float()
    asks = asks.double().reshape(n, groups, kv_heads, rep, d).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, rep * groups, d)
    mt = means.double().reshape(n, nb, kv_heads, d).permute(0, 2, 3, 1).contiguous().reshape(n * kv_heads, d, nb)
    score = (asks @ mt).reshape(n, heads, groups, nb)
    score = torch.where(score.isnan(), torch.full_like(score, -math.inf), score)
    score, at = score.sort(dim=-1, descending=True, stable=True)
    top = min(top, nb)
    return at[..., :top], score[..., :top] > -math.inf


def _plain_sparse(q, k, v, heads, kv_heads, block, group, top, mask, means):
    n, lq, c = q.shape
    lk, d, rep, groups = k.shape[1], c // heads, heads // kv_heads, -(-lq // group)
    if means is None:
        means = _plain_means(k, block, mask)
    at, there = _plain_chosen(q, means, heads, kv_heads, group, top)
    top = at.shape[-1]
    nb = means.shape[1]
    if mask is not None:
        k, v = k.masked_fill(~mask[..., None], 0), v.masked_fill(~mask[..., None], 0)
    out = torch.zeros(n, heads, lq, d, device=q.device)
    qh = q.reshape(n, lq, heads, d)
    for i in range(n):
        keep = torch.ones(lk, dtype=torch.bool, device=q.device) if mask is None else mask[i]
        keep = torch.nn.functional.pad(keep, (0, nb * block - lk)).reshape(nb, block)
        for h in range(heads):
            q1 = torch.nn.functional.pad(qh[i, :, h].float(), (0, 0, 0, groups * group - lq)).reshape(groups, group, d) * d ** -0.5
            k1, v1 = (t[i].reshape(lk, kv_heads, d)[:, h // rep].float() for t in (k, v))
            if group >= 16 or lq < 64:  # the chosen blocks fetched, some groups at a time
                k1, v1 = (torch.nn.functional.pad(t, (0, 0, 0, nb * block - lk)).reshape(nb, block, d) for t in (k1, v1))
                step = max(1, (1 << 28) // (top * block * max(d, group)))
                done = []
                for a in range(0, groups, step):
                    pick = at[i, h, a:a + step]
                    seen = (keep[pick] & there[i, h, a:a + step, :, None]).flatten(1)[:, None]
                    kt = k1[pick].flatten(1, 2).transpose(-1, -2).contiguous()
                    done.append(_plain_softmax(torch.bmm(q1[a:a + step], kt), seen, v1[pick].flatten(1, 2)))
                out[i, h] = torch.cat(done).reshape(-1, d)[:lq]
            else:  # every key under the choice as a mask, some queries at a time
                kt = k1.t().contiguous()
                step = max(1, (1 << 28) // lk // group)
                done = []
                for a in range(0, groups, step):
                    pick = torch.zeros(at[i, h, a:a + step].shape[0], nb, dtype=torch.bool, device=q.device)
                    pick.scatter_(1, at[i, h, a:a + step], there[i, h, a:a + step])
                    seen = (pick[:, :, None] & keep).flatten(1)[:, :lk].repeat_interleave(group, 0)
                    done.append(_plain_softmax(q1[a:a + step].flatten(0, 1) @ kt, seen, v1))
                out[i, h] = torch.cat(done)[:lq]
    return out.permute(0, 2, 1, 3).reshape(n, lq, c).to(q.dtype)


def _plain_softmax(s, seen, v):
    s = s.masked_fill(~seen, -math.inf)
    most = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = s.sum(-1, keepdim=True)
    return (s @ v) / torch.where(total == 0, torch.ones_like(total), total)


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if own:
            return _ops(state["x"].dtype).rotary(state["x"], case["heads"], state["sections"], positions=state["positions"],
                                                 base=BASE, pairs=case["pairs"])
        return _plain_rotary(state["x"], case["heads"], state["sections"], state["positions"], case["pairs"])
    if case["op"] == "add_norm":
        if own:
            kinds = {"none": False, "ln": True, "rms": "rms"}
            r, h = _ops(DTYPES[case["dtype"]]).add_norm(
                state["x"], state["y"], gate=state["gate"], scale=0.75, post=kinds[case["post"]],
                post_weight=state["post_weight"] if case["post"] != "none" else None, ln=kinds[case["pre"]],
                weight=state["weight"], bias=state["bias"], eps=EPS)
        else:
            r, h = _plain_add_norm(state, case)
        return {name: t for name, t in (("sum", None if case["first"] else r), ("norm", h)) if t is not None}
    q, k, v = state["q"], state["k"], state["v"]
    if case["op"] == "linear_attention":
        if own:
            out, s = _ops(q.dtype).linear_attention(q, k, v, state["log_decay"], case["heads"], kv_heads=case["kv_heads"],
                                                    state=state["state"])
        else:
            out, s = _plain_linear(q, k, v, state["log_decay"], case["heads"], case["kv_heads"], state["state"])
        return {"out": out, "state": s}
    if own:
        return _ops(q.dtype).sparse_attention(q, k, v, case["heads"], case["top"], kv_heads=case["kv_heads"], block=case["block"],
                                              group=case["group"], mask=state["mask"], means=state["means"])
    return _plain_sparse(q, k, v, case["heads"], case["kv_heads"], case["block"], case["group"], case["top"], state["mask"],
                         state["means"])


# ------------------------------------------------------------------------------- what a pass needs
def work(case):
    es, n = 2 if case["dtype"] == "bf16" else 4, case["n"]
    if case["op"] == "rotary":
        tokens = n * math.prod(_ints(case["grid"], "x"))
        pairs = sum(_ints(case["sections"], ","))
        given = (4 if case["dtype"] == "fp32" else 8) * len(_ints(case["sections"], ",")) if case["given"] else 0
        return {"bytes": tokens * (2 * case["heads"] * case["d"] * es + given), "flops": 6 * tokens * case["heads"] * pairs}
    if case["op"] == "add_norm":
        elems, xs = n * case["rows"] * case["c"], 2 if case["x_dtype"] == "bf16" else 4
        moved = xs + (es if case["pre"] != "none" else 0) + (0 if case["first"] else es + xs)
        return {"bytes": elems * moved + 4 * case["c"] * (4 if case["first"] else 6), "flops": 16 * elems}
    heads, kv = case["heads"], case["kv_heads"]
    if case["op"] == "linear_attention":
        tokens, dk, dv = n * case["length"], case["dk"], case["dv"]
        states = n * kv * dk * dv * 4 * (2 if case["carried"] else 1)
        # a token's product with the state and its addition to it
        return {"bytes": tokens * es * (heads * (dk + dv) + kv * (dk + dv)) + states, "flops": 2 * tokens * dk * dv * (heads + kv)}
    lq, lk, d, block = case["lq"], case["lk"], case["d"], case["block"]
    groups, pairs, rows, keys = -(-lq // case["group"]), 0, 0, _kept_keys(case) if case["padded"] else [lk] * n
    scored = 0
    for left in keys:
        seen = min(left, case["top"] * block)
        pairs += lq * seen
        scored += groups * -(-left // block)
        rows += min(left, heads // kv * groups * seen)  # a key that no query chooses need not be read but for its mean
    k_rows = rows if case["kept"] else sum(keys)
    small = 4 * sum(-(-left // block) for left in keys) * kv * d if case["kept"] else 0
    return {"bytes": es * d * (2 * n * lq * heads + (k_rows + rows) * kv) + small + (n * lk if case["padded"] else 0),
            "flops": (4 * pairs + 2 * scored) * heads * d}


# ------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    t = prepare(case, seed)
    if case["op"] == "rotary":
        x = t["x"].double()
        n, heads, d = case["n"], case["heads"], case["d"]
        grid = _ints(case["grid"], "x")
        z = x.reshape(n, -1, heads, d)
        length, out = z.shape[1], z.clone()
        index, first, p = torch.arange(length, device=x.device), 0, sum(t["sections"])
        stride = length
        for axis, size in enumerate(t["sections"]):
            if t["positions"] is None:
                stride //= grid[axis]
                at = (index // stride % grid[axis]).double()[None]
            else:
                at = t["positions"][..., axis].double()
            for i in range(size):
                j = first + i
                ca, cb = (2 * j, 2 * j + 1) if case["pairs"] == "adjacent" else (j, p + j)
                turn = torch.polar(torch.ones_like(at), at / BASE ** (i / size))[..., None]
                w = torch.complex(z[..., ca], z[..., cb]) * turn
                out[..., ca], out[..., cb] = w.real, w.imag
            first += size
        return out.reshape(x.shape)
    if case["op"] == "add_norm":
        def normed(u, kind):
            if kind == "none":
                return u
            mean = u.mean(-1, keepdim=True) if kind == "ln" else 0.0
            return (u - mean) / torch.sqrt(((u - mean) ** 2).mean(-1, keepdim=True) + EPS)

        def wide(u):
            return u.double().expand(case["n"], case["c"])[:, None]
        r = t["x"].double()
        if t["y"] is not None:
            y = normed(t["y"].double(), case["post"])
            r = r + 0.75 * wide(t["gate"]) * (y if case["post"] == "none" else y * t["post_weight"].double())
        out = {} if case["first"] else {"sum": r}
        if case["pre"] != "none":
            out["norm"] = normed(r, case["pre"]) * wide(t["weight"]) + wide(t["bias"])
        return out
    heads, kv = case["heads"], case["kv_heads"]
    rep = heads // kv
    if case["op"] == "linear_attention":
        n, length, dk, dv = case["n"], case["length"], case["dk"], case["dv"]
        out = torch.zeros(n, length, heads, dv, dtype=torch.float64, device=t["q"].device)
        last = torch.zeros(n, kv, dk, dv, dtype=torch.float64, device=t["q"].device)
        place = torch.arange(length, device=t["q"].device, dtype=torch.float64)
        step = max(1, (1 << 26) // length)
        for i in range(n):
            for h in range(kv):
                g = t["log_decay"][h].double()
                keys = t["k"][i, :, h * dk:(h + 1) * dk].double()
                vals = t["v"][i, :, h * dv:(h + 1) * dv].double()
                last[i, h] = (keys * torch.exp(g * (length - 1 - place))[:, None]).t().contiguous() @ vals
                if t["state"] is not None:
                    last[i, h] += t["state"][i, h].double() * torch.exp(g * length)
                for j in range(h * rep, (h + 1) * rep):
                    asks = t["q"][i, :, j * dk:(j + 1) * dk].double() / math.sqrt(dk)
                    for a in range(0, length, step):
                        b = min(a + step, length)  # every pair of tokens (i, j <= i), by the sum's definition
                        w = asks[a:b] @ keys[:b].t().contiguous()
                        gap = place[a:b, None] - place[None, :b]
                        w = w * torch.exp(g * gap.clamp_min(0)) * (gap >= 0)
                        out[i, a:b, j] = w @ vals[:b]
                    if t["state"] is not None:
                        out[i, :, j] += (asks * torch.exp(g * (place + 1))[:, None]) @ t["state"][i, h].double()
        return {"out": out.reshape(n, length, heads * dv), "state": last}
    n, lq, lk, d, block, group = (case[i] for i in ("n", "lq", "lk", "d", "block", "group"))
    out = torch.zeros(n, lq, heads, d, dtype=torch.float64, device=t["q"].device)
    nb = -(-lk // block)
    inside = torch.arange(nb * block, device=out.device).reshape(nb, block)
    for i in range(n):
        kept = torch.ones(lk, dtype=torch.bool, device=out.device) if t["mask"] is None else t["mask"][i]
        kept = torch.cat([kept, torch.zeros(nb * block - lk, dtype=torch.bool, device=out.device)])[inside]
        inner = inside.clamp(max=lk - 1)
        full = kept.any(-1)
        if not full.any():
            continue
        for h in range(heads):
            head, at = slice(h * d, (h + 1) * d), slice(h // rep * d, (h // rep + 1) * d)
            keys, vals = t["k"][i, :, at].double()[inner], t["v"][i, :, at].double()[inner]
            if t["means"] is None:
                mean = ((keys * kept[..., None]).sum(1) / kept.sum(1)[:, None]).float().double()
            else:
                mean = t["means"][i, :, at].double()
            mean = torch.where(full[:, None], mean, torch.zeros_like(mean))
            asks = t["q"][i, :, head].double()
            score = torch.stack([a.mean(0) for a in asks.split(group)]).float().double() if group > 1 else asks
            score = (score @ mean.t().contiguous()).masked_fill(~full, -math.inf)
            order = torch.argsort(score, dim=-1, descending=True, stable=True)[:, :case["top"]]
            order = order[:, :int(full.sum())]
            step = max(1, (1 << 26) // (order.shape[1] * block * max(d, group)))
            for a in range(0, order.shape[0], step):
                pick = order[a:a + step]
                rows = min(lq, (a + pick.shape[0]) * group) - a * group
                ask = torch.zeros(pick.shape[0] * group, d, dtype=torch.float64, device=out.device)
                ask[:rows] = asks[a * group:a * group + rows]
                z = torch.bmm(ask.reshape(-1, group, d) / math.sqrt(d), keys[pick].flatten(1, 2).transpose(1, 2).contiguous())
                w = torch.softmax(z.masked_fill(~kept[pick].flatten(1)[:, None], -1e300), -1)
                out[i, a * group:a * group + rows, h] = torch.bmm(w, vals[pick].flatten(1, 2)).reshape(-1, d)[:rows]
    return out.reshape(n, lq, heads * d)
