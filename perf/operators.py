"""Timed calls of the operators that a conditioned restoration model runs between its convs and 1x1 linears:

  group_norm       group norm of an NHWC feature map with its activation, the affine per channel or per image
  cross_attention  every pixel (or a few tokens) attends the states of an encoder: prompt tokens, or another
                   feature map, of another length

`run` computes them in a plain form, elementary torch operations in 32 bits rounded once at the end; with `own`
set it makes the calls of the framework's operator dispatch instead. Forward only, as the framework is.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
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
def _gn(dtype, n, h, w, c, groups, act, per_image=False):
    return {"op": "group_norm", "dtype": dtype, "n": n, "h": h, "w": w, "c": c, "groups": groups, "act": act,
            "per_image": per_image}


def _xa(dtype, n, lq, lk, heads, kv_heads, d, mask="none", joint=False):
    return {"op": "cross_attention", "dtype": dtype, "n": n, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "d": d, "mask": mask, "joint": joint}


def listed():
    return [
        # the deepest map of a thumbnail: launches and latency
        {"name": "gn_bf16_16x24_c512", **_gn("bf16", 1, 16, 24, 512, 32, "silu")},
        # the level at which most of a width-64 network's blocks run on a 720p frame
        {"name": "gn_bf16_90x160_c512", **_gn("bf16", 1, 90, 160, 512, 32, "silu")},
        # two odd-sized images in fp32, each with a scale and shift of its own (conditioned on a noise level)
        {"name": "gn_f32_2x173x251_c128", **_gn("fp32", 2, 173, 251, 128, 32, "silu", True)},
        # four photos of odd size, three channels in a group, no activation (the norm before an attention)
        {"name": "gn_bf16_4x251x333_c96", **_gn("bf16", 4, 251, 333, 96, 32, "none")},
        # the full-size map of a 720p frame
        {"name": "gn_bf16_720x1280_c64", **_gn("bf16", 1, 720, 1280, 64, 16, "gelu")},
        # a tile's deepest pixels ask one prompt: the smallest call
        {"name": "xa_bf16_48q_77k", **_xa("bf16", 1, 48, 77, 4, 4, 32)},
        # every pixel of a 180 x 320 map asks one prompt: short keys, bound by q and the output
        {"name": "xa_bf16_57600q_77k", **_xa("bf16", 1, 57600, 77, 4, 4, 64, "none", True)},
        # a batch with prompts padded to one length, one of them empty; heads of 40
        {"name": "xa_bf16_4x3600q_300k_pad", **_xa("bf16", 4, 3600, 300, 8, 8, 40, "keys", True)},
        # a 90 x 160 map asks a 45 x 80 one
        {"name": "xa_bf16_14400q_3600k", **_xa("bf16", 1, 14400, 3600, 8, 8, 64)},
        # a 180 x 320 map asks a 45 x 80 one with wide heads: the largest
        {"name": "xa_bf16_57600q_3600k_d128", **_xa("bf16", 1, 57600, 3600, 4, 4, 128)},
        # one token for each of eight images asks a long context whose heads are shared by four
        {"name": "xa_bf16_8x1q_30001k", **_xa("bf16", 8, 1, 30001, 16, 4, 128)},
        # fp32, regions of the image with prompts of their own, some pixels with none
        {"name": "xa_f32_2x3600q_1000k_regions", **_xa("fp32", 2, 3600, 1000, 4, 4, 48, "regions")},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.4:
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        c = rng.choice([32, 48, 64, 96, 128, 192, 256, 320, 384, 512, 768, 1024])
        n = rng.choice([1, 1, 2, 4])
        area = _log_int(rng, 64, 720 * 1280 * 64 // ((2 if dtype == "fp32" else 1) * n * c))
        h = max(1, min(area, int(math.sqrt(area * math.exp(rng.uniform(math.log(0.4), math.log(2.5)))))))
        return _gn(dtype, n, h, area // h, c, rng.choice([g for g in (8, 16, 32) if c % g == 0]),
                   rng.choice(["silu", "silu", "gelu", "none"]), rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    d = rng.choice([32, 40, 48, 64, 64, 80, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    kind = rng.choice(["prompt", "prompt", "map", "token"])
    n = rng.choice([1, 1, 2, 4])
    if kind == "token":
        lq, lk = rng.choice([1, 1, 2, 5, 16]), _log_int(rng, 64, 245760 * 512 // (n * kv_heads * d * (2 if dtype == "fp32" else 1)))
    else:
        lk = _log_int(rng, 1, 1000) if kind == "prompt" else _log_int(rng, 200, 14400)
        lq = _log_int(rng, 16, 57600)
        most = 57600 * 3600 * 4 * (128 if dtype == "bf16" else 12)  # products of q and k, and scores, of the largest
        while n * heads * lq * lk * max(d, 128 if dtype == "bf16" else 12) > most:
            lq = max(1, lq * 3 // 4)
    return _xa(dtype, n, lq, lk, heads, kv_heads, d, rng.choice(["none", "none", "keys", "regions"]), rng.random() < 0.5)


# ------------------------------------------------------------------------------- inputs
def _kept(case):
    """Kept keys of each image under "keys": full prompts down to an empty one (one image: three quarters)."""
    n, lk = case["n"], case["lk"]
    return [lk - lk // 4] if n == 1 else [lk * (n - 1 - i) // (n - 1) for i in range(n)]


def _regions(case):
    """Under "regions" the queries fall into four bands and the keys into three prompts: band b sees prompt b,
    the last band sees none. The first query and first key of each."""
    return [case["lq"] * b // 4 for b in range(4)], [case["lk"] * b // 3 for b in range(4)]


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device=dev).mul_(scale).add_(shift)
    if case["op"] == "group_norm":
        n, c = case["n"], case["c"]
        chan = randn(c)  # feature maps have channels with means and sizes of their own
        x = (randn(n, case["h"], case["w"], c) * (0.5 + randn(c).abs()) + chan).to(dt)
        ab = (n, c) if case["per_image"] else (c,)
        return {"case": case, "x": x, "weight": randn(*ab, scale=0.2, shift=1.0), "bias": randn(*ab, scale=0.2)}
    n, lq, lk, d = case["n"], case["lq"], case["lk"], case["d"]
    ck = case["kv_heads"] * d
    q = randn(n, lq, case["heads"] * d, scale=1.5).to(dt)
    if case["joint"]:  # one projection made both: k and v are slices of its rows
        kv = randn(n, lk, 2 * ck).to(dt)
        k, v = kv[..., :ck], kv[..., ck:]
    else:
        k, v = randn(n, lk, ck).to(dt), randn(n, lk, ck).to(dt)
    mask = None
    if case["mask"] == "keys":
        mask = torch.arange(lk, device=dev)[None] < torch.tensor(_kept(case), device=dev)[:, None]
    elif case["mask"] == "regions":
        qs, ks = _regions(case)
        at, key = torch.arange(lq, device=dev), torch.arange(lk, device=dev)
        band = sum((at >= s).long() for s in qs[1:])
        prompt = sum((key >= s).long() for s in ks[1:3])
        mask = (band[:, None] == prompt[None]).expand(n, lq, lk)
    return {"case": case, "q": q, "k": k, "v": v, "mask": mask}


# ------------------------------------------------------------------------------- one pass
def _plain_group_norm(x, groups, weight, bias, act):
    n, h, w, c = x.shape
    y = x.float().reshape(n, h * w, groups, c // groups)
    y = y - y.mean((1, 3), keepdim=True)
    y = y * torch.rsqrt(y.square().mean((1, 3), keepdim=True) + EPS)
    y = y.reshape(n, h, w, c) * weight.reshape(-1, 1, 1, c) + bias.reshape(-1, 1, 1, c)
    if act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "gelu":
        y = y * (0.5 + 0.5 * torch.erf(y * math.sqrt(0.5)))
    return y.to(x.dtype)


def _plain_attention(q, k, v, heads, kv_heads, mask):
    n, lq, c = q.shape
    lk, d, rep = k.shape[1], c // heads, heads // kv_heads
    if mask is not None and mask.dim() == 2:
        v = v.masked_fill(~mask[..., None], 0)
        mask = mask[:, None]
    qh = q.float().reshape(n, lq, kv_heads, rep, d).permute(0, 2, 3, 1, 4).reshape(n * kv_heads, rep * lq, d)
    kt = k.float().reshape(n, lk, kv_heads, d).permute(0, 2, 3, 1).contiguous().reshape(n * kv_heads, d, lk)
    vh = v.float().reshape(n, lk, kv_heads, d).permute(0, 2, 1, 3).contiguous().reshape(n * kv_heads, lk, d)
    s = torch.bmm(qh, kt).mul_(d ** -0.5)
    if mask is not None:
        s.view(n, heads, lq, lk).masked_fill_(~mask[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.bmm(s, vh) / torch.where(total == 0, torch.ones_like(total), total)
    return o.reshape(n, kv_heads, rep, lq, d).permute(0, 3, 1, 2, 4).reshape(n, lq, c).to(q.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "group_norm":
        act = case["act"]
        if own:
            return _ops(state["x"].dtype).group_norm(state["x"], case["groups"], state["weight"], state["bias"], eps=EPS,
                                                     act=None if act == "none" else act)
        return _plain_group_norm(state["x"], case["groups"], state["weight"], state["bias"], act)
    q, k, v, mask = state["q"], state["k"], state["v"], state["mask"]
    if own:
        return _ops(q.dtype).cross_attention(q, k, v, case["heads"], kv_heads=case["kv_heads"], mask=mask)
    return _plain_attention(q, k, v, case["heads"], case["kv_heads"], mask)


# ------------------------------------------------------------------------------- what a pass needs
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "group_norm":
        elems = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": 2 * elems * es + 8 * case["c"] * (case["n"] if case["per_image"] else 1), "flops": 10 * elems}
    n, lq, lk, d, heads, kv = (case[i] for i in ("n", "lq", "lk", "d", "heads", "kv_heads"))
    pairs, rows, mask = n * lq * lk, n * lk, 0
    if case["mask"] == "keys":  # masked keys are not needed
        rows = sum(_kept(case))
        pairs, mask = lq * rows, n * lk
    elif case["mask"] == "regions":
        qs, ks = _regions(case)
        pairs, mask = n * sum((qs[b + 1] - qs[b]) * (ks[b + 1] - ks[b]) for b in range(3)), lq * lk
    return {"bytes": es * d * (2 * n * lq * heads + 2 * rows * kv) + mask, "flops": 4 * pairs * heads * d}


# ------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    t = prepare(case, seed)
    if case["op"] == "group_norm":
        x = t["x"].double()
        out = torch.empty_like(x)
        size = case["c"] // case["groups"]
        wt, bs = (t[i].double().expand(case["n"], case["c"]) for i in ("weight", "bias"))
        for i in range(case["n"]):
            for g in range(case["groups"]):
                sl = slice(g * size, (g + 1) * size)
                var, mean = torch.var_mean(x[i, ..., sl], correction=0)
                out[i, ..., sl] = (x[i, ..., sl] - mean) / torch.sqrt(var + EPS) * wt[i, sl] + bs[i, sl]
        if case["act"] == "silu":
            return out * torch.sigmoid(out)
        return out * torch.special.ndtr(out) if case["act"] == "gelu" else out
    d, rep = case["d"], case["heads"] // case["kv_heads"]
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device=t["q"].device)
    step = max(1, (1 << 27) // case["lk"])
    for i in range(case["n"]):
        for h in range(case["heads"]):
            at, kv = slice(h * d, (h + 1) * d), slice(h // rep * d, (h // rep + 1) * d)
            keys, vals = t["k"][i, :, kv].double(), t["v"][i, :, kv].double()
            for a in range(0, case["lq"], step):
                z = (t["q"][i, a:a + step, at].double() / math.sqrt(d)) @ keys.t().contiguous()
                seen = torch.ones_like(z, dtype=torch.bool)
                if t["mask"] is not None:
                    seen &= t["mask"][i, a:a + step] if t["mask"].dim() == 3 else t["mask"][i][None]
                z = torch.softmax(z.masked_fill(~seen, -1e300), -1) * seen
                out[i, a:a + step, at] = z @ vals
    return out
