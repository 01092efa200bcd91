"""TEST ORACLE: the reference PyTorch backend's semantics for the GEMM-family ops, in fp32.

Restated from python/clarus/ops/torch_ref.py (cited per method). Math runs in fp32 on the
device of the inputs (the CPU in tests and in bench.py's cpu_baseline) and is cast to the
output dtype at the end of each op, exactly where the reference casts. Only tests/, smoke()
and bench.py's cpu_baseline may use this module.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F


@dataclass
class Small:
    """TLC local-mean map (torch_ref.py:18-33): data [N, oh, ow, C]; full-resolution value at
    (y, x) = data[clamp(y - pt, 0, oh - 1), clamp(x - pl, 0, ow - 1)]."""

    data: torch.Tensor
    pt: int
    pl: int
    H: int
    W: int

    def with_data(self, data):
        return Small(data, self.pt, self.pl, self.H, self.W)


def box_geometry(h: int, w: int, k):
    """torch_ref.py:36-41: (k1, k2, oh, ow, pt, pl) of a (kh, kw) valid local mean."""
    kh, kw = (k, k) if isinstance(k, int) else k
    k1, k2 = min(h, kh), min(w, kw)
    oh, ow = h - k1 + 1, w - k2 + 1
    return k1, k2, oh, ow, (h - oh) // 2, (w - ow) // 2


def _is_small(x) -> bool:
    return not torch.is_tensor(x) and hasattr(x, "data") and hasattr(x, "pt")


def _to_nchw(x):
    return x.permute(0, 3, 1, 2)


def _to_nhwc(x):
    return x.permute(0, 2, 3, 1).contiguous()


class TorchRef:
    """The reference backend's op semantics; `dtype` is the activation dtype."""

    name = "oracle"

    def __init__(self, dtype: torch.dtype = torch.float32, device="cpu"):
        self.dtype = dtype
        self.device = torch.device(device)

    # ---------------------------------------------------------------- helpers
    @staticmethod
    def expand(s) -> torch.Tensor:
        """torch_ref.py:85-91: replicate-pad the local-mean map to full resolution."""
        oh, ow = s.data.shape[1], s.data.shape[2]
        rows = torch.clamp(torch.arange(s.H, device=s.data.device) - s.pt, 0, oh - 1)
        cols = torch.clamp(torch.arange(s.W, device=s.data.device) - s.pl, 0, ow - 1)
        return s.data[:, rows][:, :, cols]

    @staticmethod
    def ln(x, eps=1e-6, rms=False):
        """torch_ref.py:93-100: two-pass LayerNorm (no affine) or RMS norm over the last dim."""
        x = x.float()
        if rms:
            return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        centred = x - x.mean(-1, keepdim=True)
        return centred * torch.rsqrt(centred.square().mean(-1, keepdim=True) + eps)

    def _odt(self, out_dtype):
        return out_dtype or self.dtype

    # ---------------------------------------------------------------- GEMM family
    def linear(self, x, w, bias=None, ln=False, act=None, gate=False, scale=None,
               residual=None, mul=None, out_dtype=None, ln_eps=1e-6):
        """torch_ref.py:103-131. Order: (* expand(mul)) -> LN -> @ w -> + bias -> gate -> GELU
        -> * scale -> + residual -> cast."""
        if _is_small(x):
            return x.with_data(self.linear(x.data, w, bias, ln, act, gate, scale, residual, mul, out_dtype, ln_eps))
        a = x.float()
        if mul is not None:
            a = a * self.expand(mul).float()
        if ln:
            a = self.ln(a, ln_eps, rms=(ln == "rms"))
        y = a @ w.float()
        if bias is not None:
            y = y + bias
        if gate:
            half = y.shape[-1] // 2
            y = y[..., :half] * y[..., half:]
        if act == "gelu":
            y = F.gelu(y)
        if scale is not None:
            y = y * scale
        if residual is not None:
            y = residual.float() + y
        return y.to(self._odt(out_dtype))

    def intro(self, inp, w, b, out_dtype=None):
        """torch_ref.py:157-158: 3x3 conv (pad 1) of the NCHW image -> NHWC."""
        return _to_nhwc(F.conv2d(inp.float(), w.float(), b, padding=1)).to(self._odt(out_dtype))

    def down(self, x, w4d, b, out_dtype=None):
        """torch_ref.py:160-161: 2x2 stride-2 conv."""
        return _to_nhwc(F.conv2d(_to_nchw(x).float(), w4d.float(), b, stride=2)).to(self._odt(out_dtype))

    def up(self, x, w, residual=None, out_dtype=None):
        """torch_ref.py:163-171: 1x1 conv to 4C' (N ordered (dy, dx, c')) + PixelShuffle(2)."""
        n, h, wd, _ = x.shape
        y = x.float() @ w.float()
        cq = y.shape[-1] // 4
        y = y.reshape(n, h, wd, 2, 2, cq).permute(0, 1, 3, 2, 4, 5).reshape(n, 2 * h, 2 * wd, cq)
        if residual is not None:
            y = y + residual.float()
        return y.to(self._odt(out_dtype))

    def ending(self, x, w, b, inp):
        """torch_ref.py:173-175: final 3x3 conv + global residual -> fp32 NCHW."""
        return F.conv2d(_to_nchw(x).float(), w.float(), b, padding=1) + inp

    def conv3x3(self, x, w, b=None, out_dtype=None, act=None, residual=None, out_scale=1.0, up2=False,
                out=None, slope=0.2):
        """torch_ref.py:178-199: y = act(conv3x3(up2?(x)) + b) * out_scale (+ residual)."""
        xi = _to_nchw(x).float()
        if up2:
            xi = F.interpolate(xi, scale_factor=2, mode="nearest")
        y = F.conv2d(xi, w.float(), b, padding=1).permute(0, 2, 3, 1)
        if act == "lrelu":
            y = F.leaky_relu(y, slope)
        if out_scale != 1.0:
            y = y * out_scale
        if residual is not None:
            y = y + residual.float()
        if out is not None:
            out.copy_(y)
            return out
        return y.contiguous().to(self._odt(out_dtype))

    def group_norm(self, x, groups, weight=None, bias=None, eps=1e-5, act=None, out_dtype=None):
        """No reference op: torch's group norm (biased variance, eps inside the root) of x [N, ..., C]
        channels last, weight and bias [C] or [N, C], then SiLU / GELU."""
        n, c = x.shape[0], x.shape[-1]
        y = x.float().reshape(n, -1, groups, c // groups)
        y = y - y.mean((1, 3), keepdim=True)
        y = (y * torch.rsqrt(y.square().mean((1, 3), keepdim=True) + eps)).reshape(n, -1, c)
        if weight is not None:
            y = y * weight.float().reshape(-1, 1, c)
        if bias is not None:
            y = y + bias.float().reshape(-1, 1, c)
        y = F.silu(y) if act == "silu" else F.gelu(y) if act == "gelu" else y
        return y.reshape(x.shape).to(self._odt(out_dtype))

    def cross_attention(self, q, k, v, heads, kv_heads=None, mask=None, scale=None, out_dtype=None):
        """No reference op: softmax(scale q k^T) v per head over the kept keys, 0 where none is kept; a key
        that a [N, Lk] mask drops counts for nothing whatever it holds."""
        kv_heads = kv_heads or heads
        n, d, rep = q.shape[0], q.shape[-1] // heads, heads // kv_heads
        qh = q.float().reshape(n, -1, heads, d).permute(0, 2, 1, 3)
        kh, vh = (t.float().reshape(n, -1, kv_heads, d).permute(0, 2, 1, 3).repeat_interleave(rep, 1) for t in (k, v))
        s = (qh @ kh.transpose(-1, -2).contiguous()) * (d ** -0.5 if scale is None else scale)
        if mask is not None:
            if mask.dim() == 2:
                vh = vh.masked_fill(~mask[:, None, :, None], 0)
            s = s.masked_fill(~(mask[:, None, None] if mask.dim() == 2 else mask[:, None]), float("-inf"))
        none = torch.isneginf(s).all(-1, keepdim=True)
        p = torch.softmax(s.masked_fill(none, 0), -1).masked_fill(none, 0)
        return (p @ vh).permute(0, 2, 1, 3).reshape(q.shape).to(self._odt(out_dtype))

    def rotary(self, x, heads, sections, positions=None, base=10000.0, pairs="adjacent", out_dtype=None):
        """No reference op: pairs of each head's columns turned by position * base^(-i / pairs of the axis)."""
        n, d, p = x.shape[0], x.shape[-1] // heads, sum(sections)
        y = x.float().reshape(n, -1, heads, d)
        if positions is None:
            positions = torch.cartesian_prod(*[torch.arange(s, device=x.device) for s in x.shape[1:-1]]).reshape(-1, x.dim() - 2)
        t = torch.cat([positions[..., a, None].double() * base ** (-torch.arange(s, device=x.device).double() / s)
                       for a, s in enumerate(sections)], -1).reshape(-1, y.shape[1], 1, p)
        cos, sin = t.cos().float(), t.sin().float()
        z = y[..., :2 * p]
        a, b = z.unflatten(-1, (p, 2)).unbind(-1) if pairs == "adjacent" else z.chunk(2, -1)
        a, b = a * cos - b * sin, b * cos + a * sin
        z = torch.stack((a, b), -1).flatten(-2) if pairs == "adjacent" else torch.cat((a, b), -1)
        return torch.cat((z, y[..., 2 * p:]), -1).reshape(x.shape).to(self._odt(out_dtype))

    def add_norm(self, x, y=None, gate=None, scale=1.0, post=False, post_weight=None, post_bias=None, ln=True, weight=None,
                 bias=None, eps=1e-6, out_dtype=None):
        """No reference op: (x + scale gate (post(y) pw + pb), ln(that) w + b), vectors [C] or [N, C]."""
        n, c = x.shape[0], x.shape[-1]

        def norm(v, kind, w, b):
            if kind:
                v = v - v.mean(-1, keepdim=True) if kind != "rms" else v
                v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
            v = v if w is None else v * w.float().reshape(-1, 1, c)
            return v if b is None else v + b.float().reshape(-1, 1, c)
        r = x.float().reshape(n, -1, c)
        if y is not None:
            add = norm(y.float().reshape(n, -1, c), post, post_weight, post_bias) * scale
            r = r + (add if gate is None else add * gate.float().reshape(-1, 1, c))
        h = norm(r, ln, weight, bias).reshape(x.shape).to(self._odt(out_dtype)) if ln else None
        return r.reshape(x.shape).to(x.dtype), h

    def block_means(self, k, block=64, mask=None):
        """No reference op: means of the kept rows of each block, in 64 bits, as fp32."""
        k = k.reshape(k.shape[0], -1, k.shape[-1]).double()
        keep = torch.ones(k.shape[:2], dtype=torch.bool, device=k.device) if mask is None else mask
        k = k.masked_fill(~keep[..., None], 0)
        return torch.stack([a.sum(1) / b.sum(1, keepdim=True) for a, b in zip(k.split(block, 1), keep.split(block, 1))], 1).float()

    def sparse_attention(self, q, k, v, heads, top, kv_heads=None, block=64, group=1, mask=None, means=None, scale=None, out_dtype=None,
                         return_blocks=False):
        """No reference op: cross_attention under a mask that keeps, for each head and group of queries, the blocks of keys
        of the `top` largest products of means."""
        kv_heads = kv_heads or heads
        n, d, rep = q.shape[0], q.shape[-1] // heads, heads // kv_heads
        q3, k3, v3 = (t.reshape(n, -1, t.shape[-1]) for t in (q, k, v))
        lq, lk = q3.shape[1], k3.shape[1]
        m = (self.block_means(k3, block, mask) if means is None else means).double()
        a = torch.stack([t.double().mean(1) for t in q3.split(group, 1)], 1).float().double() if group > 1 else q3.double()
        kept = torch.ones(n, lk, dtype=torch.bool, device=q.device) if mask is None else mask
        out, chosen = torch.zeros(n, lq, heads * d, device=q.device), []
        for h in range(heads):
            sl, kv = slice(h * d, h * d + d), slice(h // rep * d, h // rep * d + d)
            score = a[..., sl] @ m[..., kv].transpose(1, 2).contiguous()
            score = score.nan_to_num(nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
            order = score.sort(dim=-1, descending=True, stable=True)[1][..., :top]
            pick = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True) & (score > -float("inf"))
            chosen.append(pick)
            see = pick.repeat_interleave(group, 1)[:, :lq].repeat_interleave(block, 2)[..., :lk] & kept[:, None]
            out[..., sl] = self.cross_attention(q3[..., sl], k3[..., kv].masked_fill(~kept[..., None], 0),
                                                v3[..., kv].masked_fill(~kept[..., None], 0), 1, mask=see,
                                                scale=d ** -0.5 if scale is None else scale, out_dtype=torch.float32)
        out = out.reshape(q.shape).to(self._odt(out_dtype))
        return (out, torch.stack(chosen, 1)) if return_blocks else out

    def linear_attention(self, q, k, v, log_decay, heads, kv_heads=None, state=None, scale=None, state_out=None, out_dtype=None):
        """No reference op: S <- e^g S + k v^T, out = scale q^T S, token after token."""
        kv_heads = kv_heads or heads
        n, rep, dk = q.shape[0], heads // kv_heads, q.shape[-1] // heads
        qh = q.float().reshape(n, -1, kv_heads, rep, dk) * (dk ** -0.5 if scale is None else scale)
        kh, vh = (t.float().reshape(n, qh.shape[1], kv_heads, -1) for t in (k, v))
        s = torch.zeros(n, kv_heads, dk, vh.shape[-1], device=q.device) if state is None else state.clone()
        f = log_decay.float().exp()[:, None, None]
        out = []
        for t in range(qh.shape[1]):
            s = s * f + kh[:, t, :, :, None] * vh[:, t, :, None]
            out.append(qh[:, t] @ s)
        y = torch.stack(out, 1).reshape(*q.shape[:-1], -1).to(self._odt(out_dtype))
        return (y, s) if state_out is None else (y, state_out.copy_(s))

    def channel_attention(self, qkv, heads, temperature):
        """torch_ref.py:220-235: softmax((q/|q|)(k/|k|)^T * t) per image and head, fp32."""
        n, h, w, c3 = qkv.shape
        c = c3 // 3
        ch = c // heads
        q = qkv[..., :c].reshape(n, h * w, heads, ch).float().permute(0, 2, 3, 1)      # [n, hd, ch, P]
        k = qkv[..., c:2 * c].reshape(n, h * w, heads, ch).float().permute(0, 2, 1, 3)  # [n, hd, P, ch]
        g = torch.matmul(q, k)
        nq = q.square().sum(-1).clamp_min(1e-24).rsqrt()
        nk = k.square().sum(-2).clamp_min(1e-24).rsqrt()
        g = g * nq[..., :, None] * nk[..., None, :] * temperature.reshape(1, heads, 1, 1).float()
        return torch.softmax(g, dim=-1)

    def linear_per_image(self, x, w, residual=None, out_dtype=None, bias=None):
        """torch_ref.py:237-245: per image x[i] @ w[i] (+ bias, + residual)."""
        n, h, wd, k = x.shape
        y = torch.bmm(x.reshape(n, h * wd, k).float(), w.float()).reshape(n, h, wd, -1)
        if bias is not None:
            y = y + bias
        if residual is not None:
            y = y + residual.float()
        return y.to(self._odt(out_dtype))

    def patch_filter(self, x, f, residual=None, out_dtype=None):
        """torch_ref.py:253-270: per p x p patch and channel irfft2(rfft2(patch) * f[c]),
        reflect-padding sizes that are not multiples of p (result cropped)."""
        n, h, w, c = x.shape
        p = f.shape[1]
        xi = _to_nchw(x).float()
        ph, pw = (-h) % p, (-w) % p
        if ph or pw:
            xi = F.pad(xi, (0, pw, 0, ph), mode="reflect")
        hh, ww = h + ph, w + pw
        patches = xi.reshape(n, c, hh // p, p, ww // p, p).permute(0, 1, 2, 4, 3, 5)
        spec = torch.fft.rfft2(patches) * f.float().reshape(1, c, 1, 1, p, p // 2 + 1)
        y = torch.fft.irfft2(spec, s=(p, p))
        y = y.permute(0, 2, 4, 3, 5, 1).reshape(n, hh, ww, c)[:, :h, :w]
        if residual is not None:
            y = y + residual.float()
        return y.contiguous().to(self._odt(out_dtype))

    def linear_patch_filter(self, x, w, bias, f, ln=False, ln_eps=1e-6, residual=None):
        """torch_ref.py:272-276: patch_filter(linear(x, w, bias, ln) kept fp32, f, residual)."""
        y = self.linear(x, w, bias, ln=ln, ln_eps=ln_eps, out_dtype=torch.float32)
        return self.patch_filter(y, f, residual=residual)

    def patch_corr(self, x, c, p=8):
        """torch_ref.py:278-288: per patch irfft2(rfft2(q) * rfft2(k)) -> fp32 [N, H, W, c]."""
        n, h, w, _ = x.shape

        def patches(t):
            return _to_nchw(t).float().reshape(n, c, h // p, p, w // p, p).permute(0, 1, 2, 4, 3, 5)
        spec = torch.fft.rfft2(patches(x[..., :c])) * torch.fft.rfft2(patches(x[..., c:2 * c]))
        y = torch.fft.irfft2(spec, s=(p, p))
        return y.permute(0, 2, 4, 3, 5, 1).reshape(n, h, w, c).contiguous()

    def ln_mul_linear(self, x, ln_w, ln_b, m, w, bias=None, m_act=None, residual=None, ln_eps=1e-5,
                      out_dtype=None):
        """torch_ref.py:290-302: ((LN(x) * ln_w + ln_b) * act(m)) @ w (+ bias, + residual)."""
        a = self.ln(x, ln_eps) * ln_w + ln_b
        mm = m.float()
        a = a * (F.gelu(mm) if m_act == "gelu" else mm)
        y = a @ w.float()
        if bias is not None:
            y = y + bias
        if residual is not None:
            y = y + residual.float()
        return y.to(self._odt(out_dtype))

    # ---------------------------------------------------------------- non-GEMM ops of the harnesses
    def boxmean(self, x, k):
        """torch_ref.py:133-141: valid local mean via a 2-D prefix sum (TLC)."""
        n, h, w, c = x.shape
        k1, k2, oh, ow, pt, pl = box_geometry(h, w, k)
        s = F.pad(x.float().cumsum(dim=2).cumsum(dim=1), (0, 0, 1, 0, 1, 0))
        win = s[:, k1:, k2:] + s[:, :-k1, :-k2] - s[:, :-k1, k2:] - s[:, k1:, :-k2]
        return Small((win / (k1 * k2)).to(self.dtype), pt, pl, h, w)

    def dwconv(self, x, w, b, dil=1, gate=False, act=None):
        """torch_ref.py:143-155: depthwise conv ('same'), optional gate / GELU."""
        kh, kw = w.shape[-2:]
        y = F.conv2d(_to_nchw(x).float(), w.float(), b, padding=(dil * (kh // 2), dil * (kw // 2)),
                     dilation=dil, groups=x.shape[-1]).permute(0, 2, 3, 1)
        if gate:
            half = y.shape[-1] // 2
            first = F.gelu(y[..., :half]) if gate == "gelu" else y[..., :half]
            y = first * y[..., half:]
        if act == "gelu":
            y = F.gelu(y)
        return y.contiguous().to(self.dtype)

    def selective_scan(self, u, dbl, dt_w, dt_bias, A, D, chunk=32):
        """torch_ref.py:312-341: Mamba selective scan along each crop's raster sequence, computed
        chunk by chunk in closed form: within a chunk, h_l = exp(S_l) h_in + sum_{s <= l}
        exp(S_l - S_s) delta_s B_s u_s with S the running sum of delta A; y_l = C_l . h_l + D u_l.
        delta = softplus(dt_raw @ dt_w^T + dt_bias); dbl = (dt_raw | B | C). Returns fp32."""
        t, hh, ww, d = u.shape
        L, r, ns = hh * ww, dt_w.shape[1], A.shape[1]
        u = u.reshape(t, L, d).float()
        dbl = dbl.reshape(t, L, -1).float()
        delta = F.softplus(dbl[..., :r] @ dt_w.float().t() + dt_bias.float())
        bm, cm = dbl[..., r:r + ns], dbl[..., r + ns:r + 2 * ns]
        a = A.float()
        state = torch.zeros(t, d, ns, device=u.device)
        out = []
        for s0 in range(0, L, chunk):
            dl, uc = delta[:, s0:s0 + chunk], u[:, s0:s0 + chunk]
            c = dl.shape[1]
            run = (dl[..., None] * a).cumsum(1)                                 # [t, c, d, n]
            inj = (dl * uc)[..., None] * bm[:, s0:s0 + c, None, :]            # [t, c, d, n]
            gap = run[:, :, None] - run[:, None, :]                            # [t, l, s, d, n]
            low = torch.ones(c, c, dtype=torch.bool, device=u.device).tril()
            decay = torch.where(low[None, :, :, None, None], gap, float("-inf")).exp()
            hs = run.exp() * state[:, None] + torch.einsum("tlsdn,tsdn->tldn", decay, inj)
            out.append(torch.einsum("tldn,tln->tld", hs, cm[:, s0:s0 + c]))
            state = hs[:, -1]
        y = torch.cat(out, 1) + u * D.float()
        return y.view(t, hh, ww, d)
