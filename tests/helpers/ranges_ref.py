"""The attention-block operators in 64 bits, from their definitions, with the error bounds their roundings allow."""
import math

import torch

U = 2.0 ** -8            # half a step of bf16, relative


def rotate64(x, pos, freq, axis, halves, sign=1.0):
    """x [B, L, H, D] float64; pos [B or 1, L, axes]"""
    P = freq.numel()
    ang = pos.double()[..., axis.long()] * freq
    c, s = ang.cos()[:, :, None], sign * ang.sin()[:, :, None]
    i0 = torch.arange(P) if halves else 2 * torch.arange(P)
    i1 = i0 + P if halves else i0 + 1
    y = x.clone()
    y[..., i0] = c * x[..., i0] - s * x[..., i1]
    y[..., i1] = s * x[..., i0] + c * x[..., i1]
    return y


def heads64(x, w, pos, freq, axis, halves, eps=1e-6, scale=1.0):
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    return rotate64(x, pos, freq, axis, halves) * scale


def scores64(q, k, mask, scale, bias, pos, cap):
    """(t with -inf where hidden, tanh or None, visible) [B, H, Lq, Lk]"""
    B, Lq, H, D = q.shape
    Lk, G = k.shape[1], H // k.shape[2]
    kk = k.double().repeat_interleave(G, 2)
    t = torch.einsum("bihd,bjhd->bhij", q.double(), kk) * scale
    th = None
    if cap:
        th = torch.tanh(t / cap)
        t = cap * th
    seen = torch.ones(B, 1, Lq, Lk, dtype=torch.bool) if mask is None else mask[:, None].expand(B, 1, Lq, Lk)
    seen = seen.expand(B, H, Lq, Lk)
    if bias is not None:
        R = bias.shape[1] // 2
        p = (torch.arange(Lq)[None] + Lk - Lq) if pos is None else pos.long()
        idx = (torch.arange(Lk) - p[..., None]).clamp(-R, R) + R                  # [B or 1, Lq, Lk]
        b = bias.double()[:, idx].transpose(0, 1)                                # [B or 1, H, Lq, Lk]
        seen = seen & (b > -1e30)
        t = t + b.clamp(min=-1e30)
    return torch.where(seen, t, -math.inf), th, seen


def attention64(q, k, v, mask=None, scale=None, bias=None, pos=None, cap=0.0):
    """out [B, Lq, H, D], lse [B, H, Lq], bound on the error of the kernel's out (P and the result rounded to bf16 once each;
    2^-13 covers the 32-bit scores, exponentials and sums)"""
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    t, _, seen = scores64(q, k, mask, scale, bias, pos, cap)
    vv = v.double().repeat_interleave(q.shape[2] // k.shape[2], 2).transpose(1, 2)   # [B, H, Lk, D]
    if t.shape[-1] == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, torch.full(t.shape[:3], -math.inf, dtype=torch.float64), z
    lse = torch.logsumexp(t, -1)
    p = torch.where(seen, torch.exp(t - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)

    def product(p, vv):
        if torch.isfinite(vv).all():
            return p @ vv
        return torch.where(seen[..., None], p[..., None] * vv[:, :, None], 0.0).sum(-2)    # hidden keys do not enter at all
    o, mag = product(p, vv).transpose(1, 2), product(p, vv.abs()).transpose(1, 2)
    return o, lse, U * (mag + o.abs()) + 2.0 ** -13 * mag + 1e-30


def attention_grad64(do, q, k, v, out, lse, mask=None, scale=None, bias=None, pos=None, cap=0.0):
    """dict name -> (gradient, bound on the kernel's error): P and dZ rounded once as operands, the result once"""
    B, Lq, H, D = q.shape
    Hkv, G = k.shape[2], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    t, th, seen = scores64(q, k, mask, scale, bias, pos, cap)
    lse = lse.double()[..., None]
    p = torch.where(seen, torch.exp(t - torch.where(lse == -math.inf, 0.0, lse)), 0.0)
    dod, qd = do.double().transpose(1, 2), q.double().transpose(1, 2)
    kd, vd = (x.double().repeat_interleave(G, 2).transpose(1, 2) for x in (k, v))
    delta = (dod * out.double().transpose(1, 2)).sum(-1, keepdim=True)
    dp = dod @ vd.transpose(-1, -2)
    dt = torch.where(seen, p * (dp - delta), 0.0)
    dz = dt if th is None else dt * (1 - th * th)
    # 32-bit error of dT itself: P to 2^-14, dP - delta to 2^-20 of the sums of magnitudes
    mag = torch.where(seen, p * (dod.abs() @ vd.abs().transpose(-1, -2) + (dod * out.double().transpose(1, 2)).abs().sum(-1, keepdim=True)), 0.0)
    slack = 2.0 ** -14 * dt.abs() + 2.0 ** -20 * mag

    def shared(x):                                            # [B, H, Lk, D] -> [B, Lk, Hkv, D]
        return x.unflatten(1, (Hkv, G)).sum(2).transpose(1, 2)
    dq, dk, dv = (dz @ kd * scale).transpose(1, 2), shared(dz.transpose(-1, -2) @ qd * scale), shared(p.transpose(-1, -2) @ dod)
    ez = U * dz.abs() + slack
    eq = (ez @ kd.abs() * scale).transpose(1, 2)
    ek = shared(ez.transpose(-1, -2) @ qd.abs() * scale)
    ev = shared((U + 2.0 ** -13) * p.transpose(-1, -2) @ dod.abs())
    # sums over n terms in 32 bits stay far below the 2^-13 of the magnitudes that the slack holds
    r = dict(dq=(dq, eq + U * dq.abs() + 1e-30), dk=(dk, ek + U * dk.abs() + 1e-30), dv=(dv, ev + U * dv.abs() + 1e-30))
    if bias is not None:
        R = bias.shape[1] // 2
        pp = (torch.arange(Lq)[None] + k.shape[1] - Lq) if pos is None else pos.long()
        idx = ((torch.arange(k.shape[1]) - pp[..., None]).clamp(-R, R) + R).expand(B, Lq, k.shape[1])
        db, eb = torch.zeros(H, 2 * R + 1, dtype=torch.float64), torch.zeros(H, 2 * R + 1, dtype=torch.float64)
        for b in range(B):
            for h in range(H):
                db[h].index_add_(0, idx[b].flatten(), dt[b, h].flatten())
                eb[h].index_add_(0, idx[b].flatten(), (slack[b, h] + 2.0 ** -20 * dt[b, h].abs()).flatten())
        r["dbias"] = (db, eb + 1e-30)
    return r


def within(got, want, bound):
    """largest error in units of its bound; infinities and NaN have to agree in kind"""
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), "finite in different places"
    if not fine.any():
        return 0.0
    return ((got - want).abs()[fine] / bound.expand_as(want)[fine]).max().item()
