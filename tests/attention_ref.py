"""The soft reads from their definitions, in 64 bits on the host or the device of the inputs, and how far 16-bit
kernels may be from them."""
import math

import torch


def visible(lengths, b, lq, lk, causal, device):
    """[b, lq, lk]: which keys a query sees."""
    n = torch.full((b,), lk, device=device) if lengths is None else lengths.to(device).long().clamp(0, lk)
    end = n.view(b, 1).expand(b, lq)
    if causal:
        end = end - lq + 1 + torch.arange(lq, device=device)
    return torch.arange(lk, device=device) < end.unsqueeze(-1)


def heads_first(x, heads):
    """[b, n, hk, d] -> [b, heads, n, d] in 64 bits."""
    return x.double().permute(0, 2, 1, 3).repeat_interleave(heads // x.shape[2], 1)


def scores(q, k, lengths, scale, causal):
    """[b, heads, lq, lk], -inf where hidden; what lies in hidden rows has no influence."""
    s = heads_first(q, q.shape[2]) @ heads_first(k, q.shape[2]).transpose(-1, -2) * scale
    seen = visible(lengths, q.shape[0], q.shape[1], k.shape[1], causal, q.device).unsqueeze(1)
    return torch.where(seen, s, torch.full_like(s, -math.inf))


def softmax(s):
    lse = torch.logsumexp(s, -1) if s.shape[-1] else s.new_full(s.shape[:-1], -math.inf)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse).unsqueeze(-1))
    return p, lse


def live(x, seen_any):
    """Rows that no query sees as zeros, so that NaN in them does not come through 0 * NaN."""
    return torch.where(seen_any.view(*seen_any.shape, 1, 1), x, torch.zeros_like(x))


def attend(q, k, v, lengths=None, scale=None, causal=False, shared=None):
    """out [b, lq, h, d], lse [b, lq, h] and the mean absolute weight-value sum that errors scale with."""
    b, lq, h, d = q.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    s = scores(q, k, lengths, scale, causal)
    seen = visible(lengths, b, lq, k.shape[1], causal, q.device).any(1)
    vv = heads_first(live(v, seen), h)
    if shared is not None:
        sk, sv = (x.unsqueeze(0).expand(b, *x.shape) for x in shared)
        s = torch.cat([scores(q, sk, None, scale, False), s], -1)
        vv = torch.cat([heads_first(sv, h), vv], -2)
    p, lse = softmax(s)
    return (p @ vv).permute(0, 2, 1, 3), lse.permute(0, 2, 1), (p @ vv.abs()).permute(0, 2, 1, 3)


def backward(grad, q, k, v, lengths=None, scale=None):
    """grad_q, grad_k, grad_v and, for each, the sum of the absolute terms."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    seen = visible(lengths, b, lq, lk, False, q.device).any(1) if lq else torch.zeros(b, lk, dtype=torch.bool, device=q.device)
    k, v = live(k, seen), live(v, seen)
    p, _ = softmax(scores(q, k, lengths, scale, False))
    g, qq, kk, vv = heads_first(grad, h), heads_first(q, h), heads_first(k, h), heads_first(v, h)
    dp = g @ vv.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    ads = p * (g.abs() @ vv.abs().transpose(-1, -2) + (p * (g.abs() @ vv.abs().transpose(-1, -2))).sum(-1, keepdim=True)) * scale

    def group(x):
        return x.view(b, hk, h // hk, lk, d).sum(2).permute(0, 2, 1, 3)

    out = ((ds @ kk).permute(0, 2, 1, 3), group(ds.transpose(-1, -2) @ qq), group(p.transpose(-1, -2) @ g))
    size = ((ads @ kk.abs()).permute(0, 2, 1, 3), group(ads.transpose(-1, -2) @ qq.abs()), group(p.transpose(-1, -2) @ g.abs()))
    return out, size


def mass(q, k, lse, lengths=None, scale=None, causal=False, start=None):
    b, lq, h, d = q.shape
    hk = k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    s = scores(q, k, lengths, scale, causal)
    row = lse.double().permute(0, 2, 1).unsqueeze(-1)
    p = torch.exp(s - torch.where(row == -math.inf, torch.zeros_like(row), row))
    out = p.view(b, hk, h // hk * lq, k.shape[1]).sum(2)
    return out + (0 if start is None else start.double())


def evict(k, v, m, lengths, keep, recent):
    b, n, hk, d = k.shape
    ok, ov = torch.zeros(b, keep, hk, d, dtype=k.dtype), torch.zeros(b, keep, hk, d, dtype=k.dtype)
    om, rows, new = torch.zeros(b, hk, keep), torch.full((b, hk, keep), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        top = n if lengths is None else min(max(int(lengths[i]), 0), n)
        new[i] = min(top, keep)
        for h in range(hk):
            w = m[i, h, :max(top - recent, 0)].tolist()
            if top <= keep:
                chosen = list(range(top))
            else:
                best = sorted(range(top - recent), key=lambda j: (0 if w[j] != w[j] else 1, -w[j] if w[j] == w[j] else 0, j))
                chosen = sorted(best[:keep - recent]) + list(range(top - recent, top))
            for s, j in enumerate(chosen):
                ok[i, s, h], ov[i, s, h], om[i, h, s], rows[i, h, s] = k[i, j, h], v[i, j, h], m[i, h, j], j
    return ok, ov, om, rows, new
