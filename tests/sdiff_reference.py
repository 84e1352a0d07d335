"""Plain 64-bit forms of softmax differential attention and of the 4-bit cache
for the tests; written from the formulas, no code of the package."""
import math

import torch

GROUP = 32


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    n = b.norm()
    return float((a - b).norm() / n) if n > 0 else float((a - b).norm())


def attention64(q1, q2, k1, k2, v, lam, scale=None, causal=True, lengths=None, dout=None):
    """out, or (out, dq1, dq2, dk1, dk2, dv, dlam (B, H)) by autograd in 64 bits."""
    B, H, Sq, D = q1.shape
    Hkv, Sk = k1.shape[1], k1.shape[2]
    g = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    j = torch.arange(Sk, device=q1.device)
    i = torch.arange(Sq, device=q1.device)
    keep = torch.ones(B, 1, Sq, Sk, dtype=torch.bool, device=q1.device)
    if causal:
        keep = keep & (j[None, :] <= i[:, None] + Sk - Sq)
    if lengths is not None:
        live = j[None, :] < lengths.to(q1.device).long()[:, None]
        keep = keep & live[:, None, None, :]
        # what lies past a sequence's length takes no part, whatever it holds
        k1, k2, v = (torch.where(live[:, None, :, None], t.double(), torch.zeros((), dtype=torch.float64, device=t.device))
                     for t in (k1, k2, v))
    xs = [t.detach().double().clone().requires_grad_(dout is not None) for t in (q1, q2, k1, k2, v)]
    l = lam if isinstance(lam, torch.Tensor) else torch.tensor(float(lam))
    l = l.detach().double().to(q1.device)
    l = l[(None,) * (4 - l.dim())].expand(B, H, 1, 1).clone().requires_grad_(dout is not None)
    rep = [t.repeat_interleave(g, 1) for t in xs[2:]]
    none = ~keep.any(-1, keepdim=True)
    maps = []
    for q, k in ((xs[0], rep[0]), (xs[1], rep[1])):
        s = (q @ k.transpose(-1, -2)) * scale
        s = s.masked_fill(~keep, -math.inf).masked_fill(none, 0.0)
        maps.append(torch.softmax(s, -1).masked_fill(none, 0.0).masked_fill(~keep, 0.0))
    out = maps[0] @ rep[2] - l * (maps[1] @ rep[2])
    if dout is None:
        return out
    gr = torch.autograd.grad(out, xs + [l], dout.double())
    return (out.detach(), *gr[:5], gr[5].reshape(B, H))


def quantise64(x, normalize=False):
    """(codes, bf16 scales) of rows: round(7 x / amax), half to even, and bf16(amax / 7)."""
    w = x.double()
    g = w.reshape(w.shape[:-1] + (w.shape[-1] // GROUP, GROUP))
    top = g.abs().amax(-1, keepdim=True)
    code = torch.round(g * 7.0 / torch.where(top == 0, torch.ones_like(top), top))
    s = (top / 7.0).squeeze(-1)
    if normalize:
        s = s / w.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    return code.reshape(x.shape), s.float().to(torch.bfloat16)


def values64(code, scale):
    g = code.reshape(code.shape[:-1] + (code.shape[-1] // GROUP, GROUP))
    return (g * scale.double()[..., None]).reshape(code.shape)


def decode64(q1, q2, k1, k2, v, lam, threshold=False, beta=1.0, power=2.0, normalize=False, scale=None):
    """One request: q (H, D) over k, v (n, Hkv, D), lam (H,)."""
    H, D = q1.shape
    n, Hkv = k1.shape[:2]
    out = torch.zeros(H, D, dtype=torch.float64, device=q1.device)
    if n == 0:
        return out
    for h in range(H):
        c = h // (H // Hkv)
        p = []
        for q, k in ((q1[h].double(), k1[:, c].double()), (q2[h].double(), k2[:, c].double())):
            if threshold:
                if normalize:
                    q = q / q.norm().clamp_min(1e-12)
                z = torch.relu(k @ q - beta * math.sqrt(2.0 * math.log(n) / D))
                p.append(torch.where(z > 0, z ** power, torch.zeros_like(z)))
            else:
                p.append(torch.softmax((k @ q) * (D ** -0.5 if scale is None else scale), 0))
        l = lam[h].double().clamp(0, 1) if threshold else lam[h].double()
        out[h] = p[0] @ v[:, c].double() - l * (p[1] @ v[:, c].double())
    return out
