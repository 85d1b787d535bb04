"""64-bit restatement of the dense operators around the MoE layer (test infrastructure only): the W8A8 linear layer, the
block norms with their gradients, the router with its losses and gradient.  Written from the formulas, in plain torch.

Where a test needs to know how far 32-bit arithmetic may be off, the functions return next to a value its `size`: the same
formula with every difference turned into a sum of magnitudes, so that a bound on the roundings is a multiple of 2^-24 size."""
from __future__ import annotations

import torch


def quantize_int8(x):
    """[..., K] -> (q as float64 whole numbers, scale float32): scale = max(fl32(max|x| / 127), 2^-100), q = rint(x / scale)."""
    v = x.double()
    scale = (v.abs().amax(dim=-1) / 127.0).float().clamp(min=2.0 ** -100)
    q = torch.round(v / scale.double().unsqueeze(-1))
    bad = ~torch.isfinite(v).all(dim=-1)
    scale = torch.where(bad, torch.full_like(scale, float("nan")), scale)
    return torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q), scale


def linear_int8(q, scale, weight, weight_scale, bias=None):
    """-> (y, size) in 64 bits; the sums of products of 8-bit integers are exact there."""
    y = (q.double() @ weight.double().t()) * (scale.double().unsqueeze(-1) * weight_scale.double())
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def block_norm(y, residual=None, weight=None, gate=None, alpha=1.0, eps=1e-6, next_weight=None):
    """-> dict of float64 tensors: h, n and their sizes, and what the gradients need."""
    y = y.double()
    o = dict(y=y)
    o["ry"] = 1.0 / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + eps)
    o["u"] = y if weight is None else y * o["ry"] * weight.double()
    g = torch.ones((), dtype=torch.float64, device=y.device) if gate is None else gate.double()
    o["g"] = g
    gu = g * o["u"]
    o["h"] = gu if residual is None else alpha * residual.double() + gu
    o["h_size"] = gu.abs() if residual is None else (alpha * residual.double()).abs() + gu.abs()
    o["rh"] = 1.0 / torch.sqrt((o["h"] * o["h"]).mean(dim=-1, keepdim=True) + eps)
    if next_weight is not None:
        o["n"] = o["h"] * o["rh"] * next_weight.double()
        o["n_size"] = o["h_size"] * o["rh"] * next_weight.double().abs()
    return o


def block_norm_grads(o, residual, weight, gate, alpha, next_weight, dh=None, dn=None):
    """Gradients for block_norm's result `o` -> {name: (value, size)}."""
    y, h, g, u, ry, rh = (o[k] for k in ("y", "h", "g", "u", "ry", "rh"))
    H = y.shape[-1]
    zero = torch.zeros_like(h)
    d = zero if dh is None else dh.double()
    ds = d.abs()
    out = {}
    if next_weight is not None and dn is not None:
        wd = next_weight.double() * dn.double()
        d = d + rh * wd - h * rh ** 3 * (wd * h).sum(-1, keepdim=True) / H
        ds = ds + rh * wd.abs() + o["h_size"] * rh ** 3 * (wd.abs() * o["h_size"]).sum(-1, keepdim=True) / H
    if next_weight is not None:
        e = dn.double() if dn is not None else zero
        out["next_weight"] = ((e * h * rh).flatten(0, -2).sum(0), (e.abs() * o["h_size"] * rh).flatten(0, -2).sum(0))
    if residual is not None:
        out["residual"] = (alpha * d, abs(alpha) * ds)
    du, dus = d * g, ds * g.abs()
    if weight is None:
        out["y"] = (du, dus)
    else:
        w = weight.double()
        out["y"] = (ry * w * du - y * ry ** 3 * (w * du * y).sum(-1, keepdim=True) / H,
                    ry * w.abs() * dus + y.abs() * ry ** 3 * (w.abs() * dus * y.abs()).sum(-1, keepdim=True) / H)
        out["weight"] = ((du * y * ry).flatten(0, -2).sum(0), (dus * y.abs() * ry).flatten(0, -2).sum(0))
    if gate is not None:
        dg, dgs = d * u, ds * u.abs()
        if gate.dim() == 1 and y.dim() > 1:
            dg, dgs = dg.flatten(0, -2).sum(0), dgs.flatten(0, -2).sum(0)
        elif gate.shape[-1] == 1 and H > 1:
            dg, dgs = dg.sum(-1, keepdim=True), dgs.sum(-1, keepdim=True)
        out["gate"] = (dg.reshape(gate.shape), dgs.reshape(gate.shape))
    return out


def router(logits, K, scoring="softmax", renormalize=True, token_mask=None, cu_seqlens=None, dw=None, db=0.0, dz=0.0):
    """-> dict: weights, ids, counts, balance, z, dlogits (for gradients dw [T,K], db, dz) and `dsize`, all float64 but the ids
    and counts.  Walks over the tokens one by one."""
    T, E = logits.shape
    x = logits.detach().double().cpu()
    mask = torch.ones(T, dtype=torch.bool) if token_mask is None else token_mask.cpu()
    cu = [0, T] if cu_seqlens is None else cu_seqlens.tolist()
    S = len(cu) - 1
    weights, ids = torch.zeros(T, K, dtype=torch.float64), torch.arange(K).repeat(T, 1)
    counts, psum = torch.zeros(S, E, dtype=torch.int64), torch.zeros(S, E, dtype=torch.float64)
    n = [0] * S
    z, rows = 0.0, []
    for s in range(S):
        for t in range(cu[s], cu[s + 1]):
            if not mask[t] or bool((x[t] == float("-inf")).all()):
                continue
            row = [(-float(v), e) for e, v in enumerate(x[t])]
            ids[t] = torch.tensor([e for _, e in sorted(row)[:K]])
            sig = torch.sigmoid(x[t])
            a = x[t] if scoring == "softmax" else torch.nn.functional.logsigmoid(x[t])
            p = torch.softmax(a, 0)
            c = ids[t]
            weights[t] = torch.softmax(a[c], 0) if renormalize else (p[c] if scoring == "softmax" else sig[c])
            counts[s, c] += 1
            psum[s] += p
            n[s] += 1
            lse = torch.logsumexp(x[t], 0)
            z += float(lse) ** 2
            rows.append((s, t, p, sig, lse))
    used, total = sum(v > 0 for v in n), max(sum(n), 1)
    balance = sum(E / (K * n[s] ** 2) * float((counts[s].double() * psum[s]).sum()) for s in range(S) if n[s]) / max(used, 1)
    out = dict(weights=weights, ids=ids, counts=counts if cu_seqlens is not None else counts[0], balance=balance, z=z / total)
    g, size = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    dw = torch.zeros(T, K, dtype=torch.float64) if dw is None else dw.double().cpu()
    for s, t, p, sig, lse in rows:
        w, c = weights[t], ids[t]
        q = db * E / (K * n[s] ** 2) / used * counts[s].double()
        da, das = p * (q - (p * q).sum()), p * (q.abs() + (p * q.abs()).sum())
        if renormalize:
            da[c] += w * (dw[t] - (w * dw[t]).sum())
            das[c] += w * (dw[t].abs() + (w * dw[t].abs()).sum())
        else:
            da[c] += w * dw[t]
            das[c] += w * dw[t].abs()
            if scoring == "softmax":
                da -= p * (w * dw[t]).sum()
                das += p * (w * dw[t].abs()).sum()
        if scoring == "sigmoid":
            da, das = da * (1 - sig), das * (1 - sig)
        zz = dz * 2 * lse / total * torch.softmax(x[t], 0)
        g[t], size[t] = da + zz, das + zz.abs()
    return dict(out, dlogits=g, dsize=size)
