"""Cases, plain forms and exact values of the dense operators around the MoE layer:

  linear       W8A8 linear layer: tokens quantised to 8-bit integers, integer product, one scale per token and channel
  norm         RMS norms after and before a block, with the branch's gate, the residual and its scale, and their gradients
  norm_linear  a block's input norm that hands its rows to the W8A8 layer as 8-bit integers
  router       top-k routing with per-expert counts, the balance loss and the z-loss, and the gradient of the logits

`run` computes each in plain torch operations (`own` false) or by the calls that a user of the package makes (`own` true).
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def listed():
    return [
        # one decoded token through a square projection of the 2880-wide layer: latency alone counts
        dict(name="linear one token", op="linear", T=1, K=2880, N=2880, x="bf16", bias=False),
        # a decode batch through the wide projection of a 4096-wide layer: the weights' bytes bound it
        dict(name="linear decode batch", op="linear", T=64, K=4096, N=14336, x="bf16", bias=False),
        # a ragged batch with a bias; neither side is a whole number of tiles
        dict(name="linear ragged fp16", op="linear", T=333, K=1040, N=1001, x="fp16", bias=True),
        # a long prefill through the same wide projection: the integer products bound it
        dict(name="linear prefill", op="linear", T=16384, K=4096, N=14336, x="bf16", bias=False),
        # decode: the branch is added to the residual stream and the sum normalised for the next block
        dict(name="pre-norm decode", op="norm", T=64, H=2880, x="bf16", w="bf16", post=False, gate="none", nxt=True,
             alpha=1.0, train=False),
        # prefill: norm after a block with a gate per channel, the residual sum, and the next block's input norm
        dict(name="post-norm prefill", op="norm", T=8192, H=2880, x="bf16", w="fp32", post=True, gate="channel", nxt=True,
             alpha=1.0, train=False),
        # one training step of the norms on both sides of a block with a gate per token
        dict(name="norms training", op="norm", T=4096, H=7168, x="bf16", w="bf16", post=True, gate="token", nxt=True,
             alpha=0.5, train=True),
        # the same in full precision, an odd width and a gate for each value
        dict(name="norms training fp32 odd", op="norm", T=515, H=1001, x="fp32", w="fp32", post=True, gate="full", nxt=False,
             alpha=0.7071, train=True),
        # a block's input norm and its W8A8 projection, ordinary prefill chunk
        dict(name="norm and linear", op="norm_linear", T=1000, K=7168, N=2048, x="bf16", w="bf16"),
        # the router of a decode batch, with the counts that a load monitor reads
        dict(name="router decode", op="router", T=64, E=128, K=4, x="fp32", scoring="softmax", renorm=True, mask=False, seqs=0,
             train=False),
        # router training on packed sequences with padding tokens; sigmoid scores
        dict(name="router sequences", op="router", T=4096, E=256, K=8, x="bf16", scoring="sigmoid", renorm=True, mask=True,
             seqs=13, train=True),
        # router training on a large batch with few experts
        dict(name="router training", op="router", T=16384, E=8, K=2, x="fp32", scoring="softmax", renorm=True, mask=False,
             seqs=0, train=True),
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "norm", "norm_linear", "router", "router"])
    if op == "linear":
        return dict(op=op, T=_log_size(rng, 1, 8192), K=16 * _log_size(rng, 8, 512), N=_log_size(rng, 32, 14336),
                    x=rng.choice(["bf16", "bf16", "fp16"]), bias=rng.random() < 0.4)
    if op == "norm_linear":
        return dict(op=op, T=_log_size(rng, 1, 4096), K=16 * _log_size(rng, 8, 448), N=_log_size(rng, 32, 7168),
                    x=rng.choice(["bf16", "fp16"]), w=rng.choice(["fp32", "same"]))
    if op == "norm":
        post = rng.random() < 0.7
        return dict(op=op, T=_log_size(rng, 1, 8192), H=_log_size(rng, 33, 7168), x=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    w=rng.choice(["fp32", "same"]), post=post, gate=rng.choice(["none", "channel", "token", "full"]),
                    nxt=(not post) or rng.random() < 0.6, alpha=rng.choice([1.0, 0.5]), train=rng.random() < 0.5)
    E, K = _log_size(rng, 8, 512), rng.randint(1, 8)
    # one renormalised weight is 1 whatever the logits are, and has no gradient to speak of
    return dict(op=op, T=_log_size(rng, 1, 16384), E=E, K=K, x=rng.choice(["fp32", "bf16"]),
                scoring=rng.choice(["softmax", "sigmoid"]), renorm=K > 1 and rng.random() < 0.7, mask=rng.random() < 0.5,
                seqs=rng.choice([0, 0, 1, 5, 31]), train=rng.random() < 0.6)


def _type(case, key):
    return TYPES[case["x"] if case[key] == "same" else case[key]]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)

    s = dict(case=case)
    op = case["op"]
    xt = _type(case, "x")
    if op in ("linear", "norm_linear"):
        T, K, N = case["T"], case["K"], case["N"]
        # weights of width 0.02 with their largest magnitude at 127, one scale per output channel
        w = torch.randn(N, K, generator=g, device=DEV)
        amax = w.abs().amax(dim=1, keepdim=True)
        s["weight"] = (w * (127.0 / amax)).round().clamp(-127, 127).to(torch.int8)
        s["weight_scale"] = (amax[:, 0] * (0.02 / 127.0)).contiguous()
        del w
        s["x"] = randn(T, K, dtype=xt)
        if op == "linear":
            s["bias"] = randn(N, scale=0.1) if case["bias"] else None
        else:
            s["residual"] = randn(T, K, dtype=xt, scale=2.0)
            s["norm_weight"] = randn(K, dtype=_type(case, "w"), scale=0.1, shift=1.0)
    elif op == "norm":
        T, H = case["T"], case["H"]
        wt = _type(case, "w")
        s["y"] = randn(T, H, dtype=xt, scale=0.7)
        s["residual"] = randn(T, H, dtype=xt, scale=2.0)
        s["weight"] = randn(H, dtype=wt, scale=0.1, shift=1.0) if case["post"] else None
        shape = dict(none=None, channel=(H,), token=(T, 1), full=(T, H))[case["gate"]]
        s["gate"] = None if shape is None else randn(*shape, dtype=xt, scale=0.2, shift=0.5)
        s["next_weight"] = randn(H, dtype=wt, scale=0.1, shift=1.0) if case["nxt"] else None
        if case["train"]:
            s["dh"] = randn(T, H, dtype=xt, scale=0.1)
            s["dn"] = randn(T, H, dtype=xt, scale=0.1) if case["nxt"] else None
            for name in ("y", "residual", "weight", "gate", "next_weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    else:
        T, E = case["T"], case["E"]
        # a router that favours some experts, as one does before it is balanced
        s["logits"] = (torch.randn(T, E, generator=g, device=DEV) + torch.randn(E, generator=g, device=DEV) * 0.7).to(xt)
        s["mask"] = (torch.rand(T, generator=g, device=DEV) < 0.9) if case["mask"] else None
        if case["seqs"]:
            # ragged lengths, now and then an empty sequence, and some rows behind the last one
            cut = torch.rand(case["seqs"], generator=g, device=DEV).sort().values * (0.97 * T)
            cut[::5] = cut[0]
            s["cu_seqlens"] = torch.cat([torch.zeros(1, device=DEV), cut.sort().values.ceil()]).clamp(max=T).to(torch.int32)
        else:
            s["cu_seqlens"] = None
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["dw"] = randn(T, case["K"], scale=1.0 / T)
            s["db"] = torch.full((), 0.01, device=DEV)
            s["dz"] = torch.full((), 0.001, device=DEV)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_quant(v):
    """Rows of 32-bit values -> whole numbers in [-127, 127] and the rows' scales; divided in 64 bits next to the borders."""
    scale = (v.abs().amax(dim=-1, keepdim=True).double() / 127.0).float().clamp(min=2.0 ** -100)
    return (v.double() / scale.double()).round().float(), scale


def _plain_linear(q, scale, s, dtype, bias=None):
    y = (q @ s["weight"].float().t()) * scale * s["weight_scale"]
    if bias is not None:
        y = y + bias
    return y.to(dtype)


def _rms(v):
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS)


def _plain_norm(s, alpha):
    u = s["y"].float()
    if s["weight"] is not None:
        u = _rms(u) * s["weight"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = alpha * s["residual"].float() + u
    return h, None if s["next_weight"] is None else _rms(h) * s["next_weight"].float()


def _plain_router(s, c):
    T, E, K = c["T"], c["E"], c["K"]
    logits = s["logits"].float()
    rows = torch.arange(T, device=DEV)
    live = torch.ones(T, dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"]
    if s["cu_seqlens"] is None:
        seg, S = torch.zeros(T, dtype=torch.long, device=DEV), 1
    else:
        S = c["seqs"]
        seg = (rows[:, None] >= s["cu_seqlens"][None, 1:]).sum(dim=1)
        live = live & (seg < S)
    ids = torch.sort(s["logits"].detach(), dim=1, descending=True, stable=True).indices[:, :K]
    ids = torch.where(live[:, None], ids, torch.arange(K, device=DEV)[None])
    a = logits if c["scoring"] == "softmax" else torch.clamp(logits, max=0.0) - torch.log1p(torch.exp(-logits.abs()))
    e = torch.exp(a - a.amax(dim=1, keepdim=True).detach())
    p = e / e.sum(dim=1, keepdim=True)
    picked = e.gather(1, ids)
    if c["renorm"]:
        w = picked / picked.sum(dim=1, keepdim=True)
    else:
        w = p.gather(1, ids) if c["scoring"] == "softmax" else torch.exp(a.gather(1, ids))
    w = w * live[:, None]
    member = ((seg[:, None] == torch.arange(S, device=DEV)[None]) & live[:, None]).float()      # [T, S]
    n = member.sum(dim=0)
    chosen = torch.zeros(T, E, device=DEV).scatter_(1, ids, 1.0)
    counts = member.t() @ chosen                                                              # [S, E]
    mean_p = (member.t() @ p) / n.clamp(min=1.0)[:, None]
    of_seq = (counts / (K * n.clamp(min=1.0))[:, None] * mean_p).sum(dim=1) * E
    balance = of_seq.sum() / (n > 0).sum().clamp(min=1)
    top = logits.amax(dim=1, keepdim=True).detach()
    lse = (top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True)))[:, 0]
    z = (lse * lse * live).sum() / n.sum().clamp(min=1.0)
    counts = counts.to(torch.int32)
    return w, ids.to(torch.int32), counts if s["cu_seqlens"] is not None else counts[0], balance, z


def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if own:
        import pyhip_b200 as fw
    if op == "linear":
        if own:
            return fw.linear_int8(s["x"], s["weight"], s["weight_scale"], bias=s["bias"])
        q, scale = _plain_quant(s["x"].float())
        return _plain_linear(q, scale, s, s["x"].dtype, s["bias"])
    if op == "norm_linear":
        if own:
            q, scale, h = fw.fused_pre_norm(s["x"], s["norm_weight"], residual=s["residual"], eps=EPS, quant="int8")
            return fw.linear_int8(q, s["weight"], s["weight_scale"], x_scale=scale, out_dtype=s["x"].dtype), h
        h = s["x"].float() + s["residual"].float()
        q, scale = _plain_quant(_rms(h) * s["norm_weight"].float())
        return _plain_linear(q, scale, s, s["x"].dtype), h.to(s["x"].dtype)
    if op == "norm":
        leaves = [s[k] for k in ("y", "residual", "weight", "gate", "next_weight") if s[k] is not None]
        if own:
            h = fw.fused_post_norm(s["y"], s["residual"], s["weight"], gate=s["gate"], residual_scale=c["alpha"], eps=EPS,
                                   next_weight=s["next_weight"])
            h, n = h if c["nxt"] else (h, None)
        elif c["train"]:
            with torch.enable_grad():
                h, n = _plain_norm(s, c["alpha"])
                h, n = h.to(s["y"].dtype), None if n is None else n.to(s["y"].dtype)
        else:
            h, n = _plain_norm(s, c["alpha"])
            h, n = h.to(s["y"].dtype), None if n is None else n.to(s["y"].dtype)
        out = [h] if n is None else [h, n]
        if not c["train"]:
            return out
        grads = torch.autograd.grad(out, leaves, [s["dh"]] if n is None else [s["dh"], s["dn"]])
        return [o.detach() for o in out], list(grads)
    if own:
        w, ids, counts, balance, z = fw.fused_router(s["logits"], c["K"], renormalize=c["renorm"], scoring=c["scoring"],
                                                     token_mask=s["mask"], cu_seqlens=s["cu_seqlens"])
    else:
        w, ids, counts, balance, z = _plain_router(s, c)
    if not c["train"]:
        return [w, ids, counts, balance, z]
    grad, = torch.autograd.grad([w, balance, z], [s["logits"]], [s["dw"], s["db"], s["dz"]])
    return [w.detach(), ids, counts, balance.detach(), z.detach(), grad]


# ------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    size = dict(bf16=2, fp16=2, fp32=4)
    b = size[c["x"]]
    if c["op"] in ("linear", "norm_linear"):
        T, K, N = c["T"], c["K"], c["N"]
        moved = T * K * b + N * K + 4 * N + T * N * b
        flops = 2 * T * K * N
        if c["op"] == "linear":
            return {"bytes": moved + (4 * N if c["bias"] else 0), "flops": flops}
        return {"bytes": moved + 2 * T * K * b + K * (b if c["w"] == "same" else size[c["w"]]), "flops": flops + 8 * T * K}
    if c["op"] == "norm":
        T, H = c["T"], c["H"]
        w = b if c["w"] == "same" else size[c["w"]]
        params = ((H if c["post"] else 0) + (H if c["nxt"] else 0)) * w
        gate = dict(none=0, channel=H, token=T, full=T * H)[c["gate"]] * b
        fwd = (2 + 1 + (1 if c["nxt"] else 0)) * T * H * b + params + gate
        if not c["train"]:
            return {"bytes": fwd, "flops": 12 * T * H}
        # the outputs' gradients are read, the inputs' written; the inputs are read once for both directions
        return {"bytes": fwd + (1 + (1 if c["nxt"] else 0)) * T * H * b + 2 * T * H * b + params + gate, "flops": 40 * T * H}
    T, E, K = c["T"], c["E"], c["K"]
    counts = 4 * E * max(1, c["seqs"])
    fwd = T * E * b + 8 * T * K + counts + (T if c["mask"] else 0) + 4 * (c["seqs"] + 1) + 8
    if not c["train"]:
        return {"bytes": fwd, "flops": 10 * T * E}
    return {"bytes": fwd + T * E * b + 4 * T * K, "flops": 22 * T * E}


# ------------------------------------------------------------------------------------------ exact values, in 64 bits
def _exact_int8(v):
    """The 8-bit rows of 64-bit values: the scale is a 32-bit number by definition, the quotient's nearest whole number the value."""
    scale = torch.clamp((v.abs().max(dim=-1).values / 127).float(), min=2.0 ** -100).double()
    return torch.round(v / scale[:, None]), scale


def _exact_product(q, scale, s):
    out = torch.empty(q.shape[0], s["weight"].shape[0], dtype=torch.float64, device=DEV)
    for lo in range(0, q.shape[0], 4096):
        out[lo:lo + 4096] = torch.mm(q[lo:lo + 4096], s["weight"].double().t())
    return out * (scale[:, None] * s["weight_scale"].double()[None, :])


def _inv_rms(v):
    return 1.0 / torch.sqrt(v.square().sum(dim=1, keepdim=True) / v.shape[1] + EPS)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    with torch.no_grad():
        if c["op"] == "linear":
            out = _exact_product(*_exact_int8(s["x"].double()), s)
            return out if s["bias"] is None else out + s["bias"].double()[None, :]
        if c["op"] == "norm_linear":
            h = s["x"].double() + s["residual"].double()
            return _exact_product(*_exact_int8(h * _inv_rms(h) * s["norm_weight"].double()), s), h
        return _exact_norm(s, c) if c["op"] == "norm" else _exact_router(s, c)


def _exact_norm(s, c):
    y, r = s["y"].double(), s["residual"].double()
    T, H = y.shape
    iy = _inv_rms(y)
    u = y if s["weight"] is None else y * iy * s["weight"].double()
    gate = 1.0 if s["gate"] is None else s["gate"].double()
    h = c["alpha"] * r + gate * u
    out = [h]
    if c["nxt"]:
        ih, wn = _inv_rms(h), s["next_weight"].double()
        out.append(h * ih * wn)
    if not c["train"]:
        return out
    dh = s["dh"].double()
    if c["nxt"]:
        # n = wn h / rms(h): the part of the gradient along h drops out
        dn = s["dn"].double()
        dh = dh + ih * (wn * dn) - h * ih ** 3 * (wn * dn * h).sum(dim=1, keepdim=True) / H
        dwn = (dn * h * ih).sum(dim=0)
    du = dh * gate
    grads = [du if s["weight"] is None else None, c["alpha"] * dh]
    if s["weight"] is not None:
        wu = s["weight"].double() * du
        grads[0] = iy * wu - y * iy ** 3 * (wu * y).sum(dim=1, keepdim=True) / H
        grads.append((du * y * iy).sum(dim=0))
    if s["gate"] is not None:
        dg = dh * u
        grads.append(dict(channel=lambda: dg.sum(dim=0), token=lambda: dg.sum(dim=1, keepdim=True), full=lambda: dg)[c["gate"]]())
    if c["nxt"]:
        grads.append(dwn)
    return out, grads


def _exact_router(s, c):
    T, E, K = c["T"], c["E"], c["K"]
    x = s["logits"].double()
    live = torch.ones(T, dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"].clone()
    bounds = [0, T] if s["cu_seqlens"] is None else s["cu_seqlens"].tolist()
    live[bounds[-1]:] = False
    # ties go to the lower expert: a key that falls with the index decides among equal logits
    order = torch.empty(T, E, dtype=torch.long, device=DEV)
    for lo in range(0, T, 2048):
        part = x[lo:lo + 2048]
        first = torch.argsort(torch.arange(E, device=DEV).expand_as(part), dim=1)
        order[lo:lo + 2048] = first.gather(1, torch.argsort(part.neg(), dim=1, stable=True))
    ids = order[:, :K].clone()
    ids[~live] = torch.arange(K, device=DEV)
    soft = torch.softmax(x, dim=1)
    lse = torch.logsumexp(x, dim=1)
    if c["scoring"] == "softmax":
        score, p = soft, soft
    else:
        score = torch.sigmoid(x)
        p = score / score.sum(dim=1, keepdim=True)
    w = score.gather(1, ids)
    total = w.sum(dim=1, keepdim=True)
    if c["renorm"]:
        w = w / total
    w = torch.where(live[:, None], w, torch.zeros_like(w))
    counts, balance, pull, used = [], 0.0, torch.zeros(T, E, dtype=torch.float64, device=DEV), 0
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        inside = torch.arange(lo, hi, device=DEV)[live[lo:hi]]
        got = torch.bincount(ids[inside].reshape(-1), minlength=E)
        counts.append(got.to(torch.int32))
        if len(inside):
            used += 1
            f = got.double() * E / (K * len(inside))
            balance = balance + (f * p[inside].mean(dim=0)).sum()
            pull[inside] = f / len(inside)                     # d(loss of the sequence) / dp
    balance = torch.as_tensor(balance / max(used, 1), dtype=torch.float64, device=DEV)
    pull = pull / max(used, 1)
    n = max(int(live.sum()), 1)
    z = (lse.square() * live).sum() / n
    counts = torch.stack(counts) if s["cu_seqlens"] is not None else counts[0]
    if not c["train"]:
        return [w, ids.to(torch.int32), counts, balance, z]
    dscore = torch.zeros(T, E, dtype=torch.float64, device=DEV)
    dw = s["dw"].double()
    if c["renorm"]:
        dw = (dw - (dw * w).sum(dim=1, keepdim=True)) / total
    dscore.scatter_(1, ids, dw)
    db = s["db"].double() * pull
    if c["scoring"] == "softmax":
        dscore = dscore + db
        dx = soft * (dscore - (dscore * soft).sum(dim=1, keepdim=True))
    else:
        dscore = dscore + (db - (db * p).sum(dim=1, keepdim=True)) / score.sum(dim=1, keepdim=True)
        dx = dscore * score * (1.0 - score)
    dx = dx + s["dz"].double() * 2.0 * lse[:, None] * soft / n
    return [w, ids.to(torch.int32), counts, balance, z, dx * live[:, None]]
