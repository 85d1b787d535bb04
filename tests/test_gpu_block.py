"""GPU tier: the dense operators and the MoE layer run together, as a model runs them: a serving block (input norm to 8-bit rows,
W8A8 projection, router, fused MoE, gated output norm with the next block's input norm) eagerly and in a CUDA graph, and a
training step of what surrounds frozen experts (norms, gate, router)."""
import pytest
import torch

from oracle import dense_oracle as orc
from oracle import moe_oracle
from pyhip_b200 import (QuantType, fused_moe, fused_post_norm, fused_pre_norm, fused_router, linear_int8, quantize_int8, synth)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(H, I, E, seed):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s, scale=1.0, shift=0.0: torch.randn(*s, generator=g) * scale + shift  # noqa: E731
    m = dict(pre=rnd(H, scale=0.1, shift=1.0), post=rnd(H, scale=0.1, shift=1.0), nxt=rnd(H, scale=0.1, shift=1.0),
             gate=rnd(H, scale=0.2, shift=0.5), router=rnd(E, H, scale=H ** -0.5))
    m = {k: v.to(torch.bfloat16).to(DEV) for k, v in m.items()}
    m["proj"], m["proj_scale"] = quantize_int8((rnd(H, H) * H ** -0.5).to(DEV))
    m["experts_host"] = synth.make_weights_mxfp4(E, H, I, seed=seed)
    m["experts"] = tuple(t.to(DEV) for t in m["experts_host"])
    return m


def _block(m, x, residual, K):
    q, scale, h = fused_pre_norm(x, m["pre"], residual=residual, quant="int8")
    y = linear_int8(q, m["proj"], m["proj_scale"], x_scale=scale)
    logits = y @ m["router"].t()
    r = fused_router(logits, K)
    w1, s1, w2, s2 = m["experts"]
    z = fused_moe(y, w1, w2, r.topk_weights, r.topk_ids, quant_type=QuantType.per_1x32, w1_scale=s1, w2_scale=s2)
    h2, n = fused_post_norm(z, h, m["post"], gate=m["gate"], next_weight=m["nxt"])
    return dict(h=h, y=y, logits=logits, z=z, h2=h2, n=n, **r._asdict())


@pytest.mark.parametrize("T", [1, 48, 700])
def test_serving_block(T):
    H, I, E, K = 512, 256, 16, 4
    m = _model(H, I, E, 5)
    x = synth.make_hidden(T, H, 1).to(DEV)
    residual = synth.make_hidden(T, H, 2).to(DEV)
    o = _block(m, x, residual, K)
    # every step against the oracle on that step's own inputs
    ref = orc.block_norm(x, residual, None, None, 1.0, 1e-6, m["pre"])
    assert (o["h"].double() - ref["h"]).abs().max() <= 2.0 ** -8 * ref["h"].abs().max()
    y64, _ = orc.linear_int8(*orc.quantize_int8(ref["n"].float()), m["proj"], m["proj_scale"])
    # the norm's 32-bit roundings may move a value by one step of the 8-bit grid: K of them at most, each |w| <= 127 scales
    step = ref["n"].abs().amax(-1, keepdim=True) / 127
    assert ((o["y"].double() - y64).abs() <= 2.0 ** -8 * y64.abs() + step * 127 * m["proj_scale"].double() * 2).all()
    r64 = orc.router(o["logits"], K)
    assert torch.equal(o["topk_ids"].cpu().long(), r64["ids"]) and torch.equal(o["counts"].cpu().long(), r64["counts"])
    assert int(o["counts"].sum()) == T * K
    want = moe_oracle.torch_moe_oracle_mxfp4(o["y"].cpu(), *m["experts_host"], o["topk_weights"].cpu(), o["topk_ids"].cpu())
    assert moe_oracle.cosine(o["z"].cpu(), want) >= 0.9995
    ref = orc.block_norm(o["z"], o["h"], m["post"], m["gate"], 1.0, 1e-6, m["nxt"])
    for name in ("h", "n"):
        got = o["h2" if name == "h" else "n"].double()
        assert ((got - ref[name]).abs() <= 2.0 ** -8 * ref[name].abs() + 512 * 2.0 ** -24 * ref[name + "_size"]).all()
    # the same bits in a graph, on a side stream, with new inputs
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _block(m, x, residual, K)
    torch.cuda.synchronize()
    assert all(torch.equal(again[k], o[k]) for k in o)
    xs, rs = torch.zeros_like(x), torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = _block(m, xs, rs, K)
    xs.copy_(x), rs.copy_(residual)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g[k], o[k]) for k in o)


def test_training_step_around_frozen_experts():
    """Router, norms and gate take gradients of a loss that holds the routing weights, the balance loss and the z-loss; the
    chain through torch's own products is compared with the same chain in 64 bits from the oracle."""
    T, H, E, K = 300, 256, 8, 2
    g = torch.Generator().manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    x, res, up, dw = rnd(T, H), rnd(T, H), rnd(T, H), rnd(T, K)
    leaves = dict(pre=rnd(H).mul_(0.1).add_(1), post=rnd(H).mul_(0.1).add_(1), gate=rnd(T, 1), router=rnd(E, H) * H ** -0.5)
    for v in leaves.values():
        v.requires_grad_(True)
    n, h = fused_pre_norm(x, leaves["pre"], residual=res)
    logits = n @ leaves["router"].t()
    r = fused_router(logits, K)
    out = fused_post_norm(n, h, leaves["post"], gate=leaves["gate"], residual_scale=0.5)
    got = torch.autograd.grad([out, r.topk_weights, r.balance_loss, r.z_loss], list(leaves.values()),
                              [up, dw, torch.tensor(0.1, device=DEV), torch.tensor(0.01, device=DEV)])
    d = {k: v.detach() for k, v in leaves.items()}
    a = orc.block_norm(x, res, None, None, 1.0, 1e-6, d["pre"])
    # the inputs of each step are those that the device computed: what is compared is the gradients, not a chain of roundings
    b = orc.block_norm(n.detach(), h.detach(), d["post"], d["gate"], 0.5, 1e-6)
    gb = orc.block_norm_grads(b, h.detach(), d["post"], d["gate"], 0.5, None, up)
    gr = orc.router(logits.detach(), K, dw=dw, db=0.1, dz=0.01)
    dl = gr["dlogits"].to(DEV)
    dn = gb["y"][0] + dl @ d["router"].double()
    ga = orc.block_norm_grads(a, res, None, None, 1.0, d["pre"], gb["residual"][0].float(), dn.float())
    want = dict(pre=ga["next_weight"][0], post=gb["weight"][0], gate=gb["gate"][0], router=dl.t() @ n.detach().double())
    for (name, w), v in zip(want.items(), got):
        # each chain has a handful of 32-bit steps, each off by 2^-24 times the square root of at most T terms and more
        assert float((v.double() - w).norm() / w.norm()) <= 2e-5, name


def test_frozen_parts_take_no_gradient():
    x = torch.randn(6, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    h, n = fused_post_norm(x, x.detach(), w, next_weight=w)
    n.sum().backward()
    assert x.grad is not None and w.grad is None
    y = fused_post_norm(x, x.detach(), w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    y = x * 1.0
    out = fused_pre_norm(y, w)
    y.add_(1)                                            # the saved input changes in place
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
