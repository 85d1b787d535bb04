"""GPU tier: the router with counts, losses and gradient against the 64-bit oracle, which walks over the tokens one by one.

Bounds, with u = 2^-24: the exponent's argument l - max is off by u |l - max| <= 40 u here, exp and log by 2 ulp, sums of up to
1024 positive terms over 32 lanes by 40 u, so a probability or weight is within 128 u of itself and a gradient within 512 u of
its size (all terms' magnitudes).  A loss adds fewer than 100 terms in any one chain: 512 u of itself.  Ids and counts are equal."""
import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import fused_router, fused_topk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _logits(T, E, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * scale + torch.randn(E, generator=g)).to(dtype)


def _check(x, K, scoring, renorm, mask=None, cu=None, db=0.3, dz=0.07, seed=0):
    T, E = x.shape
    dw = torch.randn(T, K, generator=torch.Generator().manual_seed(seed))
    ref = orc.router(x, K, scoring, renorm, mask, cu, dw, db, dz)
    leaf = x.to(DEV).requires_grad_(True)
    dev = dict(token_mask=None if mask is None else mask.to(DEV), cu_seqlens=None if cu is None else cu.to(DEV))
    out = fused_router(leaf, K, renormalize=renorm, scoring=scoring, **dev)
    with torch.no_grad():
        plain = fused_router(leaf, K, renormalize=renorm, scoring=scoring, **dev)
    assert not any(t.requires_grad for t in plain) and all(torch.equal(a, b) for a, b in zip(out, plain))
    w, ids, counts, balance, z = (t.detach().cpu() for t in out)
    assert ids.dtype == torch.int32 and counts.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.long(), ref["ids"])
    assert torch.equal(counts.long(), ref["counts"])
    assert ((w.double() - ref["weights"]).abs() <= 128 * U * ref["weights"] + 2.0 ** -140).all()
    assert abs(float(balance) - ref["balance"]) <= 512 * U * abs(ref["balance"])
    assert abs(float(z) - ref["z"]) <= 512 * U * abs(ref["z"])
    grad, = torch.autograd.grad([out.topk_weights, out.balance_loss, out.z_loss], [leaf],
                                [dw.to(DEV), torch.tensor(db, device=DEV), torch.tensor(dz, device=DEV)])
    assert grad.dtype == x.dtype and grad.shape == x.shape
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -140}[x.dtype]
    off = (grad.cpu().double() - ref["dlogits"]).abs() - (torch.finfo(x.dtype).eps / 2 * ref["dlogits"].abs() + 512 * U * ref["dsize"] + tiny)
    assert float(off.max()) <= 0, f"gradient: {int((off > 0).sum())} out of bounds, worst {float(off.max()):.3e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 2), (5, 3, 3), (37, 8, 8), (33, 11, 4), (64, 17, 6), (50, 33, 32), (70, 64, 6), (130, 100, 8),
                                   (64, 128, 4), (90, 256, 8), (40, 300, 10), (20, 600, 5), (9, 1024, 32)])
def test_router_matches_64_bits(T, E, K, scoring, renorm, dtype):
    _check(_logits(T, E, dtype, T + E), K, scoring, renorm, seed=T)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K", [(1500, 8, 2), (700, 60, 4), (900, 256, 8)])
def test_many_tokens_masks_and_sequences(T, E, K, scoring):
    g = torch.Generator().manual_seed(T)
    x = _logits(T, E, torch.float32, T)
    mask = torch.rand(T, generator=g) < 0.8
    _check(x, K, scoring, True, mask=mask)
    cu = torch.tensor([0, 1, 1, 17, 300, 300, 301, T - 40, T - 20], dtype=torch.int32)
    _check(x, K, scoring, False, cu=cu)
    mask[1:17] = False                                        # a sequence without live tokens
    _check(x, K, scoring, True, mask=mask, cu=cu)
    _check(x, K, scoring, True, mask=mask, cu=torch.tensor([13, T], dtype=torch.int32))
    _check(x, K, scoring, True, cu=torch.arange(0, T + 1, 3, dtype=torch.int32)[:400])   # more sequences than chunks


def test_equal_logits_go_to_the_lower_expert():
    x = torch.tensor([[0.0, 1.0, 1.0, -0.0, 1.0, 0.0, -1.0, 1.0], [2.0] * 8, [-0.0, 0.0] * 4])
    for dtype in (torch.float32, torch.bfloat16):
        for wide in (1, 3, 9):                                # one lane group per row, and values spread over lanes
            _check(x.repeat(1, wide).to(dtype), 5, "softmax", True)
    x = _logits(200, 256, torch.bfloat16, 1).round()
    _check(x, 8, "sigmoid", True)


def test_empty_rows_and_values_in_masked_places():
    inf, nan = float("inf"), float("nan")
    x = _logits(40, 32, torch.float32, 3)
    x[3] = -inf                                               # no expert allowed
    x[4, 2:] = -inf                                           # fewer than K
    x[5, ::2] = -inf
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            _check(x, 4, scoring, renorm)
    mask = torch.ones(40, dtype=torch.bool)
    mask[[0, 7, 8, 9, 39]] = False
    y = x.clone()
    y[0], y[7], y[8, 3], y[9], y[39, 0] = nan, inf, nan, -inf, -inf
    want = [t.clone() for t in fused_router(x.to(DEV), 4, token_mask=mask.to(DEV))]
    got = fused_router(y.to(DEV), 4, token_mask=mask.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = y.to(DEV).requires_grad_(True)
    out = fused_router(leaf, 4, token_mask=mask.to(DEV))
    g, = torch.autograd.grad([out.topk_weights.sum(), out.balance_loss, out.z_loss], [leaf], [torch.ones((), device=DEV)] * 3)
    assert torch.isfinite(g).all() and (g[~mask.to(DEV)] == 0).all() and (g[3] == 0).all()
    cu = torch.tensor([2, 30], dtype=torch.int32, device=DEV)
    y[31:] = nan
    y[1] = nan
    out = fused_router(y[:, :].to(DEV), 4, cu_seqlens=cu, token_mask=mask.to(DEV))
    assert all(torch.isfinite(t.float()).all() for t in out)
    assert (out.topk_ids[31:].cpu() == torch.arange(4, dtype=torch.int32)).all() and (out.topk_weights[31:] == 0).all()


def test_nothing_live():
    x = _logits(20, 16, torch.float32, 0).to(DEV)
    mask = torch.zeros(20, dtype=torch.bool, device=DEV)
    leaf = x.clone().requires_grad_(True)
    out = fused_router(leaf, 2, token_mask=mask)
    g, = torch.autograd.grad([out.balance_loss, out.z_loss], [leaf], [torch.ones((), device=DEV)] * 2)
    assert (out.balance_loss == 0) and (out.z_loss == 0) and (out.counts == 0).all() and (g == 0).all()
    out = fused_router(x[:0], 2)
    assert out.topk_ids.shape == (0, 2) and (out.counts == 0).all() and float(out.balance_loss) == 0 and float(out.z_loss) == 0
    leaf = x[:0].clone().requires_grad_(True)
    out = fused_router(leaf, 2)
    g, = torch.autograd.grad([out.balance_loss], [leaf])
    assert g.shape == (0, 16)


def test_nan_and_infinite_logits_of_live_tokens_stay_in_range():
    x = _logits(12, 40, torch.float32, 5)
    x[2, 7], x[4], x[6, 3], x[6, 9] = float("nan"), float("nan"), float("inf"), float("inf")
    out = fused_router(x.to(DEV), 6)
    assert ((out.topk_ids >= 0) & (out.topk_ids < 40)).all()
    assert all(len(set(r)) == 6 for r in out.topk_ids.tolist())
    rows = [0, 1, 3, 5, 7, 8, 9, 10, 11]
    clean = fused_router(x[rows].to(DEV), 6)
    assert torch.equal(out.topk_weights[rows], clean.topk_weights) and torch.equal(out.topk_ids[rows], clean.topk_ids)
    assert int(out.counts.sum()) == 12 * 6 and out.balance_loss.isnan()


def test_extreme_scores_do_not_underflow():
    """Sigmoid scores that are all below the smallest float, and softmax rows far from zero."""
    x = _logits(30, 24, torch.float32, 9) - 300.0
    _check(x, 3, "sigmoid", True, dz=0.0)
    _check(x + 700.0, 3, "sigmoid", True, dz=0.0)
    _check(x, 3, "softmax", True)


@pytest.mark.parametrize("bad", [[5, 3, 9, 1, 40], [-7, 500, 10, 10, 99], [0, 0, 0, 0, 0], [40, 30, 20, 10, 0]])
def test_sequences_out_of_order_stay_in_range(bad):
    x = _logits(40, 16, torch.float32, 2).to(DEV).requires_grad_(True)
    out = fused_router(x, 4, cu_seqlens=torch.tensor(bad, dtype=torch.int32, device=DEV))
    assert ((out.topk_ids >= 0) & (out.topk_ids < 16)).all()
    g, = torch.autograd.grad([out.topk_weights.sum()], [x])
    assert g.shape == x.shape


def test_strided_rows_and_agreement_with_fused_topk():
    big = _logits(100, 300, torch.float32, 4).to(DEV)
    for x in (big[:, 7:135], big[::3, :64], big.t()[:60, :100], big[:1, :32].expand(50, 32)):
        a, b = fused_router(x, 4), fused_router(x.contiguous(), 4)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        w, ids = fused_topk(None, x.contiguous(), 4)
        assert torch.equal(ids, a.topk_ids) and torch.allclose(w, a.topk_weights, rtol=1e-5, atol=1e-7)
    leaf = big[:, 7:135].detach().requires_grad_(True)
    g1, = torch.autograd.grad(fused_router(leaf, 4).z_loss, leaf)
    leaf2 = big[:, 7:135].contiguous().requires_grad_(True)
    g2, = torch.autograd.grad(fused_router(leaf2, 4).z_loss, leaf2)
    assert torch.equal(g1, g2)


def test_each_gradient_alone():
    x = _logits(60, 48, torch.float32, 6)
    dw = torch.randn(60, 5, generator=torch.Generator().manual_seed(1))
    for which in ("topk_weights", "balance_loss", "z_loss"):
        leaf = x.to(DEV).requires_grad_(True)
        out = fused_router(leaf, 5)
        up = dw.to(DEV) if which == "topk_weights" else torch.ones((), device=DEV)
        g, = torch.autograd.grad(getattr(out, which), leaf, up)
        ref = orc.router(x, 5, dw=dw if which == "topk_weights" else None, db=float(which == "balance_loss"), dz=float(which == "z_loss"))
        assert ((g.cpu().double() - ref["dlogits"]).abs() <= 512 * U * ref["dsize"] + U * ref["dlogits"].abs() + 2.0 ** -140).all()
    leaf = x.to(DEV).requires_grad_(True)
    out = fused_router(leaf, 5)
    out.balance_loss.backward()
    with pytest.raises(RuntimeError):
        out.counts.float().sum().backward()


def test_formula_matches_differences():
    """The oracle's gradient (64 bits) against central differences of its values, away from ties."""
    x = _logits(6, 7, torch.float32, 8).double()
    dw = torch.randn(6, 3, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    cu, mask = torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([True, True, False, True, True, True])
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            args = (3, scoring, renorm, mask, cu)
            g = orc.router(x, *args, dw, 0.7, 0.2)["dlogits"]
            for at in range(x.numel()):
                v = []
                for step in (1e-5, -1e-5):
                    y = x.clone()
                    y.view(-1)[at] += step
                    o = orc.router(y, *args)
                    v.append(float((o["weights"] * dw).sum()) + 0.7 * o["balance"] + 0.2 * o["z"])
                # third derivatives below 100: 1e-10 * 100 / 6, and 1e-15 * |values| / 1e-5
                assert abs((v[0] - v[1]) / 2e-5 - float(g.view(-1)[at])) < 1e-7


def test_same_bits_every_time_streams_and_graphs():
    x = _logits(3000, 200, torch.bfloat16, 2).to(DEV)
    cu = torch.tensor([0, 700, 701, 2900], dtype=torch.int32, device=DEV)
    leaf = x.clone().requires_grad_(True)
    one = torch.ones((), device=DEV)

    def step():
        o = fused_router(leaf, 6, cu_seqlens=cu)
        return [*o, *torch.autograd.grad([o.topk_weights.sum(), o.balance_loss, o.z_loss], [leaf], [one] * 3)]

    first = [t.detach().clone() for t in step()]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            runs += [[t.detach() for t in step()] for _ in range(4)]
    torch.cuda.synchronize()
    for r in runs:
        assert all(torch.equal(a, b) for a, b in zip(r, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_refusals():
    x = torch.zeros(4, 16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    for call in (lambda: fused_router(x, 0), lambda: fused_router(x, 17), lambda: fused_router(torch.zeros(2, 64, device=DEV), 33),
                 lambda: fused_router(torch.zeros(2, 1025, device=DEV), 2), lambda: fused_router(x[0], 2), lambda: fused_router(x, 2, scoring="tanh"),
                 lambda: fused_router(x, 2, token_mask=torch.ones(4, **i32)), lambda: fused_router(x, 2, token_mask=torch.ones(3, dtype=torch.bool, device=DEV)),
                 lambda: fused_router(x, 2, cu_seqlens=torch.zeros(1, **i32)), lambda: fused_router(x, 2, cu_seqlens=torch.zeros(3, device=DEV)),
                 lambda: fused_router(x, 2, cu_seqlens=torch.zeros(3, dtype=torch.int32)), lambda: fused_router(torch.zeros(2, 0, device=DEV), 1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        fused_router(x.double(), 2)
